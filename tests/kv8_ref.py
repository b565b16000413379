"""The 8-bit paged KV cache in NumPy, 64 bits: its layout (include/nlgpu.h),
the quantisation, and the attention over it."""
import math

import numpy as np

F32 = np.float32
I8, E4M3 = 0, 1
TOP = {I8: 127.0, E4M3: 448.0}


def _e4m3_values():
    """The numbers of the 256 e4m3 codes (sign, 4 exponent bits of bias 7, 3 bits; 0x7f and 0xff are NaN)."""
    v = np.zeros(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7)
        v[c] = math.nan if c & 0x7f == 0x7f else (-x if c & 0x80 else x)
    return v


E4M3_VALUES = _e4m3_values()


def values(codes, fmt):
    return codes.view(np.int8).astype(np.float64) if fmt == I8 else E4M3_VALUES[codes]


def quantise(x, fmt):
    """Rows x [..., hd] (64 bits) as (codes uint8, scales f32); non-finite rows: codes 0, scale NaN."""
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        f = x.astype(F32)
        odd = ~np.isfinite(f).all(axis=-1)
        amax = np.abs(np.where(odd[..., None], 0, f)).max(axis=-1)
        scale = (amax.astype(np.float64) / TOP[fmt]).astype(F32)
        s = scale.astype(np.float64)[..., None]
        u = np.where(odd[..., None] | (s == 0), 0.0, x / s)
    if fmt == I8:
        codes = np.clip(np.rint(u), -127, 127).astype(np.int8).view(np.uint8)
    else:
        _, e = np.frexp(u)
        e = np.maximum(e, -5) - 4
        y = np.clip(np.ldexp(np.rint(np.ldexp(u, -e)), e), -448, 448)
        order = np.argsort(E4M3_VALUES[:127])
        codes = order[np.searchsorted(E4M3_VALUES[:127][order], np.abs(y))].astype(np.uint8)
        codes = np.where(np.signbit(y), codes | 0x80, codes).astype(np.uint8)
    return codes, np.where(odd, F32(np.nan), scale)


class Pools:
    """Both pools as uint8 [npool, kvheads, bs / 16, 16 * (hd + 4)], and their rows."""

    def __init__(self, npool, kvheads, hd, bs, fmt, fill=0):
        self.npool, self.kvheads, self.hd, self.bs, self.fmt = npool, kvheads, hd, bs, fmt
        shape = (npool, kvheads, bs // 16, 16 * (hd + 4))
        self.k, self.v = np.full(shape, fill, np.uint8), np.full(shape, fill, np.uint8)

    def copy(self):
        p = Pools(0, self.kvheads, self.hd, self.bs, self.fmt)
        p.npool, p.k, p.v = self.npool, self.k.copy(), self.v.copy()
        return p

    def find(self, table, b, pos):
        """(block, tile, row in it) of a position, None without one."""
        if not 0 <= b < table.shape[0] or not 0 <= pos < table.shape[1] * self.bs:
            return None
        blk = int(table[b, pos // self.bs])
        return (blk, pos % self.bs // 16, pos % 16) if 0 <= blk < self.npool else None

    def _codes(self, tile, which, at):
        n = 16 * self.hd
        return tile[:, :n].reshape(-1, 16, self.hd)[:, at] if which == "k" else \
            tile[:, :n].reshape(-1, self.hd, 16)[:, :, at]

    def _scale(self, tile, at):
        n = 16 * self.hd + 4 * at
        return tile[:, n:n + 4]

    def write(self, table, b, pos, which, codes, scale):
        """One position's codes [kvheads, hd] and scales [kvheads]."""
        w = self.find(table, b, pos)
        if w is None:
            return
        tile = getattr(self, which)[w[0], :, w[1]]
        self._codes(tile, which, w[2])[:] = codes
        self._scale(tile, w[2])[:] = np.ascontiguousarray(scale, F32).view(np.uint8).reshape(-1, 4)

    def raw(self, table, b, pos, which):
        w = self.find(table, b, pos)
        if w is None:
            return None
        tile = getattr(self, which)[w[0], :, w[1]]
        scale = np.ascontiguousarray(self._scale(tile, w[2])).view(F32)[:, 0]
        return self._codes(tile, which, w[2]).copy(), scale

    def row(self, table, b, pos, which):
        """Values [kvheads, hd] in 64 bits; zeros without a block."""
        r = self.raw(table, b, pos, which)
        if r is None:
            return np.zeros((self.kvheads, self.hd))
        return values(r[0], self.fmt) * r[1].astype(np.float64)[:, None]

    def rows(self, table, b, n, which):
        return np.stack([self.row(table, b, p, which) for p in range(n)]) if n else \
            np.zeros((0, self.kvheads, self.hd))

    def fill_rows(self, table, b, positions, rng, sigma=1.0):
        """Quantised normal rows at the given positions of sequence b."""
        n = len(positions)
        for which in "kv":
            c, s = quantise(rng.standard_normal((n, self.kvheads, self.hd)) * sigma, self.fmt)
            for i, p in enumerate(positions):
                self.write(table, b, p, which, c[i], s[i])


def norm_rope(x, gain, eps, co, si, half):
    """Head rows x [..., hd] (64 bits) normed (gain None: not) and rotated by co, si [..., hd / 2]."""
    hd = x.shape[-1]
    if gain is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * gain.astype(np.float64)
    y = np.empty_like(x)
    a, b = (slice(0, hd // 2), slice(hd // 2, hd)) if half else (slice(0, hd, 2), slice(1, hd, 2))
    y[..., a] = x[..., a] * co - x[..., b] * si
    y[..., b] = x[..., a] * si + x[..., b] * co
    return y


def attend(q, k, v, seen):
    """q [heads, hd], k and v [n, kvheads, hd], seen [n]: the output [heads, hd] in 64 bits, and what bounds a
    kernel's error: per head, the largest |v| attended and the largest root of sum (q k)^2 / hd."""
    heads, hd = q.shape
    grp = heads // k.shape[1]
    out, vmax, amp = np.zeros((heads, hd)), np.zeros(heads), np.zeros(heads)
    idx = np.flatnonzero(seen)
    if not idx.size:
        return out, vmax, amp
    for h in range(heads):
        kk, vv, qq = k[idx, h // grp], v[idx, h // grp], q[h].astype(np.float64)
        s = kk @ qq / math.sqrt(hd)
        p = np.exp(s - s.max())
        out[h] = p @ vv / p.sum()
        vmax[h] = np.abs(vv).max()
        amp[h] = np.sqrt(((kk * qq) ** 2).sum(axis=1) / hd).max()
    return out, vmax, amp


def tolerance(n, vmax, amp):
    """How far a row's output may be off.  A score: q carries 22 bits (half a step 2^-23 of each product, in 128
    directions), its coefficient and scale three roundings, the sum of the products some forty, each at most 2^-24 of
    a partial sum that is of the size of amp: about 12 amp 2^-24 in root mean square, six times that for the worst
    of a test's scores.  It moves the probabilities by that share, twice (numerator and sum).  Each probability is an
    exponential (two steps) and carries 22 bits; n of them are summed in 16 chains a lane (random: sqrt n)."""
    return vmax * 2.0 ** -24 * (150.0 * amp + 64.0 + 4.0 * math.sqrt(max(n, 1)))
