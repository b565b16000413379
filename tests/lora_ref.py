"""Adapters beside a shared linear in 64 bits, and how far 32-bit kernels may
be from them: a sum of n products whose chain has k links is off by at most
(k + 1) 2^-24 of the sum of their magnitudes."""
import numpy as np

F32, F64 = np.float32, np.float64
H = 2.0 ** -24


def to16(a, bf):
    """Values rounded to a 16-bit format: its bits (uint16), and they in float64."""
    if not bf:
        h = a.astype(np.float16)
        return h.view(np.uint16), h.astype(F64)
    w = np.ascontiguousarray(a, F32).view(np.uint32)
    h = ((w + 0x7fff + (w >> 16 & 1)) >> 16).astype(np.uint16)
    return h, (h.astype(np.uint32) << 16).view(F32).astype(F64)


def owners(seq, start, adapter, adapters):
    """Each row's adapter, -1 for none."""
    of = np.full(seq, -1)
    first = np.arange(len(adapter) + 1) if start is None else np.asarray(start)
    for i, a in enumerate(adapter):
        rows = np.arange(max(first[i], 0), max(min(first[i + 1], seq), 0))
        of[rows] = a if 0 <= a < adapters else -1
    return of


class Sums:
    """Values with bounds of their 32-bit errors."""

    def __init__(self, value, off=0.0):
        self.value, self.off = value, np.broadcast_to(np.asarray(off, F64), np.shape(value))

    def matmul(self, other, links):
        """A product whose sums have at most so many links."""
        a, b, ea, eb = np.abs(self.value), np.abs(other.value), self.off, other.off
        return Sums(self.value @ other.value, ea @ (b + eb) + a @ eb + (links + 1) * H * ((a + ea) @ (b + eb)))

    def times(self, s):
        return Sums(self.value * s, np.abs(s) * (self.off * (1 + H) + H * np.abs(self.value)))

    def plus(self, r):
        v = self.value + r
        return Sums(v, self.off * (1 + H) + H * (np.abs(v) + self.off))


def down(x, a, links):
    return Sums(x).matmul(Sums(a.T.copy()), links)


def forward(x, a, b, scale, rank, of, res):
    """y and u, as Sums; res a Sums or None."""
    seq, out = x.shape[0], b.shape[1]
    y = np.zeros((seq, out)) if res is None else res.value.copy()
    ey = np.zeros((seq, out)) if res is None else res.off.copy()
    u, eu = np.zeros((seq, a.shape[1])), np.zeros((seq, a.shape[1]))
    for k in range(a.shape[0]):
        at, r = np.flatnonzero(of == k), rank[k]
        if not at.size:
            continue
        h = down(x[at], a[k, :r], x.shape[1])
        u[at, :r], eu[at, :r] = h.value, h.off
        d = h.matmul(Sums(b[k, :, :r].T.copy()), r).times(scale[k]).plus(y[at])
        y[at], ey[at] = d.value, ey[at] + d.off
    return Sums(y, ey), Sums(u, eu)


def backward(x, u, dy, a, b, scale, rank, of, dres):
    """dx, da, db as Sums; u a Sums (what the call is given, or computes)."""
    dx = np.zeros(x.shape) if dres is None else dres.astype(F64)
    edx = np.zeros(x.shape)
    da, eda, db, edb = np.zeros(a.shape), np.zeros(a.shape), np.zeros(b.shape), np.zeros(b.shape)
    for k in range(a.shape[0]):
        at, r = np.flatnonzero(of == k), rank[k]
        if not at.size:
            continue
        du = Sums(dy[at]).matmul(Sums(b[k, :, :r]), dy.shape[1]).times(scale[k])
        d = du.matmul(Sums(a[k, :r]), r).plus(dx[at])
        dx[at], edx[at] = d.value, d.off
        p = Sums(du.value.T.copy(), du.off.T.copy()).matmul(Sums(x[at]), at.size)
        da[k, :r], eda[k, :r] = p.value, p.off
        p = Sums(dy[at].T.copy()).matmul(Sums(u.value[at, :r], u.off[at, :r]), at.size).times(scale[k])
        db[k, :, :r], edb[k, :, :r] = p.value, p.off
    return Sums(dx, edx), Sums(da, eda), Sums(db, edb)
