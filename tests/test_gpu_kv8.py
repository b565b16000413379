"""The 8-bit paged KV cache on the GPU against its NumPy form in 64 bits
(kv8_ref.py): appended bytes exactly, attention within the tolerance derived
there, commit and read-back exactly, and a run of them together."""
import numpy as np
import pytest

import kv8_ref as ref
import nlgpu

pytestmark = pytest.mark.gpu
F32 = np.float32
FORMATS = [ref.I8, ref.E4M3]


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def up(a):
    return nlgpu.to_device(a) if a is not None else None


def down(d, dtype, shape):
    return d.download(dtype, int(np.prod(shape))).reshape(shape)


def same(a, b):
    return np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8))


def rope(rows, hd):
    a = np.arange(rows)[:, None] * 500000.0 ** (-2.0 * np.arange(hd // 2) / hd)[None, :]
    return np.cos(a).astype(F32), np.sin(a).astype(F32)


def tables(rng, batch, mbps, npool):
    return rng.permutation(npool)[:batch * mbps].reshape(batch, mbps).astype(np.int32)


# ------------------------------------------------------------------ append

def append(pools, table, qkv, gains, eps, co, si, seq, slot, rpos, heads, half, stream=None):
    """The call, on copies: q [rows, heads * hd] and the pools after it."""
    rows, hd, kvh = slot.size, pools.hd, pools.kvheads
    dk, dv, dq = up(pools.k), up(pools.v), nlgpu.DeviceArray(rows * heads * hd * 4)
    nlgpu.qk_norm_rope_append_paged_q8(up(qkv), up(gains[0]), up(gains[1]), eps, up(co), up(si), co.shape[0], up(slot),
                                       up(table), pools.npool, dq, dk, dv, rows, table.shape[0], heads, kvh, hd,
                                       pools.bs, table.shape[1], seq=up(seq), rpos=up(rpos), half=half, fmt=pools.fmt,
                                       stream=stream)
    nlgpu.sync(stream)
    out = pools.copy()
    out.k, out.v = down(dk, np.uint8, pools.k.shape), down(dv, np.uint8, pools.v.shape)
    return down(dq, F32, (rows, heads * hd)), out


def append_ref(pools, table, qkv, gains, eps, co, si, seq, slot, rpos, heads, half):
    rows, hd, kvh = slot.size, pools.hd, pools.kvheads
    x = qkv.astype(np.float64).reshape(rows, heads + 2 * kvh, hd)
    at = slot if rpos is None else rpos
    eps = float(F32(eps))  # the call's argument is a 32-bit number
    ok = (at >= 0) & (at < co.shape[0])
    c, s = (np.where(ok[:, None], t[np.where(ok, at, 0)], 0).astype(np.float64)[:, None] for t in (co, si))
    with np.errstate(invalid="ignore", over="ignore"):
        q = ref.norm_rope(x[:, :heads], gains[0], eps, c, s, half)
        k = ref.norm_rope(x[:, heads:heads + kvh], gains[1], eps, c, s, half)
    out = pools.copy()
    for which, y in (("k", k), ("v", x[:, heads + kvh:])):
        codes, scale = ref.quantise(y, pools.fmt)
        for r in range(rows):
            out.write(table, r if seq is None else int(seq[r]), int(slot[r]), which, codes[r], scale[r])
    return q.reshape(rows, -1), out


def check_append(*args):
    got_q, got = append(*args)
    want_q, want = append_ref(*args)
    # one rounding to 32 bits of a value that 64-bit sums leave 2^-50 off
    with np.errstate(invalid="ignore", over="ignore"):
        want32 = want_q.astype(F32)
        step = np.spacing(np.abs(want32))
    fine = np.isfinite(want32)
    assert np.array_equal(np.isnan(got_q), np.isnan(want32))
    assert np.array_equal(got_q[~fine & ~np.isnan(want32)], want32[~fine & ~np.isnan(want32)])
    assert (np.abs(got_q[fine].astype(np.float64) - want_q[fine]) <= 0.51 * step[fine] +
            2.0 ** -48 * np.abs(want_q[fine]).max(initial=0)).all()
    assert same(got.k, want.k) and same(got.v, want.v)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,batch,heads,kvh,hd,bs,mbps,gains", [
    (1, 1, 20, 5, 128, 16, 4, "qk"), (37, 3, 32, 8, 128, 32, 3, "qk"), (130, 4, 6, 2, 64, 48, 2, "q"),
    (9, 9, 1, 1, 64, 16, 1, ""), (65, 2, 3, 3, 128, 16, 5, "k"), (200, 2, 8, 1, 64, 64, 2, "qk")])
def test_append(fmt, half, rows, batch, heads, kvh, hd, bs, mbps, gains):
    rng = np.random.default_rng(rows + hd + fmt)
    pools = ref.Pools(batch * mbps + 2, kvh, hd, bs, fmt, fill=0x5a)
    cap = bs * mbps
    where = rng.permutation(batch * cap)[:rows]
    seq, slot = (where // cap).astype(np.int32), (where % cap).astype(np.int32)
    qkv = (rng.standard_normal((rows, (heads + 2 * kvh) * hd)) * np.exp(rng.uniform(-6, 6, (rows, 1)))).astype(F32)
    co, si = rope(cap, hd)
    g = [rng.uniform(0.5, 1.5, hd).astype(F32) if w in gains else None for w in "qk"]
    check_append(pools, tables(rng, batch, mbps, pools.npool), qkv, g, 1e-6, co, si, seq, slot, None, heads, half)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("hd", [64, 128])
def test_append_out_of_range(fmt, hd):
    """Rows that cache nothing (padding, past the table, another sequence, no block), rotations past the tables, rows
    of zeros, with a NaN, an infinity, values past f32 once normed; everything else is left as it was."""
    rng = np.random.default_rng(hd)
    heads, kvh, bs, mbps, batch = 4, 2, 16, 3, 3
    pools = ref.Pools(12, kvh, hd, bs, fmt, fill=0xa5)
    table = tables(rng, batch, mbps, 12)
    table[1, 1], table[2, 0], table[2, 2] = -1, 12, 2 ** 31 - 1
    seq = np.array([0, 0, 1, 1, 2, 2, 2, 3, -1, 0, 0, 0, 0, 0, 0], np.int32)
    slot = np.array([-1, 48, 20, 5, 3, 17, 40, 0, 0, 7, 8, 9, 10, 11, -2 ** 31], np.int32)
    rpos = np.array([0, 1, 2, 3, 4, 5, 6, 7, 8, -1, 100, 99, 2, 3, 4], np.int32)
    qkv = rng.standard_normal((seq.size, (heads + 2 * kvh) * hd)).astype(F32)
    qkv[3] = 0
    qkv[5, 1], qkv[5, (heads + 1) * hd + 3], qkv[5, -1] = np.nan, np.nan, np.inf
    qkv[12, heads * hd:] *= F32(1e-42)
    qkv[13, heads * hd:] *= F32(1e37)
    co, si = rope(100, hd)
    gain = np.full(hd, 3e38, F32)
    for g in ([None, None], [gain, gain]):
        check_append(pools, table, qkv, g, 0.0 if g[0] is None else 1e-6, co, si, seq, slot, rpos, heads, False)
        check_append(pools, table, qkv, g, 0.0 if g[0] is None else 1e-6, co, si, seq, slot, rpos, heads, True)
    rows = slice(9, 12)  # without seq: row r is sequence r
    check_append(pools, table, qkv[rows], [gain, None], 1e-6, co, si, None, slot[rows], None, heads, True)


def test_append_whole_steps():
    """Quotients that lie on the border between two codes are rounded to even, whatever the scale."""
    hd, kvh = 64, 1
    for fmt, top in ((ref.I8, 127.0), (ref.E4M3, 448.0)):
        pools = ref.Pools(1, kvh, hd, 16, fmt)
        qkv = np.zeros((16, 3 * hd), F32)
        for r, s in enumerate([1, 2, 3, 5, 7, 11, 0.75, 96, 1 / 1024, 13, 17, 19, 21, 23, 25, 27]):
            v = np.concatenate([[top], np.arange(hd - 1) - 30.5]) * s
            qkv[r, hd:2 * hd] = qkv[r, 2 * hd:] = v.astype(F32)
        co, si = np.ones((16, hd // 2), F32), np.zeros((16, hd // 2), F32)
        slot = np.arange(16, dtype=np.int32)
        check_append(pools, np.zeros((1, 1), np.int32), qkv, [None, None], 0.0, co, si, np.zeros(16, np.int32), slot,
                     None, 1, False)


# ------------------------------------------------------------------ read-back

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kvh,hd,bs,mbps", [(5, 128, 16, 4), (1, 64, 48, 2), (8, 64, 32, 3)])
def test_read(fmt, kvh, hd, bs, mbps):
    """Every byte pattern, scales among them, comes back as its value rounded to fp16; absent rows as zeros."""
    rng = np.random.default_rng(hd + fmt)
    batch, npool = 3, 3 * mbps + 1
    pools = ref.Pools(npool, kvh, hd, bs, fmt)
    for p in (pools.k, pools.v):
        p[..., :16 * hd] = rng.integers(0, 256, p[..., :16 * hd].shape)
        s = np.exp(rng.uniform(-15, 5, p.shape[:3] + (16,))).astype(F32)
        s[0, 0, 0, 3] = np.nan
        p[..., 16 * hd:] = s.view(np.uint8)
    table = tables(rng, batch, mbps, npool)
    table[1, 0], table[2, 1] = -3, npool
    cap = bs * mbps
    seq = np.repeat(np.arange(-1, batch + 1), cap + 2).astype(np.int32)
    slot = np.tile(np.arange(-1, cap + 1), batch + 2).astype(np.int32)
    order = rng.permutation(seq.size)
    for n in (seq.size, 1, 17):
        s, t = np.ascontiguousarray(seq[order][:n]), np.ascontiguousarray(slot[order][:n])
        dk, dv = nlgpu.DeviceArray(n * kvh * hd * 2), nlgpu.DeviceArray(n * kvh * hd * 2)
        nlgpu.cache_read_paged_q8(up(pools.k), up(pools.v), up(t), up(table), npool, dk, dv, n, batch, kvh, hd, bs, mbps,
                                  seq=up(s), fmt=fmt)
        for which, d in (("k", dk), ("v", dv)):
            got = down(d, np.float16, (n, kvh, hd))
            with np.errstate(over="ignore", invalid="ignore"):
                want = np.stack([pools.row(table, int(b), int(p), which) if b >= 0 else np.zeros((kvh, hd))
                                 for b, p in zip(s, t)]).astype(F32).astype(np.float16)
            assert np.array_equal(got, want, equal_nan=True)
    n = batch  # without seq: row r is sequence r
    dk, dv = nlgpu.DeviceArray(n * kvh * hd * 2), nlgpu.DeviceArray(n * kvh * hd * 2)
    nlgpu.cache_read_paged_q8(up(pools.k), up(pools.v), up(np.full(n, 21, np.int32)), up(table), npool, dk, dv, n, batch,
                              kvh, hd, bs, mbps, fmt=fmt)
    want = np.stack([pools.row(table, b, 21, "v") for b in range(n)]).astype(F32).astype(np.float16)
    assert np.array_equal(down(dv, np.float16, (n, kvh, hd)), want, equal_nan=True)


# ------------------------------------------------------------------ attention

def cached(rng, lengths, kvh, hd, bs, mbps, fmt, sigma=1.0):
    """Pools whose positions below `lengths` hold rows and all others bytes 0xff (e4m3 NaN codes, NaN scales)."""
    batch = len(lengths)
    pools = ref.Pools(batch * mbps + 1, kvh, hd, bs, fmt, fill=0xff)
    table = tables(rng, batch, mbps, pools.npool)
    for b, n in enumerate(lengths):
        pools.fill_rows(table, b, range(min(max(n, 0), bs * mbps)), rng, sigma)
    return pools, table


def decode(pools, table, q, lens, stream=None, dev=None):
    batch, heads = q.shape[0], q.shape[1] // pools.hd
    kvh, hd, bs, mbps = pools.kvheads, pools.hd, pools.bs, table.shape[1]
    out = nlgpu.DeviceArray(q.nbytes).upload(np.full(q.shape, 7.0, F32))
    ws = nlgpu.DeviceArray(max(16, nlgpu.decode_attn_paged_q8_workspace(batch, heads, kvh, hd, bs, mbps)))
    ws.upload(np.full(ws.nbytes // 4, np.nan, F32))
    nlgpu.decode_attn_paged_q8(up(q), up(pools.k), up(pools.v), up(lens), up(table), pools.npool, out, batch, heads, kvh,
                               hd, bs, mbps, ws, fmt=pools.fmt)
    return down(out, F32, q.shape)


def close(got, q, k, v, seen, label):
    """One query row [heads * hd] within its tolerance of the 64-bit result."""
    hd = k.shape[2]
    want, vmax, amp = ref.attend(q.reshape(-1, hd), k, v, seen)
    err = np.abs(got.reshape(-1, hd).astype(np.float64) - want).max(axis=1)
    tol = ref.tolerance(int(seen.sum()), vmax, amp)
    assert np.isfinite(got).all() and (err <= tol).all(), (label, err.max(), tol[err.argmax()])


def check_decode(pools, table, q, lens):
    got = decode(pools, table, q, lens)
    cap = table.shape[1] * pools.bs
    for b in range(q.shape[0]):
        n = min(max(int(lens[b]) + 1, 0), cap)
        k, v = pools.rows(table, b, n, "k"), pools.rows(table, b, n, "v")
        close(got[b], q[b], k, v, np.ones(n, bool), ("sequence", b, "of", n))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kvh,hd,bs,mbps,lens", [
    (20, 5, 128, 16, 48, [0, 14, 15, 16, 62, 63, 64, 255, 256, 600, 767, -1]),
    (32, 8, 128, 64, 20, [1279, 700]), (16, 16, 64, 16, 9, [143, 1, 130]), (8, 2, 64, 32, 5, [159, 33, 95, 5000]),
    (3, 1, 128, 48, 6, [287, 47, 48]), (24, 1, 64, 16, 30, [479, 200]), (40, 1, 128, 16, 20, [319, 3]),
    (1, 1, 64, 16, 1, [0]), (10, 2, 128, 16, 70, [1119])])
def test_decode(fmt, heads, kvh, hd, bs, mbps, lens):
    rng = np.random.default_rng(heads + hd + fmt)
    pools, table = cached(rng, [n + 1 for n in lens], kvh, hd, bs, mbps, fmt)
    q = (rng.standard_normal((len(lens), heads * hd)) * 2).astype(F32)
    check_decode(pools, table, q, np.array(lens, np.int32))


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_pages(fmt):
    """Blocks outside the pool read as zero rows; sequences share a prefix; entries behind the length are not read."""
    rng = np.random.default_rng(8)
    heads, kvh, hd, bs, mbps = 8, 2, 128, 32, 12
    pools, table = cached(rng, [384, 384, 300, 70], kvh, hd, bs, mbps, fmt)
    table[1, :4] = table[0, :4]
    table[0, 5], table[1, 0], table[2, 7] = -1, pools.npool, 2 ** 31 - 1
    table[3, 3:] = -1
    q = rng.standard_normal((4, heads * hd)).astype(F32)
    check_decode(pools, table, q, np.array([383, 370, 299, 69], np.int32))


@pytest.mark.parametrize("fmt", FORMATS)
def test_decode_magnitudes(fmt):
    """Sharp and flat scores, rows of very different sizes, heads of very different queries, zero rows, a zero query."""
    rng = np.random.default_rng(9)
    heads, kvh, hd, bs, mbps = 16, 4, 128, 16, 40
    pools, table = cached(rng, [640, 500], kvh, hd, bs, mbps, fmt)
    for p in range(0, 640, 7):
        pools.fill_rows(table, 0, [p], rng, sigma=float(np.exp(rng.uniform(-4, 4))))
    zero = np.zeros((kvh, hd), np.uint8), np.zeros(kvh, F32)
    for p in (3, 64, 65, 499):
        pools.write(table, 1, p, "k", *zero)
        pools.write(table, 1, p, "v", *zero)
    q = (rng.standard_normal((2, heads, hd)) * np.exp(rng.uniform(-8, 3, (2, heads, 1)))).astype(F32)
    q[1, 3], q[0, 0] = 0, q[0, 0] * F32(1e-30)
    check_decode(pools, table, q.reshape(2, -1), np.array([639, 499], np.int32))


def test_decode_not_a_number():
    """A cached row that is no number, and a query that holds one, reach the rows that attend them and no others."""
    rng = np.random.default_rng(10)
    heads, kvh, hd, bs, mbps = 8, 2, 64, 16, 20
    pools, table = cached(rng, [320, 320], kvh, hd, bs, mbps, ref.E4M3)
    c, s = ref.quantise(np.full((kvh, hd), np.nan), ref.E4M3)
    s[1] = 0  # the second kv head's row is fine
    pools.write(table, 0, 100, "k", c, s)
    q = rng.standard_normal((2, heads, hd)).astype(F32)
    q[1, 5, 7] = np.inf
    q[1, 6, 7] = np.nan
    got = decode(pools, table, q.reshape(2, -1), np.array([319, 319], np.int32)).reshape(2, heads, hd)
    bad = np.zeros((2, heads), bool)
    bad[0, :4] = bad[1, 5] = bad[1, 6] = True
    assert np.array_equal(np.isnan(got).all(axis=2), bad) and np.array_equal(np.isnan(got).any(axis=2), bad)
    got = decode(pools, table, q.reshape(2, -1), np.array([99, 10], np.int32)).reshape(2, heads, hd)
    assert not np.isnan(got[0]).any()  # past its length


def tree(pools, table, q, base, nodes, mask, dout=None, stream=None):
    batch, tmax = q.shape[:2]
    kvh, hd, bs, mbps = pools.kvheads, pools.hd, pools.bs, table.shape[1]
    heads = q.shape[2] // hd
    out = nlgpu.DeviceArray(q.nbytes).upload(np.full(q.shape, 7.0, F32))
    ws = nlgpu.DeviceArray(max(16, nlgpu.tree_attn_paged_q8_workspace(batch, tmax, heads, kvh, hd, bs, mbps)))
    ws.upload(np.full(ws.nbytes // 4, np.nan, F32))
    nlgpu.tree_attn_paged_q8(up(q), up(pools.k), up(pools.v), up(base), up(table), pools.npool, out, batch, tmax, heads,
                             kvh, hd, bs, mbps, ws, nodes=up(nodes), mask=up(mask), fmt=pools.fmt, stream=stream)
    nlgpu.sync(stream)
    return down(out, F32, q.shape)


def check_tree(pools, table, q, base, nodes, mask, rows=None):
    got = tree(pools, table, q, base, nodes, mask)
    batch, tmax = q.shape[:2]
    cap = table.shape[1] * pools.bs
    for b in range(batch):
        nn = min(max(tmax if nodes is None else int(nodes[b]), 0), tmax) if base[b] >= 0 else 0
        end = min(int(base[b]) + nn, cap) if nn else 0
        k, v = pools.rows(table, b, end, "k"), pools.rows(table, b, end, "v")
        at = np.arange(end) - int(base[b])
        for i in range(tmax):
            if i >= nn:
                assert (got[b, i] == 7.0).all()
                continue
            if rows is not None and i not in rows:
                continue
            bit = at <= i if mask is None else np.array([j < 0 or bool(int(mask[b, i]) >> int(j) & 1) for j in at], bool)
            close(got[b, i], q[b, i], np.nan_to_num(k), np.nan_to_num(v), bit[:end], (b, i, nn, end))


def words(rng, batch, tmax):
    """Trees: each node attends itself and its ancestors."""
    m = np.zeros((batch, tmax), np.uint64)
    for b in range(batch):
        for i in range(tmax):
            p = i - 1 - int(rng.integers(0, 5))
            m[b, i] = (m[b, p] if p >= 0 else np.uint64(0)) | np.uint64(1) << np.uint64(i)
    return m


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kvh,hd,bs,mbps,tmax,base,nodes", [
    (20, 5, 128, 16, 24, 16, [300, 17, 0, 47], [16, 1, 5, 9]), (32, 8, 128, 32, 9, 64, [200, 33], [64, 63]),
    (8, 8, 64, 16, 20, 33, [250, 240, -1, 5], [33, 2, 3, 0]), (8, 1, 64, 48, 4, 7, [185, 60], None),
    (6, 2, 128, 16, 40, 1, [600, 63, 64], None), (5, 1, 64, 16, 4, 50, [0, 1], [50, 44])])
def test_tree(fmt, heads, kvh, hd, bs, mbps, tmax, base, nodes):
    rng = np.random.default_rng(tmax + hd + fmt)
    batch = len(base)
    full = [b + (tmax if nodes is None else nodes[i]) for i, b in enumerate(base)]
    pools, table = cached(rng, full, kvh, hd, bs, mbps, fmt)
    q = (rng.standard_normal((batch, tmax, heads * hd)) * 2).astype(F32)
    n = None if nodes is None else np.array(nodes, np.int32)
    check_tree(pools, table, q, np.array(base, np.int32), n, words(rng, batch, tmax))


@pytest.mark.parametrize("fmt", FORMATS)
def test_tree_masks(fmt):
    """Rows that attend nothing are zero; bits past the nodes count for nothing; arbitrary masks; a masked row that is
    no number stays out of the others'."""
    rng = np.random.default_rng(3)
    heads, kvh, hd, bs, mbps, tmax = 8, 2, 128, 16, 6, 20
    pools, table = cached(rng, [20, 60, 36], kvh, hd, bs, mbps, fmt)
    mask = rng.integers(0, 1 << 63, (3, tmax), dtype=np.uint64) | np.uint64(1 << 63)
    mask[0, 3] = mask[0, 7] = 0
    mask[0, 4] = np.uint64(1 << 63)
    c, s = ref.quantise(np.full((kvh, hd), np.inf), fmt)
    for which in "kv":
        pools.write(table, 1, 45, which, c, s)
    mask[1] &= ~np.uint64(1 << 5)  # position 45 is node 5
    q = rng.standard_normal((3, tmax, heads * hd)).astype(F32)
    base, nodes = np.array([0, 40, 17], np.int32), np.array([20, 20, 19], np.int32)
    check_tree(pools, table, q, base, nodes, mask)
    assert (tree(pools, table, q, base, nodes, mask)[0, [3, 4, 7]] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("huge", [1e4, 1e9, 1e17])
@pytest.mark.parametrize("heads,kvh,hd,tmax,base", [(4, 2, 64, 12, 0), (8, 2, 64, 6, 70), (8, 2, 64, 20, 1000),
                                                    (8, 1, 64, 30, 130), (2, 2, 128, 9, 1200), (20, 5, 128, 16, 61)])
def test_masked_rows_of_any_size(fmt, huge, heads, kvh, hd, tmax, base):
    """V rows, however large, that a node does not attend (another branch's, a later token's) leave its output alone:
    the tolerance is of the rows attended."""
    rng = np.random.default_rng(tmax)
    bs, mbps = 16, (base + tmax + 15) // 16
    pools, table = cached(rng, [base + tmax], kvh, hd, bs, mbps, fmt)
    big = tmax // 2
    for i, f in ((big, huge), (big + 1, huge ** 0.5), (tmax - 1, huge * 100)):
        codes, scale = ref.quantise(rng.standard_normal((kvh, hd)) * f, fmt)
        pools.write(table, 0, base + i, "v", codes, scale)
    q = rng.standard_normal((1, tmax, heads * hd)).astype(F32)
    at = np.array([base], np.int32)
    check_tree(pools, table, q, at, None, None)
    mask = words(rng, 1, tmax)
    mask[0, big + 2:tmax - 1] &= ~np.uint64(3 << big)
    check_tree(pools, table, q, at, None, mask)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kvh,hd,bs,mbps,tmax,base,nodes", [
    (20, 5, 128, 16, 24, 130, [200, 0, 17], [130, 129, 3]), (8, 8, 64, 16, 20, 97, [100, 3], None),
    (4, 1, 128, 32, 30, 300, [600, 0], [300, 257]), (2, 2, 64, 16, 80, 1200, [0], None)])
def test_causal_chunk(fmt, heads, kvh, hd, bs, mbps, tmax, base, nodes):
    rng = np.random.default_rng(tmax + hd)
    batch = len(base)
    full = [b + (tmax if nodes is None else nodes[i]) for i, b in enumerate(base)]
    pools, table = cached(rng, full, kvh, hd, bs, mbps, fmt)
    q = (rng.standard_normal((batch, tmax, heads * hd)) * 2).astype(F32)
    rows = set(rng.integers(0, tmax, 40).tolist()) | {0, 1, 2, 15, 16, 63, 64, 127, 128, tmax - 1}
    check_tree(pools, table, q, np.array(base, np.int32), None if nodes is None else np.array(nodes, np.int32), None,
               rows)


def test_tree_past_the_table():
    """Nodes whose positions lie past the block table have no rows; those below it are attended."""
    rng = np.random.default_rng(4)
    heads, kvh, hd, bs, mbps, tmax = 4, 2, 64, 16, 4, 12
    pools, table = cached(rng, [64, 64], kvh, hd, bs, mbps, ref.I8)
    q = rng.standard_normal((2, tmax, heads * hd)).astype(F32)
    for mask in (None, words(rng, 2, tmax)):
        check_tree(pools, table, q, np.array([58, 64], np.int32), None, mask)


def test_one_node_is_a_decoded_token():
    """A tree of one node gives the decode attention's bits."""
    rng = np.random.default_rng(5)
    heads, kvh, hd, bs, mbps = 20, 5, 128, 16, 40
    pools, table = cached(rng, [640, 77], kvh, hd, bs, mbps, ref.I8)
    q = rng.standard_normal((2, heads * hd)).astype(F32)
    last = np.array([639, 76], np.int32)
    want = decode(pools, table, q, last)
    for mask in (None, np.ones((2, 1), np.uint64)):
        got = tree(pools, table, q[:, None], last, None, mask)[:, 0]
        assert np.abs(got - want).max() <= 1e-6 * np.abs(want).max()


# ------------------------------------------------------------------ commit

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kvh,hd,bs,mbps,tmax", [(8, 128, 16, 6, 64), (2, 64, 48, 2, 31), (1, 64, 16, 3, 1)])
def test_commit(fmt, kvh, hd, bs, mbps, tmax):
    """Rising paths, any order, entries twice and out of range, accepted counts past tmax, absent blocks."""
    rng = np.random.default_rng(tmax)
    batch, npool = 7, 7 * mbps + 1
    pools = ref.Pools(npool, kvh, hd, bs, fmt)
    pools.k[:], pools.v[:] = (rng.integers(0, 256, pools.k.shape) for _ in "kv")
    table = tables(rng, batch, mbps, npool)
    table[4, 1] = -1
    base = np.array([0, 5, 16, 30, 3, -1, bs * mbps - 2], np.int32)
    path = rng.integers(0, tmax, (batch, tmax)).astype(np.int32)
    path[0] = np.sort(path[0])
    path[1] = rng.permutation(tmax)
    path[3, ::3], path[3, 1::3] = -1, tmax
    accepted = np.array([tmax, tmax, max(1, tmax // 2), tmax + 9, tmax, tmax, tmax], np.int32)
    want = pools.copy()
    for b in range(batch):
        if base[b] < 0:
            continue
        for i in range(min(int(accepted[b]), tmax)):
            p = int(path[b, i])
            if not 0 <= p < tmax or pools.find(table, b, int(base[b]) + i) is None:
                continue
            for which in "kv":
                row = pools.raw(table, b, int(base[b]) + p, which)
                if row is not None:
                    want.write(table, b, int(base[b]) + i, which, *row)
    dk, dv = up(pools.k), up(pools.v)
    nlgpu.tree_commit_paged_q8(dk, dv, up(base), up(path), up(accepted), up(table), npool, batch, tmax, kvh, hd, bs, mbps)
    assert same(down(dk, np.uint8, pools.k.shape), want.k) and same(down(dv, np.uint8, pools.v.shape), want.v)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("fmt", FORMATS)
def test_a_drafting_run(fmt):
    """Two prompts enter the cache and attend themselves, trees are drafted, verified and committed, a token is
    decoded: every attention within its tolerance, and the cache at the end byte for byte that of the accepted tokens
    appended one after the other."""
    rng = np.random.default_rng(12)
    heads, kvh, hd, bs, mbps, batch, tmax = 8, 2, 128, 16, 8, 2, 12
    h = heads + 2 * kvh
    co, si = rope(bs * mbps, hd)
    gains = [rng.uniform(0.5, 1.5, hd).astype(F32) for _ in "qk"]
    pools = ref.Pools(batch * mbps, kvh, hd, bs, fmt, fill=0xff)
    table = tables(rng, batch, mbps, pools.npool)
    prompt = [37, 50]
    x = rng.standard_normal((sum(prompt), h * hd)).astype(F32)
    seq = np.repeat(np.arange(batch), prompt).astype(np.int32)
    slot = np.concatenate([np.arange(n) for n in prompt]).astype(np.int32)
    start = (pools, table, x, gains, 1e-6, co, si, seq, slot, None, heads, True)
    check_append(*start)
    q, pools = append(*start)
    qq = np.zeros((batch, max(prompt), heads * hd), F32)
    for b in range(batch):
        qq[b, :prompt[b]] = q[seq == b]
    check_tree(pools, table, qq, np.zeros(batch, np.int32), np.array(prompt, np.int32), None, {0, 1, 15, 16, 36, 49})
    # trees: depth behind the context is the rotation's position
    mask = words(rng, batch, tmax)
    depth = np.array([[bin(int(w)).count("1") - 1 for w in r] for r in mask])
    base = np.array(prompt, np.int32)
    draft = rng.standard_normal((batch * tmax, h * hd)).astype(F32)
    seq = np.repeat(np.arange(batch), tmax).astype(np.int32)
    slot = (base[:, None] + np.arange(tmax)).reshape(-1).astype(np.int32)
    rpos = (base[:, None] + depth).reshape(-1).astype(np.int32)
    before = pools.copy()
    step = (pools, table, draft, gains, 1e-6, co, si, seq, slot, rpos, heads, True)
    check_append(*step)
    q, pools = append(*step)
    check_tree(pools, table, q.reshape(batch, tmax, -1), base, None, mask)
    # the path to each sequence's deepest node is accepted
    path, accepted = np.zeros((batch, tmax), np.int32), np.zeros(batch, np.int32)
    for b in range(batch):
        nodes = [j for j in range(tmax) if int(mask[b, depth[b].argmax()]) >> j & 1]
        path[b, :len(nodes)], accepted[b] = nodes, len(nodes)
    dk, dv = up(pools.k), up(pools.v)
    nlgpu.tree_commit_paged_q8(dk, dv, up(base), up(path), up(accepted), up(table), pools.npool, batch, tmax, kvh, hd, bs,
                               mbps)
    pools.k, pools.v = down(dk, np.uint8, pools.k.shape), down(dv, np.uint8, pools.v.shape)
    rows = [b * tmax + path[b, i] for b in range(batch) for i in range(accepted[b])]
    seq = np.repeat(np.arange(batch), accepted).astype(np.int32)
    slot = np.concatenate([base[b] + np.arange(accepted[b]) for b in range(batch)]).astype(np.int32)
    _, straight = append(before, table, draft[rows], gains, 1e-6, co, si, seq, slot, None, heads, True)
    for b in range(batch):
        for p in range(int(base[b] + accepted[b])):
            for which in "kv":
                one, two = pools.raw(table, b, p, which), straight.raw(table, b, p, which)
                assert same(one[0], two[0]) and same(one[1], two[1])
    # the next token
    last = (base + accepted).astype(np.int32)
    token = (pools, table, rng.standard_normal((batch, h * hd)).astype(F32), gains, 1e-6, co, si, None, last, None, heads,
             True)
    check_append(*token)
    q, pools = append(*token)
    check_decode(pools, table, q, last)


def test_blocks_copied():
    """nlg_block_copy_f16 moves blocks of 8-bit pools, given kvheads * (hd + 4) / 2 as its row."""
    rng = np.random.default_rng(6)
    pools = ref.Pools(9, 3, 64, 32, ref.I8)
    pools.k[:], pools.v[:] = (rng.integers(0, 256, pools.k.shape) for _ in "kv")
    dk, dv = up(pools.k), up(pools.v)
    nlgpu.block_copy_f16(dk, dv, up(np.array([2, 7, 0, 8], np.int32)), 2, 9, 32, 3 * 68 // 2)
    for p in (pools.k, pools.v):
        p[7], p[8] = p[2], p[0]
    assert same(down(dk, np.uint8, pools.k.shape), pools.k) and same(down(dv, np.uint8, pools.v.shape), pools.v)


def test_captured():
    """A step (append, attention over two chunks, tree, commit, read) captured into a graph and replayed between eager
    calls on the same buffers gives the eager call's bits each time, at lengths that change on the device."""
    rng = np.random.default_rng(7)
    heads, kvh, hd, bs, mbps, batch, tmax, fmt = 20, 5, 128, 16, 24, 3, 8, ref.E4M3
    pools, table = cached(rng, [384] * batch, kvh, hd, bs, mbps, fmt)
    co, si = rope(bs * mbps, hd)
    st = nlgpu.lib().nlg_stream_create()
    d = {"qkv": up(rng.standard_normal((batch, (heads + 2 * kvh) * hd)).astype(F32)), "co": up(co), "si": up(si),
         "k": up(pools.k), "v": up(pools.v), "table": up(table), "at": nlgpu.DeviceArray(4 * batch),
         "q": nlgpu.DeviceArray(batch * heads * hd * 4), "out": nlgpu.DeviceArray(batch * heads * hd * 4),
         "tq": up(rng.standard_normal((batch, tmax, heads * hd)).astype(F32)),
         "tout": nlgpu.DeviceArray(batch * tmax * heads * hd * 4), "mask": up(words(rng, batch, tmax)),
         "path": up(np.tile(np.array([1, 3, 4, 0, 0, 0, 0, 0], np.int32), (batch, 1))),
         "acc": up(np.full(batch, 3, np.int32)), "rk": nlgpu.DeviceArray(batch * kvh * hd * 2),
         "rv": nlgpu.DeviceArray(batch * kvh * hd * 2)}
    ws = nlgpu.DeviceArray(nlgpu.decode_attn_paged_q8_workspace(batch, heads, kvh, hd, bs, mbps))
    wt = nlgpu.DeviceArray(nlgpu.tree_attn_paged_q8_workspace(batch, tmax, heads, kvh, hd, bs, mbps))
    size = (heads, kvh, hd, bs, mbps)

    def step():
        nlgpu.qk_norm_rope_append_paged_q8(d["qkv"], None, None, 1e-6, d["co"], d["si"], bs * mbps, d["at"], d["table"],
                                           pools.npool, d["q"], d["k"], d["v"], batch, batch, *size, fmt=fmt, stream=st)
        nlgpu.decode_attn_paged_q8(d["q"], d["k"], d["v"], d["at"], d["table"], pools.npool, d["out"], batch, *size, ws,
                                   fmt=fmt, stream=st)
        nlgpu.tree_attn_paged_q8(d["tq"], d["k"], d["v"], d["at"], d["table"], pools.npool, d["tout"], batch, tmax, *size,
                                 wt, mask=d["mask"], fmt=fmt, stream=st)
        nlgpu.tree_commit_paged_q8(d["k"], d["v"], d["at"], d["path"], d["acc"], d["table"], pools.npool, batch, tmax,
                                   *size[1:], stream=st)
        nlgpu.cache_read_paged_q8(d["k"], d["v"], d["at"], d["table"], pools.npool, d["rk"], d["rv"], batch, batch,
                                  *size[1:], fmt=fmt, stream=st)

    def run(go, at):
        for n, a in (("k", pools.k), ("v", pools.v), ("at", np.array(at, np.int32))):
            d[n].upload(a)
        for n in ("q", "out", "tout", "rk", "rv"):
            d[n].zero(st)
        go()
        nlgpu.sync(st)
        return [d[n].download(np.uint8) for n in ("q", "out", "tout", "k", "v", "rk", "rv")]

    nlgpu.graph_begin(st)
    step()
    g = nlgpu.graph_end(st)
    for at in ([370, 5, 256], [0, 300, 255], [370, 5, 256], [17, 17, 17]):
        eager = run(step, at)
        for _ in range(2):
            assert all(same(a, b) for a, b in zip(run(lambda: nlgpu.graph_launch(g, st), at), eager))
    nlgpu.graph_destroy(g)
    nlgpu.lib().nlg_stream_destroy(st)


def test_two_streams():
    """Calls that overlap on two streams, each with its own workspace, give the bits of calls alone."""
    rng = np.random.default_rng(8)
    heads, kvh, hd, bs, mbps, batch = 32, 8, 128, 16, 64, 4
    pools, table = cached(rng, [300, 1000, 77, 512], kvh, hd, bs, mbps, ref.I8)
    lens = up(np.array([299, 999, 76, 511], np.int32))
    dk, dv, dt = up(pools.k), up(pools.v), up(table)
    qs = [rng.standard_normal((batch, heads * hd)).astype(F32) for _ in range(2)]
    want = [decode(pools, table, q, np.array([299, 999, 76, 511], np.int32)) for q in qs]
    streams = [nlgpu.lib().nlg_stream_create() for _ in qs]
    need = nlgpu.decode_attn_paged_q8_workspace(batch, heads, kvh, hd, bs, mbps)
    dq, ws = [up(q) for q in qs], [nlgpu.DeviceArray(need) for _ in qs]
    outs = [[nlgpu.DeviceArray(qs[0].nbytes) for _ in range(20)] for _ in qs]
    for r in range(20):
        for i, st in enumerate(streams):
            nlgpu.decode_attn_paged_q8(dq[i], dk, dv, lens, dt, pools.npool, outs[i][r], batch, heads, kvh, hd, bs, mbps,
                                       ws[i], stream=st)
    for st in streams:
        nlgpu.sync(st)
    for i in range(2):
        assert all(same(down(o, F32, qs[0].shape), want[i]) for o in outs[i])
    for st in streams:
        nlgpu.lib().nlg_stream_destroy(st)


def test_offsets_past_four_gib():
    """Blocks whose bytes lie past 2^32 of a pool."""
    rng = np.random.default_rng(11)
    heads, kvh, hd, bs, mbps, fmt = 4, 1, 64, 16, 6, ref.I8
    tile = 16 * (hd + 4)
    npool = (1 << 32) // tile + 64
    assert nlgpu.kv_q8_pool_bytes(npool, kvh, hd, bs) == npool * tile > 1 << 32
    small = ref.Pools(mbps, kvh, hd, bs, fmt)
    local = np.arange(mbps, dtype=np.int32)[None]
    small.fill_rows(local, 0, range(90), rng)
    table = (local + npool - mbps).astype(np.int32)
    dk, dv = nlgpu.DeviceArray(npool * tile), nlgpu.DeviceArray(npool * tile)
    for d, p in ((dk, small.k), (dv, small.v)):
        d.upload(p, offset=(npool - mbps) * tile)
    qkv = rng.standard_normal((1, (heads + 2 * kvh) * hd)).astype(F32)
    co, si = rope(96, hd)
    slot = np.array([90], np.int32)
    dq, out = nlgpu.DeviceArray(heads * hd * 4), nlgpu.DeviceArray(heads * hd * 4)
    nlgpu.qk_norm_rope_append_paged_q8(up(qkv), None, None, 0.0, up(co), up(si), 96, up(slot), up(table), npool, dq, dk,
                                       dv, 1, 1, heads, kvh, hd, bs, mbps)
    nlgpu.decode_attn_paged_q8(dq, dk, dv, up(slot), up(table), npool, out, 1, heads, kvh, hd, bs, mbps, None)
    q, want = append_ref(small, local, qkv, [None, None], 0.0, co, si, None, slot, None, heads, False)
    for d, p in ((dk, want.k), (dv, want.v)):
        assert same(d.download(np.uint8, mbps * tile, offset=(npool - mbps) * tile), p.reshape(-1))
    close(down(out, F32, (heads * hd,)), q[0].astype(F32), want.rows(local, 0, 91, "k"), want.rows(local, 0, 91, "v"),
          np.ones(91, bool), "far blocks")
    path = np.full((1, 64), 50, np.int32)  # the row at 40 + 50 goes to 40
    nlgpu.tree_commit_paged_q8(dk, dv, up(np.array([40], np.int32)), up(path), up(np.array([1], np.int32)), up(table),
                               npool, 1, 64, kvh, hd, bs, mbps)
    rk, rv = nlgpu.DeviceArray(2 * hd * 2), nlgpu.DeviceArray(2 * hd * 2)
    nlgpu.cache_read_paged_q8(dk, dv, up(np.array([40, 90], np.int32)), up(table), npool, rk, rv, 2, 1, kvh, hd, bs, mbps,
                              seq=up(np.zeros(2, np.int32)))
    for d, which in ((rk, "k"), (rv, "v")):
        row = want.row(local, 0, 90, which).astype(F32).astype(np.float16)
        assert np.array_equal(down(d, np.float16, (2, hd)), np.concatenate([row, row]))


# ------------------------------------------------------------------ how the work is laid out

@pytest.mark.parametrize("batch,tmax,heads,kvh,hd", [(150, 1, 8, 2, 64), (70, 5, 8, 2, 64), (65, 17, 4, 2, 128)])
def test_many_sequences(batch, tmax, heads, kvh, hd):
    """More sequences than a wave has lanes, few of them long: the layout is counted over several rounds of 64."""
    rng = np.random.default_rng(batch)
    bs, mbps = 16, 70
    base = rng.integers(-1, 90, batch)
    base[[0, 63, 64, batch - 1]] = [1119 - tmax, 700, 1100 - tmax, 300]
    pools, table = cached(rng, base + tmax, kvh, hd, bs, mbps, ref.I8)
    if tmax == 1:
        q = rng.standard_normal((batch, heads * hd)).astype(F32)
        check_decode(pools, table, q, base.astype(np.int32))
        return
    q = rng.standard_normal((batch, tmax, heads * hd)).astype(F32)
    nodes = rng.integers(0, tmax + 1, batch).astype(np.int32)
    nodes[[0, 63, 64]] = tmax
    check_tree(pools, table, q, base.astype(np.int32), nodes, words(rng, batch, tmax), rows=(0, tmax - 1))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tmax", [1, 40])
def test_long_chunks(fmt, tmax):
    """So many kv heads that a chunk of one sequence is longer than the 1,024 positions whose tiles a wave looks up at
    once; five heads are compared."""
    rng = np.random.default_rng(13 + tmax)
    kvh, hd, bs, n = 256, 64, 16, 2350
    pools = ref.Pools(150, kvh, hd, bs, fmt)
    table = rng.permutation(150)[:148].reshape(1, 148).astype(np.int32)
    for p in (pools.k, pools.v):
        c = rng.integers(0, 255, p.shape[:3] + (16 * hd,)).astype(np.uint8)
        # (any int8 but -128; any e4m3 but the NaN codes, and none over 30)
        c = np.where(c == 0x80, 0, c) if fmt == ref.I8 else (c & 0x80) | (c & 0x7f) % 0x5f
        p[..., :16 * hd] = c
        s = rng.uniform(0.5, 1.5, p.shape[:3] + (16,)) / (74.0 if fmt == ref.I8 else 8.0)
        p[..., 16 * hd:] = np.ascontiguousarray(s.astype(F32)).view(np.uint8)
    q = rng.standard_normal((1, tmax, kvh * hd)).astype(F32)
    base = np.array([n - tmax], np.int32)
    got = decode(pools, table, q[0], base)[None] if tmax == 1 else tree(pools, table, q, base, None, None)
    some = [0, 1, 100, 254, 255]
    part = ref.Pools(150, len(some), hd, bs, fmt)
    part.k, part.v = (np.ascontiguousarray(p[:, some]) for p in (pools.k, pools.v))
    k, v = (part.rows(table, 0, n, w) for w in "kv")
    for i in {0, tmax // 2, tmax - 1}:
        g, x = (t[0, i].reshape(kvh, hd)[some].reshape(-1) for t in (got, q))
        close(g, x, k, v, np.arange(n) <= n - tmax + i, (i, n))


@pytest.mark.parametrize("fmt,hd,bs,mbps", [(ref.I8, 64, 16, 1 << 15), (ref.E4M3, 128, 64, 1 << 12)])
def test_table_of_many_blocks(fmt, hd, bs, mbps):
    """A table whose positions would be over 256 MB, of which few have blocks: those without one are zero rows."""
    rng = np.random.default_rng(mbps)
    heads, kvh, batch = 16, 4, 2
    n = 1280 // bs
    pools = ref.Pools(2 * n, kvh, hd, bs, fmt, fill=0xff)
    table = np.full((batch, mbps), -1, np.int32)
    table[:, :n] = rng.permutation(2 * n).reshape(2, n)
    lens = np.array([1279, 1500], np.int32)
    for b in range(batch):
        pools.fill_rows(table, b, range(1280), rng)
    assert batch * mbps * bs * kvh * 2 * (hd + 4) > 1 << 28
    check_decode(pools, table, rng.standard_normal((batch, heads * hd)).astype(F32), lens)


def test_two_graphs_of_one_workspace():
    """Two captured calls that share a workspace, replayed in turn on one stream, give the bits of calls alone."""
    rng = np.random.default_rng(17)
    heads, kvh, hd, bs, mbps, batch = 20, 5, 128, 16, 80, 3
    lens = np.array([1250, 30, 800], np.int32)
    pools, table = cached(rng, lens + 1, kvh, hd, bs, mbps, ref.I8)
    qs = [rng.standard_normal((batch, heads * hd)).astype(F32) for _ in range(2)]
    want = [decode(pools, table, q, lens) for q in qs]
    st = nlgpu.lib().nlg_stream_create()
    dk, dv, dt, dl = up(pools.k), up(pools.v), up(table), up(lens)
    need = nlgpu.decode_attn_paged_q8_workspace(batch, heads, kvh, hd, bs, mbps)
    ws, dq, outs = nlgpu.DeviceArray(need), [up(q) for q in qs], [nlgpu.DeviceArray(q.nbytes) for q in qs]
    assert need > 0
    graphs = []
    for i in range(2):
        nlgpu.graph_begin(st)
        nlgpu.decode_attn_paged_q8(dq[i], dk, dv, dl, dt, pools.npool, outs[i], batch, heads, kvh, hd, bs, mbps, ws,
                                   stream=st)
        graphs.append(nlgpu.graph_end(st))
    for _ in range(3):
        for o in outs:
            o.zero(st)
        for g in graphs:
            nlgpu.graph_launch(g, st)
        nlgpu.sync(st)
        assert all(same(down(o, F32, w.shape), w) for o, w in zip(outs, want))
    for g in graphs:
        nlgpu.graph_destroy(g)
    nlgpu.lib().nlg_stream_destroy(st)
