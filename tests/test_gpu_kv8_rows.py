"""The 8-bit paged KV cache's forms for many rows (read-back in sixteens, queries
stored past the caches), V rows that are no number, and one node against one
decoded token."""
import numpy as np
import pytest

import kv8_ref as ref
import nlgpu
from test_gpu_kv8 import F32, FORMATS, cached, check_append, decode, down, rope, same, tables, tree, up, words

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def read_back(pools, table, seq, slot):
    n, kvh, hd = slot.size, pools.kvheads, pools.hd
    shape = (n, kvh, hd)
    # (a guard behind each: the last group of sixteen rows is not whole)
    dk, dv = (nlgpu.DeviceArray(n * kvh * hd * 2 + 64).upload(np.full(n * kvh * hd + 32, 0x5a5a, np.uint16)) for _ in "kv")
    nlgpu.cache_read_paged_q8(up(pools.k), up(pools.v), up(slot), up(table), pools.npool, dk, dv, n, table.shape[0], kvh,
                              hd, pools.bs, table.shape[1], seq=up(seq), fmt=pools.fmt)
    out = []
    for d in (dk, dv):
        got = d.download(np.uint16, n * kvh * hd + 32)
        assert (got[n * kvh * hd:] == 0x5a5a).all()
        out.append(got[:n * kvh * hd].view(np.float16).reshape(shape))
    return out


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kvh,hd,bs", [(16, 128, 16), (24, 64, 48), (40, 128, 32)])
@pytest.mark.parametrize("order", ["rising", "falling", "shuffled"])
def test_read_many(fmt, kvh, hd, bs, order):
    """At least 16,384 head rows: sequences that end inside a group of sixteen rows, in order or not, rows out of range
    and without a block at the first and last places of groups, a last group that is not whole."""
    rng = np.random.default_rng(kvh + fmt)
    lengths, batch, npool = [501, 37, 16, 470, 1, 44], 6, 160
    mbps = 512 // bs + 1
    pools = ref.Pools(npool, kvh, hd, bs, fmt)
    for p in (pools.k, pools.v):
        p[..., :16 * hd] = rng.integers(0, 256, p[..., :16 * hd].shape)
        s = np.exp(rng.uniform(-15, 3, p.shape[:3] + (16,))).astype(F32)
        p[..., 16 * hd:] = s.view(np.uint8)
    table = rng.integers(0, npool, (batch, mbps)).astype(np.int32)
    table[0, 3], table[3, 0], table[3, 5] = -1, npool, 2 ** 31 - 1
    seq = np.repeat(np.arange(batch), lengths)
    slot = np.concatenate([np.arange(n) for n in lengths])
    if order == "falling":
        seq, slot = seq[::-1], slot[::-1]
    if order == "shuffled":
        p = rng.permutation(seq.size)
        seq, slot = seq[p], slot[p]
    seq, slot = seq.astype(np.int32), slot.astype(np.int32)
    n = seq.size
    assert n * kvh >= 16384 and n % 16
    for at, (b, p) in {0: (0, -1), 15: (batch, 3), 32: (-1, 5), 47: (2, bs * mbps), 64: (1, 2 ** 31 - 1),
                       n - 1: (1, -2 ** 31)}.items():
        seq[at], slot[at] = b, p
    got = read_back(pools, table, seq, slot)
    with np.errstate(over="ignore", invalid="ignore"):
        for which, g in zip("kv", got):
            want = np.stack([pools.row(table, int(b), int(p), which) if 0 <= b < batch else np.zeros((kvh, hd))
                             for b, p in zip(seq, slot)]).astype(F32).astype(np.float16)
            bad = np.flatnonzero(~((g == want) | (np.isnan(g) & np.isnan(want))).all(axis=(1, 2)))
            assert not bad.size, (which, bad[:8])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kvh,hd,half", [(32, 1, 128, True), (64, 2, 64, False)])
def test_append_past_the_caches(fmt, heads, kvh, hd, half):
    """Queries of more than 32 MiB."""
    rng = np.random.default_rng(heads)
    rows, batch, bs, mbps = 2075, 3, 16, 44
    assert rows * heads * hd * 4 > 32 << 20
    pools = ref.Pools(batch * mbps + 2, kvh, hd, bs, fmt, fill=0x5a)
    where = rng.permutation(batch * bs * mbps)[:rows]
    seq, slot = (where // (bs * mbps)).astype(np.int32), (where % (bs * mbps)).astype(np.int32)
    qkv = rng.standard_normal((rows, (heads + 2 * kvh) * hd)).astype(F32)
    co, si = rope(bs * mbps, hd)
    gains = [rng.uniform(0.5, 1.5, hd).astype(F32) for _ in "qk"]
    check_append(pools, tables(rng, batch, mbps, pools.npool), qkv, gains, 1e-6, co, si, seq, slot, None, heads, half)


# heads, kv heads, head dim, queries, positions: as in one launch, chunks, 32 rows, 64 and 128 rows to a workgroup
LAYOUTS = [(20, 5, 128, 1, 300), (8, 2, 64, 1, 1300), (8, 2, 64, 6, 700), (8, 2, 128, 20, 400), (8, 2, 64, 40, 1300)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", ["first", "middle", "last"])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_a_value_that_is_no_number(fmt, bad, heads, kvh, hd, tmax, n):
    """V of one position and of kv head 0 is no number, its K is: the queries that attend it give NaN in that kv head's
    heads, and all else is what it is without it."""
    rng = np.random.default_rng(n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    q = rng.standard_normal((1, tmax, heads * hd)).astype(F32)
    base = np.array([n - tmax], np.int32)
    pos = {"first": 0, "middle": n // 2, "last": n - 1 - tmax // 2}[bad]
    mask = words(rng, 1, tmax)
    runs = [lambda: decode(pools, table, q[0], base)[None]] if tmax == 1 else \
        [lambda: tree(pools, table, q, base, None, None), lambda: tree(pools, table, q, base, None, mask)]
    want = [r().reshape(tmax, heads, hd) for r in runs]
    c, s = pools.raw(table, 0, pos, "v")
    c[0], s[0] = 0, np.nan
    pools.write(table, 0, pos, "v", c, s)
    for r, w in zip(runs, want):
        got = r().reshape(tmax, heads, hd)
        node = pos - (n - tmax)
        none = np.zeros((tmax, heads), bool)
        for i in range(tmax):
            on = node < 0 or (bool(int(mask[0, i]) >> node & 1) if r is not runs[0] else i >= node)
            none[i, :heads // kvh] = on
        assert none.any() and not none.all()
        assert np.isnan(got[none]).all() and same(got[~none], w[~none])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kvh,hd,bs,mbps,last", [(20, 5, 128, 16, 40, [639, 76]), (8, 2, 64, 32, 60, [1900, 5])])
def test_one_node_and_one_token(fmt, heads, kvh, hd, bs, mbps, last):
    """A tree of one node and the decode attention give the same bits."""
    rng = np.random.default_rng(5)
    pools, table = cached(rng, [n + 1 for n in last], kvh, hd, bs, mbps, fmt)
    q = rng.standard_normal((len(last), heads * hd)).astype(F32)
    at = np.array(last, np.int32)
    want = decode(pools, table, q, at)
    for mask in (None, np.ones((len(last), 1), np.uint64)):
        assert same(tree(pools, table, q[:, None], at, None, mask)[:, 0], want)
