"""Attention over the 8-bit paged KV cache where sizes lie far apart or near the
ends of the f32 range, against 64 bits and relative to what the output itself is
made of."""
import math

import numpy as np
import pytest

import kv8_ref as ref
import nlgpu
from test_gpu_kv8 import cached, decode, tree, words

pytestmark = pytest.mark.gpu
F32 = np.float32
FORMATS = [ref.I8, ref.E4M3]


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


# heads, kv heads, head dim, queries, positions: one query in one launch and in chunks, its group of 16 rows half
# and quite full; 32 rows sharing waves; 64 and 128 rows to a workgroup, the last with a row's chunks joined by one thread each.
LAYOUTS = [(20, 5, 128, 1, 300), (8, 2, 64, 1, 1300), (32, 2, 128, 1, 64), (8, 2, 64, 6, 700), (8, 2, 128, 20, 400),
           (8, 2, 64, 40, 200), (32, 4, 64, 150, 330)]


def attended(q, k, v):
    """One query head row [hd] over k, v [n, hd]: the output in 64 bits; the weighted sum of the rows' largest |v|; the
    largest root of sum (q k)^2 / hd."""
    qq = q.astype(np.float64)
    s = k @ qq / math.sqrt(q.size)
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, float(p @ np.abs(v).max(axis=1)), float(np.sqrt(((k * qq) ** 2).sum(axis=1) / q.size).max())


def close(got, q, k, v, label):
    """The query row's error against a bound relative to its own products.  Scores, exponentials and sums as in
    kv8_ref.tolerance, but each moves its own product p |v| alone, so their weighted sum stands for the largest |v|.
    A product of a probability and a V scale is two halves, the second with steps of 2^-24: half a step, where the
    row's largest is at least 1, is 2^-25 of it for each of n positions."""
    hd = k.shape[2]
    heads = q.size // hd
    q, got = q.reshape(heads, hd), got.reshape(heads, hd).astype(np.float64)
    n = k.shape[0]
    for h in range(heads):
        g = h // (heads // k.shape[1])
        want, size, amp = attended(q[h], k[:, g], v[:, g])
        tol = 2.0 ** -24 * (150.0 * amp + 64.0 + 4.0 * math.sqrt(n) + n) * size + 2.0 ** -149
        err = np.abs(got[h] - want).max()
        assert np.isfinite(got[h]).all() and err <= tol, (label, h, err, tol, size)


def check(pools, table, q, n):
    """q [1, tmax, heads * hd], the queries at positions n - tmax .. n - 1, as a decoded token, a causal chunk and a
    masked tree."""
    tmax = q.shape[1]
    k, v = pools.rows(table, 0, n, "k"), pools.rows(table, 0, n, "v")
    base = np.array([n - tmax], np.int32)
    if tmax == 1:
        close(decode(pools, table, q[0], base)[0], q[0, 0], k, v, "decode")
        return
    rows = sorted({0, 1, tmax // 2, tmax - 1} | set(range(0, tmax, 7)))
    got = tree(pools, table, q, base, None, None)
    for i in rows:
        close(got[0, i], q[0, i], k[:n - tmax + i + 1], v[:n - tmax + i + 1], ("causal", i))
    if tmax > 64:
        return
    mask = words(np.random.default_rng(1), 1, tmax)
    got = tree(pools, table, q, base, None, mask)
    for i in rows:
        on = np.array([p < n - tmax or int(mask[0, i]) >> (p - n + tmax) & 1 for p in range(n)], bool)
        close(got[0, i], q[0, i], k[on], v[on], ("masked", i))


def put(pools, table, pos, which, row):
    """One position's row [kvheads, hd], quantised."""
    c, s = ref.quantise(row, pools.fmt)
    pools.write(table, 0, pos, which, c, s)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [3e38, 1e37, 1e-20, 1e-30, 1e-35])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_values_of_any_size(fmt, size, heads, kvh, hd, tmax, n):
    """V up to the largest f32 numbers, under flat scores that many positions share: no sum on the way overflows; V of
    next to nothing keeps its bits.  (The largest magnitude of a row is 3/4 of `size`.)"""
    rng = np.random.default_rng(n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    for pos in range(n):
        put(pools, table, pos, "v", rng.uniform(-0.75, 0.75, (kvh, hd)) * size)
    q = (0.1 * rng.standard_normal((1, tmax, heads * hd))).astype(F32)
    check(pools, table, q, n)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("binades", [12, 20, 28, 40, 66, 90])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_large_rows_of_no_weight(fmt, binades, heads, kvh, hd, tmax, n):
    """V rows 2^binades above the others, attended with a probability near 2^-100: the first position, some in the
    middle, the last below the queries."""
    rng = np.random.default_rng(binades + n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    low = 100 * math.log(2) / math.sqrt(hd)
    for pos in {0, n // 3, n // 3 + 1, n - tmax - 1}:
        put(pools, table, pos, "k", np.full((kvh, hd), -low))
        put(pools, table, pos, "v", rng.standard_normal((kvh, hd)) * 2.0 ** binades)
    q = (1 + 0.1 * rng.standard_normal((1, tmax, heads * hd))).astype(F32)
    check(pools, table, q, n)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("nats", [12, 25, 60])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_a_heavy_position_without_value(fmt, nats, heads, kvh, hd, tmax, n):
    """The position that takes nearly all the weight has a V row of zeros (or a tiny one): the output is what the others
    leave."""
    rng = np.random.default_rng(nats + n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    put(pools, table, 0, "k", np.full((kvh, hd), nats / math.sqrt(hd)))
    put(pools, table, 0, "v", np.zeros((kvh, hd)))
    put(pools, table, n // 2, "k", np.full((kvh, hd), nats / math.sqrt(hd)))
    put(pools, table, n // 2, "v", rng.standard_normal((kvh, hd)) * 2.0 ** -90)
    q = (1 + 0.1 * rng.standard_normal((1, tmax, heads * hd))).astype(F32)
    check(pools, table, q, n)


def fill(pools, table, n, which, rows):
    """All n positions of a side: rows [n, kvheads, hd]."""
    c, s = ref.quantise(rows, pools.fmt)
    for pos in range(n):
        pools.write(table, 0, pos, which, c[pos], s[pos])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [3e38, 4e37, 1e30, 1e-30, 1e-35])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_keys_of_any_size(fmt, size, heads, kvh, hd, tmax, n):
    """K of any size with queries that make ordinary scores of it."""
    rng = np.random.default_rng(n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    fill(pools, table, n, "k", rng.uniform(-0.75, 0.75, (n, kvh, hd)) * size)
    q = (rng.standard_normal((1, tmax, heads * hd)) * (6 / size)).astype(F32)
    check(pools, table, q, n)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("sign", [1, -1, 0])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_scores_near_the_end_of_f32(fmt, sign, heads, kvh, hd, tmax, n):
    """Equal scores of 3e38 in base 2, all positive, all negative, or every third positive: the weight is shared by the
    largest.  (K of one magnitude and q of one value: the sums are exact and the scores the same.)"""
    rng = np.random.default_rng(n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    side = np.where(np.arange(n) % 3 == 0, 1.0, -1.0) if sign == 0 else np.full(n, float(sign))
    fill(pools, table, n, "k", np.broadcast_to(side[:, None, None] * 1e38, (n, kvh, hd)))
    q = np.full((1, tmax, heads * hd), 3e38 / (1e38 * math.sqrt(hd) * math.log2(math.e)), F32)
    v = pools.rows(table, 0, n, "v")
    base = np.array([n - tmax], np.int32)
    got = decode(pools, table, q[0], base)[None] if tmax == 1 else tree(pools, table, q, base, None, None)
    for i in {0, tmax // 2, tmax - 1}:
        on = np.flatnonzero(side[:n - tmax + i + 1] == side[0])
        want = v[on].mean(axis=0)
        # as in close(), with weights that are exact
        tol = 2.0 ** -24 * (64.0 + 4.0 * math.sqrt(n) + n) * np.abs(v[on]).max(axis=2).mean(axis=0)
        err = np.abs(got[0, i].reshape(kvh, heads // kvh, hd) - want[:, None]).max(axis=(1, 2))
        assert (err <= tol).all(), (i, err.max(), tol.min())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("binades", [8, 14, 18])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_queries_of_one_large_element(fmt, binades, heads, kvh, hd, tmax, n):
    """An element of q 2^binades above the others, where K is zero: the others make the scores.  They are multiplied as
    two halves whose last step is 2^-24 where the largest is some 2^12: half a step is 2^-37 of it, 2^-19 of an element
    of size 1 at most, against the 2^-24 * 150 amp of the bound, amp about 1; over hd products it grows as the root."""
    rng = np.random.default_rng(n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    k = rng.standard_normal((n, kvh, hd))
    k[:, :, 3] = 0
    fill(pools, table, n, "k", k)
    q = rng.standard_normal((1, tmax, heads, hd))
    q[..., 3] = 2.0 ** binades
    check(pools, table, q.reshape(1, tmax, -1).astype(F32), n)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("small", [1.0, 1e-4, 1e-10, 1e-18])
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", [x for x in LAYOUTS if x[3] > 1])
def test_masked_keys_of_any_size(fmt, small, heads, kvh, hd, tmax, n):
    """K rows near the end of f32 that a node does not attend (another branch's, a later token's) beside ordinary and
    very small ones that it does."""
    rng = np.random.default_rng(n)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    k = rng.standard_normal((n, kvh, hd)) * small
    big = n - tmax // 2
    k[big] = rng.uniform(-3e38, 3e38, (kvh, hd))
    fill(pools, table, n, "k", k)
    q = (rng.standard_normal((1, tmax, heads * hd)) * 3 / small).astype(F32)
    base = np.array([n - tmax], np.int32)
    k, v = pools.rows(table, 0, n, "k"), pools.rows(table, 0, n, "v")
    node = big - (n - tmax)
    got = tree(pools, table, q, base, None, None)
    for i in range(0, node, 3):
        close(got[0, i], q[0, i], k[:n - tmax + i + 1], v[:n - tmax + i + 1], ("causal", i))
    if tmax > 64:
        return
    mask = words(rng, 1, tmax) & ~np.uint64(1 << node)
    got = tree(pools, table, q, base, None, mask)
    for i in range(0, tmax, 3):
        on = np.array([p < n - tmax or int(mask[0, i]) >> (p - n + tmax) & 1 for p in range(n)], bool)
        close(got[0, i], q[0, i], k[on], v[on], ("masked", i))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("heads,kvh,hd,tmax,n", LAYOUTS)
def test_rows_of_all_sizes(fmt, seed, heads, kvh, hd, tmax, n):
    """Each position's K, V and each query of its own random size, over 2^72 for V, scores up to some 60 and next to
    nothing, zero rows among them."""
    rng = np.random.default_rng(100 * n + seed)
    pools, table = cached(rng, [n], kvh, hd, 16, (n + 15) // 16, fmt)
    for which, span in (("k", 4), ("v", 25)):
        rows = rng.standard_normal((n, kvh, hd)) * np.exp(rng.uniform(-span, span if which == "v" else 2, (n, kvh, 1)))
        rows[rng.random(n) < 0.05] = 0
        fill(pools, table, n, which, rows)
    q = rng.standard_normal((1, tmax, heads, hd)) * np.exp(rng.uniform(-3, 1, (1, tmax, heads, 1)))
    check(pools, table, q.reshape(1, tmax, -1).astype(F32), n)
