"""That the bounds of single products (lora_parts.py) hold for the parts' sums in 32 bits, and for nothing less: without any
one of the parts' products hundreds of values are out of them."""
import numpy as np
import pytest

import lora_parts as parts

F32 = np.float32


@pytest.mark.parametrize("bf", [False, True])
def test_bounds(bf):
    rng = np.random.default_rng(7)
    x, w = parts.values(rng, 200000, 24).astype(F32), parts.values(rng, 200000, 8 if bf else 11).astype(F32)
    exact = x.astype(float) * w.astype(float)
    bad = lambda got: int((np.abs(got.astype(float) - exact) > parts.product(bf) * np.abs(exact)).sum())  # noqa: E731
    assert bad(parts.parts_product(x, w, bf)) == 0
    for left_out in [(i, 0) for i in range(3)] + ([] if bf else [(0, 1), (1, 1)]):
        assert bad(parts.parts_product(x, w, bf, without=(left_out,))) > 100000, left_out
    # what the sums leave out in earnest: at most 2^-22, 2^-25 of the product on average
    if not bf:
        p, q = parts.split(x, 3), parts.split(w, 2)
        lost = np.abs(p[2].astype(float) * q[1]) / np.abs(exact)
        assert 2.0 ** -23 < lost.max() < 2.0 ** -22 and 2.0 ** -26 < lost.mean() < 2.0 ** -24


def test_singles_are_single():
    c = parts.Singles([30, 41], 2, 16, out=50, cols=40, bf=False)
    want = c.x.astype(float) @ c.a[0].T
    u, w = c.down_factors()
    assert np.array_equal((u.astype(float) * w)[:30], want[:30])
    given = np.random.default_rng(1).standard_normal((c.seq, c.rmax)).astype(F32)
    u, w, sc = c.up_factors(given)
    assert np.array_equal(u.astype(float)[30:] * w[30:], given[30:].astype(float) @ c.b[1].T)
    d, w, sc, a = c.back_factors()
    du = c.dy.astype(float)[:30] @ c.b[0]
    assert np.array_equal((du @ c.a[0]), (d.astype(float) * w)[:30, None] * a[:30])
