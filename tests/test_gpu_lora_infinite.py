"""An infinity in a row of x (or of dy) on the GPU: NaN in the row's u (du) and in what follows from it, whichever form the
call's size takes, and the bits of other rows as they are without it."""
import numpy as np
import pytest

import nlgpu
from test_gpu_lora import Case, same, ternary, up

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


# a launch for a few rows, a wave a row, tiles of 32 rows; ranks up to 8, 64 and 128
SHAPES = [dict(lengths=[1], adapter=[0], adapters=1, rmax=16, out=70, cols=136),
          dict(lengths=[1] * 3, adapter=[0, 1, 0], adapters=2, rmax=64, out=65, cols=520),
          dict(lengths=[1] * 12, adapter=[0, 1, 2] * 4, adapters=3, rmax=8, out=70, cols=256),
          dict(lengths=[1] * 150, adapter=[i % 4 for i in range(150)], adapters=4, rmax=64, out=130, cols=1024),
          dict(lengths=[90, 33, 60], adapter=[1, 0, 2], adapters=3, rmax=128, out=100, cols=328),
          dict(lengths=[200, 133, 260], adapter=[1, 0, 2], adapters=3, rmax=104, out=340, cols=2944),
          dict(lengths=[600, 500], adapter=[1, 0], adapters=2, rmax=32, out=520, cols=4096)]


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_infinity_in_a_row(i, value, bf):
    c = Case(bf=bf, **SHAPES[i])
    calls = {"beside": lambda: c.forward(), "with the linear": lambda: ternary(c, False, False)[:2]}
    before = {k: f() for k, f in calls.items()}
    row = c.seq // 2
    rest = np.arange(c.seq) != row
    c.x[row, 5] = value
    for k, f in calls.items():
        for got, old in zip(f(), before[k]):
            got, old = got.reshape(c.seq, -1), old.reshape(c.seq, -1)
            assert np.isnan(got[row]).all(), (k, got[row][:4])
            assert same(got[rest], old[rest]), k


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_infinity_in_a_gradient(i, bf):
    c = Case(bf=bf, **SHAPES[i])
    u = c.forward()[1]
    before = c.backward(u=u)[0].reshape(c.seq, -1)
    row = c.seq // 2
    rest = np.arange(c.seq) != row
    c.dy[row, 5] = -np.inf
    got = c.backward(u=u)[0].reshape(c.seq, -1)
    assert np.isnan(got[row]).all() and same(got[rest], before[rest])


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_infinity_where_u_is_found_again(i):
    """Without u the gradient finds it from x: dB has NaN in the row's adapter alone."""
    c = Case(**SHAPES[i])
    before = c.backward()[2].reshape(c.b.shape)
    row = c.seq // 2
    c.x[row, 5] = np.inf
    got = c.backward()[2].reshape(c.b.shape)
    assert np.isnan(got[c.of[row]]).all()
    others = np.arange(c.n) != c.of[row]
    assert same(got[others], before[others])
