"""That the rows' scale beside the adapters is the quotient of their largest value and 127, and no product with 127's
reciprocal: values that lie on a border of the int8 codes by the one and not by the other, and the projection's bits."""
import numpy as np
import pytest

import loss_ref
import nlgpu

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def codes(x, g):
    return np.floor((np.abs((x / g).astype(F32)) + F32(0.5)).astype(F32))


def rows_on_borders(n, cols, seed):
    """Rows whose scale by the reciprocal is another number, with a value in column 1 whose code then is another too."""
    rng = np.random.default_rng(seed)
    top = rng.uniform(1, 2, 400000).astype(F32)
    g, h = top / F32(127), top * (F32(1) / F32(127))
    top = top[g != h]
    g, h = (top / F32(127))[:, None], (top * (F32(1) / F32(127)))[:, None]
    v = ((rng.integers(1, 126, (top.size, 1)) + 0.5) * g).astype(F32)
    steps = (v.view(np.int32) + np.arange(-3, 4, dtype=np.int32)).view(F32)  # its neighbours
    differ = codes(steps, g) != codes(steps, h)
    at = np.flatnonzero(differ.any(axis=1))[:n]
    assert at.size == n
    x = np.zeros((n, cols), F32)
    x[:, 0], x[:, 1] = top[at], steps[at, differ[at].argmax(axis=1)]
    return x


# a wave a row and tiles, on both layouts of the columns
@pytest.mark.parametrize("rows,out,cols,rmax", [(1, 40, 256, 16), (64, 40, 256, 16), (333, 300, 4352, 64), (600, 520, 704, 64),
                                                (500, 701, 1024, 64)])
def test_scale_is_a_quotient(rows, out, cols, rmax):
    x = rows_on_borders(rows, cols, rows)
    w = np.zeros((out, cols), np.int64)
    w[:, 0], w[:, 1] = np.arange(out) % 2, 1  # the code of column 1 alone, and with that of column 0
    rng = np.random.default_rng(out)
    beta = rng.uniform(0.5, 1, out).astype(F32)
    n = 3
    up = nlgpu.to_device
    y = up(np.full((rows, out), np.nan, F32))
    d = dict(x=x, w=nlgpu.pack_ternary(w), beta=beta, a=np.zeros((n, rmax, cols), np.uint16),
             b=np.zeros((n, out, rmax), np.uint16), scale=np.ones(n, F32), adapter=np.arange(2).astype(np.int32),
             start=np.array([0, rows // 2, rows], np.int32))
    d = {k: up(v) for k, v in d.items()}
    ws = nlgpu.DeviceArray(nlgpu.ternary_linear_lora_workspace(rows, out, cols, rmax, 2))
    nlgpu.ternary_linear_lora(d["x"], d["w"], None, d["beta"], d["a"], d["b"], d["scale"], d["adapter"], y, rows, out, cols, n,
                              rmax, 2, ws, start=d["start"], beta_per_row=True)
    nlgpu.sync()
    q, g = loss_ref.quantise(x)
    assert np.array_equal(np.abs(q[:, 1]), codes(x[:, 1:2], x[:, :1] / F32(127))[:, 0])
    want = (beta[None, :] * g).astype(F32) * (q @ w.T).astype(F32)
    assert np.array_equal(y.download(F32).reshape(rows, out), want)
