"""That rows and gradients keep their 24 bits, and f16 adapters their eleven, on the bf16 matrix cores: outputs that are one
product each, within the bounds of lora_parts.py, which the sums miss without any one of the parts' products."""
import numpy as np
import pytest

import nlgpu
from lora_parts import H, Singles, product
from test_gpu_lora import up

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def near(got, factors, off, name):
    want = 1.0
    for f in factors:
        want = want * f.astype(float)
    bad = np.abs(got.reshape(want.shape).astype(float) - want) > off * np.abs(want)
    assert not bad.any(), (name, bad.sum(), np.argwhere(bad)[:3])


def forward(c, ternary):
    """y and u; the ternary linear's weights are zeros, so that y is the adapters' alone."""
    y, u = up(np.full((c.seq, c.out), np.nan, F32)), up(np.full((c.seq, c.rmax), np.nan, F32))
    d = {k: up(getattr(c, k)) for k in ("x", "a16", "b16", "scale", "adapter", "start", "rank")}
    fmt, n = nlgpu.LORA_BF16 if c.bf else nlgpu.LORA_F16, len(c.adapter)
    if ternary:
        w, beta = up(np.zeros((c.out, c.cols // 16), np.uint32)), up(np.ones(1, F32))
        ws = nlgpu.DeviceArray(nlgpu.ternary_linear_lora_workspace(c.seq, c.out, c.cols, c.rmax, n))
        nlgpu.ternary_linear_lora(d["x"], w, None, beta, d["a16"], d["b16"], d["scale"], d["adapter"], y, c.seq, c.out, c.cols,
                                  c.n, c.rmax, n, ws, start=d["start"], rank=d["rank"], u=u, fmt=fmt)
    else:
        ws = nlgpu.DeviceArray(nlgpu.lora_linear_workspace(c.seq, c.out, c.cols, c.rmax, n))
        nlgpu.lora_linear(d["x"], d["a16"], d["b16"], d["scale"], d["adapter"], None, y, c.seq, c.out, c.cols, c.n, c.rmax, n,
                          ws, start=d["start"], rank=d["rank"], u=u, fmt=fmt)
    nlgpu.sync()
    return y.download(F32).reshape(c.seq, c.out), u.download(F32).reshape(c.seq, c.rmax)


# each width of the ranks on the way down in tiles; a wave a row
BESIDE = [dict(lengths=[1000, 1100], rmax=8, out=100, cols=8200), dict(lengths=[400, 700], rmax=24, out=200, cols=5000),
          dict(lengths=[333, 367], rmax=64, out=300, cols=2904), dict(lengths=[250, 250], rmax=128, out=140, cols=2008),
          dict(lengths=[30, 31], rmax=40, out=50, cols=616)]
# with the ternary linear, whose epilogue adds the adapters: split columns, tiles of 64 and 32 rows, rows of 64s in both
TERNARY = [dict(lengths=[100, 233], rmax=128, out=300, cols=4352), dict(lengths=[513, 700], rmax=16, out=6700, cols=256),
           dict(lengths=[300, 200], rmax=64, out=701, cols=1024), dict(lengths=[1000, 1000], rmax=8, out=2560, cols=4096),
           dict(lengths=[600, 1200], rmax=24, out=4000, cols=704), dict(lengths=[150, 160], rmax=128, out=1000, cols=576)]


def test_the_cases_take_tiles():
    size = lambda c: sum(c["lengths"]) * c["rmax"] * (c["cols"] + c["out"])  # noqa: E731
    assert [size(c) > 1 << 27 for c in BESIDE] == [True] * 4 + [False]
    assert all(size(c) > 3 << 24 for c in TERNARY)


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(BESIDE) + len(TERNARY)))
def test_forward(i, bf):
    c = Singles(adapters=2, bf=bf, **(BESIDE + TERNARY)[i])
    y, u = forward(c, i >= len(BESIDE))
    near(u, c.down_factors(), product(bf), "u")
    # the product, the scale, and what it is added to (zeros)
    near(y, c.up_factors(u), product(bf) + 2 * H, "y")


# one pass over dy at each width of the ranks, whole vectors and not; a pass for du alone past 64 ranks
BACK = [dict(lengths=[90, 151], rmax=8, out=512, cols=64), dict(lengths=[90, 151], rmax=8, out=301, cols=72),
        dict(lengths=[200, 300], rmax=24, out=700, cols=136), dict(lengths=[200, 300], rmax=32, out=333, cols=136),
        dict(lengths=[150, 90], rmax=64, out=260, cols=64), dict(lengths=[150, 90], rmax=56, out=515, cols=64),
        dict(lengths=[300, 333], rmax=104, out=1000, cols=64), dict(lengths=[300, 333], rmax=128, out=777, cols=80)]


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(BACK)))
def test_backward(i, bf):
    c = Singles(adapters=2, bf=bf, **BACK[i])
    d = {k: up(getattr(c, k)) for k in ("x", "dy", "a16", "b16", "scale", "adapter", "start", "rank")}
    dx, da, db = (up(np.full(s, np.nan, F32)) for s in (c.x.shape, c.a.shape, c.b.shape))
    n = len(c.adapter)
    ws = nlgpu.DeviceArray(nlgpu.lora_linear_grad_workspace(c.seq, c.out, c.cols, c.n, c.rmax, n))
    nlgpu.lora_linear_grad(d["x"], None, d["dy"], d["a16"], d["b16"], d["scale"], d["adapter"], da, db, c.seq, c.out, c.cols,
                           c.n, c.rmax, n, ws, dx=dx, start=d["start"], rank=d["rank"],
                           fmt=nlgpu.LORA_BF16 if bf else nlgpu.LORA_F16)
    nlgpu.sync()
    dv, b, scale, a = c.back_factors()
    # du's product and scale, A's product in 32 bits
    near(dx.download(F32), (dv[:, None], b[:, None], scale[:, None], a), (product(bf) + 2 * H) * (1 + 4 * H), "dx")
