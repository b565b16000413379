"""The ternary linear with adapters over weights with a registered tiled copy: the row layout's bits, in every form that
adds the adapters in the projection's epilogue or beside it, eager and captured."""
import numpy as np
import pytest

import nlgpu
from test_gpu_lora import Case, same, up

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


# split columns, tiles of 64 and of 32 rows, with tiles of adapters and a wave a row; the forms of fewer rows
CASES = [dict(lengths=[100, 200, 33], adapter=[0, -1, 1], adapters=2, rmax=128, out=300, cols=4352, mixed=True),
         dict(lengths=[60, 100, 40], adapter=[1, 0, -1], adapters=2, rmax=16, out=257, cols=4096),
         dict(lengths=[513, 700], adapter=[1, 0], adapters=2, rmax=16, out=6700, cols=256, first=5),
         dict(lengths=[300, 200], adapter=[1, 0], adapters=2, rmax=64, out=701, cols=1024, behind=3),
         dict(lengths=[130, 20], adapter=[0, 1], adapters=2, rmax=8, out=330, cols=512),
         dict(lengths=[60, 68], adapter=[1, 0], adapters=2, rmax=128, out=2560, cols=2560),
         dict(lengths=[60, 40], adapter=[1, 0], adapters=2, rmax=128, out=2001, cols=2048),
         dict(lengths=[1] * 9, adapter=[i % 3 - 1 for i in range(9)], adapters=2, rmax=24, out=100, cols=768),
         dict(lengths=[1, 1], adapter=[0, 1], adapters=2, rmax=16, out=64, cols=256)]


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_the_row_layouts_bits(i, bf):
    c = Case(bf=bf, **CASES[i])
    n = len(c.adapter)
    rng = np.random.default_rng(c.seq)
    d = {k: up(getattr(c, k)) for k in ("x", "a16", "b16", "scale", "adapter", "start", "rank")}
    w, beta = up(nlgpu.pack_ternary(nlgpu.trits(c.out, (c.out, c.cols)))), up(rng.uniform(0.01, 0.05, c.out).astype(F32))
    bias = up(rng.standard_normal(c.out).astype(F32))
    ws = nlgpu.DeviceArray(nlgpu.ternary_linear_lora_workspace(c.seq, c.out, c.cols, c.rmax, n))
    y, u = nlgpu.DeviceArray(4 * c.seq * c.out), nlgpu.DeviceArray(4 * c.seq * c.rmax)
    st = nlgpu.lib().nlg_stream_create()

    def call():
        nlgpu.ternary_linear_lora(d["x"], w, bias, beta, d["a16"], d["b16"], d["scale"], d["adapter"], y, c.seq, c.out, c.cols,
                                  c.n, c.rmax, n, ws, start=d["start"], rank=d["rank"], u=u, fmt=c.fmt, beta_per_row=True,
                                  stream=st)

    def run(go):
        y.zero(st)
        u.zero(st)
        go()
        nlgpu.sync(st)
        return y.download(F32), u.download(F32)

    rows = run(call)
    nlgpu.ternary_tiled_register(w, c.out, c.cols, st)
    tiled = run(call)
    nlgpu.graph_begin(st)
    call()
    g = nlgpu.graph_end(st)
    graph = [run(lambda: nlgpu.graph_launch(g, st)) for _ in range(3)]
    nlgpu.graph_destroy(g)
    nlgpu.ternary_tiled_unregister(w)
    for got in [tiled] + graph + [run(call)]:
        assert all(same(a, b) for a, b in zip(got, rows))
    assert np.isfinite(rows[0]).all() and np.abs(rows[0]).max() > 0
    nlgpu.lib().nlg_stream_destroy(st)
