"""The ternary linear with adapters where its projection splits the columns: everything of a call is in its workspace, so
graphs captured on one stream may be replayed on others, beside each other and beside eager calls on that stream."""
import numpy as np
import pytest

import lora_ref as ref
import nlgpu
from test_gpu_lora import Case, close, up

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


# 22 tiles of 17 chunks in four slices, with tiles of adapters and a wave a row; 160 tiles in three
CASES = [dict(lengths=[100, 200, 33], adapter=[0, -1, 1], adapters=2, rmax=128, out=300, cols=4352, mixed=True),
         dict(lengths=[60, 100, 40], adapter=[1, 0, -1], adapters=2, rmax=16, out=257, cols=4096),
         dict(lengths=[400, 100], adapter=[0, 1], adapters=2, rmax=32, out=2560, cols=4096)]


class Call:
    """A call's arguments, outputs and workspace on the device."""

    def __init__(self, c):
        rng = np.random.default_rng(c.seq)
        self.c, self.words = c, nlgpu.pack_ternary(nlgpu.trits(c.out, (c.out, c.cols)))
        self.beta = rng.uniform(0.01, 0.05, 1).astype(F32)
        self.d = {k: up(getattr(c, k)) for k in ("x", "a16", "b16", "scale", "adapter", "start", "rank")}
        self.d.update(w=up(self.words), beta=up(self.beta))
        self.y = nlgpu.DeviceArray(4 * c.seq * c.out)
        need = nlgpu.ternary_linear_lora_workspace(c.seq, c.out, c.cols, c.rmax, len(c.adapter))
        assert need - nlgpu.lora_linear_workspace(c.seq, c.out, c.cols, c.rmax, len(c.adapter)) > 2 * c.seq * c.cols
        self.ws = up(np.full(need, 0xA5, np.uint8))  # (nothing in it may be taken for zero)

    def go(self, stream=None):
        c, d = self.c, self.d
        nlgpu.ternary_linear_lora(d["x"], d["w"], None, d["beta"], d["a16"], d["b16"], d["scale"], d["adapter"], self.y,
                                  c.seq, c.out, c.cols, c.n, c.rmax, len(c.adapter), self.ws, start=d["start"],
                                  rank=d["rank"], fmt=c.fmt, stream=stream)

    def base(self):
        c, d = self.c, self.d
        y, ws = nlgpu.DeviceArray(4 * c.seq * c.out), nlgpu.DeviceArray(nlgpu.ternary_linear_workspace(c.seq, c.cols))
        nlgpu.ternary_linear(d["x"], d["w"], None, d["beta"], y, c.seq, c.out, c.cols, workspace=ws)
        nlgpu.sync()
        return y.download(F32).reshape(c.seq, c.out)

    def bits(self):
        return self.y.download(np.uint32)


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_values(i, bf):
    c = Case(bf=bf, **CASES[i])
    call = Call(c)
    base = call.base()
    want = ref.forward(c.x.astype(float), c.a, c.b, c.scale.astype(float), c.rank, c.of, ref.Sums(base.astype(float)))[0]
    for _ in range(2):  # (the second finds the counters as the first left them)
        call.y.zero()
        call.go()
        nlgpu.sync()
        y = call.y.download(F32).reshape(c.seq, c.out)
        close(y, want, "y")
        assert np.array_equal(y[c.of < 0], base[c.of < 0])


@pytest.mark.parametrize("i", range(len(CASES)))
def test_graphs_of_one_stream_replayed_on_two(i):
    calls = [Call(Case(**{**CASES[i], "seed": k})) for k in range(3)]
    want = []
    for call in calls:
        call.go()
        nlgpu.sync()
        want.append(call.bits())
    assert not np.array_equal(want[0], want[1])
    lib = nlgpu.lib()
    st = [lib.nlg_stream_create() for _ in range(3)]
    graphs = []
    for call in calls[:2]:  # both captured on stream 0
        nlgpu.graph_begin(st[0])
        call.go(st[0])
        graphs.append(nlgpu.graph_end(st[0]))
    for _ in range(4):
        for call in calls:
            call.y.zero()
            call.ws.upload(np.full(call.ws.nbytes, 0xA5, np.uint8))
        nlgpu.sync()
        for _ in range(6):
            nlgpu.graph_launch(graphs[0], st[1])
            nlgpu.graph_launch(graphs[1], st[2])
            calls[2].go(st[0])
        for s in st:
            nlgpu.sync(s)
        for call, w in zip(calls, want):
            assert np.array_equal(call.bits(), w)
    for g in graphs:
        nlgpu.graph_destroy(g)
    for s in st:
        lib.nlg_stream_destroy(s)
