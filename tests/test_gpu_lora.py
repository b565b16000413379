"""Low-rank adapters of many requests on the GPU against their form in 64 bits
(lora_ref.py), within the bounds derived there."""
import numpy as np
import pytest

import lora_ref as ref
import nlgpu

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def up(a):
    return nlgpu.to_device(a) if a is not None else None


def close(got, want, name=""):
    off = np.abs(got.astype(np.float64).reshape(want.value.shape) - want.value)
    bad = off > want.off + 2.0 ** -140
    assert not bad.any(), (name, np.argwhere(bad)[:3], off[bad][:3], want.off[bad][:3])


class Case:
    """Requests of the given lengths over rows that begin at `first`, each with its adapter."""

    def __init__(self, lengths, adapter, adapters, rmax, out, cols, bf=False, mixed=False, first=0, behind=0, seed=0):
        rng = np.random.default_rng([sum(lengths), adapters, rmax, out, cols, seed])
        self.start = (first + np.concatenate([[0], np.cumsum(lengths)])).astype(np.int32)
        self.seq, self.out, self.cols = int(self.start[-1]) + behind, out, cols
        self.adapter = np.asarray(adapter, np.int32)
        self.n, self.rmax, self.bf = adapters, rmax, bf
        self.rank = (rng.integers(0, rmax + 1, adapters) if mixed else np.full(adapters, rmax)).astype(np.int32)
        self.scale = rng.uniform(-2, 2, adapters).astype(F32)
        self.a16, self.a = ref.to16(rng.standard_normal((adapters, rmax, cols)) * cols ** -0.5, bf)
        self.b16, self.b = ref.to16(rng.standard_normal((adapters, out, rmax)) * 0.1, bf)
        # what lies behind the ranks is not used: NaN
        for k in range(adapters):
            self.a16[k, self.rank[k]:] = 0x7fff
            self.b16[k, :, self.rank[k]:] = 0x7fff
        self.x = (rng.standard_normal((self.seq, cols)) * np.exp(rng.uniform(-3, 3, (self.seq, 1)))).astype(F32)
        self.dy = (rng.standard_normal((self.seq, out)) * np.exp(rng.uniform(-3, 3, (self.seq, 1)))).astype(F32)
        self.res = rng.standard_normal((self.seq, out)).astype(F32)
        self.dres = rng.standard_normal((self.seq, cols)).astype(F32)
        self.of = ref.owners(self.seq, self.start, self.adapter, adapters)
        self.fmt = nlgpu.LORA_BF16 if bf else nlgpu.LORA_F16

    def forward(self, res=True, inplace=False, keep=True, start=True, stream=None):
        y = up(self.res if inplace else np.full((self.seq, self.out), np.nan, F32))
        u = up(np.full((self.seq, self.rmax), np.nan, F32)) if keep else None
        ws = nlgpu.DeviceArray(nlgpu.lora_linear_workspace(self.seq, self.out, self.cols, self.rmax, len(self.adapter)))
        nlgpu.lora_linear(up(self.x), up(self.a16), up(self.b16), up(self.scale), up(self.adapter),
                          y if inplace else up(self.res) if res else None, y, self.seq, self.out, self.cols, self.n,
                          self.rmax, len(self.adapter), ws, start=up(self.start) if start else None, rank=up(self.rank),
                          u=u, fmt=self.fmt, stream=stream)
        nlgpu.sync(stream)
        return y.download(F32), u.download(F32) if keep else None

    def backward(self, u=None, dres=True, dx=True, inplace=False, stream=None):
        da, db = (up(np.full(s, np.nan, F32)) for s in (self.a.shape, self.b.shape))
        d = up(self.dres if inplace else np.full((self.seq, self.cols), np.nan, F32)) if dx else None
        ws = nlgpu.DeviceArray(nlgpu.lora_linear_grad_workspace(self.seq, self.out, self.cols, self.n, self.rmax,
                                                                len(self.adapter)))
        nlgpu.lora_linear_grad(up(self.x), up(u), up(self.dy), up(self.a16), up(self.b16), up(self.scale),
                               up(self.adapter), da, db, self.seq, self.out, self.cols, self.n, self.rmax,
                               len(self.adapter), ws, dres=d if inplace else up(self.dres) if dres else None, dx=d,
                               start=up(self.start), rank=up(self.rank), fmt=self.fmt, stream=stream)
        nlgpu.sync(stream)
        return d.download(F32) if dx else None, da.download(F32), db.download(F32)

    def want(self, res=True):
        return ref.forward(self.x.astype(float), self.a, self.b, self.scale.astype(float), self.rank, self.of,
                           ref.Sums(self.res.astype(float)) if res else None)

    def want_grad(self, u, dres=True):
        return ref.backward(self.x.astype(float), u, self.dy.astype(float), self.a, self.b, self.scale.astype(float),
                            self.rank, self.of, self.dres if dres else None)


CASES = [dict(lengths=[1], adapter=[0], adapters=1, rmax=8, out=1, cols=8),
         dict(lengths=[1] * 5, adapter=[2, 0, -1, 2, 7], adapters=3, rmax=16, out=257, cols=64, mixed=True),
         dict(lengths=[1] * 70, adapter=[i % 9 for i in range(70)], adapters=9, rmax=64, out=300, cols=264, mixed=True),
         dict(lengths=[17, 0, 40, 3, 1], adapter=[1, 0, 0, -5, 1], adapters=2, rmax=24, out=130, cols=200, first=3, behind=9),
         dict(lengths=[100, 33], adapter=[0, 0], adapters=1, rmax=32, out=256, cols=512),
         dict(lengths=[64, 64, 70], adapter=[3, 1, 3], adapters=5, rmax=128, out=72, cols=1000, mixed=True),
         dict(lengths=[5, 6, 7], adapter=[0, 1, 2], adapters=3, rmax=40, out=333, cols=96, behind=40),
         # long enough for tiles of 32 rows, at each width of the ranks
         dict(lengths=[400, 0, 5, 700, 90], adapter=[1, 0, 2, 0, -1], adapters=3, rmax=8, out=514, cols=14000, mixed=True),
         dict(lengths=[9] * 150, adapter=[i % 7 for i in range(150)], adapters=7, rmax=16, out=1003, cols=5304, first=2, behind=30),
         dict(lengths=[333, 500, 250], adapter=[1, -1, 0], adapters=2, rmax=24, out=260, cols=5000, mixed=True),
         dict(lengths=[4] * 190, adapter=[i % 11 for i in range(190)], adapters=11, rmax=64, out=801, cols=2048, mixed=True),
         dict(lengths=[100, 33, 170], adapter=[0, 2, 1], adapters=3, rmax=128, out=640, cols=2904, behind=3)]


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_forward(i, bf):
    c = Case(bf=bf, **CASES[i])
    y, u = c.forward()
    want, wu = c.want()
    close(u, wu, "u")
    close(y, want, "y")
    assert np.array_equal(c.forward(inplace=True, keep=False)[0], y)  # y = res itself, u in the workspace
    close(c.forward(res=False)[0], c.want(res=False)[0], "alone")


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_backward(i, bf):
    c = Case(bf=bf, **CASES[i])
    u = c.want()[1]
    given = u.value.astype(F32)
    got = c.backward(u=given)
    for g, w, n in zip(got, c.want_grad(ref.Sums(given.astype(float))), ("dx", "da", "db")):
        close(g, w, n)
    for k in range(c.n):  # behind the ranks, and where no row is
        assert not got[1].reshape(c.a.shape)[k, c.rank[k]:].any() and not got[2].reshape(c.b.shape)[k, :, c.rank[k]:].any()
        if not (c.of == k).any():
            assert not got[1].reshape(c.a.shape)[k].any() and not got[2].reshape(c.b.shape)[k].any()
    again = c.backward(u=given, inplace=True)
    assert all(np.array_equal(x, y) for x, y in zip(again, got))
    # u computed again, no dres, no dx
    for g, w, n in zip(c.backward(dres=False), c.want_grad(u, dres=False), ("dx", "da", "db")):
        close(g, w, n)
    assert c.backward(u=given, dx=False)[0] is None


@pytest.mark.parametrize("rmax", [8, 24, 64])
def test_backward_of_long_prompts(rmax):
    """x, dres and dx of more than 128 MiB together: dA and dx in passes of their own."""
    c = Case([300, 0, 411, 2], [1, 0, 0, 1], 2, rmax, out=40, cols=16388 - 4 * 5, mixed=True, first=1, behind=2)
    assert 12 * c.seq * c.cols > 128 << 20
    u = ref.Sums(c.want()[1].value.astype(F32).astype(float))
    got = c.backward(u=u.value.astype(F32))
    for g, w, n in zip(got, c.want_grad(u), ("dx", "da", "db")):
        close(g, w, n)
    again = c.backward(u=u.value.astype(F32), inplace=True)
    assert all(np.array_equal(x, y) for x, y in zip(again, got))
    none = c.of < 0
    assert np.array_equal(got[0].reshape(c.dres.shape)[none], c.dres[none])


# ------------------------------------------------------------------ beside the ternary linear

def ternary(c, per_row, bias, keep=True, stream=None):
    """The whole call on a Case (with weights made here); y, u, and the base alone as nlg_ternary_linear gives it."""
    rng = np.random.default_rng(c.seq + c.out)
    w = nlgpu.pack_ternary(nlgpu.trits(c.out, (c.out, c.cols)))
    beta = rng.uniform(0.01, 0.05, c.out if per_row else 1).astype(F32)
    bo = rng.standard_normal(c.out).astype(F32) if bias else None
    d = {k: up(v) for k, v in dict(x=c.x, w=w, beta=beta, bias=bo).items()}
    base, y = up(np.full((c.seq, c.out), np.nan, F32)), up(np.full((c.seq, c.out), np.nan, F32))
    ws = nlgpu.DeviceArray(max(16, nlgpu.ternary_linear_workspace(c.seq, c.cols)))
    nlgpu.ternary_linear(d["x"], d["w"], d["bias"], d["beta"], base, c.seq, c.out, c.cols, beta_per_row=per_row, workspace=ws)
    nlgpu.sync()
    u = up(np.full((c.seq, c.rmax), np.nan, F32)) if keep else None
    ws = nlgpu.DeviceArray(nlgpu.ternary_linear_lora_workspace(c.seq, c.out, c.cols, c.rmax, len(c.adapter)))
    nlgpu.ternary_linear_lora(d["x"], d["w"], d["bias"], d["beta"], up(c.a16), up(c.b16), up(c.scale), up(c.adapter), y,
                              c.seq, c.out, c.cols, c.n, c.rmax, len(c.adapter), ws, start=up(c.start), rank=up(c.rank),
                              u=u, fmt=c.fmt, beta_per_row=per_row, stream=stream)
    nlgpu.sync(stream)
    return y.download(F32), u.download(F32) if keep else None, base.download(F32).reshape(c.seq, c.out)


# one row; a few; rows of a step; column tiles cut; prompts on the wide kernel (64-token tiles, split columns, one phase)
BESIDE = [dict(lengths=[1], adapter=[0], adapters=1, rmax=16, out=100, cols=256),
          dict(lengths=[1, 1, 1], adapter=[1, -1, 0], adapters=2, rmax=8, out=64, cols=72),
          dict(lengths=[1] * 33, adapter=[i % 5 - 1 for i in range(33)], adapters=4, rmax=40, out=320, cols=512, mixed=True),
          dict(lengths=[1] * 6, adapter=[0, 1] * 3, adapters=2, rmax=16, out=70, cols=192),
          dict(lengths=[40, 60], adapter=[0, 1], adapters=2, rmax=24, out=200, cols=768, mixed=True),
          dict(lengths=[70, 1, 0, 200], adapter=[2, 1, 0, 0], adapters=3, rmax=32, out=520, cols=1024, mixed=True, behind=3),
          dict(lengths=[100, 200, 33], adapter=[0, -1, 1], adapters=2, rmax=128, out=300, cols=4352, mixed=True),
          dict(lengths=[513, 700], adapter=[1, 0], adapters=2, rmax=16, out=6700, cols=256, first=5),
          # rows of 64s: one unit, half a chunk, chunks and a rest; tiles of 32 and of 64 tokens
          dict(lengths=[30, 41], adapter=[0, 1], adapters=2, rmax=16, out=300, cols=64),
          dict(lengths=[200, 0, 90], adapter=[1, 1, 0], adapters=2, rmax=24, out=257, cols=128, behind=4),
          dict(lengths=[1] * 40, adapter=[i % 3 for i in range(40)], adapters=3, rmax=16, out=130, cols=320),
          dict(lengths=[600, 500, 700], adapter=[0, -1, 1], adapters=2, rmax=16, out=4000, cols=704),
          dict(lengths=[1000, 777], adapter=[0, 1], adapters=2, rmax=8, out=4000, cols=1088),
          dict(lengths=[150, 100, 60], adapter=[2, 0, 1], adapters=3, rmax=128, out=1000, cols=576, mixed=True),
          # the other forms of the projection beside tiles of adapters: 32-token tiles, one phase, few tokens
          dict(lengths=[300, 200], adapter=[1, 0], adapters=2, rmax=64, out=701, cols=1024),
          dict(lengths=[60, 68], adapter=[1, 0], adapters=2, rmax=128, out=2560, cols=2560),
          dict(lengths=[60, 40], adapter=[1, 0], adapters=2, rmax=128, out=2001, cols=2048)]


def test_forms_of_the_cases():
    """That the cases are on both sides of what decides between a wave a row and tiles of 32."""
    size = [sum(c["lengths"]) * c["rmax"] * (c["cols"] + c["out"]) for c in CASES]
    assert sum(s > 1 << 27 for s in size) >= 5 and sum(s <= 1 << 27 for s in size) >= 7
    size = [sum(c["lengths"]) * c["rmax"] * (c["cols"] + c["out"]) for c in BESIDE]
    assert sum(s > 3 << 24 for s in size) >= 8 and sum(s <= 3 << 24 for s in size) >= 8


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("i", range(len(BESIDE)))
def test_beside_ternary(i, bf):
    c = Case(bf=bf, **BESIDE[i])
    y, u, base = ternary(c, per_row=i % 2 == 0, bias=i % 3 == 0)
    want, wu = ref.forward(c.x.astype(float), c.a, c.b, c.scale.astype(float), c.rank, c.of, ref.Sums(base.astype(float)))
    close(u, wu, "u")
    close(y, want, "y")
    none = c.of < 0
    assert np.array_equal(y.reshape(c.seq, c.out)[none], base[none])  # the linear's own bits
    assert np.array_equal(ternary(c, i % 2 == 0, i % 3 == 0, keep=False)[0], y)


# ------------------------------------------------------------------ what the documentation allows besides

def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


# the few-row forms, the tiles of 32 rows, both backward forms
SHAPES = [dict(lengths=[1] * 12, adapter=[0, 1, 2] * 4, adapters=3, rmax=16, out=70, cols=136),
          dict(lengths=[1] * 150, adapter=[i % 4 for i in range(150)], adapters=4, rmax=8, out=130, cols=256),
          dict(lengths=[20, 3, 40, 50], adapter=[0, 1, 2, 1], adapters=3, rmax=32, out=96, cols=264),
          dict(lengths=[33, 20, 60], adapter=[1, 0, 2], adapters=3, rmax=104, out=100, cols=328),
          dict(lengths=[200, 33, 160], adapter=[1, 0, 2], adapters=3, rmax=104, out=340, cols=3000 - 56)]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_a_row_of_nan(i):
    """Reaches its own row's outputs and its adapter's gradients, and nothing else."""
    c = Case(**SHAPES[i])
    y, u = c.forward()
    g = c.backward(u=u)
    row = c.seq // 2
    rest = np.arange(c.seq) != row
    ad = c.of[row]
    c.x[row, 3], c.dy[row, 1] = np.nan, np.inf
    by, bu = c.forward()
    by, bu, y, u = (v.reshape(c.seq, -1) for v in (by, bu, y, u))
    assert np.isnan(by[row]).all() and same(by[rest], y[rest]) and same(bu[rest], u[rest])
    bg = c.backward(u=np.where(rest[:, None], u, np.nan).astype(F32))
    a, b = (v[0].reshape(c.seq, -1) for v in (bg, g))
    assert not np.isfinite(a[row]).any() and same(a[rest], b[rest])
    others = np.arange(c.n) != ad
    for k, shape in ((1, c.a.shape), (2, c.b.shape)):
        assert same(bg[k].reshape(shape)[others], g[k].reshape(shape)[others])
    assert np.isnan(bg[1].reshape(c.a.shape)[ad, :, 3]).all() and np.isnan(bg[2].reshape(c.b.shape)[ad]).all()


@pytest.mark.parametrize("rmax", [8, 32, 72])
def test_many_requests(rmax):
    """More requests than a wave looks at together, most of them empty."""
    rng = np.random.default_rng(rmax)
    lengths = np.where(rng.random(700) < 0.8, 0, rng.integers(1, 9, 700))
    c = Case(list(lengths), rng.integers(-1, 6, 700), 5, rmax, out=84, cols=72, mixed=True, first=2, behind=5)
    y, u = c.forward()
    want, wu = c.want()
    close(u, wu, "u")
    close(y, want, "y")
    for g, w, n in zip(c.backward(u=u), c.want_grad(ref.Sums(u.reshape(c.seq, rmax).astype(float))), ("dx", "da", "db")):
        close(g, w, n)


@pytest.mark.parametrize("rmax", [16, 128])
def test_rows_that_are_not_there(rmax):
    """Requests that begin before the first row or end behind the last have the rows between; no request at all has none."""
    c = Case([40], [0], 2, rmax, out=50, cols=64, mixed=False)
    c.start, c.adapter = np.array([-7, 5, 33, 2 ** 31 - 1], np.int32), np.array([1, 0, 1], np.int32)
    c.of = ref.owners(c.seq, c.start, c.adapter, c.n)
    assert (c.of >= 0).all()
    for _ in range(2):
        y, u = c.forward()
        close(y, c.want()[0], "y")
        for g, w, n in zip(c.backward(u=u), c.want_grad(ref.Sums(u.reshape(c.seq, rmax).astype(float))), ("dx", "da", "db")):
            close(g, w, n)
        c.start = np.array([2 ** 31 - 3, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31 - 1], np.int32)
        c.of = ref.owners(c.seq, c.start, c.adapter, c.n)
        assert (c.of < 0).all()


class Part:
    """An array `off` bytes into a larger one, with bytes on both sides that nothing may write."""

    def __init__(self, nbytes, off=0, a=None):
        self.off, self.nbytes, self.all = off, nbytes, nlgpu.DeviceArray(nbytes + off + 4096)
        whole = np.full(nbytes + off + 4096, 0xA5, np.uint8)
        if a is not None:
            whole[off:off + nbytes] = a.reshape(-1).view(np.uint8)
        self.all.upload(whole)
        self.ptr = self.all.ptr + off

    def get(self):
        v = self.all.download(np.uint8)
        assert (v[:self.off] == 0xA5).all() and (v[self.off + self.nbytes:] == 0xA5).all()
        return v[self.off:self.off + self.nbytes].view(F32)


@pytest.mark.parametrize("i", range(len(SHAPES)))
@pytest.mark.parametrize("seq_out", [0, 2])
def test_alignment_and_ends(i, seq_out):
    """y, res and dy a word off their vectors' alignment, every array and workspace exactly as long as it must be."""
    c = Case(**{**SHAPES[i], "out": SHAPES[i]["out"] // 4 * 4 + seq_out})
    n = len(c.adapter)
    d = {k: up(getattr(c, k)) for k in ("x", "a16", "b16", "scale", "adapter", "start", "rank", "dres")}
    res, dy = Part(c.res.nbytes, 4, c.res), Part(c.dy.nbytes, 4, c.dy)
    y, u = Part(c.res.nbytes, 4), Part(4 * c.seq * c.rmax)
    ws = Part(nlgpu.lora_linear_workspace(c.seq, c.out, c.cols, c.rmax, n))
    nlgpu.lora_linear(d["x"], d["a16"], d["b16"], d["scale"], d["adapter"], res, y, c.seq, c.out, c.cols, c.n, c.rmax, n, ws,
                      start=d["start"], rank=d["rank"], u=u, fmt=c.fmt)
    nlgpu.sync()
    want, wu = c.want()
    close(y.get(), want, "y")
    close(u.get(), wu, "u")
    ws.get()
    da, db, dx = Part(4 * c.a.size), Part(4 * c.b.size), Part(c.x.nbytes)
    ws = Part(nlgpu.lora_linear_grad_workspace(c.seq, c.out, c.cols, c.n, c.rmax, n))
    nlgpu.lora_linear_grad(d["x"], None, dy, d["a16"], d["b16"], d["scale"], d["adapter"], da, db, c.seq, c.out, c.cols, c.n,
                           c.rmax, n, ws, dres=d["dres"], dx=dx, start=d["start"], rank=d["rank"], fmt=c.fmt)
    nlgpu.sync()
    for g, w, name in zip((dx, da, db), c.want_grad(wu), ("dx", "da", "db")):
        close(g.get(), w, name)
    ws.get()


def test_row_is_its_request():
    """No `start`: request i is row i, and rows behind the last request have no adapter."""
    c = Case([1] * 30, [i % 3 for i in range(30)], 3, 16, out=40, cols=64, behind=6)
    y, u = c.forward(start=False)
    want, wu = c.want()
    close(u, wu, "u")
    close(y, want, "y")


@pytest.mark.parametrize("i", [0, 2, 4])
def test_captured(i):
    """Two captured calls that share a workspace (a projection with its adapters, their gradients), replayed in turn and
    between eager calls while rows, adapters and requests change: the eager bits each time."""
    c = Case(**SHAPES[i])
    n = len(c.adapter)
    st = nlgpu.lib().nlg_stream_create()
    w = up(nlgpu.pack_ternary(nlgpu.trits(c.out, (c.out, c.cols))))
    d = {k: up(getattr(c, k)) for k in ("x", "a16", "b16", "scale", "adapter", "start", "rank", "dres", "dy")}
    beta = up(np.array([0.03], F32))
    need = max(nlgpu.ternary_linear_lora_workspace(c.seq, c.out, c.cols, c.rmax, n),
               nlgpu.lora_linear_grad_workspace(c.seq, c.out, c.cols, c.n, c.rmax, n))
    ws = nlgpu.DeviceArray(need)
    o = [nlgpu.DeviceArray(4 * k) for k in (c.seq * c.out, c.seq * c.rmax, c.x.size, c.a.size, c.b.size)]

    def forward():
        nlgpu.ternary_linear_lora(d["x"], w, None, beta, d["a16"], d["b16"], d["scale"], d["adapter"], o[0], c.seq, c.out,
                                  c.cols, c.n, c.rmax, n, ws, start=d["start"], rank=d["rank"], u=o[1], stream=st)

    def backward():
        nlgpu.lora_linear_grad(d["x"], o[1], d["dy"], d["a16"], d["b16"], d["scale"], d["adapter"], o[3], o[4], c.seq, c.out,
                               c.cols, c.n, c.rmax, n, ws, dres=d["dres"], dx=o[2], start=d["start"], rank=d["rank"],
                               stream=st)

    def run(*go):
        for a in o:
            a.zero(st)
        for g in go:
            g()
        nlgpu.sync(st)
        return [a.download(F32) for a in o]

    run(forward, backward)  # (before a capture: the base's column split wants its scratch from an eager call)
    graphs = []
    for f in (forward, backward):
        nlgpu.graph_begin(st)
        f()
        graphs.append(nlgpu.graph_end(st))
    rng = np.random.default_rng(1)
    seen = None
    for k in range(4):
        if k:
            d["x"].upload(c.x * F32(k + 1))
            d["a16"].upload(rng.permutation(c.a16.reshape(c.n, -1)))
            d["adapter"].upload(rng.permutation(c.adapter))
        eager = run(forward, backward)
        for _ in range(2):
            got = run(*[lambda g=g: nlgpu.graph_launch(g, st) for g in graphs])
            assert all(same(a, b) for a, b in zip(got, eager))
        assert seen is None or not same(seen, eager[0])
        seen = eager[0]
    for g in graphs:
        nlgpu.graph_destroy(g)
    nlgpu.lib().nlg_stream_destroy(st)


def test_two_streams():
    """Calls that overlap on two streams, each with its own workspace, give the bits of calls alone."""
    cs = [Case(**{**SHAPES[2], "seed": k}) for k in range(2)]
    want = [(c.forward(), c.backward(u=c.forward()[1])) for c in cs]
    st = [nlgpu.lib().nlg_stream_create() for _ in cs]
    got = [(c.forward(stream=s), c.backward(u=w[0][1], stream=s)) for c, s, w in zip(cs, st, want)]
    for g, w in zip(got, want):
        assert all(same(a, b) for x, y in zip(g, w) for a, b in zip(x, y))
    n = len(cs[0].adapter)
    runs = []
    for c, s in zip(cs, st):
        d = {k: up(getattr(c, k)) for k in ("x", "a16", "b16", "scale", "adapter", "start", "rank", "res")}
        d["y"], d["ws"] = nlgpu.DeviceArray(c.res.nbytes), nlgpu.DeviceArray(
            nlgpu.lora_linear_workspace(c.seq, c.out, c.cols, c.rmax, n))
        runs.append((c, s, d))
    nlgpu.sync()
    for _ in range(5):
        for c, s, d in runs:
            nlgpu.lora_linear(d["x"], d["a16"], d["b16"], d["scale"], d["adapter"], d["res"], d["y"], c.seq, c.out, c.cols,
                              c.n, c.rmax, n, d["ws"], start=d["start"], rank=d["rank"], fmt=c.fmt, stream=s)
    for (c, s, d), w in zip(runs, want):
        nlgpu.sync(s)
        assert same(d["y"].download(F32), w[0][0].ravel())
        nlgpu.lib().nlg_stream_destroy(s)
