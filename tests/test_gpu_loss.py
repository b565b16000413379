"""The losses over a ternary head on the GPU against their form in 64 bits
(loss_ref.py), within the tolerances derived there."""
import numpy as np
import pytest

import loss_ref as ref
import nlgpu

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def up(a):
    return nlgpu.to_device(a) if a is not None else None


class Case:
    """Rows that lean to their first target, over `vocab` rows of weights; codes 10 (-2) among them if asked."""

    def __init__(self, rows, vocab, cols, top=None, tau=1.0, whole=False, per_row=False, bias=False, twos=False, seed=0):
        rng = np.random.default_rng([rows, vocab, cols, top or 0, seed])
        self.rows, self.vocab, self.cols, self.top, self.tau = rows, vocab, cols, top, float(F32(tau))
        self.w = nlgpu.trits(seed + 17, (vocab, cols)).astype(np.int64)
        if twos:
            self.w[rng.random((vocab, cols)) < 0.02] = -2
        self.words = nlgpu.pack_ternary(self.w)
        self.beta = (rng.uniform(1.5, 3.0, vocab if per_row else 1) * cols ** -0.5).astype(F32)
        if per_row:
            self.beta[rng.random(vocab) < 0.1] *= F32(-0.03)
        self.per_row = per_row
        self.bias = rng.standard_normal(vocab).astype(F32) if bias else None
        k = top or 1
        self.index = np.stack([rng.permutation(vocab)[:k] if k <= vocab else rng.integers(0, vocab, k)
                               for _ in range(rows)]).astype(np.int32)
        self.x = (rng.standard_normal((rows, cols)) +
                  rng.uniform(0, 3, (rows, 1)) * cols ** -0.5 * self.w[self.index[:, 0]]).astype(F32)
        self.dloss = rng.uniform(-1, 2, rows).astype(F32)
        self.teacher = (rng.standard_normal((rows, k)) * 3).astype(F32) if top else None
        self.teacher_lse = None
        if whole:
            y = self.teacher.astype(np.float64) / self.tau
            self.teacher_lse = (np.log(np.exp(y).sum(axis=1)) + rng.uniform(0, 1, rows)).astype(F32)

    def call(self, grad=True, stream=None, lse=True, dloss=True, buffers=None):
        """The call's outputs (loss, lse, dx), each filled with NaN before."""
        b = buffers or {k: up(getattr(self, k)) for k in ("x", "words", "beta", "bias", "index", "dloss", "teacher",
                                                          "teacher_lse")}
        nan = lambda *n: up(np.full(n, np.nan, F32))  # noqa: E731
        out = nan(self.rows), nan(self.rows) if lse else None, nan(self.rows, self.cols) if grad else None
        if self.top is None:
            ws = nlgpu.DeviceArray(nlgpu.ternary_xent_workspace(self.rows, self.vocab, self.cols, grad))
            nlgpu.ternary_xent(b["x"], b["words"], b["bias"], b["beta"], b["index"], out[0], out[1], self.rows,
                               self.vocab, self.cols, ws, dx=out[2], dloss=b["dloss"] if dloss else None,
                               beta_per_row=self.per_row, stream=stream)
        else:
            ws = nlgpu.DeviceArray(nlgpu.ternary_distill_workspace(self.rows, self.vocab, self.cols, self.top, grad))
            nlgpu.ternary_distill(b["x"], b["words"], b["bias"], b["beta"], b["index"], b["teacher"], self.top, self.tau,
                                  out[0], out[1], self.rows, self.vocab, self.cols, ws, teacher_lse=b["teacher_lse"],
                                  dx=out[2], dloss=b["dloss"] if dloss else None, beta_per_row=self.per_row,
                                  stream=stream)
        nlgpu.sync(stream)
        got = [o.download(F32) if o is not None else None for o in out]
        if grad:
            got[2] = got[2].reshape(self.rows, self.cols)
        return got

    def want(self):
        """(loss, lse, dx) in 64 bits and their bounds."""
        beta = self.beta if self.per_row else np.repeat(self.beta, self.vocab)
        q, g = ref.quantise(self.x)
        t = ref.teacher_weights(self.index, self.teacher, self.teacher_lse, self.tau, self.vocab)
        loss, lse, dx, p = ref.loss_of(q * g, self.w, self.bias, beta, self.index, t, self.tau)
        tol = ref.tolerances(self.x, self.w, self.bias, beta, self.index, self.teacher, self.teacher_lse, t, self.tau, p)
        d = self.dloss.astype(np.float64)[:, None]
        return (loss, lse, dx * d), (tol[0], tol[1], tol[2] * np.abs(d) + 2.0 ** -140)


def check(c, got, rows=slice(None), what=("loss", "lse", "dx")):
    want, tol = c.want()
    for name, g, w, t in zip(("loss", "lse", "dx"), got, want, tol):
        if g is None or name not in what:
            continue
        off = np.abs(g.astype(np.float64) - w)[rows]
        assert (off <= t[rows]).all(), (name, off.max(), t[rows][np.unravel_index(np.argmax(off - t[rows]), off.shape)])


SIZES = [(1, 1, 64), (1, 300, 256), (3, 257, 64), (33, 1000, 320), (64, 511, 512), (65, 2049, 192), (130, 777, 576),
         (300, 513, 1280), (31, 4099, 2560)]


@pytest.mark.parametrize("rows,vocab,cols", SIZES)
@pytest.mark.parametrize("per_row,bias", [(False, False), (True, True)])
def test_xent(rows, vocab, cols, per_row, bias):
    c = Case(rows, vocab, cols, per_row=per_row, bias=bias, twos=bias)
    check(c, c.call())


@pytest.mark.parametrize("rows,vocab,cols", SIZES)
@pytest.mark.parametrize("top,tau,whole,per_row", [(1, 1.0, False, False), (7, 2.0, True, True), (130, 0.7, False, False)])
def test_distill(rows, vocab, cols, top, tau, whole, per_row):
    c = Case(rows, vocab, cols, top=top, tau=tau, whole=whole, per_row=per_row, bias=per_row)
    check(c, c.call())


def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


@pytest.mark.parametrize("rows", [40, 300, 600])
@pytest.mark.parametrize("per_row", [False, True])
def test_rows_without_a_label(rows, per_row):
    """Labels outside the vocabulary: loss 0, gradient 0, lse as ever; what their rows hold reaches no other row."""
    c = Case(rows, 700, 320, per_row=per_row, bias=True)
    rng = np.random.default_rng(rows)
    out = rng.random(rows) < 0.6
    c.index[out, 0] = rng.choice([-1, 700, -100, 2 ** 31 - 1, -2 ** 31], out.sum())
    got = c.call()
    check(c, got)
    assert not got[0][out].any() and not got[2][out].any()
    c.x[out, ::3] = np.inf
    c.x[out, 1::3] = np.nan
    bad = c.call()
    assert not bad[0][out].any() and not bad[2][out].any()
    assert all(same(b[~out], g[~out]) for b, g in zip(bad, got))
    assert np.isnan(bad[1][out]).all()
    assert all(same(b, g) if g is not None else b is None for b, g in zip(c.call(lse=False)[::2], bad[::2]))


def test_no_row_has_a_label():
    for rows in (5, 300):
        c = Case(rows, 300, 128)
        c.index[:] = -1
        got = c.call()
        check(c, got, what=("lse",))
        assert not got[0].any() and not got[2].any()


def test_a_row_with_an_infinity():
    """NaN in its own outputs; the bits of the others stay."""
    for rows in (7, 290):
        c = Case(rows, 1000, 192, top=3)
        got = c.call()
        c.x[rows // 2, 5] = -np.inf
        bad = c.call()
        rest = np.arange(rows) != rows // 2
        assert all(np.isnan(b[~rest]).all() and same(b[rest], g[rest]) for b, g in zip(bad, got))


@pytest.mark.parametrize("rows,cols", [(20, 256), (270, 192)])
def test_forbidden_tokens(rows, cols):
    """A bias of -inf: a tile of the vocabulary, its first and last rows, a label or two."""
    c = Case(rows, 1030, cols, bias=True)
    c.bias[256:512] = -np.inf
    c.bias[[0, 1029, 700]] = -np.inf
    c.index[c.bias[c.index] == -np.inf] = 5
    c.index[3], c.index[rows - 1] = 300, 1029
    got = c.call()
    gone = np.isin(np.arange(rows), [3, rows - 1])
    check(c, got, rows=~gone)
    check(c, got, what=("lse", "dx"))
    assert (got[0][gone] == np.inf).all()
    assert not np.isinf(got[1]).any()


def test_every_token_forbidden():
    """lse -inf, the loss of a labelled row NaN, the gradient that of the label's logit alone."""
    c = Case(6, 300, 64, bias=True)
    c.bias[:] = -np.inf
    c.index[4] = -1
    loss, lse, dx = c.call()
    assert (lse == -np.inf).all() and loss[4] == 0 and np.isnan(np.delete(loss, 4)).all()
    want = -c.w[c.index[:, 0]].astype(F32) * c.beta[0] * c.dloss[:, None]
    want[4] = 0
    assert np.abs(dx - want).max() <= 2.0 ** -22 * np.abs(want).max()


@pytest.mark.parametrize("whole", [False, True])
def test_teacher_entries(whole):
    """Entries that name nothing (whatever their logit), one index twice, logits of -inf, a row of none."""
    c = Case(70, 555, 256, top=9, tau=1.5, whole=whole)
    c.index[::2, 3] = -1
    c.index[::3, 8] = 555
    c.teacher[::2, 3] = np.nan
    c.index[::5, 1] = c.index[::5, 0]
    c.teacher[::4, 2] = -np.inf
    c.index[11] = [-5] * 8 + [2 ** 31 - 1]
    c.teacher[11, 4] = np.inf
    got = c.call()
    check(c, got)
    assert got[0][11] == 0 and not got[2][11].any()


def test_gradient_by_differences():
    """The loss's own differences: along x a change of whole steps of the rounding's scale, at the row's largest value
    unchanged, is exact, so only the loss's rounding and its curvature (a step squared) stay."""
    c = Case(3, 400, 64, top=5, tau=2.0)
    c.dloss[:] = 1
    q, g = ref.quantise(c.x)
    c.x = (q * g).astype(F32)  # (on the grid, so a change of one step is a change of the rounded row)
    loss, _, dx = c.call()
    rng = np.random.default_rng(1)
    for col in rng.permutation(64)[:12]:
        keep, ends = c.x.copy(), []
        free = np.abs(q[:, col]) < 120
        for d in (4, -4):
            c.x = keep.copy()
            c.x[free, col] = ((q[free, col] + d) * g[free, 0]).astype(F32)
            ends.append(c.call(grad=False)[0].astype(np.float64))
        c.x = keep
        step = 8 * g[:, 0].astype(np.float64)
        # third derivatives of a log sum of z/tau: at most twice the cube of the weights' factor over tau
        slope = np.abs(c.beta[0]) / c.tau
        tol = (2 * c.want()[1][0] + 2 * (step / 2 * slope) ** 3 / 3) / step + c.want()[1][2][:, col]
        assert (np.abs((ends[0] - ends[1]) / step - dx[:, col]) <= tol)[free].all()


def test_several_chunks():
    """More rows than the probabilities are kept for at a time, some without a label: rows on both sides of the cuts."""
    vocab, cols, rows = 524288 - 40, 64, 560
    c = Case(2, vocab, cols)
    rng = np.random.default_rng(3)
    c.rows, c.index = rows, rng.integers(0, vocab, (rows, 1)).astype(np.int32)
    out = np.isin(np.arange(rows), [1, 200, 255, 400])
    c.x = (rng.standard_normal((rows, cols)) + 0.4 * c.w[c.index[:, 0]]).astype(F32)
    c.dloss = rng.uniform(-1, 2, rows).astype(F32)
    c.index[out] = -1
    got = c.call()
    assert not got[0][out].any() and not got[2][out].any() and all(np.isfinite(g).all() for g in got)
    part = [0, 199, 254, 256, 257, 258, 259, 260, 515, 516, 517, 559]
    few = Case(2, vocab, cols)
    few.rows, few.index, few.x, few.dloss = len(part), c.index[part], c.x[part], c.dloss[part]
    check(few, [g[part] for g in got])


def test_same_bits_again():
    c = Case(300, 3000, 512, top=20, per_row=True)
    assert all(same(a, b) for a, b in zip(c.call(), c.call()))


class Guarded:
    """A device array with bytes behind it that nothing may write."""

    def __init__(self, nbytes):
        self.all = nlgpu.DeviceArray(nbytes + 4096)
        self.all.upload(np.full(nbytes + 4096, 0xA5, np.uint8))
        self.ptr, self.nbytes = self.all.ptr, nbytes

    def kept(self):
        return (self.all.download(np.uint8)[self.nbytes:] == 0xA5).all()


@pytest.mark.parametrize("rows,vocab,cols,top", [(1, 100, 64, 1), (33, 511, 320, 5), (65, 1000, 64, 40), (257, 257, 576, 3)])
def test_writes_no_further(rows, vocab, cols, top):
    c = Case(rows, vocab, cols, top=top, per_row=True)
    for grad in (False, True):
        b = {k: up(getattr(c, k)) for k in ("x", "words", "beta", "index", "dloss", "teacher")}
        ws = Guarded(nlgpu.ternary_distill_workspace(rows, vocab, cols, top, grad))
        out = [Guarded(4 * rows), Guarded(4 * rows), Guarded(4 * rows * cols)]
        nlgpu.ternary_distill(b["x"], b["words"], None, b["beta"], b["index"], b["teacher"], top, c.tau, out[0], out[1], rows,
                              vocab, cols, ws, dx=out[2] if grad else None, dloss=b["dloss"], beta_per_row=True)
        nlgpu.sync()
        assert ws.kept() and all(o.kept() for o in out)
        n = [rows, rows, rows * cols]
        got = [o.all.download(F32, m) for o, m in zip(out, n)]
        got[2] = got[2].reshape(rows, cols) if grad else None
        check(c, got)
        assert nlgpu.ternary_distill_workspace(rows, vocab, cols, top, grad) > 0


def test_captured():
    """Two captured calls (labels, a teacher) that share a workspace, replayed in turn and between eager calls, at inputs
    that change: the eager bits each time."""
    rows, vocab, cols, top = 300, 2000, 320, 6
    c, t = Case(rows, vocab, cols, per_row=True), Case(rows, vocab, cols, top=top, tau=2.0, per_row=True)
    st = nlgpu.lib().nlg_stream_create()
    ws = nlgpu.DeviceArray(nlgpu.ternary_distill_workspace(rows, vocab, cols, top, True))
    d = {k: up(getattr(t, k)) for k in ("x", "words", "beta", "index", "dloss", "teacher")}
    label = up(c.index)
    outs = [[nlgpu.DeviceArray(4 * n) for n in (rows, rows, rows * cols)] for _ in range(2)]

    def xent():
        nlgpu.ternary_xent(d["x"], d["words"], None, d["beta"], label, outs[0][0], outs[0][1], rows, vocab, cols, ws,
                           dx=outs[0][2], dloss=d["dloss"], beta_per_row=True, stream=st)

    def distill():
        nlgpu.ternary_distill(d["x"], d["words"], None, d["beta"], d["index"], d["teacher"], top, 2.0, outs[1][0],
                              outs[1][1], rows, vocab, cols, ws, dx=outs[1][2], dloss=d["dloss"], beta_per_row=True, stream=st)

    def run(*go):
        for o in outs[0] + outs[1]:
            o.zero(st)
        for g in go:
            g()
        nlgpu.sync(st)
        return [o.download(F32) for o in outs[0] + outs[1]]

    graphs = []
    for f in (xent, distill):
        nlgpu.graph_begin(st)
        f()
        graphs.append(nlgpu.graph_end(st))
    rng = np.random.default_rng(1)
    first = None
    for k in range(4):
        if k:
            d["x"].upload((t.x * F32(1 + k) + rng.standard_normal(t.x.shape).astype(F32)))
            lab = c.index.copy()
            lab[rng.random(rows) < 0.3 * k] = -1
            label.upload(lab)
        eager = run(xent, distill)
        for _ in range(2):
            assert all(same(a, b) for a, b in zip(run(*[lambda g=g: nlgpu.graph_launch(g, st) for g in graphs]), eager))
        assert first is None or not same(first[0], eager[0])
        first = eager
    for g in graphs:
        nlgpu.graph_destroy(g)
    nlgpu.lib().nlg_stream_destroy(st)


def test_two_streams():
    """Calls that overlap on two streams, each with its own workspace, give the bits of calls alone."""
    cs = [Case(200, 3000, 512, seed=k) for k in range(2)]
    want = [c.call() for c in cs]
    st = [nlgpu.lib().nlg_stream_create() for _ in cs]
    bufs = [{k: up(getattr(c, k)) for k in ("x", "words", "beta", "index", "dloss")} for c in cs]
    ws = [nlgpu.DeviceArray(nlgpu.ternary_xent_workspace(200, 3000, 512, True)) for _ in cs]
    outs = [[nlgpu.DeviceArray(4 * n) for n in (200, 200, 200 * 512)] for _ in cs]
    nlgpu.sync()
    for _ in range(5):
        for b, w, o, s in zip(bufs, ws, outs, st):
            nlgpu.ternary_xent(b["x"], b["words"], None, b["beta"], b["index"], o[0], o[1], 200, 3000, 512, w, dx=o[2],
                               dloss=b["dloss"], stream=s)
    for o, s, w in zip(outs, st, want):
        nlgpu.sync(s)
        assert all(same(a.download(F32), b.ravel()) for a, b in zip(o, w))
        nlgpu.lib().nlg_stream_destroy(s)
