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
