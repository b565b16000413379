"""Adapters of a frozen ternary model tuned from labels or a teacher, and then
served: two projections with their requests' adapters, the head's loss, and
the gradients back through both, each stage against its form in 64 bits
(lora_ref.py, loss_ref.py) from what the stage before left on the device."""
import numpy as np
import pytest

import loss_ref
import lora_ref
import nlgpu

pytestmark = pytest.mark.gpu
F32 = np.float32
COLS, MID, HEAD, VOCAB, RMAX, ADAPTERS, TOP = 192, 256, 128, 777, 16, 3, 6


@pytest.fixture(scope="module", autouse=True)
def device():
    nlgpu.init()
    yield


def up(a):
    return nlgpu.to_device(np.ascontiguousarray(a))


def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


def close(got, want, name):
    off = np.abs(got.astype(np.float64).reshape(want.value.shape) - want.value)
    assert (off <= want.off + 2.0 ** -140).all(), (name, (off / (want.off + 2.0 ** -140)).max())


class Layer:
    """A frozen ternary projection and its adapters."""

    def __init__(self, rng, out, cols):
        self.out, self.cols = out, cols
        self.words = nlgpu.pack_ternary(nlgpu.trits(out + cols, (out, cols)))
        self.beta = (rng.uniform(0.5, 1.5, out) * cols ** -0.5).astype(F32)
        self.a16, self.a = lora_ref.to16(rng.standard_normal((ADAPTERS, RMAX, cols)) * cols ** -0.5, True)
        self.b16, self.b = lora_ref.to16(rng.standard_normal((ADAPTERS, out, RMAX)) * 0.2, True)
        self.blocks = np.repeat(self.beta, cols // 128 or 1)  # ternary-rows-t has a factor for each 128 columns
        self.d = {k: up(getattr(self, k)) for k in ("words", "beta", "blocks", "a16", "b16")}

    def tune(self, da, db, rate):
        """A step of gradient descent: the adapters' new values, in place on the device too."""
        self.a16, self.a = lora_ref.to16(self.a - rate * da.reshape(self.a.shape), True)
        self.b16, self.b = lora_ref.to16(self.b - rate * db.reshape(self.b.shape), True)
        self.d["a16"].upload(self.a16)
        self.d["b16"].upload(self.b16)


class Model:
    def __init__(self, lengths, adapter, teacher, stream):
        rng = np.random.default_rng(sum(lengths))
        self.teacher, self.st = teacher, stream
        self.start = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        self.adapter, self.rows = np.asarray(adapter, np.int32), int(sum(lengths))
        self.of = lora_ref.owners(self.rows, self.start, self.adapter, ADAPTERS)
        self.scale, self.rank = np.array([1.5, -0.7, 2.0], F32), np.array([16, 8, 5], np.int32)
        self.layers = [Layer(rng, MID, COLS), Layer(rng, HEAD, MID)]
        self.hw = nlgpu.trits(99, (VOCAB, HEAD)).astype(np.int64)
        self.hbeta = np.array([1.5 * HEAD ** -0.5], F32)
        self.x = rng.standard_normal((self.rows, COLS)).astype(F32)
        self.index = rng.integers(0, VOCAB, (self.rows, TOP if teacher else 1)).astype(np.int32)
        self.index[rng.random(self.rows) < 0.3] = -1  # the prompts' tokens are not learnt
        self.dloss = np.full(self.rows, 1 / max((self.index[:, 0] >= 0).sum(), 1), F32)
        self.logit = (rng.standard_normal(self.index.shape) * 2).astype(F32) if teacher else None
        self.d = {k: up(getattr(self, k)) for k in ("x", "start", "adapter", "scale", "rank", "hbeta", "index", "dloss")}
        self.d["head"] = up(nlgpu.pack_ternary(self.hw))
        if teacher:
            self.d["logit"] = up(self.logit)
        n, r = len(adapter), self.rows
        need = [nlgpu.ternary_distill_workspace(r, VOCAB, HEAD, TOP, True), nlgpu.ternary_xent_workspace(r, VOCAB, HEAD, True)]
        for y in self.layers:
            need += [nlgpu.ternary_linear_lora_workspace(r, y.out, y.cols, RMAX, n),
                     nlgpu.lora_linear_grad_workspace(r, y.out, y.cols, ADAPTERS, RMAX, n)]
        self.ws = nlgpu.DeviceArray(max(need))
        sizes = dict(h=r * MID, u1=r * RMAX, g=r * HEAD, u2=r * RMAX, loss=r, lse=r, dg=r * HEAD, base=r * MID, dh=r * MID)
        for i, y in enumerate(self.layers, 1):
            sizes[f"da{i}"], sizes[f"db{i}"] = y.a.size, y.b.size
        self.o = {k: nlgpu.DeviceArray(4 * v) for k, v in sizes.items()}

    def adapted(self, y):
        d = self.d
        return (y.d["a16"], y.d["b16"], d["scale"], d["adapter"]), dict(start=d["start"], rank=d["rank"], fmt=nlgpu.LORA_BF16,
                                                                        stream=self.st)

    def project(self, i, x, y, u):
        l = self.layers[i]
        at, kw = self.adapted(l)
        nlgpu.ternary_linear_lora(x, l.d["words"], None, l.d["beta"], *at, y, self.rows, l.out, l.cols, ADAPTERS, RMAX,
                                  len(self.adapter), self.ws, u=u, beta_per_row=True, **kw)

    def back(self, i, x, u, dy, dx):
        l = self.layers[i]
        (a, b, scale, adapter), kw = self.adapted(l)
        nlgpu.lora_linear_grad(x, u, dy, a, b, scale, adapter, self.o[f"da{i + 1}"], self.o[f"db{i + 1}"], self.rows, l.out,
                               l.cols, ADAPTERS, RMAX, len(self.adapter), self.ws, dres=dx, dx=dx, **kw)

    def step(self):
        o, d, second = self.o, self.d, self.layers[1]
        self.project(0, d["x"], o["h"], o["u1"])
        self.project(1, o["h"], o["g"], o["u2"])
        if self.teacher:
            nlgpu.ternary_distill(o["g"], d["head"], None, d["hbeta"], d["index"], d["logit"], TOP, 1.5, o["loss"], o["lse"],
                                  self.rows, VOCAB, HEAD, self.ws, dx=o["dg"], dloss=d["dloss"], stream=self.st)
        else:
            nlgpu.ternary_xent(o["g"], d["head"], None, d["hbeta"], d["index"], o["loss"], o["lse"], self.rows, VOCAB, HEAD,
                               self.ws, dx=o["dg"], dloss=d["dloss"], stream=self.st)
        for out in ("base", "dh"):  # the frozen projection's input gradient; the adapters' is added in place
            nlgpu.dispatch("ternary-rows-t", [second.d["words"], second.d["blocks"], o["dg"], o[out]],
                           [HEAD, MID, MID // 128, MID // 16, self.rows], (self.rows * MID + 63) // 64, stream=self.st)
        self.back(1, o["h"], o["u2"], o["dg"], o["dh"])
        self.back(0, d["x"], o["u1"], o["dh"], None)

    def run(self, go):
        for a in self.o.values():
            a.zero(self.st)
        go()
        nlgpu.sync(self.st)
        return {k: a.download(F32) for k, a in self.o.items()}

    def check(self, got):
        r, s64 = self.rows, self.scale.astype(float)
        x = self.x
        for i, (y, u) in enumerate((("h", "u1"), ("g", "u2"))):
            l = self.layers[i]
            base, dx = nlgpu.DeviceArray(4 * r * l.out), up(x)
            ws = nlgpu.DeviceArray(max(16, nlgpu.ternary_linear_workspace(r, l.cols)))
            nlgpu.ternary_linear(dx, l.d["words"], None, l.d["beta"], base, r, l.out, l.cols, beta_per_row=True, workspace=ws)
            nlgpu.sync()
            want, wu = lora_ref.forward(x.astype(float), l.a, l.b, s64, self.rank, self.of,
                                        lora_ref.Sums(base.download(F32).reshape(r, l.out).astype(float)))
            close(got[u], wu, u)
            close(got[y], want, y)
            x = got[y].reshape(r, l.out)
        tau = 1.5 if self.teacher else 1.0
        beta = np.repeat(self.hbeta, VOCAB)
        q, g = loss_ref.quantise(x)
        t = loss_ref.teacher_weights(self.index, self.logit, None, tau, VOCAB)
        loss, lse, dx, p = loss_ref.loss_of(q * g, self.hw, None, beta, self.index, t, tau)
        tol = loss_ref.tolerances(x, self.hw, None, beta, self.index, self.logit, None, t, tau, p)
        w = self.dloss[:, None].astype(float)
        assert (np.abs(got["loss"] - loss) <= tol[0]).all() and (np.abs(got["lse"] - lse) <= tol[1]).all()
        dg = got["dg"].reshape(r, HEAD)
        assert (np.abs(dg - dx * w) <= tol[2] * w + 2.0 ** -140).all()
        for i, xs, us, dy, out, dres in ((1, got["h"], got["u2"], dg, got["dh"], got["base"]),
                                         (0, self.x, got["u1"], got["dh"], None, None)):
            l = self.layers[i]
            want = lora_ref.backward(xs.reshape(r, l.cols).astype(float), lora_ref.Sums(us.reshape(r, RMAX).astype(float)),
                                     dy.reshape(r, l.out).astype(float), l.a, l.b, s64, self.rank, self.of,
                                     None if dres is None else dres.reshape(r, l.cols))
            if out is not None:
                close(out, want[0], "dh")
            close(got[f"da{i + 1}"], want[1], f"da{i + 1}")
            close(got[f"db{i + 1}"], want[2], f"db{i + 1}")


@pytest.mark.parametrize("teacher", [False, True])
@pytest.mark.parametrize("lengths,adapter", [([20, 0, 33, 7], [1, 0, 0, 2]), ([130, 200], [2, -1]), ([1] * 9, [0, 1, 2] * 3)])
def test_steps(lengths, adapter, teacher):
    """Three steps of descent, eager and as one captured graph between them: stages right, bits the same."""
    st = nlgpu.lib().nlg_stream_create()
    m = Model(lengths, adapter, teacher, st)
    m.run(m.step)  # (before a capture: scratch of the library's own)
    nlgpu.graph_begin(st)
    m.step()
    graph = nlgpu.graph_end(st)
    losses = []
    for _ in range(3):
        eager = m.run(m.step)
        m.check(eager)
        for _ in range(2):
            replay = m.run(lambda: nlgpu.graph_launch(graph, st))
            assert all(same(replay[k], eager[k]) for k in eager)
        losses.append(eager["loss"])
        for i, l in enumerate(m.layers, 1):
            l.tune(eager[f"da{i}"], eager[f"db{i}"], 0.5)
    assert not same(losses[0], losses[1]) and not same(losses[1], losses[2])
    # served: a token of each request at a time, by the tuned adapters
    seq = len(adapter)
    x, l = m.x[:seq], m.layers[0]
    y, ws = nlgpu.DeviceArray(4 * seq * MID), nlgpu.DeviceArray(nlgpu.ternary_linear_lora_workspace(seq, MID, COLS, RMAX, seq))
    base = nlgpu.DeviceArray(4 * seq * MID)
    at, kw = m.adapted(l)
    kw["start"] = None
    nlgpu.ternary_linear_lora(up(x), l.d["words"], None, l.d["beta"], *at, y, seq, MID, COLS, ADAPTERS, RMAX, seq, ws,
                              beta_per_row=True, **kw)
    wb = nlgpu.DeviceArray(max(16, nlgpu.ternary_linear_workspace(seq, COLS)))
    nlgpu.ternary_linear(up(x), l.d["words"], None, l.d["beta"], base, seq, MID, COLS, beta_per_row=True, workspace=wb, stream=st)
    nlgpu.sync(st)
    want = lora_ref.forward(x.astype(float), l.a, l.b, m.scale.astype(float), m.rank,
                            lora_ref.owners(seq, None, m.adapter, ADAPTERS),
                            lora_ref.Sums(base.download(F32).reshape(seq, MID).astype(float)))[0]
    close(y.download(F32), want, "served")
    nlgpu.graph_destroy(graph)
    nlgpu.lib().nlg_stream_destroy(st)
