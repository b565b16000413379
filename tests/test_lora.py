"""Low-rank adapters on the CPU: every refusal, which needs no device, and the
64-bit form that the GPU tests compare with, its gradients against
differences."""
import numpy as np
import pytest

import lora_ref as ref
import nlgpu


class Ptr:
    """An address that no call reads: every refusal comes before anything is launched."""

    def __init__(self, ptr, nbytes=1 << 40):
        self.ptr, self.nbytes = ptr, nbytes


def at(n):  # far apart: no two of them overlap
    return Ptr(n << 36)


SIZES = dict(seq=10, out=20, cols=64, adapters=3, rmax=16, requests=4)
GOOD = dict(x=at(1), a=at(2), b=at(3), scale=at(4), adapter=at(5), workspace=at(9), start=at(10), rank=at(11), **SIZES)
FORWARD = dict(GOOD, res=at(6), y=at(7), u=None)
TERNARY = dict(GOOD, w2=at(12), bias=None, beta=at(13), y=at(7), u=at(8))
GRAD = dict(GOOD, u=at(8), dy=at(6), da=at(12), db=at(13), dx=at(14), dres=at(15))
NULL = Ptr(None)
OF = {"lora_linear": FORWARD, "ternary_linear_lora": TERNARY, "lora_linear_grad": GRAD}
BAD = [(dict(a=NULL), "null"), (dict(b=NULL), "null"), (dict(scale=NULL), "null"), (dict(adapter=NULL), "null"),
       (dict(x=NULL), "null"), (dict(fmt=2), "format"), (dict(fmt=-1), "format"), (dict(adapters=0), "adapters"),
       (dict(rmax=0), "rmax"), (dict(rmax=12), "rmax"), (dict(rmax=136), "rmax"), (dict(cols=0), "cols"),
       (dict(cols=60), "cols"), (dict(out=0), "out"), (dict(seq=1 << 22), "many"), (dict(out=1 << 25), "many"),
       (dict(adapters=65535), "many"), (dict(requests=1 << 25), "many"), (dict(a=Ptr(1 << 30 | 8)), "aligned"),
       (dict(b=Ptr(1 << 30 | 8)), "aligned"), (dict(x=Ptr(1 << 30 | 4)), "aligned"), (dict(scale=Ptr(6)), "aligned"),
       (dict(start=Ptr(2)), "aligned"), (dict(rank=Ptr(1)), "aligned"), (dict(adapter=Ptr(3)), "aligned"),
       (dict(workspace=NULL), "workspace"), (dict(workspace=Ptr(1 << 40, 100)), "workspace"),
       (dict(workspace=Ptr(8 | 1 << 40)), "aligned")]


@pytest.mark.parametrize("name", sorted(OF))
@pytest.mark.parametrize("change,word", BAD)
def test_refusals(name, change, word):
    with pytest.raises(nlgpu.NlgError, match=word):
        getattr(nlgpu, name)(**{**OF[name], **change})


@pytest.mark.parametrize("name,change,word", [
    ("lora_linear", dict(y=NULL), "null"), ("lora_linear", dict(y=at(1)), "overlap"), ("lora_linear", dict(u=at(1)), "overlap"),
    ("lora_linear", dict(u=at(7)), "overlap"), ("lora_linear", dict(res=Ptr((7 << 36) + 4)), "overlap"),
    ("lora_linear", dict(u=at(6)), "overlap"), ("lora_linear", dict(y=Ptr(2)), "aligned"), ("lora_linear", dict(u=Ptr(4)), "aligned"),
    ("ternary_linear_lora", dict(w2=NULL), "null"), ("ternary_linear_lora", dict(beta=NULL), "null"),
    ("ternary_linear_lora", dict(y=NULL), "null"), ("ternary_linear_lora", dict(w2=Ptr(4)), "aligned"),
    ("ternary_linear_lora", dict(beta=Ptr(6)), "aligned"), ("ternary_linear_lora", dict(cols=16392), "cols"),
    ("ternary_linear_lora", dict(u=at(7)), "overlap"), ("ternary_linear_lora", dict(y=at(1)), "overlap"),
    ("lora_linear_grad", dict(dy=NULL), "null"), ("lora_linear_grad", dict(da=NULL), "null"),
    ("lora_linear_grad", dict(db=NULL), "null"), ("lora_linear_grad", dict(dy=Ptr(2)), "aligned"),
    ("lora_linear_grad", dict(u=Ptr(4)), "aligned"), ("lora_linear_grad", dict(dx=Ptr(8)), "aligned"),
    ("lora_linear_grad", dict(dx=at(1)), "overlap"), ("lora_linear_grad", dict(da=at(1)), "overlap"),
    ("lora_linear_grad", dict(db=at(12)), "overlap"), ("lora_linear_grad", dict(dx=at(6)), "overlap"),
    ("lora_linear_grad", dict(dres=Ptr((14 << 36) + 16)), "overlap"), ("lora_linear_grad", dict(da=at(8)), "overlap")])
def test_refusals_of_one(name, change, word):
    with pytest.raises(nlgpu.NlgError, match=word):
        getattr(nlgpu, name)(**{**OF[name], **change})


def test_no_rows_is_no_call():
    for name in ("lora_linear", "ternary_linear_lora"):
        getattr(nlgpu, name)(**{**OF[name], "seq": 0})
    with pytest.raises(nlgpu.NlgError, match="seq"):  # whose gradients of zero it would have to write
        nlgpu.lora_linear_grad(**{**GRAD, "seq": 0})


def test_workspace_sizes():
    assert nlgpu.lora_linear_workspace(10, 20, 60, 16, 4) == 0 and nlgpu.lora_linear_workspace(10, 20, 64, 12, 4) == 0
    assert nlgpu.lora_linear_workspace(10, 20, 64, 16, 4) >= 10 * 16 * 4
    assert nlgpu.ternary_linear_lora_workspace(10, 20, 64, 16, 4) > nlgpu.lora_linear_workspace(10, 20, 64, 16, 4)
    assert nlgpu.lora_linear_grad_workspace(10, 20, 64, 3, 16, 4) >= 2 * 10 * 16 * 4


def test_reference_gradients_by_differences():
    """The gradients of sum(dy * y) are linear in each argument, so differences of any step have rounding alone."""
    rng = np.random.default_rng(5)
    seq, out, cols, n, rmax = 7, 6, 8, 3, 5
    x, dy = rng.standard_normal((seq, cols)), rng.standard_normal((seq, out))
    a, b = rng.standard_normal((n, rmax, cols)), rng.standard_normal((n, out, rmax))
    scale, rank = rng.standard_normal(n), np.array([5, 0, 3])
    of = ref.owners(seq, [1, 4, 4, 6], [2, 0, 0], n)
    assert of.tolist() == [-1, 2, 2, 2, 0, 0, -1]
    value = lambda x, a, b: (ref.forward(x, a, b, scale, rank, of, None)[0].value * dy).sum()  # noqa: E731
    u = ref.forward(x, a, b, scale, rank, of, None)[1]
    grads = ref.backward(x, u, dy, a, b, scale, rank, of, None)
    for k, g in enumerate(grads):
        args = [x, a, b]
        for i in np.ndindex(args[k].shape):
            e = np.zeros(args[k].shape)
            e[i] = 0.5
            up, down = (value(*[v + s * e if j == k else v for j, v in enumerate(args)]) for s in (1, -1))
            assert abs(up - down - g.value[i]) < 1e-12 * (1 + abs(value(*args))) * 10


def test_reference_rounds_to_bf16():
    v = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -2.0 ** -130, 0.0], np.float32)
    h, w = ref.to16(v, True)
    assert w.tolist() == [1.0, 1.0, 1 + 2.0 ** -6, -2.0 ** -130, 0.0]
    assert h[0] == 0x3f80
