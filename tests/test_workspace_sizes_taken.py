"""The adapters' and losses' workspace functions give 0 for exactly the sizes that the calls refuse (no device: a call whose
sizes are taken stops at its workspace, which is a byte short here)."""
import numpy as np
import pytest

import nlgpu


class Ptr:
    """An address that no call reads; far apart, so that no two arrays overlap."""

    def __init__(self, n, nbytes=1 << 50):
        self.ptr, self.nbytes = n << 56, nbytes


def arrays(*names):
    return {k: Ptr(i + 1) for i, k in enumerate(names)}


LORA = ("x", "a", "b", "scale", "adapter", "start")


def call(name, ws, **sizes):
    a = {"lora_linear": lambda: dict(arrays(*LORA, "res", "y"), **sizes),
         "ternary_linear_lora": lambda: dict(arrays(*LORA, "w2", "beta", "y"), bias=None, **sizes),
         "lora_linear_grad": lambda: dict(arrays(*LORA, "dy", "da", "db"), u=None, **sizes),
         "ternary_xent": lambda: dict(arrays("x", "w2", "beta", "label", "loss", "lse"), bias=None,
                                      dx=Ptr(20) if sizes["grad"] else None, **sizes),
         "ternary_distill": lambda: dict(arrays("x", "w2", "beta", "index", "teacher", "loss", "lse"), bias=None,
                                         temperature=1.0, dx=Ptr(20) if sizes["grad"] else None, **sizes)}[name]()
    a.pop("grad", None)
    getattr(nlgpu, name)(workspace=Ptr(30, ws), **a)


def need(name, s):
    if name in ("lora_linear", "ternary_linear_lora"):
        return getattr(nlgpu, name + "_workspace")(s["seq"], s["out"], s["cols"], s["rmax"], s["requests"])
    if name == "lora_linear_grad":
        return nlgpu.lora_linear_grad_workspace(s["seq"], s["out"], s["cols"], s["adapters"], s["rmax"], s["requests"])
    more = (s["top"],) if name == "ternary_distill" else ()
    return getattr(nlgpu, name + "_workspace")(s["rows"], s["vocab"], s["cols"], *more, s["grad"])


EDGES = dict(seq=(1, 3, 4, 40, 65536, 65535 * 32, 65535 * 32 + 1, 1 << 30), out=(0, 1, 20, 1 << 24, (1 << 24) + 1),
             cols=(0, 4, 8, 60, 64, 96, 16384, 16392, 16448, 1 << 24, (1 << 24) + 8), rmax=(0, 4, 8, 64, 72, 128, 136),
             requests=(0, 1, 1 << 24, (1 << 24) + 1), adapters=(0, 1, 65534, 65535),
             rows=(1, 100, 1 << 20, 0xffffff, 1 << 24, 0xffffffff), vocab=(0, 1, 300, 128256, 1 << 24, (1 << 24) + 1, 0xffffffff),
             top=(0, 1, 17, 1024, 1025), grad=(False, True))
COMMON = dict(seq=40, out=20, cols=64, rmax=16, requests=4, adapters=3, rows=100, vocab=1000, top=5, grad=True)
OF = {"lora_linear": ("seq", "out", "cols", "rmax", "requests", "adapters"), "ternary_xent": ("rows", "vocab", "cols", "grad"),
      "ternary_distill": ("rows", "vocab", "cols", "top", "grad")}
OF["ternary_linear_lora"] = OF["lora_linear_grad"] = OF["lora_linear"]


@pytest.mark.parametrize("name", sorted(OF))
def test_none_for_what_is_refused(name):
    rng = np.random.default_rng(1)
    sizes = [dict({k: COMMON[k] for k in OF[name]}, **{k: v}) for k in OF[name] for v in EDGES[k]]
    sizes += [{k: EDGES[k][rng.integers(len(EDGES[k]))] for k in OF[name]} for _ in range(3000)]
    taken = 0
    for s in sizes:
        n = need(name, s)
        with pytest.raises(nlgpu.NlgError) as e:
            call(name, max(n - 1, 0), **s)
        word = f"workspace holds {max(n - 1, 0)} bytes, needs {n}"
        # (the forward calls' workspace knows nothing of how many adapters there are)
        refused = name in ("lora_linear", "ternary_linear_lora") and s["adapters"] in (0, 65535)
        assert (word in str(e.value)) == (n > 0 and not refused), (s, n, str(e.value))
        taken += n > 0
    assert taken > 20


def test_none_for_what_no_launch_holds():
    """The logits' product is one launch: 256 threads for each 256 logits of 32 rows, fewer than 2^32."""
    for rows, vocab, held in ((1 << 20, 128256, True), (0xffffff, 1 << 24, False), (0xffffff, 8000, False), (0xffffff, 256, True),
                              (64, 1 << 24, True), (1 << 23, 32768, False)):
        assert (nlgpu.ternary_xent_workspace(rows, vocab, 64, False) > 0) == held, (rows, vocab)
        assert (nlgpu.ternary_distill_workspace(rows, vocab, 64, 3, True) > 0) == held, (rows, vocab)
