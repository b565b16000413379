"""Calls of the adapters and the losses whose outputs or workspace share bytes with anything else are refused (no device:
nothing is launched)."""
import pytest

import nlgpu

NAMES = ("x", "w2", "bias", "beta", "a", "b", "scale", "rank", "start", "adapter", "res", "y", "u", "dy", "dres", "dx", "da",
         "db", "label", "index", "teacher", "teacher_lse", "dloss", "loss", "lse", "workspace")


class Ptr:
    """An address that no call reads."""

    def __init__(self, ptr, nbytes=1 << 30):
        self.ptr, self.nbytes = ptr, nbytes


def apart(*names):
    return {n: Ptr((NAMES.index(n) + 1) << 36) for n in names}


LORA = dict(apart("x", "a", "b", "scale", "rank", "start", "adapter", "workspace"), seq=10, out=20, cols=64, adapters=3,
            rmax=16, requests=4)
HEAD = dict(apart("x", "w2", "bias", "beta", "dloss", "loss", "lse", "dx", "workspace"), rows=3, vocab=1000, cols=256,
            beta_per_row=True)
CALLS = {"lora_linear": (dict(LORA, **apart("res", "y", "u")), ("y", "u", "workspace")),
         "ternary_linear_lora": (dict(LORA, **apart("w2", "bias", "beta", "y", "u"), beta_per_row=True), ("y", "u", "workspace")),
         "lora_linear_grad": (dict(LORA, **apart("u", "dy", "dres", "dx", "da", "db")), ("dx", "da", "db", "workspace")),
         "ternary_xent": (dict(HEAD, **apart("label")), ("loss", "lse", "dx", "workspace")),
         "ternary_distill": (dict(HEAD, **apart("index", "teacher", "teacher_lse"), top=4, temperature=1.0),
                             ("loss", "lse", "dx", "workspace"))}
# an array's bytes, where the sizes above make them few
LAST = {"scale": 3, "rank": 3, "start": 5, "adapter": 4, "bias": 20, "beta": 20, "loss": 3, "lse": 3, "label": 3,
        "teacher_lse": 3, "dloss": 3}


@pytest.mark.parametrize("name,out", [(n, o) for n in CALLS for o in CALLS[n][1]])
def test_outputs_and_the_workspace_overlap_nothing(name, out):
    good = CALLS[name][0]
    for other, p in good.items():
        if other == out or not isinstance(p, Ptr) or (out, other) in (("y", "res"), ("dx", "dres")):
            continue
        with pytest.raises(nlgpu.NlgError, match="overlap"):
            getattr(nlgpu, name)(**dict(good, **{out: Ptr(p.ptr)}))


@pytest.mark.parametrize("name", sorted(CALLS))
def test_to_the_last_byte(name):
    """The workspace that begins 16 bytes at most before an array's end overlaps it, its whole bytes counted."""
    good = CALLS[name][0]
    for other, words in LAST.items():
        if other not in good or (name.startswith("ternary_x") or name.startswith("ternary_d")) and other in ("bias", "beta"):
            continue
        at = good[other].ptr + (4 * words - 1) // 16 * 16
        with pytest.raises(nlgpu.NlgError, match="overlap"):
            getattr(nlgpu, name)(**dict(good, workspace=Ptr(at)))


@pytest.mark.parametrize("name,out,other", [("lora_linear", "y", "res"), ("lora_linear_grad", "dx", "dres")])
def test_added_to_in_place_or_apart(name, out, other):
    """What is added to may be the output itself, but not a part of it."""
    good = CALLS[name][0]
    for off in (-16, 16):
        with pytest.raises(nlgpu.NlgError, match="overlap"):
            getattr(nlgpu, name)(**dict(good, **{out: Ptr(good[other].ptr + off)}))
