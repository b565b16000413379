"""The losses over a ternary head on the CPU: the sizes of their pieces
(nelisp-gpu_amd/csrc/nlg_loss.h, compiled here), every refusal, which needs no
device, and the gradient that the GPU tests compare with, against
differences."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

import loss_ref as ref
import nlgpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <stdio.h>
#include "nlg_loss.h"
static uint64_t seed = 1;
static uint32_t rnd(uint32_t n) { seed = seed * 6364136223846793005ull + 1442695040888963407ull; return (uint32_t)(seed >> 33) % n; }
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
static int one(uint32_t rows, uint32_t vocab, uint32_t cols, uint32_t top, bool grad) {
  const LossPlan p = loss_plan(rows, vocab, cols, top, grad);
  CHECK(p.ok && (uint64_t)p.tiles * LOSS_TILE >= vocab && (uint64_t)(p.tiles - 1) * LOSS_TILE < vocab);
  // regions in order, each as long as what it holds, 256-byte aligned
  uint64_t at[11] = {p.xq, p.gamma, p.part, p.bmax, p.lse, p.sum, p.weight, p.bytes};
  uint64_t len[11] = {(uint64_t)rows * cols, 4ull * rows, 8ull * rows * p.tiles, 4ull * p.tiles, 4ull * rows, 4ull * rows,
                      4ull * rows * top};
  int n = 7;
  if (grad) {
    CHECK(p.chunk % p.bm == 0 && (uint64_t)p.chunks * p.chunk >= rows && (uint64_t)(p.chunks - 1) * p.chunk < rows);
    const uint64_t all = (uint64_t)p.tiles * LOSS_TILE;
    // every part has vocabulary rows
    CHECK(p.share % LOSS_TILE == 0 && (uint64_t)p.share * p.splits >= all && (uint64_t)p.share * (p.splits - 1) < all);
    at[7] = p.order; len[7] = 4ull * (rows + 1);
    at[8] = p.prob; len[8] = 4ull * p.chunk * all;
    at[9] = p.acc; len[9] = 4ull * p.splits * p.chunk * cols;
    at[10] = p.bytes;
    n = 10;
  }
  for (int i = 0; i < n; i++) CHECK(at[i] % 256 == 0 && at[i] + len[i] <= at[i + 1]);
  return 0;
}
int main(void) {
  for (int i = 0; i < 20000; i++) {
    const uint32_t rows = 1 + rnd(1u << rnd(17)), vocab = 1 + rnd(1u << rnd(20)), cols = 64 * (1 + rnd(256)), top = 1 + rnd(LOSS_TOP);
    if (one(rows, vocab, cols, top, rnd(2))) { printf("%u %u %u %u\n", rows, vocab, cols, top); return 1; }
  }
  CHECK(!loss_plan(0, 1, 64, 1, 0).ok && !loss_plan(1, 0, 64, 1, 0).ok && !loss_plan(1, 1, 63, 1, 0).ok);
  CHECK(!loss_plan(1, 1, 0, 1, 0).ok && !loss_plan(1, 1, 16448, 1, 0).ok && !loss_plan(1, 1, 64, 0, 0).ok);
  CHECK(!loss_plan(1, 1, 64, LOSS_TOP + 1, 0).ok && !loss_plan(0xffffffffu, 1, 64, 1, 1).ok && !loss_plan(1, 0xffffffffu, 64, 1, 1).ok);
  CHECK(loss_plan(0, 1, 64, 1, 1).bytes == 0);
  puts("ok");
  return 0;
}
'''


def test_plan():
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        open(src, "w").write(PROGRAM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                        os.path.join(ROOT, "nelisp-gpu_amd", "csrc"), src, "-o", exe], check=True)
        out = subprocess.run([exe], capture_output=True, text=True)
        assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr


class Ptr:
    """An address that no call reads: every refusal comes before anything is launched."""

    def __init__(self, ptr=1 << 20, nbytes=1 << 40):
        self.ptr, self.nbytes = ptr, nbytes


GOOD = dict(x=Ptr(), w2=Ptr(), bias=None, beta=Ptr(), label=Ptr(), loss=Ptr(), lse=Ptr(), rows=3, vocab=1000, cols=256,
            workspace=Ptr(), dx=Ptr())
NULL = Ptr(None)
BAD = [(dict(x=NULL), "null"), (dict(w2=NULL), "null"), (dict(beta=NULL), "null"), (dict(label=NULL), "null"),
       (dict(loss=NULL), "null"), (dict(cols=0), "cols"), (dict(cols=100), "cols"), (dict(cols=16448), "cols"),
       (dict(vocab=0), "vocab"), (dict(x=Ptr(8)), "aligned"), (dict(w2=Ptr(8)), "aligned"), (dict(dx=Ptr(8)), "aligned"),
       (dict(label=Ptr(2)), "aligned"), (dict(lse=Ptr(2)), "aligned"), (dict(dloss=Ptr(2)), "aligned"),
       (dict(beta=Ptr(6)), "aligned"), (dict(bias=Ptr(1)), "aligned"), (dict(loss=Ptr(3)), "aligned"),
       (dict(workspace=NULL), "workspace"), (dict(workspace=Ptr(nbytes=1000)), "workspace"),
       (dict(workspace=Ptr(8)), "aligned"), (dict(rows=0xffffffff), "many"), (dict(vocab=0xffffffff), "many"),
       (dict(rows=1 << 24, vocab=1 << 17), "many")]


@pytest.mark.parametrize("change,word", BAD)
def test_refusals(change, word):
    with pytest.raises(nlgpu.NlgError, match=word):
        nlgpu.ternary_xent(**{**GOOD, **change})
    a = {**GOOD, **change}
    a["index"] = a.pop("label")
    with pytest.raises(nlgpu.NlgError, match=word):
        nlgpu.ternary_distill(teacher=Ptr(), top=4, temperature=1.0, **a)


@pytest.mark.parametrize("change,word", [
    (dict(teacher=NULL), "null"), (dict(top=0), "targets"), (dict(top=1025), "targets"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(teacher=Ptr(2)), "aligned"), (dict(teacher_lse=Ptr(2)), "aligned")])
def test_distill_refusals(change, word):
    a = {**GOOD, "index": Ptr(), "teacher": Ptr(), "top": 4, "temperature": 1.0}
    del a["label"]
    with pytest.raises(nlgpu.NlgError, match=word):
        nlgpu.ternary_distill(**{**a, **change})


@pytest.mark.parametrize("change", [
    dict(dx="x"), dict(loss="x"), dict(lse="loss"), dict(dx="loss"), dict(dx="lse"), dict(lse="index"), dict(loss="dloss"),
    dict(dx="w2"), dict(lse="beta"), dict(loss="bias"), dict(dx="teacher"), dict(lse="teacher_lse")])
def test_overlaps(change):
    a = {n: Ptr((i + 1) << 36) for i, n in enumerate(("x", "w2", "bias", "beta", "index", "teacher", "teacher_lse", "dloss",
                                                       "loss", "lse", "dx", "workspace"))}
    for out, other in change.items():
        a[out] = Ptr(a[other].ptr)
    a.update(rows=3, vocab=1000, cols=256, top=4, temperature=1.0)
    with pytest.raises(nlgpu.NlgError, match="overlap"):
        nlgpu.ternary_distill(**a)
    if "teacher" not in str(change):
        for k in ("teacher", "teacher_lse", "top", "temperature"):
            del a[k]
        a["label"] = a.pop("index")
        with pytest.raises(nlgpu.NlgError, match="overlap"):
            nlgpu.ternary_xent(**a)


def test_no_rows_is_no_call():
    nlgpu.ternary_xent(**{**GOOD, "rows": 0})


def test_workspace_sizes():
    assert nlgpu.ternary_xent_workspace(1, 1000, 100, True) == 0
    small, grad = nlgpu.ternary_xent_workspace(100, 128256, 2560, False), nlgpu.ternary_xent_workspace(100, 128256, 2560, True)
    assert 0 < small < grad < (1 << 40)
    # far below the logits of the same rows
    assert nlgpu.ternary_xent_workspace(8192, 128256, 2560, True) < 8192 * 128256 * 4 / 3
    assert nlgpu.ternary_distill_workspace(100, 128256, 2560, 64, False) > small
    assert isinstance(ctypes.c_size_t(grad).value, int)


@pytest.mark.parametrize("top,tau,whole,bias", [(None, 1.0, False, True), (5, 2.0, False, False), (9, 0.7, True, True)])
def test_reference_gradient_by_differences(top, tau, whole, bias):
    rng = np.random.default_rng(3)
    rows, vocab, cols, k = 4, 50, 12, top or 1
    w = rng.integers(-2, 2, (vocab, cols))
    beta = rng.uniform(-1, 1, vocab).astype(np.float32)
    b = rng.standard_normal(vocab).astype(np.float32) if bias else None
    h = rng.standard_normal((rows, cols))
    index = rng.integers(-1, vocab, (rows, k)).astype(np.int32)
    index[0, :] = index[0, 0]  # the same index twice
    teacher = rng.standard_normal((rows, k)).astype(np.float32) if top else None
    lse = rng.standard_normal(rows).astype(np.float32) + 3 if whole else None
    t = ref.teacher_weights(index, teacher, lse, tau, vocab)
    _, _, dx, _ = ref.loss_of(h, w, b, beta, index, t, tau)
    step = 2.0 ** -18  # third derivatives are some 10: off by 10 step^2 / 6, and by 2^-52 30 / step from rounding
    for c in range(cols):
        e = np.zeros(cols)
        e[c] = step
        up, down = (ref.loss_of(h + s * e, w, b, beta, index, t, tau)[0] for s in (1, -1))
        assert np.abs((up - down) / (2 * step) - dx[:, c]).max() < 1e-8
