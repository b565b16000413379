"""Fine-tuning a frozen ternary model and serving what comes of it: low-rank
adapters of many requests beside a shared 2-bit projection (forward and
backward), the softmax cross entropy of a ternary LM head in pieces of its
vocabulary, and distillation from a teacher's top logits over the same head,
each with its gradient; in elementary torch operations and as calls through
nlgpu.

A ternary linear rounds each row of its activations to int8 (g = max|x| / 127,
q = x / g rounded half away from zero, in 32 bits) and gives bias[o] +
(beta[o] g) sum_c W[o, c] q[c], with W in 2-bit fields: 00 0, 01 +1, 11 -1,
10 -2.  Adapters see the rows as they are.  The losses' gradient goes
straight through the rounding: it is that of the linear on the rounded rows.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One decoded token of one request, its adapter among eight that are resident (O projection of the 2B-class model).
        {"name": "lora_token", "kind": "lora", "fmt": "f16", "requests": 1, "shortest": 1, "longest": 1, "adapters": 8,
         "rmax": 16, "mixed": False, "out": 2560, "cols": 2560, "per_row": False},
        # A serving step: 64 requests decode together, 48 adapters of different ranks.
        {"name": "lora_step", "kind": "lora", "fmt": "bf16", "requests": 64, "shortest": 1, "longest": 1, "adapters": 48,
         "rmax": 64, "mixed": True, "out": 6912, "cols": 2560, "per_row": False},
        # Prompts of very different lengths in one batch, each with its own adapter, one of them with none.
        {"name": "lora_prompts", "kind": "lora", "fmt": "f16", "requests": 6, "shortest": 77, "longest": 1500,
         "adapters": 5, "rmax": 32, "mixed": False, "out": 4096, "cols": 4096, "per_row": True},
        # The backward pass of two short examples.
        {"name": "lora_grad_short", "kind": "lora_grad", "fmt": "bf16", "requests": 2, "shortest": 90, "longest": 151,
         "adapters": 1, "rmax": 8, "mixed": False, "out": 2560, "cols": 2560},
        # That of a batch of eight sequences that train three adapters at once (down projection's shape).
        {"name": "lora_grad_batch", "kind": "lora_grad", "fmt": "f16", "requests": 8, "shortest": 130, "longest": 1024,
         "adapters": 3, "rmax": 32, "mixed": True, "out": 2560, "cols": 6912},
        # The log-probability of one answered token.
        {"name": "xent_token", "kind": "xent", "rows": 1, "vocab": 128256, "cols": 2560, "grad": False, "per_row": False,
         "bias": False, "ignored": False},
        # A prompt's log-probabilities (perplexity, ranking of answers).
        {"name": "xent_score", "kind": "xent", "rows": 512, "vocab": 128256, "cols": 2560, "grad": False,
         "per_row": False, "bias": False, "ignored": False},
        # A short example with its prompt masked out; a vocabulary of odd size.
        {"name": "xent_short", "kind": "xent", "rows": 100, "vocab": 32003, "cols": 2048, "grad": True, "per_row": True,
         "bias": True, "ignored": True},
        # One training step's loss and gradient over the 2B-class model's head.
        {"name": "xent_train", "kind": "xent", "rows": 4096, "vocab": 128256, "cols": 2560, "grad": True,
         "per_row": False, "bias": False, "ignored": True},
        # How far a student is from its teacher on one sequence (no gradient).
        {"name": "distill_score", "kind": "distill", "rows": 333, "vocab": 32000, "cols": 4096, "grad": False, "top": 100,
         "temperature": 1.0, "whole": True, "per_row": False, "bias": False},
        # A short sequence with its teacher's eight best tokens.
        {"name": "distill_short", "kind": "distill", "rows": 37, "vocab": 32000, "cols": 2048, "grad": True, "top": 8,
         "temperature": 2.0, "whole": False, "per_row": True, "bias": False},
        # A distillation step: the teacher's 64 best tokens of each position.
        {"name": "distill_train", "kind": "distill", "rows": 2048, "vocab": 128256, "cols": 2560, "grad": True, "top": 64,
         "temperature": 1.0, "whole": False, "per_row": False, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    k = rng.choice(["lora", "lora", "lora_grad", "xent", "xent", "distill"])
    cols = 64 * _log(rng, 4, 108)
    c = {"kind": k, "cols": cols}
    if k in ("lora", "lora_grad"):
        longest = rng.choice([1, _log(rng, 2, 2048)]) if k == "lora" else _log(rng, 1, 2048)
        c.update(fmt=rng.choice(["f16", "bf16"]), out=_log(rng, 200, 14000), longest=longest,
                 requests=max(1, min(_log(rng, 1, 256), 8192 // longest)), shortest=rng.randint(1, longest),
                 adapters=_log(rng, 1, 64) if k == "lora" else _log(rng, 1, 8),
                 rmax=rng.choice([8, 16, 16, 24, 32, 64, 128]), mixed=rng.choice([True, False]))
        if k == "lora":
            c["per_row"] = rng.choice([True, False])
        return c
    vocab = _log(rng, 1000, 131072)
    c.update(vocab=vocab, rows=max(1, min(_log(rng, 1, 4096), int(4096 * 128256 * 2560 / 4 / vocab / cols))),
             grad=rng.choice([True, True, False]), per_row=rng.choice([True, False]), bias=rng.choice([True, False]))
    if k == "xent":
        return dict(c, ignored=rng.choice([True, False]))
    return dict(c, top=_log(rng, 1, 128), temperature=rng.choice([0.7, 1.0, 2.0, 4.0]), whole=rng.choice([True, False]))


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly (a batch's sizes: the same for every seed, in another order)."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(c):
    return _spread(c["requests"], c["shortest"], c["longest"])


def _ranks(c):
    return _spread(c["adapters"], max(1, c["rmax"] // 8), c["rmax"]) if c["mixed"] else [c["rmax"]] * c["adapters"]


def _adapters(c):
    """Each request's adapter; of four and more requests one has none."""
    return [-1 if i == 3 else i % c["adapters"] for i in range(c["requests"])]


# ------------------------------------------------------------------ the inputs

class Inputs:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)
        self.r = np.random.RandomState(int(seed) % (1 << 31))

    def normal(self, *shape, sigma=1.0):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=torch.float32) * sigma

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(shape, generator=self.g, device=DEV, dtype=torch.float32) * (hi - lo) + lo

    def below(self, n, *shape):
        return torch.randint(0, n, shape, generator=self.g, device=DEV, dtype=torch.int32)

    def ints(self, values):
        return torch.tensor(np.asarray(values), device=DEV, dtype=torch.int32)

    def ternary(self, out, cols):
        """2-bit words: half of the weights zero, the others +1 and -1 alike."""
        def bits():
            return torch.randint(-(1 << 31), 1 << 31, (out, cols // 16), generator=self.g, device=DEV,
                                 dtype=torch.int64).to(torch.int32)

        low = bits() & 0x55555555
        return low | ((low << 1) & bits())


def _trits(words):
    """2-bit words [n, wng] as int8 [n, 16 wng]."""
    f = (words[:, :, None] >> (2 * torch.arange(16, device=DEV, dtype=torch.int32))) & 3
    return (f - 4 * (f >> 1)).to(torch.int8).flatten(1)


def prepare(case, seed):
    c = dict(case)
    i = Inputs(seed)
    s = {"c": c}
    cols = c["cols"]
    if c["kind"] in ("lora", "lora_grad"):
        order = i.r.permutation(c["requests"])
        lengths, adapter = np.asarray(_lengths(c))[order], np.asarray(_adapters(c))[i.r.permutation(c["requests"])]
        seq, out, n, rmax = int(lengths.sum()), c["out"], c["adapters"], c["rmax"]
        t = torch.float16 if c["fmt"] == "f16" else torch.bfloat16
        s.update(seq=seq, start=i.ints(np.concatenate([[0], np.cumsum(lengths)])), adapter=i.ints(adapter),
                 rank=i.ints(_ranks(c)), scale=i.uniform(n, lo=0.5, hi=2.0),
                 a=i.normal(n, rmax, cols, sigma=cols ** -0.5).to(t), b=i.normal(n, out, rmax, sigma=0.1).to(t),
                 x=i.normal(seq, cols) * i.uniform(seq, 1, lo=0.5, hi=2.0))
        if c["kind"] == "lora":
            s.update(w2=i.ternary(out, cols), beta=i.uniform(out if c["per_row"] else 1, lo=0.02, hi=0.04),
                     y=torch.zeros(seq, out, device=DEV))
        else:
            of = adapter.repeat(lengths)
            held = torch.tensor(np.asarray(_ranks(c))[np.maximum(of, 0)] * (of >= 0), device=DEV)
            u = torch.zeros(seq, rmax, device=DEV)
            for k in range(n):  # what the forward call left
                at = torch.tensor(np.flatnonzero(of == k), device=DEV)
                u[at] = s["x"][at] @ s["a"][k].float().t()
            s["u"] = torch.where(torch.arange(rmax, device=DEV)[None, :] < held[:, None], u, 0.0)
            s.update(dy=i.normal(seq, out, sigma=0.02) * i.uniform(seq, 1, lo=0.2, hi=3.0),
                     dres=i.normal(seq, cols, sigma=0.05), dx=torch.zeros(seq, cols, device=DEV),
                     da=torch.zeros(n, rmax, cols, device=DEV), db=torch.zeros(n, out, rmax, device=DEV))
        return s
    rows, vocab = c["rows"], c["vocab"]
    s["w2"] = i.ternary(vocab, cols)
    s["beta"] = i.uniform(vocab if c["per_row"] else 1, lo=1.5, hi=3.0) * cols ** -0.5
    if c["bias"]:
        s["bias"] = i.normal(vocab, sigma=0.5)
    # what a position may go on with: distinct tokens, the first the likeliest, and states that lean to the first few
    top = c.get("top", 1)
    first, step = i.below(vocab, rows, 1).long(), 1 + i.below(max(1, vocab // max(top, 4) - 1), rows, 1).long()
    index = ((first + step * torch.arange(max(top, 4), device=DEV)) % vocab).to(torch.int32)
    x = i.normal(rows, cols)
    for k in range(min(4, vocab)):
        x += i.uniform(rows, 1, hi=5.0 / (1 + k)) * cols ** -0.5 * _trits(s["w2"][index[:, k].long()])
    s.update(x=x * i.uniform(rows, 1, lo=0.7, hi=1.5), loss=torch.zeros(rows, device=DEV), lse=torch.zeros(rows, device=DEV))
    if c["grad"]:
        s.update(dloss=i.uniform(rows, lo=0.5, hi=1.0) / rows, dx=torch.zeros(rows, cols, device=DEV))
    if c["kind"] == "xent":
        label = index[:, 0].clone()
        if c["ignored"]:
            label[: rows // 3] = -1
        s["label"] = label
    else:
        s["index"] = index[:, :top].contiguous()
        s["teacher"] = 9.0 - 1.5 * torch.log2(1.0 + torch.arange(top, device=DEV)) + i.normal(rows, top, sigma=0.8)
        if c["whole"]:  # the teacher's own normaliser: what its other tokens hold is some share of the top ones'
            of = torch.logsumexp(s["teacher"].double() / c["temperature"], dim=1)
            s["teacher_lse"] = (of + i.uniform(rows, lo=0.01, hi=0.5)).float()
    return s


# ------------------------------------------------------------------ the plain forms

def _quantised(x):
    """Rows as whole numbers of int8 (in 32 bits), and their scales [rows, 1]."""
    g = x.abs().amax(dim=1, keepdim=True) / 127.0
    q = torch.where(g > 0, x / g, 0.0)
    return torch.sign(q) * torch.floor(q.abs() + 0.5).clamp(max=127.0), g


def _linear(s):
    """The ternary linear in 32 bits (its whole sums are exact there)."""
    q, g = _quantised(s["x"])
    w = _trits(s["w2"]).float()
    z = (s["beta"][None, :] * g) * (q @ w.t())
    return (z + s["bias"] if "bias" in s else z), w


def _members(s):
    """[seq, adapters, rmax]: the adapter's scale where a row's request uses that rank of that adapter, else 0."""
    c, seq = s["c"], s["seq"]
    of = torch.repeat_interleave(s["adapter"], (s["start"][1:] - s["start"][:-1]).long(), output_size=seq)
    mine = of[:, None] == torch.arange(c["adapters"], device=DEV)[None, :]
    held = torch.arange(c["rmax"], device=DEV)[None, :] < s["rank"][:, None]
    return (mine[:, :, None] & held[None]) * s["scale"][None, :, None]


def _lora(s):
    m = _members(s).flatten(1)
    y, _ = _linear(s)
    u = (s["x"] @ s["a"].float().flatten(0, 1).t()) * m
    s["y"][:] = y + u @ s["b"].float().transpose(1, 2).flatten(0, 1)
    return s["y"]


def _lora_grad(s):
    n, rmax, cols = s["a"].shape
    m = _members(s)
    a, b = s["a"].float().flatten(0, 1), s["b"].float().transpose(1, 2).flatten(0, 1)
    du = (s["dy"] @ b.t()) * m.flatten(1)
    s["dx"][:] = s["dres"] + du @ a
    s["da"][:] = (du.t() @ s["x"]).view(n, rmax, cols)
    u = (s["u"][:, None, :] * m).flatten(1)
    s["db"][:] = (s["dy"].t() @ u).view(-1, n, rmax).transpose(0, 1)
    return {"dx": s["dx"], "da": s["da"], "db": s["db"]}


def _softmax(z):
    """log sum exp and exp(z - it), row by row."""
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    return (top + torch.log(total))[:, 0], e / total


def _loss_outputs(s):
    return {k: s[k] for k in ("loss", "lse", "dx") if k in s}


def _xent(s):
    z, w = _linear(s)
    s["lse"][:], p = _softmax(z)
    there = s["label"] >= 0
    at = torch.where(there, s["label"], 0).long()[:, None]
    s["loss"][:] = torch.where(there, s["lse"] - z.gather(1, at)[:, 0], 0.0)
    if s["c"]["grad"]:
        p.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
        s["dx"][:] = (p * (s["beta"][None, :] * torch.where(there, s["dloss"], 0.0)[:, None])) @ w
    return _loss_outputs(s)


def _distill(s):
    tau = s["c"]["temperature"]
    z, w = _linear(s)
    z = z / tau
    s["lse"][:], p = _softmax(z)
    t = s["teacher"] / tau
    if "teacher_lse" in s:
        logt = t - s["teacher_lse"][:, None]
    else:
        top = t.amax(dim=1, keepdim=True)
        logt = t - top - torch.log(torch.exp(t - top).sum(dim=1, keepdim=True))
    t, at = torch.exp(logt), s["index"].long()
    s["loss"][:] = (t * (logt - (z.gather(1, at) - s["lse"][:, None]))).sum(dim=1)
    if s["c"]["grad"]:
        p = (p * t.sum(dim=1, keepdim=True)).scatter_add_(1, at, -t)
        s["dx"][:] = (p * (s["beta"][None, :] * (s["dloss"] / tau)[:, None])) @ w
    return _loss_outputs(s)


# ------------------------------------------------------------------ the framework's calls

class View:
    """A torch tensor as the binding takes buffers (its pointer and length)."""

    def __init__(self, t):
        self.t = t.contiguous()
        self.ptr = self.t.data_ptr()
        self.nbytes = self.t.numel() * self.t.element_size()


def _binding():
    d = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nelisp-gpu_amd")
    if d not in sys.path:
        sys.path.insert(0, d)
    import nlgpu

    return nlgpu


def _views(s):
    """The state's buffers as the binding takes them, made at its first call, with the workspace that a program keeps."""
    if "views" not in s:
        n, c = _binding(), s["c"]
        n.init()
        s["views"] = {k: View(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
        if "fmt" in c:
            s["fmt"] = {"f16": n.LORA_F16, "bf16": n.LORA_BF16}[c["fmt"]]
        if c["kind"] == "lora":
            need = n.ternary_linear_lora_workspace(s["seq"], c["out"], c["cols"], c["rmax"], c["requests"])
        elif c["kind"] == "lora_grad":
            need = n.lora_linear_grad_workspace(s["seq"], c["out"], c["cols"], c["adapters"], c["rmax"], c["requests"])
        elif c["kind"] == "xent":
            need = n.ternary_xent_workspace(c["rows"], c["vocab"], c["cols"], c["grad"])
        else:
            need = n.ternary_distill_workspace(c["rows"], c["vocab"], c["cols"], c["top"], c["grad"])
        s["views"]["ws"] = View(torch.empty(max(need, 16), device=DEV, dtype=torch.uint8))
    return s["views"]


def _own(s):
    n, c, b = _binding(), s["c"], _views(s)
    k = c["kind"]
    # in the order of torch's current stream (the default one: the library's, which waits for it and it for that)
    st = torch._C._cuda_getCurrentRawStream(s["x"].device.index) or None
    if k == "lora":
        n.ternary_linear_lora(b["x"], b["w2"], None, b["beta"], b["a"], b["b"], b["scale"], b["adapter"], b["y"],
                              s["seq"], c["out"], c["cols"], c["adapters"], c["rmax"], c["requests"], b["ws"],
                              start=b["start"], rank=b["rank"], fmt=s["fmt"], beta_per_row=c["per_row"], stream=st)
        return s["y"]
    if k == "lora_grad":
        n.lora_linear_grad(b["x"], b["u"], b["dy"], b["a"], b["b"], b["scale"], b["adapter"], b["da"], b["db"], s["seq"],
                           c["out"], c["cols"], c["adapters"], c["rmax"], c["requests"], b["ws"], dres=b["dres"],
                           dx=b["dx"], start=b["start"], rank=b["rank"], fmt=s["fmt"], stream=st)
        return {"dx": s["dx"], "da": s["da"], "db": s["db"]}
    more = {"dx": b.get("dx"), "dloss": b.get("dloss"), "beta_per_row": c["per_row"], "stream": st}
    if k == "xent":
        n.ternary_xent(b["x"], b["w2"], b.get("bias"), b["beta"], b["label"], b["loss"], b["lse"], c["rows"], c["vocab"],
                       c["cols"], b["ws"], **more)
    else:
        n.ternary_distill(b["x"], b["w2"], b.get("bias"), b["beta"], b["index"], b["teacher"], c["top"], c["temperature"],
                          b["loss"], b["lse"], c["rows"], c["vocab"], c["cols"], b["ws"],
                          teacher_lse=b.get("teacher_lse"), **more)
    return _loss_outputs(s)


def run(state):
    """One pass."""
    if own:
        return _own(state)
    return {"lora": _lora, "lora_grad": _lora_grad, "xent": _xent, "distill": _distill}[state["c"]["kind"]](state)


# ------------------------------------------------------------------ the bounds

def work(case):
    c, k, cols = case, case["kind"], case["cols"]
    if k in ("lora", "lora_grad"):
        ranks, of, out = _ranks(c), _adapters(c), c["out"]
        n = sum(_lengths(c))
        used = sum(ranks[a] for a in set(of) if a >= 0)
        mean = sum(ranks[a] for a in of if a >= 0) / len(of)  # lengths and adapters meet in an order that the seed sets
        if k == "lora":
            return {"bytes": 4 * n * (cols + out) + cols * out / 4 + 2 * used * (cols + out),
                    "flops": 2 * n * cols * out + 2 * n * mean * (cols + out)}
        return {"bytes": 4 * n * (3 * cols + out + mean) + 2 * used * (cols + out) + 4 * sum(ranks) * (cols + out),
                "flops": 4 * n * mean * (cols + out)}
    # the logits, and from them the gradient with respect to the rows
    passes = 2 if c["grad"] else 1
    top = c.get("top", 1)
    return {"bytes": c["vocab"] * cols / 4 + 4 * passes * c["rows"] * cols + 8 * c["rows"] * (top + 1),
            "flops": 2 * passes * c["rows"] * c["vocab"] * cols}


# ------------------------------------------------------------------ in 64 bits

def _linear64(s, rows):
    """The ternary linear of the given rows; the rounding to int8 is defined in 32 bits: each step of it is rounded
    there."""
    x = s["x"][rows].double()
    g = (x.abs().max(dim=1, keepdim=True).values / 127.0).float().double()
    q = torch.where(g > 0, x / g, 0.0).float().double()
    q = torch.copysign((q.abs() + 0.5).float().double().floor().clamp(max=127.0), q)
    w = _weights64(s)
    z = (q @ w.t()) * g * s["beta"].double()
    return z + s["bias"].double() if "bias" in s else z


def _weights64(s):
    if "w64" not in s:
        table = torch.tensor([0.0, 1.0, -2.0, -1.0], device=DEV, dtype=torch.float64)
        parts = [table[((s["w2"] >> (2 * f)) & 3).long()] for f in range(16)]
        s["w64"] = torch.stack(parts, dim=2).flatten(1)
    return s["w64"]


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    k = c["kind"]
    if k in ("lora", "lora_grad"):
        first, of = s["start"].tolist(), s["adapter"].tolist()
        if k == "lora":
            y = _linear64(s, slice(None))
        else:
            dx, da, db = s["dres"].double(), s["da"].double(), s["db"].double()
        for i, a in enumerate(of):
            if a < 0:
                continue
            at, r, scale = slice(first[i], first[i + 1]), int(s["rank"][a]), float(s["scale"][a])
            down, up = s["a"][a, :r].double(), s["b"][a, :, :r].double()
            x = s["x"][at].double()
            if k == "lora":
                y[at] += scale * ((x @ down.t()) @ up.t())
                continue
            du = scale * (s["dy"][at].double() @ up)
            dx[at] += du @ down
            da[a, :r] += du.t() @ x
            db[a, :, :r] += scale * (s["dy"][at].double().t() @ s["u"][at, :r].double())
        return y if k == "lora" else {"dx": dx, "da": da, "db": db}
    got = {key: [] for key in ("loss", "lse", "dx")}
    for b in range(0, c["rows"], 512):
        at = slice(b, min(b + 512, c["rows"]))
        z = _linear64(s, at) / c.get("temperature", 1.0)
        l = torch.logsumexp(z, dim=1, keepdim=True)
        logp = z - l
        got["lse"].append(l[:, 0])
        if k == "xent":
            there = (s["label"][at] >= 0).double()[:, None]
            t, where = there, s["label"][at].long().clamp(min=0)[:, None]
            got["loss"].append((-there * logp.gather(1, where))[:, 0])
        else:
            where, t = s["index"][at].long(), s["teacher"][at].double() / c["temperature"]
            base = s["teacher_lse"][at].double()[:, None] if "teacher_lse" in s else torch.logsumexp(t, 1, keepdim=True)
            t = (t - base).exp()
            got["loss"].append((t * (t.log() - logp.gather(1, where))).sum(dim=1))
        if c["grad"]:
            d = logp.exp() * t.sum(dim=1, keepdim=True)
            d.scatter_add_(1, where, -t.expand(-1, where.shape[1]).contiguous())
            d *= s["beta"].double() / c.get("temperature", 1.0)
            got["dx"].append((d @ _weights64(s)) * s["dloss"][at].double()[:, None])
    return {key: torch.cat(v) for key, v in got.items() if v}
