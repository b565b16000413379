"""The 8-bit paged KV cache: its write (head norms, rotation and quantisation in
one pass), the attention that reads it (one token a sequence, a tree of drafted
tokens, a chunk of a prompt), the commit of a tree's accepted path and the
read-back, each in elementary torch operations and as calls through nlgpu.

A pool is [block][kv head][bs / 16] tiles of sixteen positions, each of
16 * (hd + 4) bytes: the codes, then one f32 scale a position.  K codes lie
[16][hd], V codes [hd][16].  A value is its code (int8 or e4m3) times its
position's scale.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
THETA = 500000.0


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One decoded token of one sequence of the 2B-class model, in one layer.
        {"name": "append_token", "kind": "append", "fmt": "e4m3", "batch": 1, "fewest": 1, "most": 1, "start": 511,
         "heads": 20, "kvheads": 5, "head_dim": 128, "bs": 16, "half": False},
        # Prompts of very different lengths, entering the cache together (q/k-normed model, split-half rotation).
        {"name": "append_prompts", "kind": "append", "fmt": "int8", "batch": 6, "fewest": 77, "most": 1500, "start": 0,
         "heads": 32, "kvheads": 8, "head_dim": 128, "bs": 16, "half": True},
        # One decode step of one sequence, a few hundred tokens in: latency.
        {"name": "decode_one", "kind": "decode", "fmt": "int8", "batch": 1, "shortest": 640, "longest": 640,
         "heads": 20, "kvheads": 5, "head_dim": 128, "bs": 16},
        # A serving step: 32 sequences of very different lengths.
        {"name": "decode_batch", "kind": "decode", "fmt": "int8", "batch": 32, "shortest": 9, "longest": 4096,
         "heads": 20, "kvheads": 5, "head_dim": 128, "bs": 16},
        # Long documents being answered: the cache is all that counts.
        {"name": "decode_long", "kind": "decode", "fmt": "e4m3", "batch": 8, "shortest": 24001, "longest": 32768,
         "heads": 32, "kvheads": 8, "head_dim": 128, "bs": 64},
        # One sequence's sixteen drafted tokens verified at once.
        {"name": "tree_one", "kind": "tree", "fmt": "int8", "batch": 1, "tmax": 16, "fewest": 16, "causal": False,
         "shortest": 1001, "longest": 1001, "heads": 32, "kvheads": 8, "head_dim": 128, "bs": 16},
        # Drafts of many sequences verified together, unequal trees over unequal contexts.
        {"name": "tree_batch", "kind": "tree", "fmt": "e4m3", "batch": 16, "tmax": 32, "fewest": 3, "causal": False,
         "shortest": 130, "longest": 4000, "heads": 20, "kvheads": 5, "head_dim": 128, "bs": 16},
        # A chunk of two long prompts over what is cached of them (head dim 64).
        {"name": "chunk_prompts", "kind": "tree", "fmt": "int8", "batch": 2, "tmax": 512, "fewest": 500, "causal": True,
         "shortest": 1024, "longest": 2047, "heads": 32, "kvheads": 8, "head_dim": 64, "bs": 32},
        # The accepted path of one sequence's tree.
        {"name": "commit_one", "kind": "commit", "fmt": "int8", "batch": 1, "tmax": 16, "start": 1001, "heads": 32,
         "kvheads": 8, "head_dim": 128, "bs": 16},
        # The accepted paths of 64 sequences' trees.
        {"name": "commit_batch", "kind": "commit", "fmt": "e4m3", "batch": 64, "tmax": 32, "start": 777, "heads": 32,
         "kvheads": 8, "head_dim": 128, "bs": 16},
        # A short shared prefix read back.
        {"name": "read_prefix", "kind": "read", "fmt": "e4m3", "batch": 1, "shortest": 100, "longest": 100, "heads": 20,
         "kvheads": 5, "head_dim": 128, "bs": 16},
        # Whole sequences read back into fp16 rows, to leave the device or for an fp16 cache.
        {"name": "read_sequences", "kind": "read", "fmt": "int8", "batch": 8, "shortest": 1000, "longest": 4096,
         "heads": 32, "kvheads": 8, "head_dim": 128, "bs": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kvheads = rng.choice([(20, 5), (32, 8), (16, 16), (16, 8), (32, 4), (8, 2)])
    c = {"kind": rng.choice(["append", "decode", "decode", "tree", "tree", "commit", "read"]),
         "fmt": rng.choice(["int8", "e4m3"]), "heads": heads, "kvheads": kvheads,
         "head_dim": rng.choice([64, 128, 128]), "bs": rng.choice([16, 16, 32, 48, 64])}
    k = c["kind"]
    if k == "append":
        batch = _log(rng, 1, 64)
        most = max(1, min(_log(rng, 1, 2048), 4096 // batch))
        return dict(c, batch=batch, most=most, fewest=rng.randint(1, most), start=rng.choice([0, rng.randint(0, 4000)]),
                    half=rng.choice([True, False]))
    if k == "decode":
        batch = _log(rng, 1, 64)
        longest = max(1, min(_log(rng, 16, 32768), (1 << 20) // (batch * kvheads)))
        return dict(c, batch=batch, longest=longest, shortest=rng.randint(1, longest))
    if k == "tree":
        causal = rng.choice([False, False, True])
        tmax = _log(rng, 1, 512) if causal else _log(rng, 2, 64)
        batch = max(1, min(_log(rng, 1, 32), 1024 // tmax))
        longest = max(1, min(_log(rng, 16, 16384), (1 << 21) // (batch * tmax)))
        return dict(c, batch=batch, tmax=tmax, fewest=rng.randint(1, tmax), causal=causal, longest=longest,
                    shortest=rng.randint(0, longest))
    if k == "commit":
        return dict(c, batch=_log(rng, 1, 64), tmax=_log(rng, 2, 64), start=rng.randint(0, 4000))
    batch = _log(rng, 1, 64)
    longest = max(1, min(_log(rng, 16, 16384), 20000 // batch))
    return dict(c, batch=batch, longest=longest, shortest=rng.randint(1, longest))


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly (the sizes of a batch: the same for every seed, in another order)."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _most(c):
    """Positions that the block table of a sequence has room for."""
    need = {"append": c.get("start", 0) + c.get("most", 0), "commit": c.get("start", 0) + c.get("tmax", 0),
            "tree": c.get("longest", 0) + c.get("tmax", 0)}.get(c["kind"], c.get("longest", 0))
    return -(-need // c["bs"]) * c["bs"]


def _accepted(c):
    return _spread(c["batch"], min(1, c["tmax"]), min(6, c["tmax"]))


# ------------------------------------------------------------------ the inputs

class Inputs:
    """Seeded inputs on the GPU."""

    def __init__(self, c, seed):
        self.c = c
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)
        self.r = np.random.RandomState(int(seed) % (1 << 31))
        self.mbps = _most(c) // c["bs"]
        self.npool = c["batch"] * self.mbps + 1

    def normal(self, *shape, sigma=1.0):
        return torch.randn(shape, generator=self.g, device=DEV, dtype=torch.float32) * sigma

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(shape, generator=self.g, device=DEV, dtype=torch.float32) * (hi - lo) + lo

    def ints(self, values):
        return torch.tensor(np.asarray(values), device=DEV, dtype=torch.int32)

    def sizes(self, lo, hi):
        return self.r.permutation(_spread(self.c["batch"], lo, hi))

    def table(self, used):
        """Blocks in any order for the `used` first positions of each sequence, -1 behind them."""
        t = self.r.permutation(self.npool)[:self.c["batch"] * self.mbps].reshape(self.c["batch"], self.mbps)
        held = -(-np.asarray(used) // self.c["bs"])
        return self.ints(np.where(np.arange(self.mbps)[None, :] < held[:, None], t, -1))

    def pool(self):
        """A pool whose every position holds a row: codes of normal values, scales that differ by position."""
        c = self.c
        n, tiles = 16 * c["head_dim"], self.npool * c["kvheads"] * c["bs"] // 16
        p = torch.empty(tiles, n + 64, device=DEV, dtype=torch.uint8)
        step = (1 << 26) // n
        for b in range(0, tiles, step):
            x = self.normal(min(step, tiles - b), n)
            if c["fmt"] == "int8":
                codes = torch.clamp(torch.round(x * 40.0), -127, 127).to(torch.int8)
            else:
                codes = torch.clamp(x * 140.0, -448, 448).to(torch.float8_e4m3fn)
            p[b:b + step, :n] = codes.view(torch.uint8)
        top = 40.0 if c["fmt"] == "int8" else 140.0
        p[:, n:] = (self.uniform(tiles, 16, lo=0.6, hi=1.6) / top).view(torch.uint8)
        return p.view(self.npool, c["kvheads"], c["bs"] // 16, n + 64)

    def rope(self, rows):
        m = np.arange(self.c["head_dim"] // 2, dtype=np.float64)
        a = np.arange(max(rows, 1), dtype=np.float64)[:, None] * THETA ** (-2.0 * m / self.c["head_dim"])[None, :]
        return [torch.tensor(f(a).astype(np.float32), device=DEV) for f in (np.cos, np.sin)]


def _drafted(i, c):
    """Base and node count of each sequence, and which nodes each node attends: itself and its ancestors."""
    tmax, batch = c["tmax"], c["batch"]
    base, nodes = i.sizes(c["shortest"], c["longest"]), i.sizes(c["fewest"], tmax)
    mask = None
    if not c["causal"]:
        words = np.zeros((batch, tmax), np.uint64)
        for n in range(tmax):
            # a parent among the last eight nodes, or the context itself
            parent = np.maximum(n - 1 - i.r.randint(0, 8, batch), -1)
            above = np.where(parent >= 0, words[np.arange(batch), np.maximum(parent, 0)], np.uint64(0))
            words[:, n] = above | (np.uint64(1) << np.uint64(n))
        mask = torch.tensor(words.view(np.int64), device=DEV)
    return i.ints(base), i.ints(nodes), mask, base + nodes


def prepare(case, seed):
    c = dict(case)
    i = Inputs(c, seed)
    k, hd = c["kind"], c["head_dim"]
    s = {"c": c, "npool": i.npool, "mbps": i.mbps}
    if k == "append":
        count = i.sizes(c["fewest"], c["most"])
        rows = int(count.sum())
        seq = np.repeat(np.arange(c["batch"]), count)
        slot = np.concatenate([np.arange(n) for n in count]) + c["start"]
        s.update(rows=rows, qkv=i.normal(rows, (c["heads"] + 2 * c["kvheads"]) * hd, sigma=1.5), seq=i.ints(seq),
                 slot=i.ints(slot), table=i.table(count + c["start"]), qgain=i.uniform(hd, lo=0.75, hi=1.25),
                 kgain=i.uniform(hd, lo=0.75, hi=1.25), q=torch.zeros(rows, c["heads"] * hd, device=DEV),
                 kpool=i.pool(), vpool=i.pool())
        s["co"], s["si"] = i.rope(c["start"] + c["most"])
    elif k == "decode":
        length = i.sizes(c["shortest"], c["longest"])
        s.update(q=i.normal(c["batch"], c["heads"] * hd, sigma=1.5), last=i.ints(length - 1), table=i.table(length),
                 kpool=i.pool(), vpool=i.pool(), out=torch.zeros(c["batch"], c["heads"] * hd, device=DEV))
    elif k == "tree":
        s["base"], s["nodes"], s["mask"], used = _drafted(i, c)
        s.update(q=i.normal(c["batch"], c["tmax"], c["heads"] * hd, sigma=1.5), table=i.table(used), kpool=i.pool(),
                 vpool=i.pool(), out=torch.zeros(c["batch"], c["tmax"], c["heads"] * hd, device=DEV))
    elif k == "commit":
        taken = np.asarray(i.r.permutation(_accepted(c)))
        # a path goes down the tree: its nodes' numbers rise
        path = np.sort(np.argsort(i.r.rand(c["batch"], c["tmax"]), axis=1)[:, :max(_accepted(c))], axis=1)
        path = np.concatenate([path, np.zeros((c["batch"], c["tmax"] - path.shape[1]), path.dtype)], axis=1)
        s.update(base=i.ints(np.full(c["batch"], c["start"])), path=i.ints(path), accepted=i.ints(taken),
                 table=i.table(np.full(c["batch"], c["start"] + c["tmax"])), kpool=i.pool(), vpool=i.pool())
    else:
        length = i.sizes(c["shortest"], c["longest"])
        rows = int(length.sum())
        s.update(rows=rows, seq=i.ints(np.repeat(np.arange(c["batch"]), length)),
                 slot=i.ints(np.concatenate([np.arange(n) for n in length])), table=i.table(length), kpool=i.pool(),
                 vpool=i.pool())
    if k in ("append", "read"):
        s["k"], s["v"] = (torch.zeros(s["rows"], c["kvheads"], hd, device=DEV, dtype=torch.float16) for _ in "kv")
    return s


# ------------------------------------------------------------------ the plain forms

def _values(c, codes):
    """8-bit codes (as bytes) as the numbers they are."""
    return codes.view(torch.int8 if c["fmt"] == "int8" else torch.float8_e4m3fn).float()


def _rows_at(s, seq, slot, which):
    """Byte offsets [rows, kvheads, hd + 4] of the rows (sequence, slot) in a pool: their codes, then their scales."""
    c = s["c"]
    bs, hd = c["bs"], c["head_dim"]
    block = s["table"].long()[seq, slot // bs]
    record = block[:, None] * c["kvheads"] + torch.arange(c["kvheads"], device=DEV)
    tile = (record * (bs // 16) + (slot % bs // 16)[:, None]) * (16 * (hd + 4))
    at = (slot % 16)[:, None]
    d = torch.arange(hd, device=DEV)
    code = at * hd + d if which == "k" else d * 16 + at
    scale = 16 * hd + 4 * at + torch.arange(4, device=DEV)
    return tile[:, :, None] + torch.cat([code, scale], dim=1)[:, None, :]


def _read(s, seq, slot, which):
    """The rows' values in 32 bits, [rows, kvheads, hd]."""
    c, hd = s["c"], s["c"]["head_dim"]
    raw = s[which + "pool"].view(-1)[_rows_at(s, seq, slot, which)]
    return _values(c, raw[..., :hd].contiguous()) * raw[..., hd:].contiguous().view(torch.float32)


def _quantised(c, x):
    """Rows of 64-bit values [rows, kvheads, hd] as bytes [rows, kvheads, hd + 4].  In 64 bits: next to a border between
    two codes 32 are not enough."""
    top = 127.0 if c["fmt"] == "int8" else 448.0
    scale = (x.abs().amax(dim=-1, keepdim=True).float().double() / top).float()
    y = torch.where(scale > 0, x / scale.double(), 0.0)
    if c["fmt"] == "int8":
        codes = torch.clamp(torch.round(y), -127, 127).to(torch.int8)
    else:
        # three bits behind the first; the smallest step is 2^-9
        step = torch.exp2(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -6))) - 3)
        codes = torch.clamp(torch.round(y / step) * step, -448, 448).float().to(torch.float8_e4m3fn)
    return torch.cat([codes.view(torch.uint8), scale.view(torch.uint8)], dim=-1)


def _append(s):
    c, hd, kvh = s["c"], s["c"]["head_dim"], s["c"]["kvheads"]
    seq, slot = s["seq"].long(), s["slot"].long()
    x = s["qkv"].double().view(s["rows"], -1, hd)
    nh = c["heads"] + kvh
    gain = torch.cat([s["qgain"].expand(c["heads"], hd), s["kgain"].expand(kvh, hd)]).double()
    y = x[:, :nh] / torch.sqrt(x[:, :nh].square().mean(dim=-1, keepdim=True) + EPS) * gain
    co, si = s["co"].double()[slot][:, None, :], s["si"].double()[slot][:, None, :]
    if c["half"]:
        a, b = y[..., :hd // 2], y[..., hd // 2:]
        y = torch.cat([a * co - b * si, a * si + b * co], dim=-1)
    else:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * co - b * si, a * si + b * co], dim=-1).flatten(-2)
    s["q"][:] = y[:, :c["heads"]].reshape(s["rows"], -1).float()
    for which, rows in (("k", y[:, c["heads"]:]), ("v", x[:, nh:])):
        s[which + "pool"].view(-1)[_rows_at(s, seq, slot, which)] = _quantised(c, rows)
        s[which][:] = _read(s, seq, slot, which).half()
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _whole(s, which):
    """The whole sequences' values in 32 bits, [batch, kvheads, positions, hd]."""
    c, hd = s["c"], s["c"]["head_dim"]
    raw = s[which + "pool"][s["table"].long().clamp(min=0)]  # [batch, mbps, kvheads, bs / 16, tile]
    scale = raw[..., 16 * hd:].contiguous().view(torch.float32)[..., None]
    codes = _values(c, raw[..., :16 * hd].contiguous())
    codes = codes.view(*raw.shape[:-1], 16, hd) if which == "k" else codes.view(*raw.shape[:-1], hd, 16).transpose(-1, -2)
    return (codes * scale).transpose(1, 2).reshape(raw.shape[0], raw.shape[2], -1, hd)


def _attend(s, q, seen):
    """q [batch, n, heads * hd] over the cache, seen [batch, n, positions]; [batch, n, heads * hd], a row that sees
    nothing as zeros."""
    c, hd, kvh = s["c"], s["c"]["head_dim"], s["c"]["kvheads"]
    batch, n = q.shape[:2]
    grp = c["heads"] // kvh
    k, v = _whole(s, "k"), _whole(s, "v")
    q = q.view(batch, n, kvh, grp, hd).permute(0, 2, 1, 3, 4).reshape(batch, kvh, n * grp, hd)
    x = (torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)).view(batch, kvh, n, grp, -1)
    x = x.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0))
    z = e.sum(dim=-1, keepdim=True)
    p = (e / torch.where(z > 0, z, 1.0)).view(batch, kvh, n * grp, -1)
    o = torch.matmul(p, v).view(batch, kvh, n, grp, hd)
    return o.permute(0, 2, 1, 3, 4).reshape(batch, n, -1)


def _seen(s):
    """Which positions each node attends, [batch, tmax, positions]."""
    c = s["c"]
    at = torch.arange(_most(c), device=DEV)[None, None, :]
    node = torch.arange(c["tmax"], device=DEV)[None, :, None]
    behind = at - s["base"].long()[:, None, None]
    if s["mask"] is None:
        return behind <= node
    bit = (s["mask"][:, :, None] >> behind.clamp(0, 63)) & 1
    return (behind < 0) | ((behind < s["nodes"].long()[:, None, None]) & (bit == 1))


def _decode(s):
    seen = torch.arange(_most(s["c"]), device=DEV)[None, None, :] <= s["last"].long()[:, None, None]
    s["out"][:] = _attend(s, s["q"][:, None], seen)[:, 0]
    return s["out"]


def _tree(s):
    there = torch.arange(s["c"]["tmax"], device=DEV)[None, :, None] < s["nodes"].long()[:, None, None]
    s["out"][:] = torch.where(there, _attend(s, s["q"], _seen(s)), s["out"])
    return s["out"]


def _commit(s):
    c = s["c"]
    n = torch.arange(c["tmax"], device=DEV)[None, :]
    to = s["base"].long()[:, None] + n
    come = torch.where(n < s["accepted"].long()[:, None], s["base"].long()[:, None] + s["path"].long(), to)
    seq = torch.arange(c["batch"], device=DEV)[:, None].expand(-1, c["tmax"]).reshape(-1)
    for which in "kv":
        p = s[which + "pool"].view(-1)
        p[_rows_at(s, seq, to.reshape(-1), which)] = p[_rows_at(s, seq, come.reshape(-1), which)]
    return _pools(s)


def _pools(s):
    """Both pools as the codes and the scales that they hold, without a copy."""
    c = s["c"]
    n = 16 * c["head_dim"]
    t = torch.int8 if c["fmt"] == "int8" else torch.float8_e4m3fn
    return {w: (s[w][..., :n].view(t), s[w][..., n:].view(torch.float32)) for w in ("kpool", "vpool")}


def _read_back(s):
    for which in "kv":
        s[which][:] = _read(s, s["seq"].long(), s["slot"].long(), which).half()
    return {"k": s["k"], "v": s["v"]}


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
        n = _binding()
        c = s["c"]
        n.init()
        s["views"] = {k: View(t) for k, t in s.items() if isinstance(t, torch.Tensor)}
        s["fmt"] = {"int8": n.KV_I8, "e4m3": n.KV_E4M3}[c["fmt"]]
        sizes = (c["heads"], c["kvheads"], c["head_dim"], c["bs"], s["mbps"])
        if c["kind"] in ("decode", "tree"):
            need = (n.decode_attn_paged_q8_workspace(c["batch"], *sizes) if c["kind"] == "decode"
                    else n.tree_attn_paged_q8_workspace(c["batch"], c["tmax"], *sizes))
            s["views"]["ws"] = View(torch.empty(max(need, 16), device=DEV, dtype=torch.uint8))
    return s["views"]


def _own(s):
    n, c, b = _binding(), s["c"], _views(s)
    k = c["kind"]
    # in the order of torch's current stream (the default one: the library's, which waits for it and it for that); its
    # number alone, a fraction of the 3 us that torch.cuda.current_stream() takes
    st = torch._C._cuda_getCurrentRawStream(s["table"].device.index) or None
    if k == "append":
        n.qk_norm_rope_append_paged_q8(b["qkv"], b["qgain"], b["kgain"], EPS, b["co"], b["si"], s["co"].shape[0],
                                       b["slot"], b["table"], s["npool"], b["q"], b["kpool"], b["vpool"], s["rows"],
                                       c["batch"], c["heads"], c["kvheads"], c["head_dim"], c["bs"], s["mbps"],
                                       seq=b["seq"], half=c["half"], fmt=s["fmt"], stream=st)
    if k in ("append", "read"):
        n.cache_read_paged_q8(b["kpool"], b["vpool"], b["slot"], b["table"], s["npool"], b["k"], b["v"], s["rows"],
                              c["batch"], c["kvheads"], c["head_dim"], c["bs"], s["mbps"], seq=b["seq"], fmt=s["fmt"],
                              stream=st)
        return {w: s[w] for w in ("q", "k", "v") if w in s}
    if k == "decode":
        n.decode_attn_paged_q8(b["q"], b["kpool"], b["vpool"], b["last"], b["table"], s["npool"], b["out"], c["batch"],
                               c["heads"], c["kvheads"], c["head_dim"], c["bs"], s["mbps"], b["ws"], fmt=s["fmt"],
                               stream=st)
        return s["out"]
    if k == "tree":
        n.tree_attn_paged_q8(b["q"], b["kpool"], b["vpool"], b["base"], b["table"], s["npool"], b["out"], c["batch"],
                             c["tmax"], c["heads"], c["kvheads"], c["head_dim"], c["bs"], s["mbps"], b["ws"],
                             nodes=b["nodes"], mask=b.get("mask"), fmt=s["fmt"], stream=st)
        return s["out"]
    n.tree_commit_paged_q8(b["kpool"], b["vpool"], b["base"], b["path"], b["accepted"], b["table"], s["npool"],
                           c["batch"], c["tmax"], c["kvheads"], c["head_dim"], c["bs"], s["mbps"], stream=st)
    return _pools(s)


def run(state):
    """One pass.  Appended rows are also read back, as the cache now gives them."""
    if own:
        return _own(state)
    return {"append": _append, "decode": _decode, "tree": _tree, "commit": _commit,
            "read": _read_back}[state["c"]["kind"]](state)


# ------------------------------------------------------------------ the bounds

def work(case):
    c, k = case, case["kind"]
    hd, kvh, heads = c["head_dim"], c["kvheads"], c["heads"]
    row = 2 * kvh * (hd + 4)  # one position's K and V
    if k == "append":
        n = sum(_spread(c["batch"], c["fewest"], c["most"]))
        return {"bytes": n * (4 * hd * (2 * heads + 2 * kvh) + 2 * row + 4 * kvh * hd + 4 * hd + 8),
                "flops": n * hd * (10 * heads + 16 * kvh)}
    if k == "decode":
        n = sum(_spread(c["batch"], c["shortest"], c["longest"]))
        return {"bytes": n * row + 8 * c["batch"] * heads * hd, "flops": 4 * n * heads * hd}
    if k == "tree":
        base, nodes = sum(_spread(c["batch"], c["shortest"], c["longest"])), _spread(c["batch"], c["fewest"], c["tmax"])
        mean = base / c["batch"]  # bases and node counts meet in an order that the seed sets
        pairs = sum(n * mean + (n * (n + 1) / 2 if c["causal"] else n) for n in nodes)
        return {"bytes": (base + sum(nodes)) * row + 8 * sum(nodes) * heads * hd, "flops": 4 * pairs * heads * hd}
    if k == "commit":
        return {"bytes": 2 * sum(_accepted(c)) * row, "flops": 0}
    n = sum(_spread(c["batch"], c["shortest"], c["longest"]))
    return {"bytes": n * (row + 4 * kvh * hd + 8), "flops": 2 * n * kvh * hd}


# ------------------------------------------------------------------ in 64 bits

def _held64(s, b, which, slots):
    """Values [kvheads, slots, hd] of sequence b's given slots."""
    c = s["c"]
    bs, hd = c["bs"], c["head_dim"]
    pool = s[which + "pool"].movedim(2, 1)  # [block, tile of the block, kvheads, bytes]
    tile = pool[s["table"][b].long()[slots // bs], slots % bs // 16]
    pick = (slots % 16)[:, None, None]
    t = torch.int8 if c["fmt"] == "int8" else torch.float8_e4m3fn
    codes = tile[..., :16 * hd].contiguous().view(t).float()
    codes = codes.view(-1, c["kvheads"], 16, hd) if which == "k" else codes.view(-1, c["kvheads"], hd, 16).mT
    codes = codes.take_along_dim(pick[..., None], dim=2)[:, :, 0].double()
    scale = tile[..., 16 * hd:].contiguous().view(torch.float32).take_along_dim(pick, dim=2)
    return (codes * scale.double()).transpose(0, 1)


def _pieces64(s, b, which, n):
    return torch.cat([_held64(s, b, which, torch.arange(p, min(p + 1024, n), device=DEV)) for p in range(0, n, 1024)],
                     dim=1)


def _attend64(s, b, q, n, hidden):
    """q [rows, heads, hd] of sequence b over its first n positions; hidden [rows, n]."""
    c, hd = s["c"], s["c"]["head_dim"]
    out = torch.zeros(q.shape[0], c["heads"], hd, device=DEV, dtype=torch.float64)
    if not n:
        return out.flatten(1)
    k, v = _pieces64(s, b, "k", n), _pieces64(s, b, "v", n)
    for h in range(c["heads"]):
        g = h // (c["heads"] // c["kvheads"])
        x = (q[:, h].double() @ k[g].t().contiguous() / math.sqrt(hd)).masked_fill(hidden, -math.inf)
        out[:, h] = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0) @ v[g]
    return out.flatten(1)


def _write64(c, x):
    """A row as the cache holds it, and the rounding to fp16 of its values, by the format's definition."""
    largest = {"int8": 127.0, "e4m3": 448.0}[c["fmt"]]
    amax = x.abs().max(dim=-1, keepdim=True).values.to(torch.float32)
    scale = (amax.double() / largest).to(torch.float32).double()
    u = x / scale.clamp(min=1e-300)
    if c["fmt"] == "int8":
        code = u.round().clamp(-127, 127)
    else:
        e = torch.frexp(u).exponent.clamp(min=-5).double() - 4
        code = torch.ldexp(torch.ldexp(u, -e).round(), e).clamp(-448, 448)
    return (code * scale).to(torch.float32).to(torch.float16)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    k, hd = c["kind"], c["head_dim"]
    if k == "append":
        x = s["qkv"].view(s["rows"], -1, hd).double()
        pos = s["slot"].long()
        turned = []
        for h in range(c["heads"] + c["kvheads"]):
            g = (s["qgain"] if h < c["heads"] else s["kgain"]).double()
            y = x[:, h] * torch.rsqrt((x[:, h] ** 2).sum(dim=1, keepdim=True) / hd + EPS) * g
            z = y.view(-1, 2, hd // 2) if c["half"] else y.view(-1, hd // 2, 2).transpose(1, 2)
            w = torch.complex(z[:, 0], z[:, 1]) * torch.complex(s["co"].double(), s["si"].double())[pos]
            z = torch.stack([w.real, w.imag], dim=1)
            turned.append((z if c["half"] else z.transpose(1, 2)).reshape(-1, hd))
        y = torch.stack(turned, dim=1)
        return {"q": y[:, :c["heads"]].flatten(1), "k": _write64(c, y[:, c["heads"]:]),
                "v": _write64(c, x[:, c["heads"] + c["kvheads"]:])}
    if k == "decode":
        rows = []
        for b in range(c["batch"]):
            n = int(s["last"][b]) + 1
            q = s["q"][b].view(1, c["heads"], hd)
            rows.append(_attend64(s, b, q, n, torch.zeros(1, n, device=DEV, dtype=torch.bool)))
        return torch.cat(rows)
    if k == "tree":
        out = torch.zeros(s["out"].shape, device=DEV, dtype=torch.float64)
        for b in range(c["batch"]):
            base, m = int(s["base"][b]), int(s["nodes"][b])
            hidden = torch.ones(m, m, device=DEV, dtype=torch.bool).triu(1)
            if s["mask"] is not None:
                word = s["mask"][b, :m].cpu().numpy().view(np.uint64)
                hidden = torch.tensor([[not (int(w) >> j) & 1 for j in range(m)] for w in word], device=DEV)
            hidden = torch.cat([torch.zeros(m, base, device=DEV, dtype=torch.bool), hidden], dim=1)
            out[b, :m] = _attend64(s, b, s["q"][b, :m].view(m, c["heads"], hd), base + m, hidden)
        return out
    if k == "commit":
        return None  # nothing is computed
    rows = [[_held64(s, b, w, s["slot"][s["seq"] == b].long()).transpose(0, 1) for b in range(c["batch"])] for w in "kv"]
    return {w: torch.cat(r).float().half() for w, r in zip("kv", rows)}
