"""The 8-bit paged KV cache on the CPU: the addressing and the masks that its
kernels use (nelisp-gpu_amd/csrc/nlg_kv8.h, compiled here) against their
definition, for every row and position of small cases; the split of large
ones; and every refusal, which needs no device."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

import kv8_ref as ref
import nlgpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r'''
#include <stdio.h>
#include <stdlib.h>
#include <vector>
#include "nlg_kv8.h"
static uint64_t seed = 1;
static uint32_t rnd(uint32_t n) { seed = seed * 6364136223846793005ull + 1442695040888963407ull; return (uint32_t)(seed >> 33) % n; }
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
// the layout: each byte of a tile once
static int division() {
  for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 8u, 40u, 48u, 65535u, 65537u, 1u << 20, (1u << 27) - 1, 0x7fffffffu, 0x80000000u, 0xffffffffu}) {
    const Kv8Div v = kv8_div(d);
    for (int i = 0; i < 20000; i++) {
      const uint32_t n = i < 5 ? i : i < 10 ? 0x7fffffffu - i : i % 2 ? rnd(1u << 31) : (uint32_t)((uint64_t)d * rnd(0x7fffffffu / d + 1) - i / 2 % 2) & 0x7fffffffu;
      CHECK(kv8_quot(v, n) == n / d);
    }
  }
  return 0;
}
static int layout(uint32_t hd) {
  for (int v = 0; v < 2; v++) {
    std::vector<int> seen(kv8_tile_bytes(hd));
    for (uint32_t at = 0; at < 16; at++) {
      for (uint32_t d = 0; d < hd; d++) seen[v ? kv8_v_byte(at, d) : kv8_k_byte(hd, at, d)]++;
      for (int i = 0; i < 4; i++) seen[kv8_scale_byte(hd, at) + i]++;
    }
    for (int n : seen) CHECK(n == 1);
  }
  return 0;
}
// one call: what the workgroups and waves attend, by sequence, row and position
static int call(bool tree, bool masked, std::vector<int32_t> at, std::vector<int32_t> nodes, uint32_t tmax, uint32_t grp,
                uint32_t bs, uint32_t mbps, uint32_t kvheads) {
  const uint32_t cap = bs * mbps, rows = tmax * grp, batch = at.size();
  const Kv8Split s = kv8_split(batch, rows, kvheads, rnd(2) ? 64 : 128, cap);
  CHECK((uint64_t)s.groups * s.rowsper >= rows && (s.groups - 1) * s.rowsper < rows && s.want >= 1 && 1u << s.rowslog == s.rowsper);
  CHECK(kv8_div_up((1ull << 47) + 12345, 7) * 7 >= (1ull << 47) + 12345);
  std::vector<Kv8Extent> e(batch);
  uint64_t total = 0, slots = 0, pairs = 0;
  for (uint32_t b = 0; b < batch; b++) {
    e[b] = kv8_extent(tree, at[b], nodes[b], tmax, cap);
    CHECK(e[b].end <= cap);
    const uint32_t g = kv8_groups(e[b], grp, s.rowslog);
    CHECK(g <= s.groups && (g == 0) == !e[b].on && (uint64_t)g * s.rowsper >= (e[b].on ? (uint64_t)e[b].nodes * grp : 0));
    total += (uint64_t)g * kv8_steps(e[b]);
    pairs += g;
  }
  CHECK(s.blocks == s.slots * kvheads);
  const Kv8Per range = kv8_per(total ? total : 1, pairs, s.want, s.least, s.unit);
  CHECK(range.first <= range.last && range.first % s.unit == 0 && range.last % s.unit == 0 && range.first >= s.least);
  uint32_t per = range.first;
  for (int i = 0; i < 4 && per < range.last; i++) {  // as the kernel does
    if (batch > 64 || i == 3) {
      per = range.last;
      break;
    }
    uint64_t n = 0;
    for (uint32_t b = 0; b < batch; b++) n += kv8_groups(e[b], grp, s.rowslog) * kv8_chunks(kv8_steps(e[b]), per);
    if (n <= s.want) break;
    const uint32_t next = kv8_more(per, n, s.want, range.last, s.unit);
    CHECK(next > per && next % s.unit == 0);
    per = next;
  }
  for (uint32_t b = 0; b < batch; b++) {
    const int64_t nn = !tree ? 1 : nodes[b] < 0 ? 0 : nodes[b] > (int64_t)tmax ? tmax : nodes[b];
    CHECK(e[b].on == (!tree || (at[b] >= 0 && nn > 0)));
    const uint32_t steps = kv8_steps(e[b]);
    uint32_t chunks = kv8_chunks(steps, per);
    slots += s.one ? s.groups : kv8_groups(e[b], grp, s.rowslog) * chunks;
    CHECK((chunks == 0) == !e[b].on);
    if (!chunks) continue;
    if (s.one) chunks = 1;
    const uint32_t share = s.one ? 1u << 25 : kv8_share(steps, chunks, s.unit);
    CHECK(s.one || (share % s.unit == 0 && share <= per && (uint64_t)share * chunks >= steps && share * (chunks - 1) < steps));
    std::vector<uint64_t> mask(tmax);
    for (auto &m : mask) m = (uint64_t)rnd(1u << 31) << 33 ^ (uint64_t)rnd(1u << 31) << 10 ^ rnd(1024);
    for (uint32_t r = 0; r < rows; r += 1 + rnd(3)) {
      const uint32_t node = r / grp;
      if (node >= nn) continue;
      std::vector<int> seen(cap + 64);
      const uint32_t g0 = r / s.rowsper * s.rowsper;
      const uint32_t stop = masked ? e[b].end : kv8_stop(e[b], (g0 + s.rowsper - 1) / grp);
      const uint32_t mine = masked ? e[b].end : kv8_stop(e[b], node);
      for (uint32_t c = 0; c < chunks; c++) {
        const uint32_t c0 = c * share * KV8_STEP;
        const uint32_t c1 = c0 >= stop ? c0 : stop - c0 < share * KV8_STEP ? stop : c0 + share * KV8_STEP;
        const uint32_t whole = e[b].base < c1 ? e[b].base : c1;
        for (uint32_t p = c0; p < c1; p += KV8_STEP)
          for (uint32_t t = 0; t < 4; t++) {
            const uint32_t q0 = p + t * 16;
            const uint32_t bits = p + KV8_STEP <= whole ? 0xffffu
                                  : kv8_bits(e[b], masked, node, masked ? kv8_word(mask[node], e[b].nodes) : 0, q0);
            CHECK(bits < 65536 && (p < mine || !bits));
            for (uint32_t j = 0; j < 16; j++) seen[q0 + j < cap + 63 ? q0 + j : cap + 63] += bits >> j & 1;
          }
      }
      for (uint32_t p = 0; p < cap + 64; p++) {
        int want;
        if (p >= cap) want = 0;
        else if (!tree) want = (int64_t)p <= at[b];
        else if ((int64_t)p < at[b]) want = 1;
        else if ((int64_t)p >= at[b] + nn) want = 0;
        else if (masked) want = mask[node] >> (p - at[b]) & 1;
        else want = p - at[b] <= node;
        CHECK(seen[p] == want);
      }
    }
  }
  CHECK(slots <= s.slots);
  return 0;
}
int main(void) {
  if (division() || layout(64) || layout(128)) return 1;
  // pages: entries outside the pool, positions behind the table
  const int32_t table[6] = {3, -1, 0, 7, 2147483647, 1};
  const Kv8Pages g = {table, 7, 3, 5, kv8_div(2)};
  CHECK(kv8_tile(g, 0, 4, 1) == (3 * 5 + 4) * 2 + 1 && kv8_tile(g, 0, 0, 4) == 0);
  CHECK(kv8_tile(g, 0, 0, 2) == KV8_NONE && kv8_tile(g, 0, 0, 6) == KV8_NONE && kv8_tile(g, 1, 0, 0) == KV8_NONE);
  CHECK(kv8_tile(g, 1, 0, 3) == KV8_NONE && kv8_tile(g, 1, 4, 5) == (1 * 5 + 4) * 2 + 1 && kv8_tile(g, 0, 0, 0x7fffffffu) == KV8_NONE);
  for (int i = 0; i < 300; i++) {
    const uint32_t bs = 16 * (1 + rnd(4)), mbps = 1 + rnd(i % 10 ? 20 : 300), cap = bs * mbps;
    const uint32_t grp = 1 + rnd(9), kvh = 1 + rnd(i % 3 ? 8 : 300), batch = 1 + rnd(i % 4 ? 4 : 90);
    const uint32_t tm = 1 + rnd(64), tc = 1 + rnd(90);
    std::vector<int32_t> at, nm, nc;
    for (uint32_t b = 0; b < batch; b++) {
      at.push_back((int32_t)rnd(cap + 20) - 2);
      nm.push_back((int32_t)rnd(tm + 4) - 1);
      nc.push_back((int32_t)rnd(tc + 4) - 1);
    }
    if (call(false, false, at, std::vector<int32_t>(batch, 1), 1, grp, bs, mbps, kvh)) return 1;
    if (call(true, true, at, nm, tm, grp, bs, mbps, kvh)) return 1;
    if (call(true, false, at, nc, tc, grp, bs, mbps, kvh)) return 1;
  }
  // extremes
  if (call(false, false, {2147483647}, {1}, 1, 1, 16, 1, 1) || call(true, false, {2147483647}, {5}, 5, 1, 16, 2, 1)) return 1;
  const Kv8Extent e = kv8_extent(true, 2147483647, 2147483647, 2147483647u, 2147483632u);
  CHECK(e.end == 2147483632u && e.base == 2147483647u && kv8_left(e, 2147483616u) == 16);
  CHECK(kv8_steps(e) == (1u << 25) && kv8_per(65535ull << 25, 1, 1, 4, 4).last == 0x7ffffffcu);
  for (uint64_t pos : {16ull, 4096ull, 2147483632ull})
    for (uint32_t batch : {1u, 65535u, 4294967295u})
      for (uint32_t rows : {1u, 16u, 17u, 33u, 65u, 2147483647u}) {
        const Kv8Split s = kv8_split(batch, rows, 8, 64, pos);
        CHECK((uint64_t)s.groups * s.rowsper >= rows && s.slots >= 1);
        CHECK(s.one == (pos <= (rows > 32 ? 128 : rows > 16 ? 256 : 1024)) && s.blocks == s.slots * 8);
      }
  printf("ok\n");
  return 0;
}
'''


def test_addressing_and_masks():
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        with open(src, "w") as f:
            f.write(PROGRAM)
        subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined,address",
                        "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "nelisp-gpu_amd", "csrc"), src, "-o",
                        exe], check=True)
        r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_reference_formats():
    """The reference's own quantisation: within half a step of the value, the largest value kept, ties to even."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((64, 128)) * np.exp(rng.uniform(-20, 20, (64, 1)))
    for fmt in (ref.I8, ref.E4M3):
        c, s = ref.quantise(x, fmt)
        y = ref.values(c, fmt) * s[:, None].astype(np.float64)
        u = np.abs(x / s[:, None].astype(np.float64))
        step = np.ones_like(u) if fmt == ref.I8 else 2.0 ** np.maximum(np.floor(np.log2(u)) - 3, -9)
        assert (np.abs(x - y) <= s[:, None].astype(np.float64) * step * 0.5 * (1 + 1e-6)).all()
        assert np.allclose(np.abs(y).max(axis=1), np.abs(x).max(axis=1), rtol=1e-6)
    c, s = ref.quantise(np.array([[127.0, 0.5, 1.5, -2.5, 0, -0.5]]), ref.I8)
    assert s[0] == 1 and c.view(np.int8).tolist() == [[127, 0, 2, -2, 0, 0]]
    for bad in (np.nan, np.inf, 1e39):
        c, s = ref.quantise(np.array([[1.0, bad]]), ref.E4M3)
        assert not c.any() and np.isnan(s[0])


def test_pool_bytes():
    f = nlgpu.kv_q8_pool_bytes
    assert f(10, 5, 128, 16) == 10 * 5 * 16 * 132 and f(3, 2, 64, 48) == 3 * 2 * 48 * 68
    assert f(0, 5, 128, 16) == f(4, 0, 128, 16) == f(4, 5, 96, 16) == f(4, 5, 128, 0) == f(4, 5, 128, 24) == 0
    assert f(1 << 27, 8, 64, 32) == (1 << 27) * 8 * 32 * 68 and f(1 << 30, 4, 64, 16) == 0


def test_workspace_bytes():
    """0 where one chunk needs none and for sizes that are refused; the bytes of all partials else."""
    w, t = nlgpu.decode_attn_paged_q8_workspace, nlgpu.tree_attn_paged_q8_workspace
    assert w(1, 20, 5, 128, 16, 64) == 0 and w(1, 20, 5, 128, 16, 65) == 5 * 5 * 16 * 130 * 4 + 8
    assert t(1, 8, 20, 5, 64, 16, 16) == 0 and t(1, 8, 20, 5, 64, 16, 17) == 2 * 5 * 32 * 66 * 4 + 8
    assert w(3, 20, 5, 128, 16, 1 << 20) == (512 // 5) * 5 * 16 * 130 * 4 + 24
    assert w(1, 20, 5, 128, 16, 65) == t(1, 1, 20, 5, 128, 16, 65)
    for bad in ((0, 1, 20, 5, 128, 16, 64), (1, 0, 20, 5, 128, 16, 64), (1, 1, 20, 3, 128, 16, 64),
                (1, 1, 20, 0, 128, 16, 64), (1, 1, 0, 5, 128, 16, 64), (1, 1, 20, 5, 96, 16, 64),
                (1, 1, 20, 5, 128, 20, 64), (1, 1, 20, 5, 128, 16, 0), (1, 1, 20, 5, 128, 16, 1 << 27),
                (1, 1 << 31, 20, 5, 128, 16, 64)):
        assert t(*bad) == 0, bad


class At:
    """A buffer at an address that no call below gets to use."""

    def __init__(self, ptr, nbytes=1 << 40):
        self.ptr, self.nbytes = ptr, nbytes


GOOD = At(1 << 20)
ODD = At((1 << 20) + 4)


def refused(call, kw, words):
    """The call is refused with these words, before any device is asked for."""
    with pytest.raises(nlgpu.NlgError) as e:
        call(**kw)
    for w in words.split("|"):
        assert w in str(e.value), (kw, str(e.value))


CACHE = dict(kpool=GOOD, vpool=GOOD, table=GOOD, npool=64, batch=2, kvheads=4, head_dim=128, bs=16, mbps=32)
BAD_CACHE = [(dict(kpool=At(None)), "null"), (dict(vpool=At(None)), "null"), (dict(table=At(None)), "null"),
             (dict(kpool=ODD), "aligned"), (dict(vpool=ODD), "aligned"), (dict(table=At((1 << 20) + 2)), "aligned"),
             (dict(head_dim=96), "head_dim"), (dict(kvheads=0), "kvheads"), (dict(bs=0), "block size"),
             (dict(bs=24), "block size"), (dict(mbps=0), "block"), (dict(mbps=1 << 27), "positions"),
             (dict(npool=0), "pool"), (dict(npool=1 << 31, kvheads=4), "pool")]


@pytest.mark.parametrize("bad,words", BAD_CACHE + [
    (dict(fmt=2), "format"), (dict(fmt=-1), "format"), (dict(qkv=At(None)), "null"), (dict(co=At(None)), "null"),
    (dict(si=At(None)), "null"), (dict(slot=At(None)), "null"), (dict(q=At(None)), "null"), (dict(heads=0), "heads"),
    (dict(batch=0), "batch"), (dict(trows=0), "trows"), (dict(qkv=At((1 << 20) + 4)), "aligned"),
    (dict(q=At((1 << 20) + 4)), "aligned"), (dict(rows=3, seq=None), "sequence"),
    (dict(rows=1 << 30), "too many"), (dict(heads=0xffffffff), "too many")])
def test_append_refuses(bad, words):
    kw = dict(CACHE, qkv=GOOD, qgain=None, kgain=None, eps=1e-6, co=GOOD, si=GOOD, trows=10, slot=GOOD, q=GOOD, rows=2,
              heads=8, seq=GOOD)
    refused(nlgpu.qk_norm_rope_append_paged_q8, dict(kw, **bad), words)


ATTN = dict(CACHE, mbps=128, q=GOOD, out=GOOD, heads=8, workspace=GOOD)
BAD_ATTN = BAD_CACHE + [
    (dict(fmt=2), "format"), (dict(q=At(None)), "null"), (dict(out=At(None)), "null"), (dict(heads=9), "heads"),
    (dict(heads=0), "heads"), (dict(q=ODD), "aligned"), (dict(out=ODD), "aligned"), (dict(workspace=ODD), "aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace=At(1 << 20, 100)), "workspace"),
    (dict(batch=1 << 28), "too many")]


@pytest.mark.parametrize("bad,words", BAD_ATTN + [(dict(lens=At(None)), "null")])
def test_decode_refuses(bad, words):
    refused(nlgpu.decode_attn_paged_q8, dict(ATTN, lens=GOOD, **{}) | bad, words)


@pytest.mark.parametrize("bad,words", BAD_ATTN + [
    (dict(base=At(None)), "null"), (dict(mask=GOOD, tmax=65), "mask"), (dict(mask=ODD), "aligned"),
    (dict(tmax=1 << 31), "queries"), (dict(tmax=1 << 26), "too many")])
def test_tree_refuses(bad, words):
    refused(nlgpu.tree_attn_paged_q8, dict(ATTN, base=GOOD, tmax=8) | bad, words)


@pytest.mark.parametrize("bad,words", BAD_CACHE + [
    (dict(base=At(None)), "null"), (dict(path=At(None)), "null"), (dict(accepted=At(None)), "null"),
    (dict(tmax=65), "at most"), (dict(batch=65536), "batch")])
def test_commit_refuses(bad, words):
    refused(nlgpu.tree_commit_paged_q8, dict(CACHE, base=GOOD, path=GOOD, accepted=GOOD, tmax=8) | bad, words)


@pytest.mark.parametrize("bad,words", BAD_CACHE + [
    (dict(fmt=2), "format"), (dict(slot=At(None)), "null"), (dict(k=At(None)), "null"), (dict(v=At(None)), "null"),
    (dict(k=ODD), "aligned"), (dict(v=ODD), "aligned"), (dict(batch=0), "batch"), (dict(rows=3, seq=None), "sequence"),
    (dict(rows=0xffffffff), "too many")])
def test_read_refuses(bad, words):
    refused(nlgpu.cache_read_paged_q8, dict(CACHE, slot=GOOD, k=GOOD, v=GOOD, rows=2, seq=GOOD) | bad, words)


def test_nothing_to_do_is_no_error():
    """No rows or sequences: nothing is checked further, nothing runs."""
    n = At(None)
    kw = dict(kpool=n, vpool=n, table=n, npool=0, kvheads=0, head_dim=0, bs=0, mbps=0)
    nlgpu.qk_norm_rope_append_paged_q8(qkv=n, qgain=None, kgain=None, eps=0.0, co=n, si=n, trows=0, slot=n, q=n, rows=0,
                                       heads=0, batch=0, **kw)
    nlgpu.decode_attn_paged_q8(q=n, lens=n, out=n, heads=0, workspace=None, batch=0, **kw)
    nlgpu.tree_attn_paged_q8(q=n, base=n, out=n, heads=0, workspace=None, batch=4, tmax=0, **kw)
    nlgpu.tree_commit_paged_q8(base=n, path=n, accepted=n, batch=0, tmax=4, **kw)
    nlgpu.cache_read_paged_q8(slot=n, k=n, v=n, rows=0, batch=0, **kw)


HALF = At((1 << 20) + 2)


@pytest.mark.parametrize("call,kw,names", [
    (nlgpu.qk_norm_rope_append_paged_q8,
     dict(CACHE, qkv=GOOD, qgain=None, kgain=None, eps=1e-6, co=GOOD, si=GOOD, trows=10, slot=GOOD, q=At(1 << 24), rows=2,
          heads=8, seq=GOOD, rpos=GOOD), ("seq", "slot", "rpos")),
    (nlgpu.decode_attn_paged_q8, dict(ATTN, lens=GOOD), ("lens",)),
    (nlgpu.tree_attn_paged_q8, dict(ATTN, base=GOOD, nodes=GOOD, tmax=8), ("base", "nodes")),
    (nlgpu.tree_commit_paged_q8, dict(CACHE, base=GOOD, path=GOOD, accepted=GOOD, tmax=8), ("base", "path", "accepted")),
    (nlgpu.cache_read_paged_q8, dict(CACHE, slot=GOOD, k=GOOD, v=GOOD, rows=2, seq=GOOD), ("seq", "slot"))])
def test_number_arrays_are_aligned(call, kw, names):
    for n in names:
        refused(call, dict(kw, **{n: HALF}), "4-byte aligned|" + n)


@pytest.mark.parametrize("q,qkv", [(1 << 20, 1 << 20), ((1 << 20) + 16, 1 << 20), (1 << 20, (1 << 20) + 8192 - 16),
                                   ((1 << 20) + 16384 - 16, 1 << 20)])
def test_append_refuses_queries_over_its_input(q, qkv):
    """Two rows of 16 heads of 128: 16,384 bytes of input, 8,192 of them queries."""
    kw = dict(CACHE, qkv=At(qkv), qgain=None, kgain=None, eps=1e-6, co=GOOD, si=GOOD, trows=10, slot=GOOD, q=At(q), rows=2,
              heads=8, seq=GOOD)
    refused(nlgpu.qk_norm_rope_append_paged_q8, kw, "overlaps")
