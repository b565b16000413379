// nlg_kv8.h -- the 8-bit paged KV cache: its layout and how the attention
// over it is split, in one place (plain C++, so both are checked on the CPU).
//
// A pool (one for K, one for V) is [block][kv head][bs / 16] tiles of sixteen
// positions; a tile is 16 * hd codes, then sixteen f32 scales.  K codes lie
// [16][hd]: a lane's sixteen bytes are matrix-operand depth.  V codes lie
// [hd][16]: in the product with the probabilities the positions are the depth,
// so a lane's sixteen bytes are that again, and neither needs a transposition
// when it is read.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define NLG_KV8_HD __host__ __device__ __forceinline__
#else
#define NLG_KV8_HD inline
#endif

#define KV8_TILE 16  // positions of a tile
#define KV8_STEP 64  // positions that a wave attends at once
#define KV8_WAVES 4  // waves of an attention workgroup that takes a chunk (eight where a sequence is one)

NLG_KV8_HD constexpr uint32_t kv8_tile_bytes(uint32_t hd) { return KV8_TILE * (hd + 4); }
// Byte of position `at` (0..15), dimension d in a tile; of its scale.
NLG_KV8_HD constexpr uint32_t kv8_k_byte(uint32_t hd, uint32_t at, uint32_t d) { return at * hd + d; }
NLG_KV8_HD constexpr uint32_t kv8_v_byte(uint32_t at, uint32_t d) { return d * KV8_TILE + at; }
NLG_KV8_HD constexpr uint32_t kv8_scale_byte(uint32_t hd, uint32_t at) { return KV8_TILE * hd + 4 * at; }

// Bytes of one pool, 0 for sizes that the cache does not take.
inline uint64_t kv8_pool_bytes(uint32_t npool, uint32_t bs, uint32_t kvheads, uint32_t hd) {
  if (!npool || !bs || bs % KV8_TILE || !kvheads || (hd != 64 && hd != 128)) return 0;
  const uint64_t tiles = (uint64_t)npool * kvheads * (bs / KV8_TILE);
  // a tile's number is held in 32 bits, the largest standing for "none"
  if ((uint64_t)npool * kvheads > 0xffffffffull || tiles >= 0xffffffffull) return 0;
  return tiles * kv8_tile_bytes(hd);
}

// Division of n < 2^31 by a number that the host knows: n * mul / 2^shift, mul
// the quotient 2^shift / d rounded up with shift = 31 + ceil(log2 d), so that
// its error, below 1 / 2^31 of a step, never reaches the next quotient.
struct Kv8Div {
  uint32_t d, mul, shift;
};
inline Kv8Div kv8_div(uint32_t d) {
  uint32_t l = 0;
  while (l < 31 && (1ull << l) < d) l++;
  return Kv8Div{d, (uint32_t)(((1ull << (31 + l)) + d - 1) / d), 31 + l};
}
NLG_KV8_HD uint32_t kv8_quot(const Kv8Div &v, uint32_t n) { return (uint32_t)(((uint64_t)n * v.mul) >> v.shift); }

// What finds a position's tile.
struct Kv8Pages {
  const int32_t *table;          // [batch][mbps]
  uint32_t npool, mbps, kvheads;
  Kv8Div bpt;                    // tiles of a block
};
#define KV8_NONE 0xffffffffu
// The tile of sequence b's tile number t (position / 16, below 2^31) and kv head h, or
// KV8_NONE outside the table or the pool.
NLG_KV8_HD uint32_t kv8_tile(const Kv8Pages &g, uint32_t b, uint32_t h, uint32_t t) {
  const uint32_t blk = kv8_quot(g.bpt, t);
  if (blk >= g.mbps) return KV8_NONE;
  const int32_t ph = g.table[(uint64_t)b * g.mbps + blk];
  if (ph < 0 || (uint32_t)ph >= g.npool) return KV8_NONE;
  return ((uint32_t)ph * g.kvheads + h) * g.bpt.d + (t - blk * g.bpt.d);
}

// The positions of a sequence: those below `base` all rows attend, those from
// base to end hold nodes; on: it takes part at all.  A decoded token is one
// node at the last position.
struct Kv8Extent {
  uint32_t base, end, nodes;
  bool on;
};
// at: the slot of node 0; cap: the block table's positions.  A sequence without
// a slot or nodes takes no part in a tree; a decoded one attends nothing.
NLG_KV8_HD Kv8Extent kv8_extent(bool tree, int32_t at, int32_t nodes, uint32_t tmax, uint32_t cap) {
  Kv8Extent e;
  e.nodes = nodes < 0 ? 0u : (uint32_t)nodes > tmax ? tmax : (uint32_t)nodes;
  e.base = at < 0 ? 0u : (uint32_t)at;
  e.end = at < 0 ? 0u : e.base + e.nodes < cap ? e.base + e.nodes : cap;
  e.on = !tree || (at >= 0 && e.nodes);
  return e;
}
// Where the rows of nodes up to `last` stop attending, without a mask.
NLG_KV8_HD uint32_t kv8_stop(const Kv8Extent &e, uint32_t last) {
  return last < e.nodes && e.base + last + 1 < e.end ? e.base + last + 1 : e.end;
}
// How many of the sixteen positions from p0 on exist.
NLG_KV8_HD int kv8_left(const Kv8Extent &e, uint32_t p0) { return p0 >= e.end ? 0 : e.end - p0 < 16 ? (int)(e.end - p0) : 16; }
// Which of the sixteen positions from p0 on a row of `node` attends; word: the
// node's mask (its bits past the nodes cleared), without one those up to itself.
NLG_KV8_HD uint32_t kv8_bits(const Kv8Extent &e, bool masked, uint32_t node, uint64_t word, uint32_t p0) {
  const uint32_t all = (1u << kv8_left(e, p0)) - 1;
  if (p0 + 16 <= e.base) return all;
  if (!masked) {
    const int64_t lim = (int64_t)e.base + node + 1 - p0;
    return all & (lim <= 0 ? 0u : lim >= 16 ? 0xffffu : (1u << (int)lim) - 1);
  }
  if (p0 < e.base) {
    const uint32_t off = e.base - p0;  // 1..15
    return all & ((uint32_t)(word << off) | ((1u << off) - 1));
  }
  return p0 - e.base < 64 ? all & (uint32_t)(word >> (p0 - e.base)) : 0u;
}
NLG_KV8_HD uint64_t kv8_word(uint64_t mask, uint32_t nodes) { return nodes < 64 ? mask & ((1ull << nodes) - 1) : mask; }

// How an attention call is laid over workgroups.  Rows (queries x query heads
// of a kv head) come in groups of `rowsper`; up to 32 of them a workgroup's
// waves share (they split the positions), from 33 on each wave has its own
// (`wide`: they share K and V).  A slot is a sequence, a group of its rows and a
// chunk of its positions; every kv head has all of them.  How many there are,
// and how long, follows from the lengths and node counts that the kernel finds
// on the device (kv8_per); a sequence's chunks are of one size.  want: the slots
// that fill the card once, two workgroups on each of its 256 CUs; slots: the most there can be.
// one: no sequence is split, and a slot is its sequence and group.
struct Kv8Split {
  uint32_t rowsper, rowslog, groups, want, least, unit;
  uint64_t slots;
  bool wide, one;
  uint64_t blocks;  // workgroups
};
inline Kv8Split kv8_split(uint32_t batch, uint32_t rows, uint32_t kvheads, uint32_t hd, uint64_t positions) {
  Kv8Split s;
  s.wide = rows > 32;
  // (head dim 128: 17-32 rows in two groups of 16, 34 us for 16 sequences of 8 nodes over 500-4,000, 32/8 heads; 46 in
  // one of 32, whose registers leave one wave a SIMD; 33-64 rows in groups of 16 57 us, 45 wide, with 16 nodes)
  s.rowsper = rows > 64 && hd == 64 ? 128 : rows > 32 ? 64 : rows > 16 && hd == 64 ? 32 : 16;
  s.rowslog = s.rowsper == 16 ? 4 : s.rowsper == 32 ? 5 : s.rowsper == 64 ? 6 : 7;
  s.groups = (uint32_t)(((uint64_t)rows + s.rowsper - 1) / s.rowsper);
  s.unit = s.wide ? 1 : KV8_WAVES;
  s.least = s.wide ? 2 : KV8_WAVES;
  const uint64_t most = (positions + KV8_STEP - 1) / KV8_STEP, pairs = (uint64_t)batch * s.groups;
  s.want = 512 / kvheads ? 512 / kvheads : 1;
  // (eight waves to a workgroup take 1,024 positions in two steps each: less than a second launch.  By the table's
  // positions, as the lengths are on the device: 640 in a table for more take the two launches, 11.0 us for 9.6)
  s.one = most <= (s.rowsper == 16 ? 16 : s.least);
  const uint64_t all = pairs * ((most + s.least - 1) / s.least);
  const uint64_t upto = pairs <= s.want / 2 ? s.want : 2ull * s.want + pairs;
  s.slots = s.one ? pairs : upto < all ? upto : all;
  s.blocks = s.slots * kvheads;
  return s;
}
// A sequence's steps and groups.
NLG_KV8_HD uint32_t kv8_steps(const Kv8Extent &e) {
  return !e.on ? 0u : e.end ? (e.end - 1) / KV8_STEP + 1 : 1u;
}
NLG_KV8_HD uint32_t kv8_groups(const Kv8Extent &e, uint32_t grp, uint32_t rowslog) {
  return e.on ? (e.nodes * grp + (1u << rowslog) - 1) >> rowslog : 0u;  // (a sequence's rows are below 2^31)
}
// Steps of a chunk: a first guess, from the steps of all groups of rows and
// their number, and the largest that is taken.  The last chunk of each may be a
// small one, so total / per + pairs bound the slots: few pairs are split so that
// there are no more than want, and all workgroups run at once; with many (over
// want / 2) there are several rounds anyway, and the chunks are made small
// against the last one's tail.
struct Kv8Per {
  uint32_t first, last;
};
NLG_KV8_HD uint32_t kv8_ceil_to(uint64_t per, uint32_t least, uint32_t unit) {
  if (per < least) per = least;
  per = (per + unit - 1) / unit * unit;
  return per > 0x7fffffffu ? 0x7fffffffu / unit * unit : (uint32_t)per;
}
// At least n / d, 0 < n < 2^48 (from 2^32 on not the least: no 64-bit division).
NLG_KV8_HD uint64_t kv8_div_up(uint64_t n, uint32_t d) {
  return n >> 32 ? ((uint64_t)((uint32_t)(n >> 16) / d) + 1) << 16 : ((uint32_t)n - 1u) / d + 1u;
}
NLG_KV8_HD Kv8Per kv8_per(uint64_t total, uint64_t pairs, uint32_t want, uint32_t least, uint32_t unit) {
  const bool few = pairs <= want / 2;
  Kv8Per p;
  p.last = kv8_ceil_to(kv8_div_up(total, few ? want - (uint32_t)pairs : 2 * want), least, unit);
  p.first = few ? kv8_ceil_to(kv8_div_up(total, want), least, unit) : p.last;
  return p;
}
// The next guess, where `per` gave `slots` > want.
NLG_KV8_HD uint32_t kv8_more(uint32_t per, uint32_t slots, uint32_t want, uint32_t last, uint32_t unit) {
  if ((uint64_t)per * slots >> 32) return last;
  uint64_t next = kv8_div_up((uint64_t)per * slots, want);
  next = (next > per ? next : per + 1) + unit - 1;
  next = next / unit * unit;
  return next < last ? (uint32_t)next : last;
}
NLG_KV8_HD uint32_t kv8_chunks(uint32_t steps, uint32_t per) { return (steps + per - 1) / per; }
NLG_KV8_HD uint32_t kv8_share(uint32_t steps, uint32_t chunks, uint32_t unit) {
  return ((steps + chunks - 1) / chunks + unit - 1) / unit * unit;
}
