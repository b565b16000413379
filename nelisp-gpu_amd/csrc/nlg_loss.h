// nlg_loss.h -- sizes of the losses over a ternary head: how the vocabulary is
// cut into pieces and where the workspace holds what.  Plain C++: also
// compiled for the CPU by tests/test_loss.py.
#pragma once

#include <stddef.h>
#include <stdint.h>

#define LOSS_TILE 256      // vocabulary rows of a workgroup of the logits' product
#define LOSS_TOP 1024      // most targets of a row
#define LOSS_COLS 16384    // most columns (the activations' quantiser's)
#define LOSS_CUT 256       // columns of a workgroup of the gradient's product

struct LossPlan {
  bool ok;
  uint32_t tiles;          // tiles of the vocabulary
  uint32_t bm;             // rows of a workgroup of the gradient's product
  uint32_t chunk, chunks;  // rows whose probabilities are held at a time (a multiple of bm)
  uint32_t splits;         // parts of the vocabulary whose sums meet at the end
  uint32_t share;          // vocabulary rows of a part (a multiple of LOSS_TILE)
  // offsets into the workspace (256-byte aligned) and its size
  uint64_t xq, gamma, part, bmax, lse, sum, weight, order, prob, acc, bytes;
};

static inline uint64_t loss_round(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// How many parts the gradient's product takes its `tiles` tiles of vocabulary in: those of the shortest time by a
// measured 13 us for 256 vocabulary rows of a 256 x 256 tile (as many such tiles as CUs side by side), 6 us to begin and
// end one, and 4 TB/s for what the parts leave and is read again.  Tiles of fewer rows are taken in proportion, 6.5 us for
// 128 and 3.25 for 64, which is less than they were traced at (8 and 5.7, in 38 and 29 us of four such steps): the parts
// are then fewer than those times alone would ask for, as their sum costs more than it gains there (37 rows in 64 parts for
// 32: the product 28 -> 25.6 us, the sum 5 -> 8.4).
static inline uint32_t loss_splits(uint32_t tiles, uint32_t bm, uint64_t workgroups, uint64_t values) {
  uint32_t best = 1;
  double least = 0;
  for (uint32_t n = 1; n <= 64 && n <= tiles; n++) {
    const double rounds = (double)((workgroups * n + 255) / 256), share = (double)((tiles + n - 1) / n);
    const double t = rounds * (share * 13 * bm / 256 + 6) + (double)n * (double)values * 8 / 4e6;
    if (n == 1 || t < least) {
      least = t;
      best = n;
    }
  }
  return best;
}

// rows x vocab logits over cols columns, top targets a row (refused sizes: ok false)
static inline LossPlan loss_plan(uint32_t rows, uint32_t vocab, uint32_t cols, uint32_t top, bool grad) {
  LossPlan p = {};
  if (!rows || !vocab || !cols || cols % 64 || cols > LOSS_COLS || !top || top > LOSS_TOP || rows > 0xffffffu ||
      vocab > 0x1000000u)
    return p;
  p.tiles = (uint32_t)((vocab + (uint64_t)LOSS_TILE - 1) / LOSS_TILE);
  // one launch of the logits' product: 256 threads a tile of 32 rows, tiles rounded up to the XCDs and their groups
  if ((((uint64_t)rows + 31) / 32 + 16) * (p.tiles + 8) * 256 >= 1ull << 32) return p;
  uint64_t at = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t a = at;
    at += loss_round(bytes, 256);
    return a;
  };
  p.xq = take((uint64_t)rows * cols);
  p.gamma = take((uint64_t)rows * 4);
  p.part = take((uint64_t)rows * p.tiles * 8);
  p.bmax = take((uint64_t)p.tiles * 4);
  p.lse = take((uint64_t)rows * 4);
  p.sum = take((uint64_t)rows * 4);
  p.weight = take((uint64_t)rows * top * 4);
  if (grad) {
    p.order = take(((uint64_t)rows + 1) * 4);
    p.bm = rows > 128 ? 256 : rows > 64 ? 128 : rows > 32 ? 64 : 32;
    // chunks of rows whose probabilities (two f16 each) are at most 512 MB, or of bm rows where those have more (256 rows
    // past 524,288 tokens, 16 GB of 2^24)
    const uint64_t row = 4ull * p.tiles * LOSS_TILE;
    uint64_t most = (512ull << 20) / row / p.bm * p.bm;
    if (most < p.bm) most = p.bm;
    p.chunks = (uint32_t)((rows + most - 1) / most);
    p.chunk = (uint32_t)loss_round((rows + (uint64_t)p.chunks - 1) / p.chunks, p.bm);
    p.chunks = (uint32_t)((rows + (uint64_t)p.chunk - 1) / p.chunk);
    const uint64_t workgroups = (uint64_t)(p.chunk / p.bm) * ((cols + LOSS_CUT - 1) / LOSS_CUT);
    p.splits = loss_splits(p.tiles, p.bm, workgroups, (uint64_t)p.chunk * cols);
    p.share = (p.tiles + p.splits - 1) / p.splits * LOSS_TILE;
    p.splits = (uint32_t)(((uint64_t)p.tiles * LOSS_TILE + p.share - 1) / p.share);
    p.prob = take(row * p.chunk);
    p.acc = take((uint64_t)p.splits * p.chunk * cols * 4);
  }
  p.bytes = at;
  p.ok = true;
  return p;
}
