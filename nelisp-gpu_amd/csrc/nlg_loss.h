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
  uint32_t rows_pad;       // rows of a piece's probabilities
  uint32_t piece;          // vocabulary rows of a piece (a multiple of LOSS_TILE)
  uint32_t pieces;
  uint32_t splits;         // parts of a piece that meet at the end, each with sums of its own
  uint32_t share;          // vocabulary rows of such a part
  // offsets into the workspace (256-byte aligned) and its size
  uint64_t xq, gamma, part, bmax, lse, sum, weight, prob, acc, bytes;
};

static inline uint64_t loss_round(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// rows x vocab logits over cols columns, top targets a row (0 refused sizes: ok false)
static inline LossPlan loss_plan(uint32_t rows, uint32_t vocab, uint32_t cols, uint32_t top, bool grad) {
  LossPlan p = {};
  if (!rows || !vocab || !cols || cols % 64 || cols > LOSS_COLS || !top || top > LOSS_TOP || rows > 0x1000000u ||
      vocab > 0x40000000u)
    return p;
  p.tiles = (uint32_t)((vocab + (uint64_t)LOSS_TILE - 1) / LOSS_TILE);
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
    p.bm = rows > 128 ? 256 : rows > 64 ? 128 : rows > 32 ? 64 : 32;
    p.rows_pad = (uint32_t)loss_round(rows, p.bm);
    // a piece's probabilities (two f16 each) are at most 128 MB where a piece of 2,048 rows of the vocabulary is: they are
    // read back from the 256 MB MALL
    uint64_t most = (128ull << 20) / (4ull * p.rows_pad) / LOSS_TILE * LOSS_TILE;
    if (most < 2048) most = 2048;
    p.pieces = (uint32_t)((vocab + most - 1) / most);
    p.piece = (uint32_t)loss_round((vocab + p.pieces - 1) / p.pieces, LOSS_TILE);
    p.pieces = (uint32_t)((vocab + (uint64_t)p.piece - 1) / p.piece);
    // parts until every CU has a workgroup, of 256 vocabulary rows at least
    const uint64_t tiles = (uint64_t)p.rows_pad / p.bm * ((cols + LOSS_CUT - 1) / LOSS_CUT);
    uint64_t n = (256 + tiles - 1) / tiles;
    const uint64_t most_parts = p.piece / LOSS_TILE;
    if (n > most_parts) n = most_parts;
    p.share = (uint32_t)loss_round((p.piece + n - 1) / n, LOSS_TILE);
    p.splits = (uint32_t)((p.piece + (uint64_t)p.share - 1) / p.share);
    p.prob = take((uint64_t)p.rows_pad * p.piece * 4);
    p.acc = take((uint64_t)p.splits * rows * cols * 4);
  }
  p.bytes = at;
  p.ok = true;
  return p;
}
