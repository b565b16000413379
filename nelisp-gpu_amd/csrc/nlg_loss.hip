// nlg_loss.hip -- losses over a ternary LM head without its logits: softmax
// cross entropy with labels, and the divergence from a teacher's top logits,
// each with its gradient.  No reference counterpart: the reference ends at
// the logits (rmsnorm-fwd, pack-act-rows, bitlinear-dp4a-1f,
// kernels.el:1249-1265, :884-932, :619-634) and takes input gradients with
// ternary-rows-t.
//
//   z[s, o] = bias[o] + (beta[o] g[s]) sum_c W[o, c] q[s, c]   (the composite linear)
//   l[s]    = log sum_o exp(z[s, o] / tau)
//   loss[s] = sum_k t_k (log t_k - (z[s, i_k] / tau - l[s]))    (labels: one k, t = 1)
//   dx[s]   = dloss[s] / tau (T sum_o p_o beta_o W[o] - sum_k t_k beta_{i_k} W[i_k])
// with p_o = exp(z_o / tau - l) and T = sum_k t_k.
//
// 1. k_act_q: the rows to int8.
// 2. k_head<LOGSUM>: the logits in 256 x 64 tiles on the int8 matrix cores;
//    of each only every row's maximum and its sum of exponentials are kept.
// 3. k_loss: a workgroup a row joins those, dots the row with its targets'
//    weights, and leaves the loss.
// Gradient:
// 4. k_order: the rows that have targets, ahead of those that have none.
// and in chunks of those rows:
// 5. k_head<PROB>: the chunk's logits again, as probabilities in two f16.
// 6. k_back: their product with the weights on the f16 matrix cores, in
//    parts of the vocabulary.
// 7. k_dx: the parts' sums, less the targets' weights.
#include <math.h>

#include <type_traits>

#include "nlg_loss.h"
#include "nlg_quant.h"
#include "nlg_scope.h"

int nlg_act_q_launch(const float *x, const float *gain, float eps, const float *attn_mz, uint32_t attn_nc, uint32_t hd,
                     int pro, uint8_t *xq, float *gamma, uint32_t seq, uint32_t cols, hipStream_t st);

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));

#define KC 256  // columns of a step of the logits' product (16 words of a row)
// s_waitcnt vmcnt(n) lgkmcnt(0)
#define WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | (0x7 << 4) | (((n) >> 4) << 14))
// no memory operation moves across it at compile time
#define ORDER() asm volatile("" ::: "memory")

// Probabilities are held as 2^15 p in two f16, the rounded value and what
// the rounding left: 22 bits of those from 2^-15 on, steps of 2^-39 below.
#define PROB_SCALE 32768.0f

struct HeadArgs {
  const uint8_t *xq;    // [rows][cols], k_act_q's order
  const float *gamma;   // [rows]
  const uint32_t *w2;   // [vocab][cols / 16]
  const float *bias;    // [vocab] or null
  const float *beta;    // [1] or [vocab]
  bool per_row;
  uint32_t rows, vocab, cols;
  float coef;           // log2(e) / tau
  uint32_t tiles;       // of the vocabulary
  uint32_t ttiles, group; // token tiles, and of how many an XCD takes one vocabulary tile in a row
  // LOGSUM
  float2 *part;         // [rows][tiles]: the largest z2 = z coef, and the sum of 2^(z2 - it)
  float *bmax;          // [tiles]: the largest |beta|
  // PROB
  const float *lse;     // [rows], base 2
  const int32_t *order; // [rows + 1] or null: the rows in order, then how many of them have targets
  uint32_t first, chunk; // this chunk's
  uint4 *prob;          // [tiles * 32][2][chunk]: eight vocabulary rows of a row, rounded and left over
};

// A maximum in which a NaN loses, so that it meets the sum and not the maximum.
__device__ __forceinline__ float max_nn(float a, float b) { return fmaxf(a, b); }

// (m, l) and (m2, l2), sums of 2^(z - m), as one.  A part that holds nothing
// but -inf has m = -inf and l = 0.
__device__ __forceinline__ void join(float &m, float &l, float m2, float l2) {
  const float t = max_nn(m, m2), r = t == -INFINITY ? 0.0f : t;
  l = l * nlg_exp2(m - r) + l2 * nlg_exp2(m2 - r);
  m = t;
}

enum { LOGSUM, PROB };

// A workgroup owns 256 vocabulary rows x MT = 32 MB tokens, each of its waves
// 64 rows x all tokens, in 32 x 32 x 32 int8 products whose first operand is
// the weights: a lane then holds one token's logits of sixteen vocabulary
// rows a block, and maxima, sums and packing stay in the lane.
// Activations go from memory straight to LDS, two stages of [MT][256 B], a
// step ahead, their 16-byte units swizzled by token; weights come two steps
// ahead into registers, where a field moved to bits 6..7 of its byte is 64
// times its value (the sums are 64 times the exact ones).
// TAIL: cols is no multiple of 256, and the last step's words past the row
// are zeroed.
// Vocabulary tiles of one token group follow each other on an XCD, so weights
// come from HBM once and activations from L2.  From 64 rows on the matrix cores
// bound it: 4,096 rows of 128,256 x 2,560 1.14 ms (2.35 POP/s), 512 rows 150 us;
// one row reads the weights, 82 MB in 19.9 us (4.1 TB/s).  PROB: 1,024 rows 336 us.
template <int MODE, int MB, bool TAIL>
__global__ __launch_bounds__(256, 2) void k_head(HeadArgs a) {
  constexpr int NB = 2, MT = 32 * MB, STAGE = MT * KC;
  constexpr int PI = STAGE / 1024 / 4;  // 1 KiB stage loads per wave and step
  constexpr int NWL = 2 * NB;           // weight loads per wave and step
  typedef uint32_t wvec __attribute__((ext_vector_type(8 * NB)));
  __shared__ __align__(1024) uint8_t s_a0[STAGE];
  __shared__ __align__(1024) uint8_t s_a1[STAGE];
  __shared__ float s_gm[MT], s_ref[MT];
  __shared__ float s_bo[LOSS_TILE], s_be[LOSS_TILE];
  __shared__ float2 s_ml[4][MT];
  __shared__ float s_red[4];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 31, lg = lane >> 5;
  // Workgroups go to the eight XCDs in turn: XCD x takes the tiles x, x + 8, ..
  // of the vocabulary, and of each tile up to sixteen token tiles in a row, so
  // that its L2 keeps those tokens and fetches each weight once for them.
  const uint32_t xcd = blockIdx.x % 8, j = blockIdx.x / 8;
  const uint32_t mine = (a.tiles + 7 - xcd) / 8;  // tiles of this XCD
  const uint32_t each = (a.tiles + 7) / 8 * a.group, g0 = j / each, in = j % each;
  const uint32_t here = min(a.group, a.ttiles - g0 * a.group);
  const uint32_t vt = in / a.group, tt = in % a.group;
  if (vt >= mine || tt >= here) return;
  const uint32_t vtile = vt * 8 + xcd, tok0 = (g0 * a.group + tt) * MT;
  // tokens: of the call, or of the chunk and then by their order
  const uint32_t count = MODE == PROB && a.order ? (uint32_t)a.order[a.rows] : a.rows;
  const uint32_t first = MODE == PROB ? a.first : 0;
  if (MODE == PROB && first + tok0 >= count) return;
  const auto row_of = [&](uint32_t t) {
    const uint32_t at = min(first + tok0 + t, count - 1);
    return MODE == PROB && a.order ? (uint32_t)a.order[at] : at;
  };
  const uint32_t vrow0 = vtile * LOSS_TILE, rbase = vrow0 + w * 64;
  const uint32_t steps = (a.cols + KC - 1) / KC, wng = a.cols / 16;
  uint32_t rc[NB];
  const uint4 *wp[NB];
#pragma unroll
  for (int nt = 0; nt < NB; nt++) {
    const uint32_t r = rbase + 32 * nt + li;
    rc[nt] = r < a.vocab ? r : a.vocab - 1;
    wp[nt] = (const uint4 *)(a.w2 + (size_t)rc[nt] * wng) + 2 * lg;
  }
  typename std::conditional<MODE == PROB, uint64_t, uint32_t>::type xo[PI];
  uint32_t xu[PI];
#pragma unroll
  for (int i = 0; i < PI; i++) {
    const uint32_t k = 4 * (w * PI + i) + lane / 16;
    xu[i] = 16 * ((lane % 16) ^ (k % 16));
    if (MODE == PROB) xo[i] = (uint64_t)row_of(k) * a.cols;
    else xo[i] = (row_of(k) - tok0) * a.cols;
  }
  const uint8_t *const xrow0 = a.xq + (MODE == PROB ? 0 : (size_t)tok0 * a.cols);
  // (macros: register sets handed to a lambda end up in scratch)
#define LOADW(c, dst)                                                                              \
  do {                                                                                             \
    if (TAIL && 16 * (c) + 16 > wng) LOADW_END(c, dst);                                            \
    else _Pragma("unroll") for (int nt = 0; nt < NB; nt++) {                                       \
      const uint4 u0 = wp[nt][4 * (c)], u1 = wp[nt][4 * (c) + 1];                                  \
      dst[8 * nt + 0] = u0.x; dst[8 * nt + 1] = u0.y; dst[8 * nt + 2] = u0.z;                      \
      dst[8 * nt + 3] = u0.w; dst[8 * nt + 4] = u1.x; dst[8 * nt + 5] = u1.y;                      \
      dst[8 * nt + 6] = u1.z; dst[8 * nt + 7] = u1.w;                                              \
    }                                                                                              \
  } while (0)
  // (a unit past the row reads the row's first; in the last step alone, as the masks wait for the loads)
#define LOADW_END(c, dst)                                                                          \
  do {                                                                                             \
    /* 16-byte units: cols is a multiple of 64 */                                                  \
    const bool in0 = 16 * (c) + 8 * lg < wng, in1 = 16 * (c) + 8 * lg + 4 < wng;                   \
    const uint32_t k0 = in0 ? 0xffffffffu : 0u, k1 = in1 ? 0xffffffffu : 0u;                       \
    _Pragma("unroll") for (int nt = 0; nt < NB; nt++) {                                            \
      const uint4 u0 = wp[nt][in0 ? (int)(4 * (c)) : -2 * lg], u1 = wp[nt][in1 ? (int)(4 * (c) + 1) : -2 * lg]; \
      dst[8 * nt + 0] = u0.x & k0; dst[8 * nt + 1] = u0.y & k0; dst[8 * nt + 2] = u0.z & k0;       \
      dst[8 * nt + 3] = u0.w & k0; dst[8 * nt + 4] = u1.x & k1; dst[8 * nt + 5] = u1.y & k1;       \
      dst[8 * nt + 6] = u1.z & k1; dst[8 * nt + 7] = u1.w & k1;                                    \
    }                                                                                              \
  } while (0)
#define LOADA(c, stage)                                                                                \
  do {                                                                                                 \
    _Pragma("unroll") for (int i = 0; i < PI; i++) {                                                   \
      uint32_t col = (c) * KC + xu[i];                                                                 \
      if (TAIL && col >= a.cols) col = 0;                                                              \
      __builtin_amdgcn_global_load_lds(                                                                \
          (const void *)(xrow0 + (xo[i] + col)),                                                       \
          (__attribute__((address_space(3))) void *)((stage) + 1024 * (w * PI + i)), 16, 0, 0);        \
    }                                                                                                  \
  } while (0)
  // the tile's rows' bias and scale, the tokens' scale and log sum
  const uint32_t vr = vrow0 + threadIdx.x;
  const float bo = a.bias && vr < a.vocab ? a.bias[vr] : 0.0f;
  const float be = a.beta[a.per_row ? min(vr, a.vocab - 1) : 0];
  const uint32_t tkc = row_of(threadIdx.x % MT);
  const float gm = a.gamma[tkc];
  const float ref = MODE == PROB ? a.lse[tkc] : 0.0f;
  wvec wA, wB, wC;
  ORDER();
  LOADW(0, wA);
  ORDER();
  LOADA(0, s_a0);
  ORDER();
  LOADW((steps > 1 ? 1 : 0), wB);
  // past the vocabulary: logits of -inf
  s_bo[threadIdx.x] = (vr < a.vocab ? bo : -INFINITY) * a.coef;
  s_be[threadIdx.x] = be;
  if (threadIdx.x < MT) {
    s_gm[threadIdx.x] = gm;
    s_ref[threadIdx.x] = ref;
  }
  v16i acc[NB][MB];
#pragma unroll
  for (int nt = 0; nt < NB; nt++)
#pragma unroll
    for (int mt = 0; mt < MB; mt++) acc[nt][mt] = (v16i){};
  const uint32_t ra = li * KC + 16 * ((8 * lg) ^ (li % 16));
#define RDA(stage, t, dst)                                       \
  do {                                                           \
    const uint8_t *sp = (stage) + (ra ^ (16 * (t)));             \
    _Pragma("unroll") for (int mt = 0; mt < MB; mt++) {          \
      const uint4 u = *(const uint4 *)(sp + 32 * KC * mt);       \
      dst[mt] = (v4i){(int)u.x, (int)u.y, (int)u.z, (int)u.w};   \
    }                                                            \
  } while (0)
#define MMA(stage, WCUR)                                                                          \
  {                                                                                               \
    v4i av[2][MB];                                                                                \
    RDA(stage, 0, av[0]);                                                                         \
    _Pragma("unroll") for (int t = 0; t < 8; t++) {                                               \
      if (t < 7) RDA(stage, t + 1, av[(t + 1) & 1]);                                              \
      __builtin_amdgcn_sched_barrier(0);                                                          \
      _Pragma("unroll") for (int nt = 0; nt < NB; nt++) {                                         \
        const uint32_t x0 = WCUR[8 * nt + t];                                                     \
        const v4i b0 = {(int)((x0 << 6) & 0xC0C0C0C0u), (int)((x0 << 4) & 0xC0C0C0C0u),           \
                        (int)((x0 << 2) & 0xC0C0C0C0u), (int)(x0 & 0xC0C0C0C0u)};                 \
        _Pragma("unroll") for (int mt = 0; mt < MB; mt++)                                         \
          acc[nt][mt] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b0, av[t & 1][mt], acc[nt][mt], 0, 0, 0); \
      }                                                                                           \
    }                                                                                             \
  }
  // step c: its stage has landed (only the weights of step c + 1, issued
  // behind it, may be out) and every wave is done with the other stage; then
  // the next loads are issued (the last repeat), then the products
#define STEP(k, SCUR, SLOAD, WCUR, WLOAD)                       \
  {                                                             \
    const uint32_t c = c0 + (k);                                \
    ORDER();                                                    \
    __builtin_amdgcn_sched_barrier(0);                          \
    WAIT_VM(NWL);                                               \
    __builtin_amdgcn_s_barrier();                               \
    ORDER();                                                    \
    LOADA((c + 1 < steps ? c + 1 : steps - 1), SLOAD);          \
    ORDER();                                                    \
    LOADW((c + 2 < steps ? c + 2 : steps - 1), WLOAD);          \
    __builtin_amdgcn_sched_barrier(0);                          \
    MMA(SCUR, WCUR);                                            \
  }
  uint32_t c0 = 0;
  for (; c0 + 6 <= steps; c0 += 6) {
    STEP(0, s_a0, s_a1, wA, wC)
    STEP(1, s_a1, s_a0, wB, wA)
    STEP(2, s_a0, s_a1, wC, wB)
    STEP(3, s_a1, s_a0, wA, wC)
    STEP(4, s_a0, s_a1, wB, wA)
    STEP(5, s_a1, s_a0, wC, wB)
  }
  if (c0 < steps) {
    STEP(0, s_a0, s_a1, wA, wC)
    if (c0 + 1 < steps) {
      STEP(1, s_a1, s_a0, wB, wA)
      if (c0 + 2 < steps) {
        STEP(2, s_a0, s_a1, wC, wB)
        if (c0 + 3 < steps) {
          STEP(3, s_a1, s_a0, wA, wC)
          if (c0 + 4 < steps) STEP(4, s_a0, s_a1, wB, wA)
        }
      }
    }
  }
#undef STEP
#undef MMA
#undef RDA
#undef LOADA
#undef LOADW
#undef LOADW_END
  WAIT_VM(0);  // the last (repeated) stage loads land before the LDS is given back
  // acc[nt][mt] register r of lane (li, lg): vocabulary row 32 nt + (r % 4) +
  // 8 (r / 4) + 4 lg of the wave's 64, token 32 mt + li
  const float c64 = a.coef * 0.015625f;
  if (MODE == LOGSUM) {
#pragma unroll
    for (int mt = 0; mt < MB; mt++) {
      const float g = s_gm[32 * mt + li] * c64;
      float z[NB * 16], m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int i = 0; i < NB * 16; i++) {
        const int r = i % 16, row = w * 64 + 32 * (i / 16) + (r % 4) + 8 * (r / 4) + 4 * lg;
        z[i] = fmaf(s_be[row] * g, (float)acc[i / 16][mt][r], s_bo[row]);
        m = max_nn(m, z[i]);
      }
      const float at = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int i = 0; i < NB * 16; i++) l += nlg_exp2(z[i] - at);
      const float2 mm = nlg_pair_f32<32>(m), ll = nlg_pair_f32<32>(l);
      m = mm.x;
      l = ll.x;
      join(m, l, mm.y, ll.y);
      if (lg == 0) s_ml[w][32 * mt + li] = make_float2(m, l);
    }
    if (a.per_row && tok0 == 0) {
      const float b = nlg_wave_max_f32(fabsf(be));
      if (lane == 0) s_red[w] = b;
    }
    __syncthreads();
    if (threadIdx.x < MT && tok0 + threadIdx.x < a.rows) {
      float2 v = s_ml[0][threadIdx.x];
#pragma unroll
      for (int k = 1; k < 4; k++) join(v.x, v.y, s_ml[k][threadIdx.x].x, s_ml[k][threadIdx.x].y);
      a.part[(size_t)(tok0 + threadIdx.x) * a.tiles + vtile] = v;
    }
    if (a.per_row && tok0 == 0 && threadIdx.x == 0)
      a.bmax[vtile] = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  } else {
    // beta, where it differs by row, goes into the probabilities, over the
    // power of two above the largest (k_loss left its reciprocal behind)
    const float bn = a.per_row ? a.bmax[0] : 0.0f;
#pragma unroll
    for (int mt = 0; mt < MB; mt++) {
      const float g = s_gm[32 * mt + li] * c64, ls = s_ref[32 * mt + li];
      const uint32_t tk = tok0 + 32 * mt + li;  // of the chunk
#pragma unroll
      for (int nt = 0; nt < NB; nt++) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
          // sixteen rows, of which the lane holds eight: j' and j' + 8 for j' =
          // 4 lg .. 4 lg + 3, as pairs, in the order k_back's weights come in
          union {
            half2v h[4];
            uint4 u;
          } hi, lo;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const int r = 8 * b + 4 * (e & 1) + (e >> 1);
            const int row = w * 64 + 32 * nt + (r % 4) + 8 * (r / 4) + 4 * lg;
            const float z = fmaf(s_be[row] * g, (float)acc[nt][mt][r], s_bo[row]);
            float p = nlg_exp2(z - ls) * PROB_SCALE;
            if (a.per_row) p *= s_be[row] * bn;
            const _Float16 h = (_Float16)p;
            hi.h[e >> 1][e & 1] = h;
            lo.h[e >> 1][e & 1] = (_Float16)(p - (float)h);
          }
          const uint32_t kg = (vrow0 + w * 64 + 32 * nt + 16 * b) / 8 + lg;
          if (tk < a.chunk) {
            uint4 *o = a.prob + (size_t)kg * 2 * a.chunk + tk;
            o[0] = hi.u;
            o[a.chunk] = lo.u;
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------ the loss

struct LossArgs {
  const uint8_t *xq;
  const float *gamma;
  const uint32_t *w2;
  const float *bias, *beta;
  bool per_row;
  uint32_t vocab, cols, tiles, top;
  float coef, itau;            // log2(e) / tau, 1 / tau
  const float2 *part;
  float *bmax;                 // [tiles] in; the first one out: what beta is multiplied by in the probabilities
  const int32_t *index;        // [rows][top]
  const float *teacher;        // [rows][top] or null: labels
  const float *teacher_lse;    // [rows] or null
  float *loss, *lse;           // out; lse may be null
  float *lse2, *sum, *weight;  // for the gradient: log sum in base 2, T, t_k
};

// A workgroup a row: the tiles' maxima and sums joined, the targets' logits
// (each wave one target at a time: the row's int8 values stay in the lanes),
// the teacher's probabilities, the loss.  It waits for the targets' rows of
// weights: W waves, so that up to 4 W of them are on the way together (333 rows
// of 100 targets: 26.4 us with four waves, 14.3 with sixteen; of one target 5 us).
template <int W>
__global__ __launch_bounds__(64 * W) void k_loss(LossArgs a) {
  __shared__ float s_z[LOSS_TOP], s_r[W], s_r2[W];
  const uint32_t s = blockIdx.x;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  // targets' logits, in base 2
  const uint32_t wng = a.cols / 16;
  const uint4 *xr = (const uint4 *)(a.xq + (size_t)s * a.cols);
  const float gm = a.gamma[s];
  // four targets at a time a wave: their weights are on the way together
  for (uint32_t k0 = 4 * w; k0 < a.top; k0 += 4 * W) {
    int32_t at[4];
    const uint32_t *wr[4];
    int q[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      at[e] = a.index[(size_t)s * a.top + min(k0 + e, a.top - 1)];
      if (at[e] < 0 || (uint32_t)at[e] >= a.vocab) at[e] = 0;  // (has no part)
      wr[e] = a.w2 + (size_t)at[e] * wng;
      q[e] = 0;
    }
    for (uint32_t i = lane; i < wng; i += 64) {
      const uint4 y = xr[i];
      uint32_t v[4];
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = wr[e][i];
#pragma unroll
      for (int e = 0; e < 4; e++) q[e] = wdot(v[e], y.x, y.y, y.z, y.w, q[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int sum = nlg_wave_sum_i32(q[e]);
      const float b = a.bias ? a.bias[at[e]] * a.coef : 0.0f;
      if (lane == 0 && k0 + e < a.top)
        s_z[k0 + e] = fmaf(a.beta[a.per_row ? at[e] : 0] * (gm * (a.coef * 0.015625f)), (float)sum, b);
    }
  }
  // the tiles' parts
  float m = -INFINITY, l = 0.0f;
  for (uint32_t i = threadIdx.x; i < a.tiles; i += 64 * W) {
    const float2 p = a.part[(size_t)s * a.tiles + i];
    join(m, l, p.x, p.y);
  }
  const float top = nlg_block_max_f32<W>(m, s_r);
  const float at = top == -INFINITY ? 0.0f : top;
  const float total = nlg_block_sum_f32<W>(l * nlg_exp2(m - at), s_r2);
  const float tail = __builtin_amdgcn_logf(total);  // base 2
  const float ln2 = 0.69314718055994531f;
  // the targets' weights
  const int32_t *ix = a.index + (size_t)s * a.top;
  const float *tl = a.teacher ? a.teacher + (size_t)s * a.top : nullptr;
  float base = 0.0f;  // log2 of the teacher's sum, less its maximum
  float tm = 0.0f;
  const float c2 = a.coef;
  if (tl && a.teacher_lse) {
    tm = a.teacher_lse[s];
  } else if (tl) {
    float mx = -INFINITY, sm = 0.0f;
    for (uint32_t k = threadIdx.x; k < a.top; k += 64 * W)
      if (ix[k] >= 0 && (uint32_t)ix[k] < a.vocab) mx = max_nn(mx, tl[k]);
    tm = nlg_block_max_f32<W>(mx, s_r);
    for (uint32_t k = threadIdx.x; k < a.top; k += 64 * W)
      if (ix[k] >= 0 && (uint32_t)ix[k] < a.vocab) sm += nlg_exp2((tl[k] - tm) * c2);
    base = __builtin_amdgcn_logf(nlg_block_sum_f32<W>(sm, s_r2));
  }
  float loss = 0.0f, sum = 0.0f;
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < a.top; k += 64 * W) {
    float t = 0.0f;
    if (ix[k] >= 0 && (uint32_t)ix[k] < a.vocab) {
      // log2 of the target's weight and of the row's probability of it
      const float lt = !tl ? 0.0f : a.teacher_lse ? (tl[k] * a.itau - tm) * NLG_LOG2E : (tl[k] - tm) * c2 - base;
      const float lp = (s_z[k] - at) - tail;
      t = !tl ? 1.0f : nlg_exp2(lt);
      sum += t;
      if (t != 0.0f) loss += t * (lt - lp);
    }
    a.weight[(size_t)s * a.top + k] = t;
  }
  loss = nlg_block_sum_f32<W>(loss, s_r);
  sum = nlg_block_sum_f32<W>(sum, s_r2);
  float bm = 0.0f;
  if (a.per_row && s == 0) {
    for (uint32_t i = threadIdx.x; i < a.tiles; i += 64 * W) bm = max_nn(bm, a.bmax[i]);
    bm = nlg_block_max_f32<W>(bm, s_r);
  }
  if (threadIdx.x == 0) {
    a.loss[s] = loss * ln2;
    if (a.lse) a.lse[s] = (top + tail) * ln2;
    a.lse2[s] = total > 0.0f ? top + tail : total == 0.0f ? INFINITY : NAN;
    a.sum[s] = sum;
    if (a.per_row && s == 0) {
      int e = 0;
      (void)frexpf(bm, &e);
      a.bmax[0] = bm > 0.0f && bm < INFINITY ? ldexpf(1.0f, -e) : 1.0f;
    }
  }
}

// The rows with targets in order, then those without; order[rows]: how many have.  (One workgroup, two passes: 5.8 us for
// 4,096 rows, where it saves a third of 4 ms.)
__global__ __launch_bounds__(1024) void k_order(const float *sum, int32_t *order, uint32_t rows) {
  __shared__ uint32_t s_n[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t have = 0;
  for (int pass = 0; pass < 2; pass++) {
    uint32_t at = pass ? have : 0;  // where the next rows of this pass go
    for (uint32_t r0 = 0; r0 < rows; r0 += 1024) {
      const uint32_t r = r0 + threadIdx.x;
      const bool put = r < rows && (sum[r] != 0.0f) == (pass == 0);  // (a NaN has targets)
      const uint64_t b = __ballot(put);
      if (lane == 0) s_n[w] = __popcll(b);
      __syncthreads();
      uint32_t before = 0, all = 0;
      for (int k = 0; k < 16; k++) {
        if (k < w) before += s_n[k];
        all += s_n[k];
      }
      if (put) order[at + before + __popcll(b & ((1ull << lane) - 1))] = (int32_t)r;
      at += all;
      __syncthreads();
    }
    if (!pass) have = at;
  }
  if (threadIdx.x == 0) order[rows] = (int32_t)have;
}

// ------------------------------------------------------------------ the gradient's product

struct BackArgs {
  const uint4 *prob;    // [tiles * 32][2][chunk]
  const uint32_t *w2;   // [vocab][wng]
  const int32_t *order; // [rows + 1] or null
  float *acc;           // [splits][chunk][cols]
  uint32_t rows, first, chunk, cols, wng, vocab;
  uint32_t count, share, splits;  // vocabulary rows (rounded up to 256), a part's
};

// 16 x 16 two-bit fields, words by rows, turned: field r of word f was field f of word r.
__device__ __forceinline__ void turn16(uint32_t (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t a = w[i], b = w[i + 8];
    w[i] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    w[i + 8] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  }
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (!(i & 4)) {
      const uint32_t a = w[i], b = w[i + 4];
      w[i] = __builtin_amdgcn_perm(b, a, 0x06020400u);
      w[i + 4] = __builtin_amdgcn_perm(b, a, 0x07030501u);
    }
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (!(i & 2)) {
      const uint32_t a = w[i], b = w[i + 2];
      w[i] = (a & 0x0f0f0f0fu) | ((b << 4) & 0xf0f0f0f0u);
      w[i + 2] = ((a >> 4) & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u);
    }
#pragma unroll
  for (int i = 0; i < 16; i++)
    if (!(i & 1)) {
      const uint32_t a = w[i], b = w[i + 1];
      w[i] = (a & 0x33333333u) | ((b << 2) & 0xccccccccu);
      w[i + 1] = ((a >> 2) & 0x33333333u) | (b & 0xccccccccu);
    }
}

// Sums over a part of the vocabulary of p W, for BM = 32 TM WM rows x 256
// columns a workgroup of 8 waves (WM x WN of them, each TM x TN blocks), in 32
// x 32 x 16 f16 products of the probabilities' two halves.  The weights are
// turned on the way: a thread loads sixteen rows' words of sixteen columns,
// turns the 16 x 16 fields in registers and leaves a word a column in LDS, 256
// vocabulary rows at a time (waves 0..3 the even ones, 4..7 the odd ones); a
// lane makes f16 of its eight fields with one byte permutation a pair (the
// high byte of 0, +1, -2, -1).  Probabilities go from memory to LDS directly,
// 32 vocabulary rows at a time, NS - 1 steps ahead: one is enough for 256 rows,
// fewer are multiplied sooner than memory answers (100 rows of 32,003 x 2,048
// with one step 43.8 us, with three 37.5; 37 rows 30.9 and 27.9; 256 rows a tile
// the same either way).
// The matrix cores bound it: 1,024 rows of 128,256 x 2,560 1.10 ms, 1.22 PFLOP/s
// of both halves.
template <int WM, int TM, int TN, int NS>
__global__ __launch_bounds__(512) void k_back(BackArgs a) {
  constexpr int WN = 8 / WM, BM = 32 * TM * WM;
  static_assert(WN * TN == 8, "256 columns");
  constexpr int STAGE = 4 * 2 * BM;                        // 16-byte units of 32 vocabulary rows
  constexpr int NL = STAGE / 64, PI = NL < 8 ? 1 : NL / 8; // loads a stage, a wave's
  // (apart: a read of one stage waits for no load of another)
  __shared__ __align__(1024) uint4 s_p0[STAGE];
  __shared__ __align__(1024) uint4 s_p1[STAGE];
  __shared__ __align__(1024) uint4 s_p2[NS > 2 ? STAGE : 1];
  __shared__ __align__(1024) uint4 s_p3[NS > 2 ? STAGE : 1];
  __shared__ __align__(16) uint32_t s_w[2 * 16 * 256];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 31, lg = lane >> 5;
  const int wm = w % WM, wn = w / WM;
  // the column tiles of one part and row tile on one XCD, in a row: its L2 then fetches the probabilities once
  const uint32_t ncol = (a.cols + LOSS_CUT - 1) / LOSS_CUT, nrow = a.chunk / BM;
  const uint32_t xcd = blockIdx.x % 8, j = blockIdx.x / 8;
  const uint32_t pair = j / ncol * 8 + xcd, ct = j % ncol;
  if (pair >= nrow * a.splits) return;
  const uint32_t rt = pair % nrow, part = pair / nrow, row0 = rt * BM;
  const uint32_t have = a.order ? (uint32_t)a.order[a.rows] : a.rows;
  if (a.first + row0 >= have) return;
  const uint32_t k0 = part * a.share;
  const uint32_t chunks = min(a.share, a.count - k0) / 256, steps = chunks * 8;
  // thread: words column wi of the tile, rows 16 wr .. 16 wr + 15 of a 256-row block, the even or the odd ones
  const uint32_t wi = threadIdx.x & 15, wr = threadIdx.x >> 4 & 15, odd = w / 4;
  const uint32_t wcol = min(ct * 16 + wi, a.wng - 1);
  uint32_t wv[16];
  const auto loadw = [&](uint32_t block) {
    const uint32_t r0 = k0 + block * 256 + wr * 16;
#pragma unroll
    for (int i = 0; i < 16; i++) wv[i] = a.w2[(size_t)min(r0 + i, a.vocab - 1) * a.wng + wcol];
  };
  const auto storew = [&] {
    turn16(wv);
#pragma unroll
    for (int q = 0; q < 4; q++)
      *(uint4 *)&s_w[odd * 4096 + wr * 256 + 16 * wi + 4 * q] = make_uint4(wv[4 * q], wv[4 * q + 1], wv[4 * q + 2], wv[4 * q + 3]);
  };
  const uint4 *const p0 = a.prob + (size_t)(k0 / 8) * 2 * a.chunk + row0;
  const auto loadp = [&](uint32_t step, uint4 *stage) {
    if (NL < 8 && w >= NL) return;
#pragma unroll
    for (int i = 0; i < PI; i++) {
      const uint32_t u = (w * PI + i) * 64, plane = (u + lane) / BM, r = (u + lane) % BM;
      __builtin_amdgcn_global_load_lds((const void *)(p0 + ((size_t)step * 8 + plane) * a.chunk + r),
                                       (__attribute__((address_space(3))) void *)(stage + u), 16, 0, 0);
    }
  };
  v16f acc[TM][TN];
#pragma unroll
  for (int m = 0; m < TM; m++)
#pragma unroll
    for (int n = 0; n < TN; n++) acc[m][n] = (v16f){};
  const auto mma = [&](uint32_t step, const uint4 *stage) {
    const uint32_t wa = step / 8 % 2 * 4096 + wn * TN * 32 + li, g = step % 8 * 2;
    uint32_t pa = 2 * lg * BM + wm * TM * 32 + li;
    asm volatile("" : "+v"(pa));
    half8v p[2][TM][2];
    uint32_t t[2][TN];
    const auto read = [&](int h) {
#pragma unroll
      for (int n = 0; n < TN; n++) {
        // (an index of its own, as of a stage in each step: of addresses derived from one another the compiler no longer
        // knows which array they are in, and waits for every load that is on its way to LDS)
        uint32_t at = wa + (g + h) * 256 + n * 32;
        asm volatile("" : "+v"(at));
        t[h][n] = s_w[at];
      }
#pragma unroll
      for (int m = 0; m < TM; m++)
#pragma unroll
        for (int q = 0; q < 2; q++)
          p[h][m][q] = __builtin_bit_cast(half8v, stage[pa + (4 * h + q) * BM + m * 32]);
    };
    read(0);
#pragma unroll
    for (int h = 0; h < 2; h++) {  // sixteen vocabulary rows
      if (h == 0) read(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < TN; n++) {
        const uint32_t f = t[h][n] >> (8 * lg);
        union {
          uint32_t u[4];
          half8v h;
        } b;
#pragma unroll
        for (int e = 0; e < 4; e++)
          b.u[e] = __builtin_amdgcn_perm(0u, 0xBCC03C00u, ((f << (8 - 2 * e)) & 0x03000300u) | 0x000c000cu);
#pragma unroll
        for (int m = 0; m < TM; m++) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[h][m][0], b.h, acc[m][n], 0, 0, 0);
#pragma unroll
        for (int m = 0; m < TM; m++) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[h][m][1], b.h, acc[m][n], 0, 0, 0);
      }
    }
  };
  // the first two blocks' weights, each by its half of the waves
  if (odd < chunks) loadw(odd);
  loadp(0, s_p0);
  if (NS > 2) {
    loadp(1, s_p1);
    loadp(2, s_p2);
  }
  if (odd < chunks) storew();
  // A step: its stage has landed (at least those of the next NS - 2 steps are newer), every wave is done with the stage
  // before, which is loaded anew (the last one again at the end).  While one block is multiplied, the half whose block is
  // done loads its next one.
#define STEP(j, SCUR, SLOAD)                                                     \
  {                                                                              \
    const uint32_t s = s0 + (j), next = s / 8 + 1;                               \
    const bool turn = s >= 8 && next < chunks && next % 2 == odd;                \
    WAIT_VM((NS - 2) * PI);                                                      \
    __builtin_amdgcn_s_barrier();                                                \
    ORDER();                                                                     \
    loadp(s + NS - 1 < steps ? s + NS - 1 : steps - 1, SLOAD);                   \
    if (turn && s % 8 == 0) loadw(next);                                         \
    if (turn && s % 8 == 7) storew();                                            \
    mma(s, SCUR);                                                                \
    ORDER();                                                                     \
  }
  if (NS == 2) {
    for (uint32_t s0 = 0; s0 < steps; s0 += 2) {
      STEP(0, s_p0, s_p1)
      STEP(1, s_p1, s_p0)
    }
  } else {
    for (uint32_t s0 = 0; s0 < steps; s0 += 4) {
      STEP(0, s_p0, s_p3)
      STEP(1, s_p1, s_p0)
      STEP(2, s_p2, s_p1)
      STEP(3, s_p3, s_p2)
    }
  }
#undef STEP
  WAIT_VM(0);  // the last (repeated) stages land before the LDS is given back
  // register r: row (r % 4) + 8 (r / 4) + 4 lg of the block, column li
#pragma unroll
  for (int m = 0; m < TM; m++)
#pragma unroll
    for (int n = 0; n < TN; n++) {
      const uint32_t col = ct * LOSS_CUT + (wn * TN + n) * 32 + li;
      if (col >= a.cols) continue;
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const uint32_t row = row0 + (wm * TM + m) * 32 + (r % 4) + 8 * (r / 4) + 4 * lg;
        a.acc[((size_t)part * a.chunk + row) * a.cols + col] = acc[m][n][r];
      }
    }
}

struct DxArgs {
  const float *acc;      // [splits][chunk][cols]
  const uint32_t *w2;
  const float *beta, *bmax, *sum, *weight, *dloss;
  const int32_t *index, *order;
  float *dx;
  uint32_t first, chunk, cols, wng, top, splits;
  float itau;
  bool per_row;
};

// dx of 1,024 columns of a row: four a thread (a byte of the targets' words),
// eight targets' loads and eight parts' at a time.  100 rows of 2,048 in 32 parts
// 5.8 us, 1,024 of 2,560 in 6 parts 14, with 64 targets each 30.
__global__ __launch_bounds__(256) void k_dx(DxArgs a) {
  __shared__ float s_f[LOSS_TOP];
  __shared__ uint32_t s_at[LOSS_TOP];
  const uint32_t i = blockIdx.x, s = a.order ? (uint32_t)a.order[a.first + i] : a.first + i;
  const uint32_t c = blockIdx.y * 256 + threadIdx.x, n4 = a.cols / 4;
  const float T = a.sum[s];
  float4 *const o = (float4 *)(a.dx + (size_t)s * a.cols);
  if (T == 0.0f) {
    if (c < n4) o[c] = make_float4(0, 0, 0, 0);
    return;
  }
  const uint32_t top8 = (a.top + 7) / 8 * 8;
  for (uint32_t k = threadIdx.x; k < top8; k += 256) {
    const float t = k < a.top ? a.weight[(size_t)s * a.top + k] : 0.0f;
    const uint32_t at = t != 0.0f ? (uint32_t)a.index[(size_t)s * a.top + k] : 0u;  // (an index out of range has no weight)
    s_at[k] = at;
    s_f[k] = t * (a.per_row ? a.beta[at] : 1.0f);
  }
  __syncthreads();
  if (c >= n4) return;
  const float tp = T / (PROB_SCALE * (a.per_row ? a.bmax[0] : 1.0f));
  const float4 *p = (const float4 *)(a.acc + (size_t)i * a.cols) + c;
  const size_t stride = (size_t)a.chunk * n4;
  float4 v = make_float4(0, 0, 0, 0);
  uint32_t q = 0;
  for (; q + 8 <= a.splits; q += 8, p += 8 * stride) {
    float4 f[8];
#pragma unroll
    for (int k = 0; k < 8; k++) f[k] = p[k * stride];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      v.x += f[k].x; v.y += f[k].y; v.z += f[k].z; v.w += f[k].w;
    }
  }
  for (; q < a.splits; q++, p += stride) {
    const float4 f = *p;
    v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
  }
  v.x *= tp; v.y *= tp; v.z *= tp; v.w *= tp;
  const uint8_t *const w = (const uint8_t *)a.w2 + c;
  for (uint32_t k0 = 0; k0 < top8; k0 += 8) {
    int b[8];
#pragma unroll
    for (int k = 0; k < 8; k++) b[k] = w[(size_t)s_at[k0 + k] * (a.wng * 4)];
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float f = s_f[k0 + k];
      v.x = fmaf(-f, (float)((b[k] << 30) >> 30), v.x);
      v.y = fmaf(-f, (float)((b[k] << 28) >> 30), v.y);
      v.z = fmaf(-f, (float)((b[k] << 26) >> 30), v.z);
      v.w = fmaf(-f, (float)((b[k] << 24) >> 30), v.w);
    }
  }
  const float g = (a.dloss ? a.dloss[s] : 1.0f) * a.itau * (a.per_row ? 1.0f : a.beta[0]);
  v.x *= g; v.y *= g; v.z *= g; v.w *= g;
  o[c] = v;
}

// ------------------------------------------------------------------ host side

template <class... P>
static bool loss_words(P... p) {
  return ((... | (uintptr_t)p) & 3) == 0;
}

template <int MODE>
static void head_go(HeadArgs &h, uint32_t tokens, hipStream_t st) {
  const bool wide = tokens > 32, tail = h.cols % KC != 0;
  h.ttiles = (tokens + (wide ? 63 : 31)) / (wide ? 64 : 32);
  h.group = h.ttiles < 16 ? h.ttiles : 16;
  const dim3 grid((uint32_t)((uint64_t)((h.ttiles + h.group - 1) / h.group) * h.group * ((h.tiles + 7) / 8) * 8));
  if (wide && tail) hipLaunchKernelGGL((k_head<MODE, 2, true>), grid, dim3(256), 0, st, h);
  else if (wide) hipLaunchKernelGGL((k_head<MODE, 2, false>), grid, dim3(256), 0, st, h);
  else if (tail) hipLaunchKernelGGL((k_head<MODE, 1, true>), grid, dim3(256), 0, st, h);
  else hipLaunchKernelGGL((k_head<MODE, 1, false>), grid, dim3(256), 0, st, h);
}

static int loss_run(const char *what, const float *x, const uint32_t *w2, const float *bias, const float *beta,
                    int beta_per_row, const int32_t *index, const float *teacher, const float *teacher_lse,
                    uint32_t top, float tau, const float *dloss, float *loss, float *lse, float *dx, uint32_t rows,
                    uint32_t vocab, uint32_t cols, void *workspace, size_t workspace_bytes, void *stream) {
  if (!rows) return NLG_OK;
  if (!x || !w2 || !beta || !index || !loss) return nlg_fail("%s: null pointer", what);
  if (cols % 64 || !cols || cols > LOSS_COLS)
    return nlg_fail("%s: cols must be a multiple of 64 in [64, %d] (got %u)", what, LOSS_COLS, cols);
  if (!vocab) return nlg_fail("%s: vocab must be nonzero", what);
  if (!top || top > LOSS_TOP) return nlg_fail("%s: %u targets a row (1 to %d)", what, top, LOSS_TOP);
  if (!(tau > 0.0f) || !(tau < INFINITY)) return nlg_fail("%s: the temperature must be positive", what);
  if (((uintptr_t)x & 15) || ((uintptr_t)w2 & 15) || ((uintptr_t)dx & 15))
    return nlg_fail("%s: x, w2 and dx must be 16-byte aligned", what);
  if (!loss_words(bias, beta, index, teacher, teacher_lse, dloss, loss, lse))
    return nlg_fail("%s: arrays must be 4-byte aligned", what);
  const LossPlan p = loss_plan(rows, vocab, cols, top, dx != nullptr);
  if (!p.ok) return nlg_fail("%s: %u rows of %u logits are too many", what, rows, vocab);
  if (!workspace || workspace_bytes < p.bytes)
    return nlg_fail("%s: workspace holds %zu bytes, needs %llu", what, workspace ? workspace_bytes : 0,
                    (unsigned long long)p.bytes);
  if ((uintptr_t)workspace & 15) return nlg_fail("%s: the workspace must be 16-byte aligned", what);
  const uint64_t nr = (uint64_t)rows * 4, nv = beta_per_row ? (uint64_t)vocab * 4 : 4;
  const NlgSpan at[] = {
      {x, nr * cols}, {w2, (uint64_t)vocab * (cols / 4)}, {bias, (uint64_t)vocab * 4}, {beta, nv}, {index, nr * top},
      {teacher, nr * top}, {teacher_lse, nr}, {dloss, nr}, {loss, nr}, {lse, nr}, {dx, nr * cols}, {workspace, p.bytes}};
  if (nlg_outputs_overlap(at, 12, 4)) return nlg_fail("%s: outputs or the workspace overlap each other or an input", what);
  NLG_SCOPE(what);
  hipStream_t st = nlg_stream(stream);
  uint8_t *const ws = (uint8_t *)workspace;
  uint8_t *const xq = ws + p.xq;
  float *const gamma = (float *)(ws + p.gamma);
  if (nlg_act_q_launch(x, nullptr, 0.0f, nullptr, 0, 0, NLG_PRO_NONE, xq, gamma, rows, cols, st)) return NLG_ERR;
  HeadArgs h{};
  h.xq = xq; h.gamma = gamma; h.w2 = w2; h.bias = bias; h.beta = beta; h.per_row = beta_per_row != 0;
  h.rows = rows; h.vocab = vocab; h.cols = cols; h.coef = NLG_LOG2E / tau;
  h.part = (float2 *)(ws + p.part); h.tiles = p.tiles; h.bmax = (float *)(ws + p.bmax);
  h.lse = (float *)(ws + p.lse); h.prob = (uint4 *)(ws + p.prob); h.chunk = p.chunk;
  head_go<LOGSUM>(h, rows, st);
  NLG_LAUNCHED(what);
  LossArgs l{};
  l.xq = xq; l.gamma = gamma; l.w2 = w2; l.bias = bias; l.beta = beta; l.per_row = h.per_row;
  l.vocab = vocab; l.cols = cols; l.tiles = p.tiles; l.top = top; l.coef = h.coef; l.itau = 1.0f / tau;
  l.part = h.part; l.bmax = h.bmax; l.index = index; l.teacher = teacher; l.teacher_lse = teacher_lse;
  l.loss = loss; l.lse = lse; l.lse2 = (float *)(ws + p.lse); l.sum = (float *)(ws + p.sum);
  l.weight = (float *)(ws + p.weight);
  if (top > 16 && nlg_fits(rows, 1024)) hipLaunchKernelGGL((k_loss<16>), dim3(rows), dim3(1024), 0, st, l);
  else hipLaunchKernelGGL((k_loss<4>), dim3(rows), dim3(256), 0, st, l);
  NLG_LAUNCHED(what);
  if (!dx) return NLG_OK;
  // one tile of rows needs no order
  int32_t *const order = rows > p.bm ? (int32_t *)(ws + p.order) : nullptr;
  if (order) {
    hipLaunchKernelGGL(k_order, dim3(1), dim3(1024), 0, st, l.sum, order, rows);
    NLG_LAUNCHED(what);
  }
  h.order = order;
  BackArgs b{};
  b.prob = h.prob; b.w2 = w2; b.order = order; b.acc = (float *)(ws + p.acc); b.rows = rows; b.chunk = p.chunk;
  b.cols = cols; b.wng = cols / 16; b.vocab = vocab; b.count = p.tiles * LOSS_TILE; b.share = p.share; b.splits = p.splits;
  DxArgs d{};
  d.acc = b.acc; d.w2 = w2; d.beta = beta; d.bmax = h.bmax; d.sum = l.sum; d.weight = l.weight; d.dloss = dloss;
  d.index = index; d.order = order; d.dx = dx; d.chunk = p.chunk; d.cols = cols; d.wng = cols / 16; d.top = top;
  d.splits = p.splits; d.itau = 1.0f / tau; d.per_row = h.per_row;
  for (uint32_t i = 0; i < p.chunks; i++) {
    h.first = b.first = d.first = i * p.chunk;
    const uint32_t n = rows - h.first < p.chunk ? rows - h.first : p.chunk;
    head_go<PROB>(h, n, st);
    NLG_LAUNCHED(what);
    const uint32_t ncol = (cols + LOSS_CUT - 1) / LOSS_CUT, pairs = p.chunk / p.bm * p.splits;
    const dim3 grid((pairs + 7) / 8 * 8 * ncol), blk(512);
    if (p.bm == 256) hipLaunchKernelGGL((k_back<2, 4, 2, 2>), grid, blk, 0, st, b);
    else if (p.bm == 128) hipLaunchKernelGGL((k_back<2, 2, 2, 4>), grid, blk, 0, st, b);
    else if (p.bm == 64) hipLaunchKernelGGL((k_back<2, 1, 2, 4>), grid, blk, 0, st, b);
    else hipLaunchKernelGGL((k_back<1, 1, 1, 4>), grid, blk, 0, st, b);
    NLG_LAUNCHED(what);
    hipLaunchKernelGGL(k_dx, dim3(n, (cols + 1023) / 1024), dim3(256), 0, st, d);
    NLG_LAUNCHED(what);
  }
  return NLG_OK;
}

extern "C" size_t nlg_ternary_xent_workspace(uint32_t rows, uint32_t vocab, uint32_t cols, int grad) {
  return (size_t)loss_plan(rows, vocab, cols, 1, grad != 0).bytes;
}
extern "C" int nlg_ternary_xent(const float *x, const uint32_t *w2, const float *bias, const float *beta,
                                int beta_per_row, const int32_t *label, const float *dloss, float *loss, float *lse,
                                float *dx, uint32_t rows, uint32_t vocab, uint32_t cols, void *workspace,
                                size_t workspace_bytes, void *stream) {
  return loss_run("ternary cross entropy", x, w2, bias, beta, beta_per_row, label, nullptr, nullptr, 1, 1.0f, dloss,
                  loss, lse, dx, rows, vocab, cols, workspace, workspace_bytes, stream);
}

extern "C" size_t nlg_ternary_distill_workspace(uint32_t rows, uint32_t vocab, uint32_t cols, uint32_t top, int grad) {
  return (size_t)loss_plan(rows, vocab, cols, top, grad != 0).bytes;
}
extern "C" int nlg_ternary_distill(const float *x, const uint32_t *w2, const float *bias, const float *beta,
                                   int beta_per_row, const int32_t *index, const float *teacher,
                                   const float *teacher_lse, uint32_t top, float temperature, const float *dloss,
                                   float *loss, float *lse, float *dx, uint32_t rows, uint32_t vocab, uint32_t cols,
                                   void *workspace, size_t workspace_bytes, void *stream) {
  const char *what = "ternary distillation";
  if (!rows) return NLG_OK;
  if (!teacher) return nlg_fail("%s: null pointer", what);
  return loss_run(what, x, w2, bias, beta, beta_per_row, index, teacher, teacher_lse, top, temperature, dloss, loss,
                  lse, dx, rows, vocab, cols, workspace, workspace_bytes, stream);
}
