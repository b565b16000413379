// nlg_lora.hip -- low-rank adapters of many requests beside a shared linear,
// forward and backward.  No reference counterpart.
//
//   u[s, j]  = sum_c A[a][j][c] x[s, c]               (j < rank[a]; 0 from there on)
//   y[s, o]  = res[s, o] + scale[a] sum_j B[a][o][j] u[s, j]
//   du[s, j] = scale[a] sum_o B[a][o][j] dy[s, o]
//   dx[s, c] = dres[s, c] + sum_j A[a][j][c] du[s, j]
//   dA[a][j][c] = sum_{s of a} du[s, j] x[s, c],  dB[a][o][j] = scale[a] sum_{s of a} dy[s, o] u[s, j]
//
// with a the adapter of row s's request.  Rows and adapters' values meet in
// 32 bits: on the bf16 matrix cores in parts (the way down in tiles, du, the way
// up in the ternary linear's epilogue), a wave a row in plain f32, else in 16 x
// 16 x 4 f32 products, where the 16-bit values are exact.
//
// v_mfma_f32_16x16x4_f32: lane 16 g + i gives A[i][g] and B[g][i]; its result
// r is C[4 g + r][i].
#include <math.h>

#include "nlg_act_q.h"
#include "nlg_lora.h"
#include "nlg_scope.h"

int nlg_act_q_launch(const float *x, const float *gain, float eps, const float *attn_mz, uint32_t attn_nc, uint32_t hd,
                     int pro, uint8_t *xq, float *gamma, uint32_t seq, uint32_t cols, hipStream_t st);

#define LORA_RANK 128            // most ranks of an adapter
#define LORA_ROWS (65535u * 32)  // most rows (a grid's y dimension)
#define LORA_REQUESTS 0x1000000u
#define LORA_TERNARY_COLS 16384  // most columns beside a ternary linear (its quantiser's)

// p[k] .. p[k + 3] of n values, or where those are not all there any others of
// the n (VEC: n is a multiple of 4 and p aligned).
template <bool VEC>
__device__ __forceinline__ float4 inside4(const float *p, uint32_t k, uint32_t n) {
  if (VEC) return *(const float4 *)(p + min(k, n - 4));
  return make_float4(p[min(k, n - 1)], p[min(k + 1, n - 1)], p[min(k + 2, n - 1)], p[min(k + 3, n - 1)]);
}
template <bool VEC>
__device__ __forceinline__ void store4(float *p, uint32_t n, float4 v) {
  if (VEC) {
    if (n) *(float4 *)p = v;
    return;
  }
  if (n > 0) p[0] = v.x;
  if (n > 1) p[1] = v.y;
  if (n > 2) p[2] = v.z;
  if (n > 3) p[3] = v.w;
}
__device__ __forceinline__ float at4(float4 v, int e) { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; }

// ------------------------------------------------------------------ down: to the ranks

struct DownArgs {
  LoraArgs l;
  const float *x;   // [seq][k]
  uint32_t k;
  bool scaled;
  float *u;         // [seq][rmax]; of several parts, one after the other
  uint32_t *zero;   // TG_SPLIT_COUNTERS words to be zeroed for the projection behind this launch, or null
};
// (256 threads)
__device__ __forceinline__ void zero_counters(const DownArgs &a) {
  static_assert(TG_SPLIT_COUNTERS == 256, "one a thread");
  if (a.zero && blockIdx.x == 0 && blockIdx.y == 0) a.zero[threadIdx.x] = 0;
}

// 32 rows a workgroup, all ranks (NT blocks of sixteen), the contraction over
// its four waves and gridDim.y workgroups.  Each adapter among the rows is one
// pass.
// A step is 128 k, a wave 32 of them, on the bf16 matrix cores
// (v_mfma_f32_16x16x32_bf16: lane 16 g + i holds k = 8 g .. 8 g + 7 of row or
// column i): x as the three bf16 that make up its 24 bits, a bf16 weight as it
// is, an f16 weight as two.  Of the products of parts only that of the last two
// is left out: under 2^-22 of a product, 2^-25 on average.
// Both operands go from memory to LDS directly in runs of 256 bytes and more,
// three stages, two on the way while one is multiplied.  (Read straight into
// the products' layout, 128 bytes of each of 32 rows at a time, 4,731 rows of
// 4,096 took 35 us, and 18.7 without the reads of x.)  An x row's 16-byte units
// are swizzled by its number.
// Waits for memory: 4,731 rows of 4,096 down to 32 ranks 31 us (2.5 TB/s of x, in
// three parts), 241 rows of 2,560 to 8 6.8 us.
// Every load is in bounds and none is masked: ranks behind the rank make sums
// that are thrown away, and a k behind the row has its weights zeroed.
// KMAJOR: weights [k][rmax] (B, in the backward pass), else [rmax][k] (A).
// Weights [k][rmax] are read as NT neighbouring ranks a lane, so block t of
// the ranks is then NT i + t.
// s_waitcnt vmcnt(n) lgkmcnt(0)
#define WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | (0x7 << 4) | (((n) >> 4) << 14))
// no memory operation moves across it at compile time
#define ORDER() asm volatile("" ::: "memory")

template <bool BF, bool KMAJOR, int NT, bool VEC>
__global__ __launch_bounds__(256) void k_lora_down(DownArgs a) {
  constexpr int MT = 2, ROWS = 16 * MT, NX = VEC ? 4 : 16, XB = ROWS * 512, STAGE = XB + NT * 4096;
  __shared__ __align__(1024) uint8_t s_0[STAGE];
  __shared__ __align__(1024) uint8_t s_1[STAGE];
  __shared__ __align__(1024) uint8_t s_2[STAGE];
  __shared__ int32_t s_ad[ROWS];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row0 = blockIdx.x * ROWS;
  zero_counters(a);
  float *const out = a.u + (size_t)blockIdx.y * a.l.seq * a.l.rmax;
  // this workgroup's steps
  const uint32_t all = (a.k + 127) / 128, s0 = (uint64_t)blockIdx.y * all / gridDim.y;
  const uint32_t n = (uint32_t)((uint64_t)(blockIdx.y + 1) * all / gridDim.y) - s0;
  const auto loadx = [&](uint32_t step, uint8_t *stage) {
    const uint32_t k0 = (s0 + min(step, n - 1)) * 128;  // (past the end the last one repeats)
#pragma unroll
    for (int q = 0; q < NX; q++) {
      // VEC: two rows of 32 units an instruction; else a quarter of a row in single values
      const uint32_t at = (w * NX + q) * (VEC ? 1024 : 256), e = at + lane * (VEC ? 16 : 4);
      const uint32_t r = e / 512, unit = e / 16 % 32 ^ (r & 15), k = k0 + 4 * unit + (VEC ? 0 : e / 4 % 4);
      const float *p = a.x + (size_t)min(row0 + r, a.l.seq - 1) * a.k + min(k, a.k - (VEC ? 4 : 1));
      if (VEC) __builtin_amdgcn_global_load_lds((const void *)p, (__attribute__((address_space(3))) void *)(stage + at), 16, 0, 0);
      else __builtin_amdgcn_global_load_lds((const void *)p, (__attribute__((address_space(3))) void *)(stage + at), 4, 0, 0);
    }
  };
  // (the first rows are on the way while their adapters are found)
  loadx(0, s_0);
  loadx(1, s_1);
  ORDER();
  if (w == 0) {
    const int32_t ad = lora_rows(a.l, row0, ROWS, lane);
    if (lane < ROWS) s_ad[lane] = ad;
  }
  __syncthreads();
  const int32_t own = lane < ROWS ? s_ad[lane] : -1;
  uint64_t todo = __ballot(own >= 0);
  const uint64_t none = ~todo;
  bool first = true;
  for (uint32_t p = threadIdx.x; p < ROWS * a.l.rmax; p += 256) {
    const uint32_t r = p / a.l.rmax;
    if ((none >> r & 1) && row0 + r < a.l.seq) out[(size_t)row0 * a.l.rmax + p] = 0.0f;
  }
  while (todo) {
    const int32_t ad = __builtin_amdgcn_readlane(own, __builtin_ctzll(todo));
    const uint64_t mine = __ballot(own == ad);
    todo &= ~mine;
    const uint32_t rank = lora_rank(a.l, ad);
    const uint16_t *const wt = (KMAJOR ? a.l.b : a.l.a) + (size_t)ad * a.l.rmax * a.k;
    v4f acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int t = 0; t < NT; t++) acc[m][t] = (v4f){0, 0, 0, 0};
    const auto loadw = [&](uint32_t step, uint8_t *stage) {
      const uint32_t k0 = (s0 + min(step, n - 1)) * 128;
#pragma unroll
      for (int q = 0; q < NT; q++) {
        const uint32_t at = (w * NT + q) * 1024, e = at + lane * 16;
        const uint16_t *p;
        if (KMAJOR) {  // 128 rows of rmax as they lie
          p = wt + min((size_t)k0 * a.l.rmax + e / 2, (size_t)a.k * a.l.rmax - 8);
        } else {  // 256 bytes of each rank, units swizzled as x's
          const uint32_t j = e / 256, unit = e / 16 % 16 ^ (j & 15);
          p = wt + (size_t)min(j, a.l.rmax - 1) * a.k + min(k0 + 8 * unit, a.k - 8);
        }
        __builtin_amdgcn_global_load_lds((const void *)p, (__attribute__((address_space(3))) void *)(stage + XB + at), 16, 0, 0);
      }
    };
    const auto mul = [&](uint32_t step, const uint8_t *stage) {
      const uint32_t kk = 32 * w + 8 * g, k = (s0 + step) * 128 + kk;  // in the stage, and of the row
      Bf8 p0[MT], p1[MT], p2[MT];
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const uint8_t *const xr = stage + (16 * m + i) * 512;
        const float4 x0 = *(const float4 *)(xr + 16 * (kk / 4 ^ i)), x1 = *(const float4 *)(xr + 16 * ((kk / 4 + 1) ^ i));
        split3(x0.x, x0.y, p0[m].u[0], p1[m].u[0], p2[m].u[0]);
        split3(x0.z, x0.w, p0[m].u[1], p1[m].u[1], p2[m].u[1]);
        split3(x1.x, x1.y, p0[m].u[2], p1[m].u[2], p2[m].u[2]);
        split3(x1.z, x1.w, p0[m].u[3], p1[m].u[3], p2[m].u[3]);
      }
      // k's of the lane that are there
      const uint32_t there = k < a.k ? a.k - k : 0u;
      Bf8 h[NT];
      if (KMAJOR) {
        // (the lane's ranks 8 i .. 8 i + 7 all lie in a row of rmax, or none does)
        static_assert(!KMAJOR || NT == 8, "eight ranks a lane");
        const uint32_t j = 8u * i < a.l.rmax ? 8 * i : 0u;
        uint32_t v[8][4];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint16_t *const p = (const uint16_t *)(stage + XB) + (kk + e) * a.l.rmax + j;
          *(uint4 *)v[e] = *(const uint4 *)p;
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int q = 0; q < 4; q++)
            h[t].u[q] = __builtin_amdgcn_perm(v[2 * q + 1][t / 2], v[2 * q][t / 2], t & 1 ? 0x07060302u : 0x05040100u);
      } else {
#pragma unroll
        for (int t = 0; t < NT; t++)
          h[t].q = *(const uint4 *)(stage + XB + (16 * t + i) * 256 + 16 * (kk / 8 ^ i));
      }
      if ((s0 + step + 1) * 128 > a.k) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int q = 0; q < 4; q++) {
            if (2 * q >= (int)there) h[t].u[q] = 0;
            else if (2 * q + 1 >= (int)there) h[t].u[q] &= 0xffffu;
          }
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        Bf8 w0, w1;
        if (BF) {
          w0 = h[t];
        } else {
#pragma unroll
          for (int q = 0; q < 4; q++) split_f16(h[t].u[q], w0.u[q], w1.u[q]);
        }
#pragma unroll
        for (int m = 0; m < MT; m++) {
          acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p0[m].v, w0.v, acc[m][t], 0, 0, 0);
          acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p1[m].v, w0.v, acc[m][t], 0, 0, 0);
          acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p2[m].v, w0.v, acc[m][t], 0, 0, 0);
          if (!BF) {
            acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p0[m].v, w1.v, acc[m][t], 0, 0, 0);
            acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p1[m].v, w1.v, acc[m][t], 0, 0, 0);
          }
        }
      }
    };
    // step s: its stage has landed (the one behind it may be on the way: of the first two stages, whose rows come ahead
    // of their weights, only the second's weights), every wave is done with the one before it, whose room the loads of step
    // s + 2 take
#define STEP(s, CUR, FREE)              \
    {                                   \
      ORDER();                          \
      if ((s) == 0) WAIT_VM(NT);        \
      else WAIT_VM(NX + NT);            \
      __builtin_amdgcn_s_barrier();     \
      ORDER();                          \
      loadx((s) + 2, FREE);             \
      loadw((s) + 2, FREE);             \
      mul(s, CUR);                      \
    }
    if (!first) {
      loadx(0, s_0);
      loadx(1, s_1);
    }
    first = false;
    loadw(0, s_0);
    loadw(1, s_1);
    for (uint32_t s = 0; s < n; s += 3) {
      STEP(s, s_0, s_2)
      if (s + 1 < n) STEP(s + 1, s_1, s_0)
      if (s + 2 < n) STEP(s + 2, s_2, s_1)
    }
#undef STEP
    ORDER();
    WAIT_VM(0);
    __syncthreads();
    float *const su = (float *)s_0;  // [2][ROWS][16 NT + 4]
    constexpr int PITCH = NT * 16 + 4;
    // a wave's sums: the first two waves', then the others' on top
    static_assert(2 * ROWS * PITCH * 4 <= STAGE, "two waves' sums in a stage");
    if (w < 2)
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) su[(w * ROWS + 16 * m + 4 * g + r) * PITCH + (KMAJOR ? NT * i + t : 16 * t + i)] = acc[m][t][r];
    __syncthreads();
    if (w >= 2)
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int r = 0; r < 4; r++) su[((w - 2) * ROWS + 16 * m + 4 * g + r) * PITCH + (KMAJOR ? NT * i + t : 16 * t + i)] += acc[m][t][r];
    __syncthreads();
    const float sc = a.scaled ? a.l.scale[ad] : 1.0f;
    for (uint32_t p = threadIdx.x; p < ROWS * a.l.rmax; p += 256) {
      const uint32_t r = p / a.l.rmax, j = p % a.l.rmax;
      if (mine >> r & 1)
        out[(size_t)row0 * a.l.rmax + p] = j < rank ? (su[r * PITCH + j] + su[(ROWS + r) * PITCH + j]) * sc : 0.0f;
    }
    __syncthreads();
  }
  WAIT_VM(0);  // (where no row has an adapter: the LDS is not given back before its loads have landed)
}

// Few rows a request: a wave a row and R ranks, the contraction over its
// lanes (eight neighbouring columns each, sixteen bytes of a rank's weights).
template <bool BF, int R>
__device__ __forceinline__ void tok_down(const DownArgs &a, const uint16_t *wt, uint32_t rank, uint32_t row, uint32_t j0,
                                         int lane, float (&u)[R]) {
  const float *const xr = a.x + (size_t)row * a.k;
#pragma unroll
  for (int t = 0; t < R; t++) u[t] = 0.0f;
#pragma unroll 2
  for (uint32_t k = 8 * lane; k < a.k; k += 512) {
    const float4 x0 = *(const float4 *)(xr + k), x1 = *(const float4 *)(xr + k + 4);
    uint4 v[R];
#pragma unroll
    for (int t = 0; t < R; t++) v[t] = *(const uint4 *)(wt + (size_t)min(j0 + t, rank - 1) * a.k + k);
#pragma unroll
    for (int t = 0; t < R; t++) {
      u[t] = fmaf(x0.x, wide<BF>(v[t].x & 0xffff), u[t]);
      u[t] = fmaf(x0.y, wide<BF>(v[t].x >> 16), u[t]);
      u[t] = fmaf(x0.z, wide<BF>(v[t].y & 0xffff), u[t]);
      u[t] = fmaf(x0.w, wide<BF>(v[t].y >> 16), u[t]);
      u[t] = fmaf(x1.x, wide<BF>(v[t].z & 0xffff), u[t]);
      u[t] = fmaf(x1.y, wide<BF>(v[t].z >> 16), u[t]);
      u[t] = fmaf(x1.z, wide<BF>(v[t].w & 0xffff), u[t]);
      u[t] = fmaf(x1.w, wide<BF>(v[t].w >> 16), u[t]);
    }
  }
  // (an infinity becomes NaN, which is what three parts of x make of it: a row's u does not depend on the form)
#pragma unroll
  for (int t = 0; t < R; t++) {
    const float v = nlg_wave_sum_f32(u[t]);
    u[t] = fmaf(v, 0.0f, v);
  }
}

#define TOK_RANKS 4
// a workgroup's 4 waves: sixteen ranks of a row, four a wave (each read of x feeds four dots, and a row of 64 ranks has
// sixteen waves), in plain f32: an adapter's rows are too few for a tile.  Waits for memory; 64 rows of 2,560 with 48
// adapters of up to 64 ranks 7.3 us with their rounding to int8 (tiles of 32 rows, a pass for each adapter among them: 324).
template <bool BF>
__device__ __forceinline__ void tok_down_group(const DownArgs &a, uint32_t row, uint32_t group) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t j0 = (group * 4 + w) * TOK_RANKS;
  if (j0 >= a.l.rmax) return;
  const int32_t ad = __builtin_amdgcn_readfirstlane(lora_rows(a.l, row, 1, lane));
  const uint32_t rank = ad < 0 ? 0u : lora_rank(a.l, ad);
  float u[TOK_RANKS] = {};
  if (j0 < rank) tok_down<BF, TOK_RANKS>(a, a.l.a + (size_t)ad * a.l.rmax * a.k, rank, row, j0, lane, u);
  if (lane < TOK_RANKS) {
    const float v = lane == 0 ? u[0] : lane == 1 ? u[1] : lane == 2 ? u[2] : u[3];
    a.u[(size_t)row * a.l.rmax + j0 + lane] = j0 + lane < rank ? v : 0.0f;
  }
}
template <bool BF>
__global__ __launch_bounds__(256) void k_lora_tok_down(DownArgs a) {  // (never ahead of a projection: no zero)
  tok_down_group<BF>(a, blockIdx.x, blockIdx.y);
}
// That beside the rounding of the same rows to int8 for the shared projection, in one launch.
template <bool BF, int G16>
__global__ __launch_bounds__(256) void k_lora_tok_down_q(DownArgs a, ActQArgs q) {
  if (blockIdx.y == 0) act_q_row<G16, NLG_PRO_NONE>(q, blockIdx.x);
  else tok_down_group<BF>(a, blockIdx.x, blockIdx.y - 1);
  zero_counters(a);
}

// ------------------------------------------------------------------ up: from the ranks

struct UpArgs {
  LoraArgs l;
  const float *u;    // [seq][rmax]
  const float *res;  // [seq][n] or null
  float *y;          // [seq][n] (may be res)
  uint32_t n;
  bool scaled;
};

// 32 rows x 256 columns a workgroup, a wave 64 columns: four neighbouring
// columns a lane, in four blocks (block e of the columns is 4 i + e), so that
// results are stored sixteen bytes a lane.  f32 matrix cores (16 x 16 x 4: no
// operand is rounded further); bound by what moves, 4,616 rows of 6,912 with
// rank up to 32 58 us (4.4 TB/s of res and y).
// KMAJOR: weights [rmax][n] (A, in the backward pass), else [n][rmax] (B).
template <bool BF, bool KMAJOR, bool VEC>
__global__ __launch_bounds__(256) void k_lora_up(UpArgs a) {
  __shared__ int32_t s_ad[32];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const uint32_t row0 = blockIdx.y * 32, col = blockIdx.x * 256 + w * 64 + 4 * i;
  const uint32_t nc = col < a.n ? min(4u, a.n - col) : 0u;
  // what is added to: on the way from the start
  float4 res[2][4];
#pragma unroll
  for (int m = 0; m < 2; m++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t row = min(row0 + 16 * m + 4 * g + r, a.l.seq - 1);
      res[m][r] = a.res ? inside4<VEC>(a.res + (size_t)row * a.n, col, a.n) : make_float4(0, 0, 0, 0);
    }
  if (w == 0) {
    const int32_t ad = lora_rows(a.l, row0, 32, lane);
    if (lane < 32) s_ad[lane] = ad;
  }
  __syncthreads();
  uint32_t todo = 0;
  for (int r = 0; r < 32; r++) {
    if (s_ad[r] >= 0) todo |= 1u << r;
  }
  if (a.y != a.res) {  // rows without an adapter
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint32_t rr = 16 * m + 4 * g + r;
        if (s_ad[rr] < 0 && row0 + rr < a.l.seq) store4<VEC>(a.y + (size_t)(row0 + rr) * a.n + col, nc, res[m][r]);
      }
  }
  while (todo) {
    const int32_t ad = __builtin_amdgcn_readfirstlane(s_ad[__builtin_ctz(todo)]);
    uint32_t mine = 0;
    for (int r = 0; r < 32; r++) mine |= s_ad[r] == ad ? 1u << r : 0u;
    todo &= ~mine;
    const uint32_t rank = lora_rank(a.l, ad);
    const uint16_t *const wt = (KMAJOR ? a.l.a : a.l.b) + (size_t)ad * a.l.rmax * a.n;
    v4f acc[2][4];
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[m][e] = (v4f){0, 0, 0, 0};
    for (uint32_t j0 = 0; j0 < rank; j0 += 16) {
      const uint32_t j = j0 + 4 * g;  // lane group g's ranks j .. j + 3
      float4 uv[2];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        const uint32_t row = min(row0 + 16 * m + i, a.l.seq - 1);
        uv[m] = *(const float4 *)(a.u + (size_t)row * a.l.rmax + min(j, a.l.rmax - 4));
      }
      uint2 v[4];  // KMAJOR: rank j + q, columns col ..; else column col + q, ranks j ..
#pragma unroll
      for (int q = 0; q < 4; q++) {
        if (KMAJOR) v[q] = *(const uint2 *)(wt + (size_t)min(j + q, a.l.rmax - 1) * a.n + min(col, a.n - 4));
        else v[q] = *(const uint2 *)(wt + (size_t)min(col + q, a.n - 1) * a.l.rmax + min(j, a.l.rmax - 4));
      }
      if (j0 + 16 > rank) {  // ranks behind the rank: neither factor counts
#pragma unroll
        for (int m = 0; m < 2; m++) {
          if (j >= rank) uv[m].x = 0.0f;
          if (j + 1 >= rank) uv[m].y = 0.0f;
          if (j + 2 >= rank) uv[m].z = 0.0f;
          if (j + 3 >= rank) uv[m].w = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const uint32_t c = KMAJOR ? j + q : j;
          if (KMAJOR) {
            if (c >= rank) v[q] = make_uint2(0, 0);
          } else {
            if (c >= rank) v[q].x &= 0xffff0000u;
            if (c + 1 >= rank) v[q].x &= 0xffffu;
            if (c + 2 >= rank) v[q].y &= 0xffff0000u;
            if (c + 3 >= rank) v[q].y &= 0xffffu;
          }
        }
      }
#pragma unroll
      for (int s = 0; s < 4; s++) {  // rank j + s
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint2 p = v[KMAJOR ? s : e];
          const int f = KMAJOR ? e : s;
          const uint32_t h = (f & 2 ? p.y : p.x) >> (16 * (f & 1)) & 0xffff;
          const float b = wide<BF>(h);
#pragma unroll
          for (int m = 0; m < 2; m++)
            acc[m][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(at4(uv[m], s), b, acc[m][e], 0, 0, 0);
        }
      }
    }
    const float sc = a.scaled ? a.l.scale[ad] : 1.0f;
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint32_t rr = 16 * m + 4 * g + r;
        if (!(mine >> rr & 1)) continue;
        const size_t o = (size_t)(row0 + rr) * a.n + col;
        float4 v = res[m][r];
        v.x = fmaf(sc, acc[m][0][r], v.x);
        v.y = fmaf(sc, acc[m][1][r], v.y);
        v.z = fmaf(sc, acc[m][2][r], v.z);
        v.w = fmaf(sc, acc[m][3][r], v.w);
        store4<VEC>(a.y + o, nc, v);
      }
  }
}

// Few rows a request: a wave a row and NC steps of 64 / L columns, L lanes a
// column (eight neighbouring ranks each: sixteen bytes), all on the way
// together.  Bound by the adapters' bytes: 64 rows of 48 adapters, up to 64
// ranks to 6,912 columns, 11.9 us (tiles of 32 rows: 120).
template <int L, int NC>
struct TokUp {
  uint4 v[NC];
  float res[NC];
  __device__ __forceinline__ void load(const UpArgs &a, const uint16_t *wt, uint32_t rank, uint32_t row, uint32_t c0,
                                       int lane) {
#pragma unroll
    for (int e = 0; e < NC; e++) {
      const uint32_t c = c0 + e * (64 / L) + lane / L;
      v[e] = make_uint4(0, 0, 0, 0);
      if (8u * (lane % L) < rank && c < a.n) v[e] = *(const uint4 *)(wt + (size_t)c * a.l.rmax + 8 * (lane % L));
      res[e] = lane % L == 0 && c < a.n && a.res ? a.res[(size_t)row * a.n + c] : 0.0f;
    }
  }
  template <bool BF>
  __device__ __forceinline__ void store(const UpArgs &a, uint32_t rank, float sc, uint32_t row, const float (&u)[8],
                                        uint32_t c0, int lane) {
#pragma unroll
    for (int e = 0; e < NC; e++) {
      const uint32_t c = c0 + e * (64 / L) + lane / L;
      float y = 0.0f;
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const uint32_t p = q < 2 ? v[e].x : q < 4 ? v[e].y : q < 6 ? v[e].z : v[e].w;
        if (8u * (lane % L) + q < rank) y = fmaf(u[q], wide<BF>(p >> (16 * (q & 1)) & 0xffff), y);
      }
      if (L >= 2) y += __int_as_float(nlg_dpp<0xB1>(__float_as_int(y)));
      if (L >= 4) y += __int_as_float(nlg_dpp<0x4E>(__float_as_int(y)));
      if (L >= 8) y += __int_as_float(nlg_dpp<0x141>(__float_as_int(y)));   // half-row mirror
      if (L >= 16) y += __int_as_float(nlg_dpp<0x140>(__float_as_int(y)));  // row mirror
      if (lane % L == 0 && c < a.n) a.y[(size_t)row * a.n + c] = fmaf(sc, y, res[e]);
    }
  }
};

template <bool BF, int L, int NC>
__global__ __launch_bounds__(256) void k_lora_tok_up(UpArgs a) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t row = blockIdx.y, c0 = (blockIdx.x * 4 + w) * (64 / L * NC);
  if (c0 >= a.n) return;
  const int32_t ad = __builtin_amdgcn_readfirstlane(lora_rows(a.l, row, 1, lane));
  if (ad < 0 && a.y == a.res) return;
  const uint32_t rank = ad < 0 ? 0u : lora_rank(a.l, ad), j = 8 * (lane % L);
  TokUp<L, NC> t;
  t.load(a, a.l.b + (size_t)max(ad, 0) * a.l.rmax * a.n, rank, row, c0, lane);
  float u[8] = {};
  if (j < a.l.rmax) {
    const float *p = a.u + (size_t)row * a.l.rmax + j;
    const float4 u0 = *(const float4 *)p, u1 = *(const float4 *)(p + 4);
    u[0] = u0.x; u[1] = u0.y; u[2] = u0.z; u[3] = u0.w; u[4] = u1.x; u[5] = u1.y; u[6] = u1.z; u[7] = u1.w;
  }
  t.template store<BF>(a, rank, ad < 0 ? 0.0f : a.l.scale[ad], row, u, c0, lane);
}

// A few rows of small adapters in one launch: every workgroup finds its row's
// u again (two ranks a wave at a time), while its columns' weights are on the
// way.  One token, 2,560 -> 2,560 at rank 16: 4.6 us, a launch and two round trips
// to memory (the call with its projection 8.2 us; with the ways down and up
// apart, of tiles, 13).
template <bool BF, int L>
__global__ __launch_bounds__(512) void k_lora_tok(DownArgs d, UpArgs a) {
  __shared__ float s_u[LORA_RANK];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t row = blockIdx.y, c0 = (blockIdx.x * 8 + w) * (64 / L);
  const int32_t ad = __builtin_amdgcn_readfirstlane(lora_rows(a.l, row, 1, lane));
  const uint32_t rank = ad < 0 ? 0u : lora_rank(a.l, ad), j = 8 * (lane % L);
  TokUp<L, 1> t;
  t.load(a, a.l.b + (size_t)max(ad, 0) * a.l.rmax * a.n, rank, row, c0, lane);
  const float sc = ad < 0 ? 0.0f : a.l.scale[ad];
  for (uint32_t j0 = 2 * w; j0 < a.l.rmax; j0 += 16) {
    float u[2] = {};
    if (j0 < rank) tok_down<BF, 2>(d, d.l.a + (size_t)ad * d.l.rmax * d.k, rank, row, j0, lane, u);
    if (lane < 2) s_u[j0 + lane] = j0 + lane < rank ? u[lane] : 0.0f;
  }
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x < a.l.rmax) d.u[(size_t)row * a.l.rmax + threadIdx.x] = s_u[threadIdx.x];
  if (ad < 0 && a.y == a.res) return;
  float u[8] = {};
  if (j < a.l.rmax) {
#pragma unroll
    for (int q = 0; q < 8; q++) u[q] = s_u[j + q];
  }
  t.template store<BF>(a, rank, sc, row, u, c0, lane);
}

// ------------------------------------------------------------------ the adapters' gradients

struct OuterArgs {
  LoraArgs l;
  const float *p;    // [seq][rmax]
  const float *q;    // [seq][n]
  float *out;        // [adapters][rmax][n], or [adapters][n][rmax]; of several parts, one after the other
  uint32_t n;
  bool scaled;
};

// Blocks of sixteen rows of an adapter, in its requests' order, every parts-th
// from part on; a wave looks at 64 requests at a time.
struct LoraBlocks {
  uint32_t r0 = 0, skip;   // the next 64 requests; how many blocks lie before the next of this part
  uint64_t mine = 0;       // those of the last 64 that are the adapter's and not yet begun
  int32_t s = 0, e = 0;    // the lane's request of the last 64
  uint32_t at = 0, end = 0;
  __device__ __forceinline__ explicit LoraBlocks(uint32_t part) : skip(part) {}
  // the next block's first row, and the end of its request's rows (the same in every lane); false: there is none
  __device__ __forceinline__ bool next(const LoraArgs &l, int32_t ad, uint32_t parts, uint32_t &row, uint32_t &stop) {
    while (at >= end) {
      while (!mine) {
        if (r0 >= l.requests) return false;
        const uint32_t i = r0 + (threadIdx.x & 63);
        const bool in = i < l.requests;
        s = !in ? 0 : l.start ? max(l.start[i], 0) : (int32_t)i;
        e = !in ? 0 : l.start ? min(l.start[i + 1], (int32_t)l.seq) : (int32_t)min(i + 1, l.seq);
        mine = __ballot(in && s < e && l.adapter[i] == ad);
        r0 += 64;
      }
      const int k = __builtin_ctzll(mine);
      mine &= mine - 1;
      at = __builtin_amdgcn_readlane(s, k);
      end = __builtin_amdgcn_readlane(e, k);
      const uint32_t n = (end - at + 15) / 16;
      at += 16 * (skip < n ? skip : n);  // (seq is under 2^21, parts at most 128)
      skip = skip < n ? (parts - (n - skip) % parts) % parts : skip - n;
    }
    row = at;
    stop = end;
    at += 16 * parts;
    return true;
  }
};

// sum over an adapter's rows of p[s, j] q[s, c], 64 columns and 16 NT ranks (of
// more than 64 the workgroups behind have the others: 128 at once spill) a workgroup, blocks of sixteen rows over the eight waves of gridDim.z
// workgroups, in 16 x 16 x 4 f32 products.  Waits for memory: 4,616 rows of 6,912, rank up to 32,
// three adapters 46 us (2.7 TB/s); in 2, 3, 4 and 8 parts 52, 49, 51 and 59.
// TURN: stored [c][j].
template <int NT, bool TURN, bool VEC>
__global__ __launch_bounds__(512) void k_lora_outer(OuterArgs a) {
  __shared__ v4f s_acc[4][NT][4][64];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t ad = blockIdx.y;
  const uint32_t rank = lora_rank(a.l, ad);
  const uint32_t ncol = (a.n + 63) / 64, j0 = blockIdx.x / ncol * 64;  // the first rank
  const uint32_t col = blockIdx.x % ncol * 64 + 4 * i, nc = col < a.n ? min(4u, a.n - col) : 0u;
  v4f acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[t][e] = (v4f){0, 0, 0, 0};
  LoraBlocks blocks(w + 8 * blockIdx.z);
  uint32_t s0, s1;
  while (blocks.next(a.l, ad, 8 * gridDim.z, s0, s1)) {
    float4 qv[4];
    float pv[4][NT];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t row = min(s0 + 4 * k + g, s1 - 1);
      qv[k] = inside4<VEC>(a.q + (size_t)row * a.n, col, a.n);
#pragma unroll
      for (int t = 0; t < NT; t++) pv[k][t] = a.p[(size_t)row * a.l.rmax + min(j0 + 16u * t + i, a.l.rmax - 1)];
    }
    if (s0 + 16 > s1) {  // rows past the request's: neither factor counts
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (s0 + 4 * k + g >= s1) {
          qv[k] = make_float4(0, 0, 0, 0);
#pragma unroll
          for (int t = 0; t < NT; t++) pv[k][t] = 0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          acc[t][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(pv[k][t], at4(qv[k], e), acc[t][e], 0, 0, 0);
  }
  // the waves' sums, by halves
#pragma unroll
  for (int half = 4; half; half /= 2) {
    if (w >= half && w < 2 * half)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) s_acc[w - half][t][e][lane] = acc[t][e];
    __syncthreads();
    if (w < half)
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[t][e] += s_acc[w][t][e][lane];
    __syncthreads();
  }
  if (w) return;
  const float sc = a.scaled ? a.l.scale[ad] : 1.0f;
  float *const o = a.out + ((size_t)blockIdx.z * a.l.adapters + ad) * a.l.rmax * a.n;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    if (TURN) {
      const uint32_t j = j0 + 16 * t + 4 * g;
      if (j >= a.l.rmax) continue;
#pragma unroll
      for (int e = 0; e < 4; e++)
        if ((uint32_t)e < nc)
          *(float4 *)(o + (size_t)(col + e) * a.l.rmax + j) =
              make_float4(j < rank ? acc[t][e][0] * sc : 0.0f, j + 1 < rank ? acc[t][e][1] * sc : 0.0f,
                          j + 2 < rank ? acc[t][e][2] * sc : 0.0f, j + 3 < rank ? acc[t][e][3] * sc : 0.0f);
    } else {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint32_t j = j0 + 16 * t + 4 * g + r;
        if (j < a.l.rmax)
          store4<VEC>(o + (size_t)j * a.n + col, nc,
                      j < rank ? make_float4(acc[t][0][r] * sc, acc[t][1][r] * sc, acc[t][2][r] * sc, acc[t][3][r] * sc)
                               : make_float4(0, 0, 0, 0));
      }
    }
  }
}

// What lies `off` bytes behind a place that is the same in every lane: the load takes both as they are, without an
// address of its own to be made in each lane.
template <class T>
__device__ __forceinline__ T behind(const void *p, uint32_t off) {
  return *(const T *)((const uint8_t *)p + off);
}

// One pass over dy [seq][n]: the adapters' dB, and du = scale B^T dy.  A
// workgroup has 256 columns (16 E a wave) of an adapter's rows, every
// gridDim.z-th block of sixteen.  dB is summed in 16 x 16 x 4 f32 products (a
// lane has E neighbouring columns, so block e of the columns is E i + e); for du the
// rows turn in LDS and meet B, which stays in registers, on the bf16 cores
// as in k_lora_down; the waves' sums for the block meet in LDS and are left in
// one of gridDim.x parts.  It waits for memory: 4,616 rows of 2560, rank up to
// 32, three adapters 28 us (1.7 TB/s of dy; a pass for each, 24 and 21); 241 rows
// 5.4 us.
// E neighbouring columns of a lane
template <int E>
struct Cols {
  typedef float vec __attribute__((ext_vector_type(E)));
};
struct GyArgs {
  LoraArgs l;
  const float *dy, *u;  // [seq][n], [seq][rmax]
  float *du;            // [gridDim.x][seq][rmax]
  float *db;            // [gridDim.z][adapters][n][rmax]
  uint32_t n;
};
template <bool BF, int NT, int E, bool VEC>
__global__ __launch_bounds__(1024 / E, NT <= 2 ? 4 : 2) void k_lora_gy(GyArgs a) {
  typedef typename Cols<E>::vec vec;
  constexpr int NW = 16 / E, H = E / 2, P = 16 * E + 4, Q = 16 * NT + 1;
  __shared__ float s_t[NW][16][P];
  __shared__ float s_du[2][NW][16][Q];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t ad = blockIdx.y;
  const uint32_t rank = lora_rank(a.l, ad), rmax = a.l.rmax;
  const uint32_t col0 = blockIdx.x * 256 + w * (16 * E), col = col0 + E * i;
  const float sc = a.l.scale[ad];
  // B of the wave's columns: lane (i, g) rank 16 t + i of columns 32 h + 8 g .. + 7
  const uint16_t *const wt = a.l.b + (size_t)ad * a.n * rmax;
  Bf8 w0[H][NT], w1[BF ? 1 : H][NT];
#pragma unroll
  for (int h = 0; h < H; h++)
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        uint32_t v[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t c = col0 + 32 * h + 8 * g + 2 * q + e;
          v[e] = wt[(size_t)min(c, a.n - 1) * rmax + min(16u * t + i, rmax - 1)];
          if (c >= a.n) v[e] = 0;
        }
        const uint32_t pair = v[0] | v[1] << 16;
        if (BF) w0[h][t].u[q] = pair;
        else split_f16(pair, w0[h][t].u[q], w1[h][t].u[q]);
      }
  v4f acc[NT][E];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < E; e++) acc[t][e] = (v4f){0, 0, 0, 0};
  float *const out = a.du + (size_t)blockIdx.x * a.l.seq * rmax;
  // (macros: register sets handed to a lambda end up in scratch)
#define LOAD(r0, stop, D, U)                                                                                     \
  do {                                                                                                           \
    const uint32_t last = stop - 1 - r0; /* of the block's rows; those behind it read that one */                \
    const float *const bd = a.dy + (size_t)r0 * a.n, *const bu = a.u + (size_t)r0 * rmax;                         \
    if (VEC && last >= 15) {                                                                                     \
      _Pragma("unroll") for (int q = 0; q < 4; q++) {                                                            \
        D[q] = behind<vec>(bd + (size_t)(4 * q) * a.n, vd);                                                      \
        _Pragma("unroll") for (int t = 0; t < NT; t++) U[q][t] = behind<float>(bu + (4 * q) * rmax, vp[t]);       \
      }                                                                                                          \
    } else {                                                                                                     \
      _Pragma("unroll") for (int q = 0; q < 4; q++) {                                                            \
        const uint32_t row = min(4u * q + g, last);                                                              \
        if (VEC) D[q] = behind<vec>(bd, 4 * (row * a.n + min(col, a.n - E)));                                    \
        else _Pragma("unroll") for (int e = 0; e < E; e++) D[q][e] = behind<float>(bd, 4 * (row * a.n + min(col + e, a.n - 1))); \
        _Pragma("unroll") for (int t = 0; t < NT; t++)                                                           \
          U[q][t] = behind<float>(bu, 4 * (row * rmax + min(16u * t + i, rmax - 1)));                            \
      }                                                                                                          \
    }                                                                                                            \
  } while (0)
  // a block, its sums left in half b of s_du (free again after the next block's barrier)
#define MUL(r0, stop, D, U, b)                                                                                   \
  do {                                                                                                           \
    if (r0 + 16 > stop || col0 + 16 * E > a.n) { /* rows past the request's, columns past the matrix: neither factor counts */ \
      _Pragma("unroll") for (int q = 0; q < 4; q++) {                                                            \
        const bool in = r0 + 4 * q + g < stop;                                                                   \
        _Pragma("unroll") for (int e = 0; e < E; e++) if (!in || col + e >= a.n) D[q][e] = 0.0f;                 \
        if (!in) _Pragma("unroll") for (int t = 0; t < NT; t++) U[q][t] = 0.0f;                                  \
      }                                                                                                          \
    }                                                                                                            \
    _Pragma("unroll") for (int q = 0; q < 4; q++) *(vec *)&s_t[w][4 * q + g][E * i] = D[q];                      \
    ORDER(); /* the wave's own rows: LDS takes a wave's accesses in order */                                     \
    _Pragma("unroll") for (int q = 0; q < 4; q++)                                                                \
      _Pragma("unroll") for (int t = 0; t < NT; t++)                                                             \
        _Pragma("unroll") for (int e = 0; e < E; e++)                                                            \
          acc[t][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(U[q][t], D[q][e], acc[t][e], 0, 0, 0);                \
    v4f du[NT];                                                                                                  \
    _Pragma("unroll") for (int t = 0; t < NT; t++) du[t] = (v4f){0, 0, 0, 0};                                    \
    _Pragma("unroll") for (int h = 0; h < H; h++) {                                                              \
      const float *const p = &s_t[w][i][32 * h + 8 * g];                                                         \
      const float4 x0 = *(const float4 *)p, x1 = *(const float4 *)(p + 4);                                       \
      Bf8 p0, p1, p2;                                                                                            \
      split3(x0.x, x0.y, p0.u[0], p1.u[0], p2.u[0]);                                                             \
      split3(x0.z, x0.w, p0.u[1], p1.u[1], p2.u[1]);                                                             \
      split3(x1.x, x1.y, p0.u[2], p1.u[2], p2.u[2]);                                                             \
      split3(x1.z, x1.w, p0.u[3], p1.u[3], p2.u[3]);                                                             \
      _Pragma("unroll") for (int t = 0; t < NT; t++) {                                                           \
        du[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p0.v, w0[h][t].v, du[t], 0, 0, 0);                       \
        du[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p1.v, w0[h][t].v, du[t], 0, 0, 0);                       \
        du[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p2.v, w0[h][t].v, du[t], 0, 0, 0);                       \
        if (!BF) {                                                                                               \
          du[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p0.v, w1[BF ? 0 : h][t].v, du[t], 0, 0, 0);            \
          du[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p1.v, w1[BF ? 0 : h][t].v, du[t], 0, 0, 0);            \
        }                                                                                                        \
      }                                                                                                          \
    }                                                                                                            \
    _Pragma("unroll") for (int t = 0; t < NT; t++)                                                               \
      _Pragma("unroll") for (int r = 0; r < 4; r++) s_du[b][w][4 * g + r][16 * t + i] = du[t][r];                \
    __syncthreads();                                                                                             \
    for (uint32_t k = threadIdx.x; k < 16 * rmax; k += 1024 / E) {                                               \
      const uint32_t r = k / rmax, j = k % rmax;                                                                 \
      if (r0 + r < stop) {                                                                                       \
        float v = 0.0f;                                                                                          \
        _Pragma("unroll") for (int q = 0; q < NW; q++) v += s_du[b][q][r][j];                                    \
        out[(size_t)r0 * rmax + k] = j < rank ? v * sc : 0.0f;                                                   \
      }                                                                                                          \
    }                                                                                                            \
  } while (0)
  // bytes from a block's q-th four rows to what the lane reads there
  const uint32_t vd = 4 * (g * a.n + min(col, a.n - min(a.n, (uint32_t)E)));
  uint32_t vp[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) vp[t] = 4 * (g * rmax + min(16u * t + i, rmax - 1));
  LoraBlocks blocks(blockIdx.z);
  vec dv[4];
  float uv[4][NT];
  uint32_t r0, s0;
  for (uint32_t b = 0; blocks.next(a.l, ad, gridDim.z, r0, s0); b ^= 1) {
    LOAD(r0, s0, dv, uv);
    MUL(r0, s0, dv, uv, b);
  }
#undef MUL
#undef LOAD
  // acc[t][e] register r: rank 16 t + 4 g + r, column col + e
  float *const o = a.db + ((size_t)blockIdx.z * a.l.adapters + ad) * rmax * a.n;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const uint32_t j = 16 * t + 4 * g;
    if (j >= rmax) continue;
#pragma unroll
    for (int e = 0; e < E; e++)
      if (col + e < a.n)
        *(float4 *)(o + (size_t)(col + e) * rmax + j) =
            make_float4(j < rank ? acc[t][e][0] * sc : 0.0f, j + 1 < rank ? acc[t][e][1] * sc : 0.0f,
                        j + 2 < rank ? acc[t][e][2] * sc : 0.0f, j + 3 < rank ? acc[t][e][3] * sc : 0.0f);
  }
}

// One pass over x [seq][n]: the adapters' dA, and dx = dres + A^T du.  A
// workgroup has 256 columns of an adapter's rows (those of none: blockIdx.y ==
// adapters), every gridDim.z-th block of sixteen, its waves 16 E columns each, E
// neighbouring ones a lane, in 16 x 16 x 4 f32 products.  x, dres and dx move
// once, a row 1 KB at a time.  It waits for memory: 241 rows of 2560 6.0 us; 4,616
// of 6912 112 to 125 us, the same with the next block's loads in flight, which is
// why larger calls take two passes.
struct GxArgs {
  LoraArgs l;
  const float *x, *du, *dres;  // [seq][n], [seq][rmax], [seq][n] or null
  float *dx;                   // [seq][n] or null
  float *da;                   // [gridDim.z][adapters][rmax][n]
  uint32_t n;
};
template <bool BF, int NT, int E>
__global__ __launch_bounds__(1024 / E, NT <= 2 ? 4 : 2) void k_lora_gx(GxArgs a) {
  typedef typename Cols<E>::vec vec;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t rmax = a.l.rmax, col = blockIdx.x * 256 + w * (16 * E) + E * i, cc = min(col, a.n - E);
  const bool here = col < a.n;
  if (blockIdx.y == a.l.adapters) {
    for (uint32_t r0 = 64 * blockIdx.z; r0 < a.l.seq; r0 += 64 * gridDim.z) {
      const int32_t ad = lora_rows(a.l, r0, 64, lane);
      uint64_t none = __ballot(ad < 0);
      for (int r = g; r < 64; r += 4)
        if ((none >> r & 1) && r0 + r < a.l.seq && here) {
          const size_t o = (size_t)(r0 + r) * a.n + col;
          *(vec *)(a.dx + o) = a.dres ? *(const vec *)(a.dres + o) : (vec)0.0f;
        }
    }
    return;
  }
  const int32_t ad = blockIdx.y;
  const uint32_t rank = lora_rank(a.l, ad);
  // A of the columns: ranks 16 t + 4 g + s
  const uint16_t *const wt = a.l.a + (size_t)ad * rmax * a.n;
  uint32_t wv[NT][4][E / 2];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int s = 0; s < 4; s++) {
      const uint32_t j = 16 * t + 4 * g + s;
#pragma unroll
      for (int e = 0; e < E / 2; e++) {
        wv[t][s][e] = *(const uint32_t *)(wt + (size_t)min(j, rmax - 1) * a.n + cc + 2 * e);
        if (j >= rank) wv[t][s][e] = 0;  // (du is 0 there)
      }
    }
  v4f acc[NT][E];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int e = 0; e < E; e++) acc[t][e] = (v4f){0, 0, 0, 0};
  // (macros: register sets handed to a lambda end up in scratch)
#define LOAD(r0, stop, X, R, U, P)                                                                                  \
  do {                                                                                                              \
    const uint32_t last = stop - 1 - r0; /* of the block's rows; those behind it read that one */                   \
    const float *const bx = a.x + (size_t)r0 * a.n, *const bu = a.du + (size_t)r0 * rmax;                            \
    const float *const br = a.dres + (size_t)r0 * a.n;                                                              \
    if (last >= 15) {                                                                                               \
      _Pragma("unroll") for (int q = 0; q < 4; q++) {                                                               \
        X[q] = behind<vec>(bx + (size_t)(4 * q) * a.n, vx);                                                         \
        _Pragma("unroll") for (int t = 0; t < NT; t++) P[q][t] = behind<float>(bu + (4 * q) * rmax, vp[t]);          \
      }                                                                                                             \
      if (a.dx) {                                                                                                   \
        _Pragma("unroll") for (int r = 0; r < 4; r++)                                                               \
          R[r] = a.dres ? behind<vec>(br + (size_t)r * a.n, vr) : (vec)0.0f;                                        \
        _Pragma("unroll") for (int t = 0; t < NT; t++) U[t] = behind<float4>(bu, vu[t]);                            \
      }                                                                                                             \
    } else {                                                                                                        \
      _Pragma("unroll") for (int q = 0; q < 4; q++) {                                                               \
        const uint32_t row = min(4u * q + g, last);                                                                 \
        X[q] = behind<vec>(bx, 4 * (row * a.n + cc));                                                               \
        _Pragma("unroll") for (int t = 0; t < NT; t++)                                                              \
          P[q][t] = behind<float>(bu, 4 * (row * rmax + min(16u * t + i, rmax - 1)));                               \
      }                                                                                                             \
      if (a.dx) {                                                                                                   \
        _Pragma("unroll") for (int r = 0; r < 4; r++)                                                               \
          R[r] = a.dres ? behind<vec>(br, 4 * (min(4u * g + r, last) * a.n + cc)) : (vec)0.0f;                      \
        _Pragma("unroll") for (int t = 0; t < NT; t++)                                                              \
          U[t] = behind<float4>(bu, 4 * (min((uint32_t)i, last) * rmax + min(16u * t + 4 * g, rmax - 4)));          \
      }                                                                                                             \
    }                                                                                                               \
  } while (0)
  // rows past the request's: neither factor counts.  (Of the way up: a rank that rmax has no room for reads another's
  // du, with weights of 0.)
#define MUL(r0, stop, X, R, U, P)                                                                                   \
  do {                                                                                                              \
    if (r0 + 16 > stop) {                                                                                           \
      _Pragma("unroll") for (int q = 0; q < 4; q++) if (r0 + 4 * q + g >= stop) {                                   \
        X[q] = (vec)0.0f;                                                                                           \
        _Pragma("unroll") for (int t = 0; t < NT; t++) P[q][t] = 0.0f;                                              \
      }                                                                                                             \
    }                                                                                                               \
    _Pragma("unroll") for (int q = 0; q < 4; q++)                                                                   \
      _Pragma("unroll") for (int t = 0; t < NT; t++)                                                                \
        _Pragma("unroll") for (int e = 0; e < E; e++)                                                               \
          acc[t][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(P[q][t], X[q][e], acc[t][e], 0, 0, 0);                   \
    if (a.dx) {                                                                                                     \
      v4f up[E];                                                                                                    \
      _Pragma("unroll") for (int e = 0; e < E; e++) up[e] = (v4f){0, 0, 0, 0};                                      \
      _Pragma("unroll") for (int t = 0; t < NT; t++)                                                                \
        _Pragma("unroll") for (int s = 0; s < 4; s++)                                                               \
          _Pragma("unroll") for (int e = 0; e < E; e++) {                                                           \
            const uint32_t h = wv[t][s][e / 2] >> (16 * (e & 1)) & 0xffff;                                          \
            up[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(at4(U[t], s), wide<BF>(h), up[e], 0, 0, 0);                \
          }                                                                                                         \
      float *const bd = a.dx + (size_t)r0 * a.n;                                                                    \
      _Pragma("unroll") for (int r = 0; r < 4; r++) {                                                               \
        vec v = R[r];                                                                                               \
        _Pragma("unroll") for (int e = 0; e < E; e++) v[e] += up[e][r];                                             \
        if (here && r0 + 4 * g + r < stop) *(vec *)((uint8_t *)(bd + (size_t)r * a.n) + vr) = v;                    \
      }                                                                                                             \
    }                                                                                                               \
  } while (0)
  // bytes from a block's first row (or the q-th four of its rows, or its r-th row) to what the lane reads there
  const uint32_t vx = 4 * (g * a.n + cc), vr = 4 * (4 * g * a.n + cc);
  uint32_t vp[NT], vu[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    vp[t] = 4 * (g * rmax + min(16u * t + i, rmax - 1));
    vu[t] = 4 * (i * rmax + min(16u * t + 4 * g, rmax - 4));
  }
  LoraBlocks blocks(blockIdx.z);
  vec xv[4], res[4];
  float4 uv[NT];
  float pv[4][NT];
  uint32_t r0, s0;
  while (blocks.next(a.l, ad, gridDim.z, r0, s0)) {
    LOAD(r0, s0, xv, res, uv, pv);
    MUL(r0, s0, xv, res, uv, pv);
  }
#undef MUL
#undef LOAD
  if (!here) return;
  float *const o = a.da + ((size_t)blockIdx.z * a.l.adapters + ad) * rmax * a.n;
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const uint32_t j = 16 * t + 4 * g + r;
      if (j < rmax) {
        vec v;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = j < rank ? acc[t][e][r] : 0.0f;
        *(vec *)(o + (size_t)j * a.n + col) = v;
      }
    }
}

struct LoraSum {
  const float4 *part;  // [parts][n4]
  float4 *out;
  uint64_t n4;
  uint32_t parts;
};
// The parts of such sums, added in order (so the bits are the same each time); of two of them in one launch, which is
// what it costs at small sizes: 4 to 7 us.
__global__ __launch_bounds__(256) void k_lora_sum(LoraSum a, LoraSum b) {
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < a.n4 + b.n4; i += gridDim.x * 256ull) {
    const bool second = i >= a.n4;
    const LoraSum &s = second ? b : a;
    const uint64_t k = second ? i - a.n4 : i;
    float4 v = s.part[k];
    for (uint32_t q = 1; q < s.parts; q++) {
      const float4 f = s.part[q * s.n4 + k];
      v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
    }
    s.out[k] = v;
  }
}

// ------------------------------------------------------------------ host side

static int lora_check(const char *what, const void *a, const void *b, int fmt, const float *scale, const int32_t *rank,
                      const int32_t *start, const int32_t *adapter, uint32_t requests, uint32_t adapters, uint32_t rmax,
                      uint32_t seq, uint32_t out, uint32_t cols, LoraArgs &l) {
  if (!a || !b || !scale || (requests && !adapter)) return nlg_fail("%s: null pointer", what);
  if (fmt != NLG_LORA_F16 && fmt != NLG_LORA_BF16) return nlg_fail("%s: unknown adapter format %d", what, fmt);
  if (!adapters) return nlg_fail("%s: adapters must be nonzero", what);
  if (!rmax || rmax % 8 || rmax > LORA_RANK)
    return nlg_fail("%s: rmax must be a multiple of 8 up to %d (got %u)", what, LORA_RANK, rmax);
  if (!cols || cols % 8) return nlg_fail("%s: cols must be a multiple of 8 (got %u)", what, cols);
  if (!out) return nlg_fail("%s: out must be nonzero", what);
  if (seq > LORA_ROWS || out > 0x1000000u || cols > 0x1000000u || adapters > 65534 || requests > LORA_REQUESTS)
    return nlg_fail("%s: too many rows, columns, requests or adapters", what);
  if (((uintptr_t)a & 15) || ((uintptr_t)b & 15)) return nlg_fail("%s: adapters must be 16-byte aligned", what);
  if (((uintptr_t)scale | (uintptr_t)rank | (uintptr_t)start | (uintptr_t)adapter) & 3)
    return nlg_fail("%s: scale, rank, start and adapter must be 4-byte aligned", what);
  l.start = start; l.adapter = adapter; l.rank = rank; l.scale = scale;
  l.a = (const uint16_t *)a; l.b = (const uint16_t *)b;
  l.requests = requests; l.adapters = adapters; l.rmax = rmax; l.seq = seq;
  return NLG_OK;
}

// sizes alone (the workspace functions have no pointers)
static bool lora_sizes(uint32_t seq, uint32_t out, uint32_t cols, uint32_t rmax, uint32_t requests) {
  return seq && out && cols && cols % 8 == 0 && rmax && rmax % 8 == 0 && rmax <= LORA_RANK && seq <= LORA_ROWS &&
         out <= 0x1000000u && cols <= 0x1000000u && requests <= LORA_REQUESTS;
}

static LoraSum lora_parts_of(const float *part, float *out, uint64_t n, uint32_t parts) {
  return {(const float4 *)part, (float4 *)out, parts > 1 ? n / 4 : 0, parts};
}
static int lora_sum(const char *what, const LoraSum &a, const LoraSum &b, hipStream_t st) {
  if (!a.n4 && !b.n4) return NLG_OK;
  const uint32_t blocks = nlg_blocks(a.n4 + b.n4, 256);
  hipLaunchKernelGGL(k_lora_sum, dim3(blocks < 2048 ? blocks : 2048), dim3(256), 0, st, a, b);
  NLG_LAUNCHED(what);
  return NLG_OK;
}

// How many parts a contraction over k columns is summed in: until two workgroups a CU have some, each of four steps at
// least.
static uint32_t lora_ksplit(uint32_t seq, uint32_t k) {
  const uint64_t tiles = ((uint64_t)seq + 31) / 32, most = k / 512;
  uint64_t n = 512 / tiles;
  if (n > most) n = most;
  return n < 1 ? 1 : n > 8 ? 8 : (uint32_t)n;
}
static size_t lora_round(size_t n) { return (n + 255) / 256 * 256; }
static size_t lora_down_bytes(uint32_t seq, uint32_t k, uint32_t rmax) {
  const uint32_t n = lora_ksplit(seq, k);
  return n > 1 ? lora_round((size_t)n * seq * rmax * 4) : 0;
}

// parts: lora_down_bytes
static int lora_down(const char *what, DownArgs d, bool bf, bool kmajor, float *parts, hipStream_t st) {
  const uint32_t np = lora_ksplit(d.l.seq, d.k);
  float *const u = d.u;
  if (np > 1) d.u = parts;
  const dim3 grid((d.l.seq + 31) / 32, np), blk(256);
  const bool vec = d.k % 4 == 0 && ((uintptr_t)d.x & 15) == 0;
  const uint32_t nt = (d.l.rmax + 15) / 16;
#define GO(BF, KM, N, V) hipLaunchKernelGGL((k_lora_down<BF, KM, N, V>), grid, blk, 0, st, d)
#define GO2(BF)                               \
  do {                                        \
    if (nt <= 1) GO(BF, false, 1, true);      \
    else if (nt <= 2) GO(BF, false, 2, true); \
    else if (nt <= 4) GO(BF, false, 4, true); \
    else GO(BF, false, 8, true);              \
  } while (0)
  // (the gradient's way down of up to 64 ranks is k_lora_gy; x has whole float4s)
  if (kmajor) {
    if (bf && vec) GO(true, true, 8, true);
    else if (bf) GO(true, true, 8, false);
    else if (vec) GO(false, true, 8, true);
    else GO(false, true, 8, false);
  } else if (bf) {
    GO2(true);
  } else {
    GO2(false);
  }
#undef GO2
#undef GO
  NLG_LAUNCHED(what);
  return lora_sum(what, lora_parts_of(parts, u, (uint64_t)d.l.seq * d.l.rmax, np), {}, st);
}

static int lora_up(const char *what, const UpArgs &d, bool bf, bool kmajor, hipStream_t st) {
  const dim3 grid((d.n + 255) / 256, (d.l.seq + 31) / 32), blk(256);
  const bool vec = d.n % 4 == 0 && (((uintptr_t)d.y | (uintptr_t)d.res) & 15) == 0;
#define GO(BF, KM, V) hipLaunchKernelGGL((k_lora_up<BF, KM, V>), grid, blk, 0, st, d)
  // (dx has whole float4s)
  if (bf && kmajor) GO(true, true, true);
  else if (kmajor) GO(false, true, true);
  else if (bf && vec) GO(true, false, true);
  else if (bf) GO(true, false, false);
  else if (vec) GO(false, false, true);
  else GO(false, false, false);
#undef GO
  NLG_LAUNCHED(what);
  return NLG_OK;
}

// How many parts an adapter's rows are summed in: until two workgroups a CU have some, each of 64 rows at least.
static uint32_t lora_parts(uint32_t seq, uint32_t n, uint32_t adapters) {
  const uint64_t wg = (uint64_t)((n + 63) / 64) * adapters, most = seq / 64;
  uint64_t k = 512 / wg;
  if (k > most) k = most;
  return k < 1 ? 1 : k > 16 ? 16 : (uint32_t)k;
}

// The launch alone: of np parts, to `parts` where that is more than one.
static int lora_outer(const char *what, OuterArgs d, bool turn, float *parts, uint32_t np, hipStream_t st) {
  if (np > 1) d.out = parts;
  const dim3 grid((d.n + 63) / 64 * ((d.l.rmax + 63) / 64), d.l.adapters, np), blk(512);
  const bool vec = d.n % 4 == 0 && ((uintptr_t)d.q & 15) == 0;
  const uint32_t nt = (d.l.rmax + 15) / 16;
  // (dB of up to 64 ranks is k_lora_gy's; x has whole float4s)
  if (turn && vec) hipLaunchKernelGGL((k_lora_outer<4, true, true>), grid, blk, 0, st, d);
  else if (turn) hipLaunchKernelGGL((k_lora_outer<4, true, false>), grid, blk, 0, st, d);
  else if (nt <= 1) hipLaunchKernelGGL((k_lora_outer<1, false, true>), grid, blk, 0, st, d);
  else if (nt <= 2) hipLaunchKernelGGL((k_lora_outer<2, false, true>), grid, blk, 0, st, d);
  else hipLaunchKernelGGL((k_lora_outer<4, false, true>), grid, blk, 0, st, d);
  NLG_LAUNCHED(what);
  return NLG_OK;
}

// A wave a row, which reads its adapter anew, or tiles of 32 rows, a pass for each adapter among them: the former while what
// is read so stays small (`most` ranks times columns), or requests have fewer than four rows.  Measured, us a call, by row
// and by tile, 2560 -> 2560 at rank 16 unless told.  Alone (most 2^27): 256 rows of a request 8.5 and 14.8, 1,024 16.7 and
// 18.3, 64 requests of 8 rows with 64 adapters 20.0 and 31.1, of 16 23.5 and 24.8, of 32 (1.25 times `most`) 30.2 and 24.4;
// 512 rows at rank 64 22.6 and 22.2; 64 requests of 2 rows 8.4 and 84.  With the ternary linear (3 2^24: tiles save reading
// and writing y again): 256 rows 19.9 and 23.2, 512 24.6 and 26.1, 1,024 37.2 and 36.3; 1,000 rows of 704 29.6 and 23.5.
// The sizes know no lengths, so requests without rows count as short ones: 4,000 rows of one request at rank 128, 4096 ->
// 4096, 104 us, among 1,023 empty ones 418.
static bool lora_by_token(const LoraArgs &l, uint32_t cols, uint32_t out, uint64_t most) {
  return l.seq <= 16 ||
         (l.seq < 65536 && ((uint64_t)l.seq * l.rmax * ((uint64_t)cols + out) <= most || l.seq < 4ull * l.requests));
}

// Whether one launch does them, each workgroup finding u again: a few rows of small adapters (four rows of 2,560 at rank 16
// 4.2 us for 6.4 in two, at rank 64 8.4 for 6.5).
static bool lora_tok_whole(const DownArgs &d) { return d.l.seq <= 4 && (uint64_t)d.l.rmax * d.k <= 65536; }

// q: the rows' rounding to int8, wanted beside
static int lora_tok_down(const char *what, const DownArgs &d, bool bf, const ActQArgs *q, hipStream_t st) {
  const uint32_t groups = (d.l.rmax + 4 * TOK_RANKS - 1) / (4 * TOK_RANKS);
  const dim3 gd(d.l.seq, groups + (q ? 1 : 0));
  if (q) {
#define GO(G)                                                                                        \
  do {                                                                                               \
    if (bf) hipLaunchKernelGGL((k_lora_tok_down_q<true, G>), gd, dim3(256), 0, st, d, *q);           \
    else hipLaunchKernelGGL((k_lora_tok_down_q<false, G>), gd, dim3(256), 0, st, d, *q);             \
  } while (0)
    if (q->cols <= 4096) GO(1);
    else if (q->cols <= 8192) GO(2);
    else GO(4);
#undef GO
  } else if (bf) {
    hipLaunchKernelGGL((k_lora_tok_down<true>), gd, dim3(256), 0, st, d);
  } else {
    hipLaunchKernelGGL((k_lora_tok_down<false>), gd, dim3(256), 0, st, d);
  }
  NLG_LAUNCHED(what);
  return NLG_OK;
}

// down and up
static int lora_tok(const char *what, const DownArgs &d, const UpArgs &p, bool bf, hipStream_t st) {
  const uint32_t lanes = p.l.rmax <= 8 ? 1 : p.l.rmax <= 16 ? 2 : p.l.rmax <= 32 ? 4 : p.l.rmax <= 64 ? 8 : 16;
  const uint32_t step = 64 / lanes;
#define BY_LANES(GO)              \
  do {                            \
    if (lanes == 1) GO(1);        \
    else if (lanes == 2) GO(2);   \
    else if (lanes == 4) GO(4);   \
    else if (lanes == 8) GO(8);   \
    else GO(16);                  \
  } while (0)
  const dim3 grid((p.n + 8 * step - 1) / (8 * step), p.l.seq);
#define GO(L)                                                                              \
  do {                                                                                     \
    if (bf) hipLaunchKernelGGL((k_lora_tok<true, L>), grid, dim3(512), 0, st, d, p);       \
    else hipLaunchKernelGGL((k_lora_tok<false, L>), grid, dim3(512), 0, st, d, p);         \
  } while (0)
  BY_LANES(GO);
#undef GO
  NLG_LAUNCHED(what);
  return NLG_OK;
}

static int lora_tok_up(const char *what, const UpArgs &p, bool bf, hipStream_t st) {
  const uint32_t lanes = p.l.rmax <= 8 ? 1 : p.l.rmax <= 16 ? 2 : p.l.rmax <= 32 ? 4 : p.l.rmax <= 64 ? 8 : 16;
  const uint32_t step = 64 / lanes;
  // eight steps a wave where that leaves the card full
  const bool many = (uint64_t)p.l.seq * p.n / (8 * step) >= 2048;
  const uint32_t per = 4 * step * (many ? 8 : 2);
  const dim3 grid((p.n + per - 1) / per, p.l.seq);
#define GO(L)                                                                                          \
  do {                                                                                                 \
    if (bf && many) hipLaunchKernelGGL((k_lora_tok_up<true, L, 8>), grid, dim3(256), 0, st, p);        \
    else if (bf) hipLaunchKernelGGL((k_lora_tok_up<true, L, 2>), grid, dim3(256), 0, st, p);           \
    else if (many) hipLaunchKernelGGL((k_lora_tok_up<false, L, 8>), grid, dim3(256), 0, st, p);        \
    else hipLaunchKernelGGL((k_lora_tok_up<false, L, 2>), grid, dim3(256), 0, st, p);                  \
  } while (0)
  BY_LANES(GO);
#undef GO
#undef BY_LANES
  NLG_LAUNCHED(what);
  return NLG_OK;
}

extern "C" size_t nlg_lora_linear_workspace(uint32_t seq, uint32_t out, uint32_t cols, uint32_t rmax, uint32_t requests) {
  return lora_sizes(seq, out, cols, rmax, requests) ? lora_round((size_t)seq * rmax * 4) + lora_down_bytes(seq, cols, rmax) : 0;
}

// ws: nlg_lora_linear_workspace
static int lora_forward(const char *what, const LoraArgs &l, const float *x, bool bf, const float *res, float *y, float *u,
                        uint32_t out, uint32_t cols, void *ws, hipStream_t st) {
  DownArgs d{};
  d.l = l; d.x = x; d.k = cols; d.scaled = false; d.u = u ? u : (float *)ws;
  UpArgs p{};
  p.l = l; p.u = d.u; p.res = res; p.y = y; p.n = out; p.scaled = true;
  if (lora_by_token(l, cols, out, 1u << 27))
    return lora_tok_whole(d) ? lora_tok(what, d, p, bf, st)
                             : lora_tok_down(what, d, bf, nullptr, st) || lora_tok_up(what, p, bf, st);
  float *const parts = (float *)((uint8_t *)ws + lora_round((size_t)l.seq * l.rmax * 4));
  return lora_down(what, d, bf, false, parts, st) || lora_up(what, p, bf, false, st);
}

extern "C" int nlg_lora_linear(const float *x, const uint16_t *a, const uint16_t *b, int fmt, const float *scale,
                               const int32_t *rank, const int32_t *start, const int32_t *adapter, uint32_t requests,
                               uint32_t adapters, uint32_t rmax, const float *res, float *y, float *u, uint32_t seq,
                               uint32_t out, uint32_t cols, void *workspace, size_t workspace_bytes, void *stream) {
  const char *what = "lora linear";
  if (!seq) return NLG_OK;
  LoraArgs l;
  if (lora_check(what, a, b, fmt, scale, rank, start, adapter, requests, adapters, rmax, seq, out, cols, l)) return NLG_ERR;
  if (!x || !y) return nlg_fail("%s: null pointer", what);
  if (((uintptr_t)x | (uintptr_t)u) & 15) return nlg_fail("%s: x and u must be 16-byte aligned", what);
  if (((uintptr_t)y | (uintptr_t)res) & 3) return nlg_fail("%s: y and res must be 4-byte aligned", what);
  const size_t need = nlg_lora_linear_workspace(seq, out, cols, rmax, requests);
  if (!workspace || workspace_bytes < need)
    return nlg_fail("%s: workspace holds %zu bytes, needs %zu", what, workspace ? workspace_bytes : 0, need);
  if ((uintptr_t)workspace & 15) return nlg_fail("%s: the workspace must be 16-byte aligned", what);
  const uint64_t r4 = (uint64_t)seq * 4, na = (uint64_t)adapters * rmax * cols, nb = (uint64_t)adapters * rmax * out;
  const NlgSpan at[] = {{x, r4 * cols}, {a, 2 * na}, {b, 2 * nb}, {scale, 4ull * adapters}, {rank, 4ull * adapters},
                        {start, 4ull * requests + 4}, {adapter, 4ull * requests}, {res == y ? nullptr : res, r4 * out},
                        {y, r4 * out}, {u, r4 * rmax}, {workspace, need}};
  if (nlg_outputs_overlap(at, 11, 3))
    return nlg_fail("%s: outputs or the workspace overlap each other or an input (y may be res itself)", what);
  NLG_SCOPE(what);
  return lora_forward(what, l, x, fmt == NLG_LORA_BF16, res, y, u, out, cols, workspace, nlg_stream(stream)) ? NLG_ERR : NLG_OK;
}

// What the projection keeps apart from its column split: rows as int8 and their scales, in either form's layout.
static size_t ternary_bytes(uint32_t seq, uint32_t cols) {
  const size_t rows = nlg_ternary_linear_workspace(seq, cols), batched = nlg_batched_scratch_bytes(seq, cols);
  return lora_round(rows > batched ? rows : batched);
}

extern "C" size_t nlg_ternary_linear_lora_workspace(uint32_t seq, uint32_t out, uint32_t cols, uint32_t rmax,
                                                    uint32_t requests) {
  const size_t u = nlg_lora_linear_workspace(seq, out, cols, rmax, requests);
  if (!u || cols > LORA_TERNARY_COLS) return 0;
  return u + ternary_bytes(seq, cols) + nlg_batched_split_bytes(seq, out, cols);
}

extern "C" int nlg_ternary_linear_lora(const float *x, const uint32_t *w2, const float *bias, const float *beta,
                                       int beta_per_row, const uint16_t *a, const uint16_t *b, int fmt,
                                       const float *scale, const int32_t *rank, const int32_t *start,
                                       const int32_t *adapter, uint32_t requests, uint32_t adapters, uint32_t rmax,
                                       float *y, float *u, uint32_t seq, uint32_t out, uint32_t cols, void *workspace,
                                       size_t workspace_bytes, void *stream) {
  const char *what = "ternary linear with adapters";
  if (!seq) return NLG_OK;
  LoraArgs l;
  if (lora_check(what, a, b, fmt, scale, rank, start, adapter, requests, adapters, rmax, seq, out, cols, l)) return NLG_ERR;
  if (!x || !w2 || !beta || !y) return nlg_fail("%s: null pointer", what);
  if (((uintptr_t)x | (uintptr_t)w2 | (uintptr_t)u) & 15) return nlg_fail("%s: x, w2 and u must be 16-byte aligned", what);
  if (((uintptr_t)y | (uintptr_t)bias | (uintptr_t)beta) & 3)
    return nlg_fail("%s: y, bias and beta must be 4-byte aligned", what);
  if (cols > LORA_TERNARY_COLS) return nlg_fail("%s: cols must be at most %d (got %u)", what, LORA_TERNARY_COLS, cols);
  const size_t nu = nlg_lora_linear_workspace(seq, out, cols, rmax, requests);
  const size_t need = nlg_ternary_linear_lora_workspace(seq, out, cols, rmax, requests);
  if (!workspace || workspace_bytes < need)
    return nlg_fail("%s: workspace holds %zu bytes, needs %zu", what, workspace ? workspace_bytes : 0, need);
  if ((uintptr_t)workspace & 15) return nlg_fail("%s: the workspace must be 16-byte aligned", what);
  const uint64_t r4 = (uint64_t)seq * 4, na = (uint64_t)adapters * rmax * cols, nb = (uint64_t)adapters * rmax * out;
  const NlgSpan at[] = {{x, r4 * cols}, {w2, (uint64_t)out * ((cols + 15) / 16) * 4}, {bias, 4ull * out},
                        {beta, beta_per_row ? 4ull * out : 4}, {a, 2 * na}, {b, 2 * nb}, {scale, 4ull * adapters},
                        {rank, 4ull * adapters}, {start, 4ull * requests + 4}, {adapter, 4ull * requests},
                        {y, r4 * out}, {u, r4 * rmax}, {workspace, need}};
  if (nlg_outputs_overlap(at, 13, 3))
    return nlg_fail("%s: outputs or the workspace overlap each other or an input", what);
  NLG_SCOPE(what);
  hipStream_t st = nlg_stream(stream);
  uint8_t *const more = (uint8_t *)workspace + nu;
  const bool bf = fmt == NLG_LORA_BF16;
  if (nlg_batched_lora(seq, cols)) {
    float *const gamma = (float *)(more + ((size_t)seq * cols + 255) / 256 * 256);
    FusedArgs f{};
    f.w2 = w2; f.bias = bias; f.beta = beta; f.beta_per_row = beta_per_row; f.seq = seq; f.out = out; f.cols = cols;
    f.y = y; f.ystride = out;
    // the projection's column split, in this call's own workspace: its counters are zeroed by the launch ahead of it
    uint32_t *const split = nlg_batched_split_bytes(seq, out, cols) ? (uint32_t *)(more + ternary_bytes(seq, cols)) : nullptr;
    if (lora_by_token(l, cols, out, 3u << 24)) {
      DownArgs d{};
      d.l = l; d.x = x; d.k = cols; d.scaled = false; d.u = u ? u : (float *)workspace; d.zero = split;
      UpArgs p{};
      p.l = l; p.u = d.u; p.res = y; p.y = y; p.n = out; p.scaled = true;
      const ActQArgs q{x, nullptr, 0.0f, nullptr, 0, 0, more, gamma, seq, cols, 0u};
      return lora_tok_down(what, d, bf, &q, st) || nlg_batched_gemm(f, more, gamma, NLG_EPI_STORE, st, split) ||
                     lora_tok_up(what, p, bf, st)
                 ? NLG_ERR
                 : NLG_OK;
    }
    DownArgs d{};
    d.l = l; d.x = x; d.k = cols; d.scaled = false; d.u = u ? u : (float *)workspace; d.zero = split;
    float *const parts = (float *)((uint8_t *)workspace + lora_round((size_t)seq * rmax * 4));
    bool done = false;
    if (nlg_act_q_launch(x, nullptr, 0.0f, nullptr, 0, 0, NLG_PRO_NONE, more, gamma, seq, cols, st) ||
        lora_down(what, d, bf, false, parts, st) || nlg_batched_gemm_lora(f, more, gamma, l, d.u, bf, split, &done, st))
      return NLG_ERR;
    if (done) return NLG_OK;
    UpArgs p{};
    p.l = l; p.u = d.u; p.res = y; p.y = y; p.n = out; p.scaled = true;
    return lora_up(what, p, bf, false, st) ? NLG_ERR : NLG_OK;
  }
  // (a row is a grid's y there)
  for (uint32_t r = 0; r < seq; r += 65535)
    if (nlg_ternary_linear(x + (size_t)r * cols, w2, bias, beta, beta_per_row, y + (size_t)r * out, nullptr,
                           seq - r < 65535 ? seq - r : 65535, out, cols, more, workspace_bytes - nu, (void *)st))
      return NLG_ERR;
  return lora_forward(what, l, x, bf, y, y, u, out, cols, workspace, st) ? NLG_ERR : NLG_OK;
}

// What a gradient call keeps: du and u, and the parts of their sums and the gradients'.  Up to 64 ranks it makes one pass over dy
// (parts: of 256 columns of dy each, and every zy-th block of rows) and, while x, dres and dx are 128 MiB or less, one over x.
// Whole calls with that pass and with one for dA and one for dx, at rank 16, two adapters, out = cols = 2560: 250 rows 24.8 and
// 30.3 us, 1,000 rows 30.8 and 35.8, 4,000 rows (117 MiB) 54.6 and 61.0; at rank 32, three adapters, 6912 -> 2560: 1,200 rows
// (95 MiB) 58.6 and 67.2, 2,400 rows (190 MiB) 91.7 and 86.9, 4,616 rows 156 and 144.  More ranks take a pass for each sum.
struct LoraGradPlan {
  bool gx;                       // one pass over x
  uint32_t gy, wx, zy, zx;       // workgroups along the columns, parts of the rows
  size_t u, du_parts, db_parts, da_parts, bytes;
};
#define LORA_GRAD_RANK 64
static LoraGradPlan lora_grad_plan(uint32_t seq, uint32_t out, uint32_t cols, uint32_t adapters, uint32_t rmax,
                                   uint32_t requests) {
  LoraGradPlan p = {};
  if (!lora_sizes(seq, out, cols, rmax, requests) || !adapters || adapters > 65534) return p;
  const size_t row = lora_round((size_t)seq * rmax * 4), down = lora_down_bytes(seq, cols, rmax);
  const uint64_t na = (uint64_t)adapters * rmax * cols, nb = (uint64_t)adapters * rmax * out, blocks = ((uint64_t)seq + 15) / 16;
  p.u = row;
  p.du_parts = 2 * row;
  if (rmax > LORA_GRAD_RANK) {
    p.zy = lora_parts(seq, out, adapters);
    p.zx = lora_parts(seq, cols, adapters);
    const size_t more = lora_down_bytes(seq, out, rmax);
    p.db_parts = p.du_parts + (down > more ? down : more);
  } else {
    // three workgroups a CU, of a block of rows at least
    const auto parts = [&](uint64_t wg) {
      uint64_t z = (768 + wg - 1) / wg;
      if (z > blocks) z = blocks;
      return (uint32_t)(z < 1 ? 1 : z > 16 ? 16 : z);
    };
    p.gy = (out + 255) / 256;
    p.zy = parts((uint64_t)p.gy * adapters);
    p.gx = 12ull * seq * cols <= (128u << 20);
    p.wx = (cols + 255) / 256;
    p.zx = p.gx ? parts((uint64_t)p.wx * adapters) : lora_parts(seq, cols, adapters);
    const size_t du = p.gy > 1 ? p.gy * ((size_t)seq * rmax * 4) : 0;
    p.db_parts = p.du_parts + lora_round(du > down ? du : down);
  }
  p.da_parts = p.db_parts + (p.zy > 1 ? lora_round(p.zy * nb * 4) : 0);
  p.bytes = p.da_parts + (p.zx > 1 ? lora_round(p.zx * na * 4) : 0);
  return p;
}

extern "C" size_t nlg_lora_linear_grad_workspace(uint32_t seq, uint32_t out, uint32_t cols, uint32_t adapters,
                                                 uint32_t rmax, uint32_t requests) {
  return lora_grad_plan(seq, out, cols, adapters, rmax, requests).bytes;
}

// du and dB of up to 64 ranks
static int lora_gy(const char *what, const LoraArgs &l, const LoraGradPlan &p, const float *u, const float *dy, float *du,
                   float *db, uint32_t out, bool bf, uint8_t *ws, hipStream_t st) {
  GyArgs y{};
  y.l = l; y.dy = dy; y.u = u; y.n = out;
  y.du = p.gy > 1 ? (float *)(ws + p.du_parts) : du;
  y.db = p.zy > 1 ? (float *)(ws + p.db_parts) : db;
  const uint32_t nt = (l.rmax + 15) / 16;
  const bool vec = out % 4 == 0 && ((uintptr_t)dy & 15) == 0;
  const dim3 grid(p.gy, l.adapters, p.zy);
#define BY_RANK(GO)           \
  do {                        \
    if (nt <= 1) GO(1);       \
    else if (nt <= 2) GO(2);  \
    else GO(4);               \
  } while (0)
#define GO(N)                                                                              \
  do {                                                                                     \
    constexpr int E = N == 1 ? 4 : 2;                                                      \
    const dim3 blk(1024 / E);                                                              \
    if (bf && vec) hipLaunchKernelGGL((k_lora_gy<true, N, E, true>), grid, blk, 0, st, y);  \
    else if (bf) hipLaunchKernelGGL((k_lora_gy<true, N, E, false>), grid, blk, 0, st, y);   \
    else if (vec) hipLaunchKernelGGL((k_lora_gy<false, N, E, true>), grid, blk, 0, st, y);  \
    else hipLaunchKernelGGL((k_lora_gy<false, N, E, false>), grid, blk, 0, st, y);          \
  } while (0)
  BY_RANK(GO);
#undef GO
  NLG_LAUNCHED(what);
  return lora_sum(what, lora_parts_of(y.du, du, (uint64_t)l.seq * l.rmax, p.gy), {}, st);
}

// dA and dx of up to 64 ranks in one pass; da: where its parts go
static int lora_gx(const char *what, const LoraArgs &l, const LoraGradPlan &p, const float *x, const float *du,
                   const float *dres, float *dx, float *da, uint32_t cols, bool bf, hipStream_t st) {
  GxArgs g{};
  g.l = l; g.x = x; g.du = du; g.dres = dres; g.dx = dx; g.n = cols; g.da = da;
  const uint32_t nt = (l.rmax + 15) / 16;
  const dim3 grid(p.wx, l.adapters + (dx && dx != dres ? 1 : 0), p.zx);
#define GO(N)                                                                                   \
  do {                                                                                          \
    constexpr int E = N == 1 ? 4 : 2;                                                           \
    if (bf) hipLaunchKernelGGL((k_lora_gx<true, N, E>), grid, dim3(1024 / E), 0, st, g);        \
    else hipLaunchKernelGGL((k_lora_gx<false, N, E>), grid, dim3(1024 / E), 0, st, g);          \
  } while (0)
  BY_RANK(GO);
#undef GO
#undef BY_RANK
  NLG_LAUNCHED(what);
  return NLG_OK;
}

extern "C" int nlg_lora_linear_grad(const float *x, const float *u, const float *dy, const uint16_t *a,
                                    const uint16_t *b, int fmt, const float *scale, const int32_t *rank,
                                    const int32_t *start, const int32_t *adapter, uint32_t requests,
                                    uint32_t adapters, uint32_t rmax, const float *dres, float *dx, float *da,
                                    float *db, uint32_t seq, uint32_t out, uint32_t cols, void *workspace,
                                    size_t workspace_bytes, void *stream) {
  const char *what = "lora linear gradient";
  if (!seq) return nlg_fail("%s: seq must be nonzero", what);
  DownArgs d{};
  if (lora_check(what, a, b, fmt, scale, rank, start, adapter, requests, adapters, rmax, seq, out, cols, d.l)) return NLG_ERR;
  if (!x || !dy || !da || !db) return nlg_fail("%s: null pointer", what);
  if (((uintptr_t)x | (uintptr_t)u | (uintptr_t)da | (uintptr_t)db | (uintptr_t)dx | (uintptr_t)dres) & 15)
    return nlg_fail("%s: x, u, dres, dx, da and db must be 16-byte aligned", what);
  if ((uintptr_t)dy & 3) return nlg_fail("%s: dy must be 4-byte aligned", what);
  const LoraGradPlan plan = lora_grad_plan(seq, out, cols, adapters, rmax, requests);
  const size_t need = plan.bytes;
  if (!workspace || workspace_bytes < need)
    return nlg_fail("%s: workspace holds %zu bytes, needs %zu", what, workspace ? workspace_bytes : 0, need);
  if ((uintptr_t)workspace & 15) return nlg_fail("%s: the workspace must be 16-byte aligned", what);
  const uint64_t r4 = (uint64_t)seq * 4, na = (uint64_t)adapters * rmax * cols, nb = (uint64_t)adapters * rmax * out;
  const NlgSpan at[] = {{x, r4 * cols}, {u, r4 * rmax}, {dy, r4 * out}, {a, 2 * na}, {b, 2 * nb}, {scale, 4ull * adapters},
                        {rank, 4ull * adapters}, {start, 4ull * requests + 4}, {adapter, 4ull * requests},
                        {dres == dx ? nullptr : dres, r4 * cols}, {dx, r4 * cols}, {da, 4 * na}, {db, 4 * nb},
                        {workspace, need}};
  if (nlg_outputs_overlap(at, 14, 4))
    return nlg_fail("%s: outputs or the workspace overlap each other or an input (dx may be dres itself)", what);
  NLG_SCOPE(what);
  hipStream_t st = nlg_stream(stream);
  const bool bf = fmt == NLG_LORA_BF16;
  uint8_t *const ws = (uint8_t *)workspace;
  float *const du = (float *)ws, *const parts = (float *)(ws + plan.du_parts);
  if (!u) {  // (in the form that this call's own size takes: the last bits may differ from the forward call's)
    d.x = x; d.k = cols; d.scaled = false; d.u = (float *)(ws + plan.u);
    u = d.u;
    if (lora_by_token(d.l, cols, 0, 1u << 27) ? lora_tok_down(what, d, bf, nullptr, st) : lora_down(what, d, bf, false, parts, st))
      return NLG_ERR;
  }
  float *const dbp = plan.zy > 1 ? (float *)(ws + plan.db_parts) : db, *const dap = plan.zx > 1 ? (float *)(ws + plan.da_parts) : da;
  if (rmax <= LORA_GRAD_RANK) {
    if (lora_gy(what, d.l, plan, u, dy, du, db, out, bf, ws, st)) return NLG_ERR;
  } else {
    d.x = dy; d.k = out; d.scaled = true; d.u = du;
    OuterArgs o{};
    o.l = d.l; o.p = u; o.q = dy; o.out = db; o.n = out; o.scaled = true;
    if (lora_down(what, d, bf, true, parts, st) || lora_outer(what, o, true, dbp, plan.zy, st)) return NLG_ERR;
  }
  if (plan.gx) {
    if (lora_gx(what, d.l, plan, x, du, dres, dx, dap, cols, bf, st)) return NLG_ERR;
  } else {
    OuterArgs o{};
    o.l = d.l; o.p = du; o.q = x; o.out = da; o.n = cols; o.scaled = false;
    if (lora_outer(what, o, false, dap, plan.zx, st)) return NLG_ERR;
    if (dx) {
      UpArgs p{};
      p.l = d.l; p.u = du; p.res = dres; p.y = dx; p.n = cols; p.scaled = false;
      if (lora_up(what, p, bf, true, st)) return NLG_ERR;
    }
  }
  const uint64_t nb4 = (uint64_t)adapters * rmax * out, na4 = (uint64_t)adapters * rmax * cols;
  return lora_sum(what, lora_parts_of(dbp, db, nb4, plan.zy), lora_parts_of(dap, da, na4, plan.zx), st);
}
