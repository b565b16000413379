// nlg_kv8.hip -- the 8-bit paged KV cache: written with the head norms, the
// rotation and the quantisation in one pass, attended by one token or by a
// tree of drafted tokens a sequence, its accepted path moved into place, and
// read back.  No reference counterpart: the reference chains rmsnorm-heads,
// rope-half and cache-append-paged-v (kernels.el:823-882, :1211-1220) on f32
// caches.  The layout is in nlg_kv8.h.
#include <math.h>

#include "nlg_internal.h"
#include "nlg_kv8.h"

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

// The device the library runs on made the calling thread's for one call.
struct DeviceScope {
  int was = -1;
  bool ok = true;
  DeviceScope() {
    const int want = nlg_device();
    if (hipGetDevice(&was) != hipSuccess) was = -1;
    if (was != want) ok = hipSetDevice(want) == hipSuccess;
    else was = -1;
  }
  ~DeviceScope() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

// ------------------------------------------------------------------ append

struct AppendArgs {
  const float *qkv, *qgain, *kgain;  // [rows][(heads + 2 kvheads) * hd]; [hd] or null
  const float *co, *si;              // [trows][hd / 2]
  const int32_t *seq, *slot, *rpos;  // [rows]; seq null: row r; rpos null: slot
  float *q;                          // [rows][heads * hd]
  uint8_t *kpool, *vpool;
  Kv8Pages pg;
  double eps;
  uint64_t rows;
  uint32_t batch, heads, trows, qblocks;
  bool past;  // q is stored past the caches
};

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Over aligned groups of L lanes (8 or 16), in every lane.
template <int L>
__device__ __forceinline__ double lanes_sum_f64(double v) {
  v = v + dpp_f64<0xB1>(v);   // quad_perm [1,0,3,2]
  v = v + dpp_f64<0x4E>(v);   // quad_perm [2,3,0,1]
  v = v + dpp_f64<0x141>(v);  // row_half_mirror
  if (L == 16) v = v + dpp_f64<0x140>(v);  // row_mirror
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t lanes_max_u32(uint32_t v) {
  v = max(v, nlg_qperm<0xB1>(v));
  v = max(v, nlg_qperm<0x4E>(v));
  v = max(v, nlg_qperm<0x141>(v));
  if (L == 16) v = max(v, nlg_qperm<0x140>(v));
  return v;
}

// x / s rounded to a code: int8 to the nearest whole number (ties to even)
// within +-127, e4m3 to its nearest value within +-448.  rs is 1 / s rounded;
// the quotient is corrected by its remainder, so that a tie stays one.
template <int FMT>
__device__ __forceinline__ double kv8_round(double x, double s, double rs) {
  double u = x * rs;
  u = fma(fma(-u, s, x), rs, u);
  if (FMT == NLG_KV_I8) return fmin(fmax(rint(u), -127.0), 127.0);
  // e4m3: steps of 2^(e - 3) from 2^e on, of 2^-9 below 2^-6
  int e = __builtin_amdgcn_frexp_exp(u);
  e = (e < -5 ? -5 : e) - 4;
  return fmin(fmax(ldexp(rint(ldexp(u, -e)), e), -448.0), 448.0);
}
template <int FMT>
__device__ __forceinline__ uint32_t kv8_code2(double a, double b) {
  if (FMT == NLG_KV_I8) return ((uint32_t)(int)a & 0xffu) | ((uint32_t)(int)b & 0xffu) << 8;
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32((float)a, (float)b, 0, false) & 0xffffu;
}

// A row's eight values of this lane as codes (two words) and the row's scale; L
// lanes hold the row.
template <int FMT, int L>
__device__ __forceinline__ float kv8_quantise(const double *y, uint2 &code) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) top = max(top, __float_as_uint((float)y[i]) & 0x7fffffffu);
  top = lanes_max_u32<L>(top);  // magnitudes in their bits' order, infinities and NaN above all
  const float scale = (float)((double)__uint_as_float(top) / (FMT == NLG_KV_I8 ? 127.0 : 448.0));
  code = make_uint2(0, 0);
  // a row with a value that is not finite: no codes, a scale that says so
  if (top >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if (scale > 0.0f) {
    const double s = scale, rs = 1.0 / s;
    double r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = kv8_round<FMT>(y[i], s, rs);
    code.x = kv8_code2<FMT>(r[0], r[1]) | kv8_code2<FMT>(r[2], r[3]) << 16;
    code.y = kv8_code2<FMT>(r[4], r[5]) | kv8_code2<FMT>(r[6], r[7]) << 16;
  }
  return scale;
}
__device__ __forceinline__ void load8(const float *p, const float *q, double *y) {
  const float4 a = *(const float4 *)p, b = *(const float4 *)q;
  y[0] = a.x; y[1] = a.y; y[2] = a.z; y[3] = a.w;
  y[4] = b.x; y[5] = b.y; y[6] = b.z; y[7] = b.w;
}

// y = x / sqrt(mean(x^2) + eps) * gain, rotated; codes of y / scale.  All in 64
// bits: a code then depends on the inputs alone and not on the order of a sum, so
// a prefix cached twice holds the same bytes.  They cost little only where lanes
// share a row's root and quotients: a head row is on HD / 8 lanes, eight values
// (four rotation pairs) each (on all 64 of a wave 97 us at 4,731 rows of 32/8
// heads of 128, 51 so).  The first qblocks workgroups take the q and
// k heads; the others V, a wave sixteen rows of one head, whose codes pass
// through LDS: a position's bytes of a tile lie sixteen apart, and a store then
// runs over 64 dimensions (8 lines) instead of one byte a line.  Bound by the
// bytes where there are many: 48 us there, 204 MB, 4.2 TB/s, in either format; one row of 20/5
// heads, 3.1 us, by the chain slot -> block -> store.
template <int HD, int FMT, bool HALF>
__global__ __launch_bounds__(256) void k_append_q8(AppendArgs a) {
  constexpr int L = HD / 8, RP = 64 / L;  // lanes a row, rows at once
  constexpr int VS = 20;                  // bytes between a dimension's codes in LDS: two lanes a bank
  __shared__ __align__(16) uint8_t s_v[4][HD * VS];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, m = lane % L;
  const uint32_t per = a.heads + 2 * a.pg.kvheads;
  if (blockIdx.x >= a.qblocks) {
    const uint64_t w = (uint64_t)(blockIdx.x - a.qblocks) * 4 + wv;
    const uint32_t h = (uint32_t)(w % a.pg.kvheads);
    const uint64_t r0 = w / a.pg.kvheads * 16;
    if (r0 >= a.rows) return;
    const int n = a.rows - r0 < 16 ? (int)(a.rows - r0) : 16;
    float4 x[16 / RP][2];
#pragma unroll
    for (int p = 0; p < 16 / RP; p++) {
      const int i = p * RP + lane / L;
      const float *src = a.qkv + ((r0 + (i < n ? i : 0)) * per + a.heads + a.pg.kvheads + h) * HD + m * 8;
      x[p][0] = *(const float4 *)src;
      x[p][1] = *(const float4 *)(src + 4);
    }
    // where row r0 + lane goes
    uint32_t tile = KV8_NONE, at = 0;
    if (lane < n) {
      const int32_t slot = a.slot[r0 + lane];
      const uint32_t b = a.seq ? (uint32_t)a.seq[r0 + lane] : (uint32_t)(r0 + lane);
      if (slot >= 0 && b < a.batch) tile = kv8_tile(a.pg, b, h, (uint32_t)slot / KV8_TILE);
      at = (uint32_t)slot % KV8_TILE;
    }
#pragma unroll
    for (int p = 0; p < 16 / RP; p++) {
      const int i = p * RP + lane / L;
      if (p * RP >= n) break;
      const double y[8] = {x[p][0].x, x[p][0].y, x[p][0].z, x[p][0].w, x[p][1].x, x[p][1].y, x[p][1].z, x[p][1].w};
      uint2 code;
      const float scale = kv8_quantise<FMT, L>(y, code);
#pragma unroll
      for (int d = 0; d < 8; d++)
        s_v[wv][(m * 8 + d) * VS + i] = (uint8_t)((d < 4 ? code.x : code.y) >> (8 * (d & 3)));
      const uint32_t to = __shfl(tile, i), ta = __shfl(at, i);
      if (m == 0 && to != KV8_NONE)
        *(float *)(a.vpool + (size_t)to * kv8_tile_bytes(HD) + kv8_scale_byte(HD, ta)) = scale;
    }
    __builtin_amdgcn_wave_barrier();  // (LDS of one wave: its operations keep their order)
    for (int i = 0; i < n; i++) {
      const uint32_t to = __builtin_amdgcn_readlane(tile, i), ta = __builtin_amdgcn_readlane(at, i);
      if (to == KV8_NONE) continue;
      uint8_t *t = a.vpool + (size_t)to * kv8_tile_bytes(HD);
#pragma unroll
      for (int d = 0; d < HD; d += 64) t[kv8_v_byte(ta, d + lane)] = s_v[wv][(d + lane) * VS + i];
    }
    return;
  }
  const uint32_t perq = a.heads + a.pg.kvheads;
  const uint64_t unit = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / L;
  if (unit >= a.rows * perq) return;
  const uint64_t row = unit / perq;
  const uint32_t h = (uint32_t)(unit % perq);
  // this lane's dimensions: 8 m .., or with HALF 4 m .. and HD / 2 + 4 m ..
  const int d0 = HALF ? 4 * m : 8 * m, d1 = HALF ? HD / 2 + 4 * m : 8 * m + 4;
  const float *x = a.qkv + (row * per + h) * HD;
  double y[8];
  load8(x + d0, x + d1, y);
  const int32_t slot = a.slot[row];
  const int32_t rp = a.rpos ? a.rpos[row] : slot;
  const bool in = rp >= 0 && (uint32_t)rp < a.trows;
  const size_t trow = (size_t)(in ? rp : 0) * (HD / 2) + 4 * m;
  const float4 c4 = *(const float4 *)(a.co + trow), s4 = *(const float4 *)(a.si + trow);
  // (looked up ahead of the arithmetic, which hides it)
  uint32_t tile = KV8_NONE;
  if (h >= a.heads) {
    const uint32_t b = a.seq ? (uint32_t)a.seq[row] : (uint32_t)row;
    if (slot >= 0 && b < a.batch) tile = kv8_tile(a.pg, b, h - a.heads, (uint32_t)slot / KV8_TILE);
  }
  const float *gain = h < a.heads ? a.qgain : a.kgain;
  if (gain) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fma(y[i], y[i], ss);
    ss = lanes_sum_f64<L>(ss);
    const double inv = 1.0 / sqrt(ss / HD + a.eps);
    double g[8];
    load8(gain + d0, gain + d1, g);
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = y[i] * inv * g[i];
  }
  const float cf[4] = {c4.x, c4.y, c4.z, c4.w}, sf[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const double c = in ? cf[i] : 0.0f, s = in ? sf[i] : 0.0f;
    double &p = y[HALF ? i : 2 * i], &r = y[HALF ? i + 4 : 2 * i + 1];
    const double t = p * c - r * s;
    r = p * s + r * c;
    p = t;
  }
  if (h < a.heads) {
    float *q = a.q + (row * a.heads + h) * HD;
    const float4 q0 = make_float4((float)y[0], (float)y[1], (float)y[2], (float)y[3]);
    const float4 q1 = make_float4((float)y[4], (float)y[5], (float)y[6], (float)y[7]);
    if (a.past) {
      nlg_st_stream_f4((float4 *)(q + d0), q0);
      nlg_st_stream_f4((float4 *)(q + d1), q1);
    } else {
      *(float4 *)(q + d0) = q0;
      *(float4 *)(q + d1) = q1;
    }
    return;
  }
  uint2 code;
  const float scale = kv8_quantise<FMT, L>(y, code);
  if (tile == KV8_NONE) return;
  const uint32_t at = (uint32_t)slot % KV8_TILE;
  uint8_t *t = a.kpool + (size_t)tile * kv8_tile_bytes(HD);
  *(uint32_t *)(t + kv8_k_byte(HD, at, d0)) = code.x;
  *(uint32_t *)(t + kv8_k_byte(HD, at, d1)) = code.y;
  if (m == 0) *(float *)(t + kv8_scale_byte(HD, at)) = scale;
}

// ------------------------------------------------------------------ attention

struct Kv8Attn {
  const float *q;  // [batch][tmax][heads * hd]
  const uint8_t *kpool, *vpool;
  const int32_t *base;    // decode: the last position; tree: the slot of node 0
  const int32_t *nodes;   // tree: [batch] or null
  const uint64_t *mask;   // tree: [batch][tmax] or null
  Kv8Pages pg;
  // partials: averages of V [slots][kvheads][rowsper][hd] (sums of them with their weights
  // could pass f32's end where V is large), maxima and sums [slots][kvheads][rowsper][2]
  float *out, *pctx, *pmz;
  uint2 *pfirst;            // [batch]: a sequence's first slot, its chunks
  uint32_t batch, tmax, heads, grp;  // grp: query heads of a kv head; a sequence's rows: tmax * grp
  uint32_t rowsper, rowslog, groups, want, least, unit;  // Kv8Split
  Kv8Div bykvheads, bygrp, bygroups;
  bool tree, one;
  float coef;  // log2(e) / sqrt(hd): scores in base 2
};

// Eight codes of a K or V row (two words) as halves, exactly: an int8 code's
// byte made unsigned and set behind 0x64 is the half 1024 + 128 + code.
template <int FMT>
__device__ __forceinline__ half8v kv8_half8(uint32_t w0, uint32_t w1) {
  union {
    half8v v;
    half2v p[4];
    uint32_t u[4];
  } r;
  if (FMT == NLG_KV_I8) {
    const uint32_t x0 = w0 ^ 0x80808080u, x1 = w1 ^ 0x80808080u;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, x0, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, x0, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, x1, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, x1, 0x04030402u);
    const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) r.p[i] = r.p[i] + off;
  } else {
    r.p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
    r.p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
    r.p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
    r.p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
  }
  return r.v;
}
// Eight f32 as halves hi + lo, each rounded to nearest: 22 bits together.
__device__ __forceinline__ void split8(const float *w, half8v &hi, half8v &lo) {
  float minus = -1.0f;  // (a factor the compiler does not see: one mixed FMA a remainder, not two instructions)
  asm("" : "+s"(minus));
  union {
    half8v v;
    half2v p[4];
  } a, b;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2v t = {w[2 * i], w[2 * i + 1]};
    a.p[i] = __builtin_convertvector(t, half2v);
    b.p[i] = {(_Float16)fmaf((float)a.p[i][0], minus, t[0]), (_Float16)fmaf((float)a.p[i][1], minus, t[1])};
  }
  hi = a.v;
  lo = b.v;
}
// Eight products of f32 as halves: rounded, and what that left, rounded (exact
// where it is representable).  Written out: each is one mixed FMA that leaves its
// half in place, where the compiler takes two instructions.  It does not look
// inside, so the waits are here too: before, for an exponential issued just
// ahead (one state); after, for a matrix instruction that reads the result (two).
__device__ __forceinline__ void split_products(const float *x, const float *y, half8v &hi, half8v &lo) {
  union {
    half8v v;
    uint32_t u[4];
  } a, b;
  asm("s_nop 0\n\t"
      "v_fma_mixlo_f16 %0, %8, %16, 0\n\t"
      "v_fma_mixhi_f16 %0, %9, %17, 0\n\t"
      "v_fma_mixlo_f16 %1, %10, %18, 0\n\t"
      "v_fma_mixhi_f16 %1, %11, %19, 0\n\t"
      "v_fma_mixlo_f16 %2, %12, %20, 0\n\t"
      "v_fma_mixhi_f16 %2, %13, %21, 0\n\t"
      "v_fma_mixlo_f16 %3, %14, %22, 0\n\t"
      "v_fma_mixhi_f16 %3, %15, %23, 0\n\t"
      "v_fma_mixlo_f16 %4, %8, %16, -%0 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %4, %9, %17, -%0 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixlo_f16 %5, %10, %18, -%1 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %5, %11, %19, -%1 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixlo_f16 %6, %12, %20, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %6, %13, %21, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixlo_f16 %7, %14, %22, -%3 op_sel:[0,0,0] op_sel_hi:[0,0,1]\n\t"
      "v_fma_mixhi_f16 %7, %15, %23, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]\n\t"
      "s_nop 1"
      : "=&v"(a.u[0]), "=&v"(a.u[1]), "=&v"(a.u[2]), "=&v"(a.u[3]), "=&v"(b.u[0]), "=&v"(b.u[1]), "=&v"(b.u[2]),
        "=&v"(b.u[3])
      : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]), "v"(y[0]), "v"(y[1]),
        "v"(y[2]), "v"(y[3]), "v"(y[4]), "v"(y[5]), "v"(y[6]), "v"(y[7]));
  hi = a.v;
  lo = b.v;
}
// Lane J of each row of sixteen, in all of them.
template <int J>
__device__ __forceinline__ float row_lane(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + J, 0xf, 0xf, true));
}
template <int I>
struct Int {
  static constexpr int value = I;
};
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(F &&f) {
  if constexpr (I < N) {
    f(Int<I>{});
    each<N, I + 1>(f);
  }
}
// (fmaxf would make each operand quiet first; a NaN may lose against any value:
// the sums take it up again)
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}
__device__ __forceinline__ float rows_max(float v) {  // over lanes 16, 32 and 48 apart
  float2 r = nlg_pair_f32<16>(v);
  v = max3(r.x, r.y, r.y);
  r = nlg_pair_f32<32>(v);
  return max3(r.x, r.y, r.y);
}
__device__ __forceinline__ float rows_sum(float v) {
  float2 r = nlg_pair_f32<16>(v);
  v = r.x + r.y;
  r = nlg_pair_f32<32>(v);
  return r.x + r.y;
}

// What a row's context is divided by: its sum; where it has attended nothing, the
// context is zero.
__device__ __forceinline__ float kv8_inverse(float z) { return z > 0.0f || z != z ? 1.0f / z : 0.0f; }

// The positions of sequence b.
__device__ __forceinline__ Kv8Extent kv8_of(const Kv8Attn &a, uint32_t b) {
  return kv8_extent(a.tree, a.base[b], a.nodes ? a.nodes[b] : (int32_t)a.tmax, a.tmax,
                    a.pg.mbps * a.pg.bpt.d * KV8_TILE);
}

// A wave's view of the split: lanes hold 64 sequences at a time.
struct Kv8Plan {
  uint32_t per;
  Kv8Extent mine;  // of sequence `lane`

  __device__ __forceinline__ Kv8Extent at(const Kv8Attn &a, uint32_t b0, int lane) const {
    if (b0 == 0) return mine;
    return of(a, b0, lane);
  }
  static __device__ __forceinline__ Kv8Extent of(const Kv8Attn &a, uint32_t b0, int lane) {
    Kv8Extent e = kv8_of(a, b0 + lane < a.batch ? b0 + lane : a.batch - 1);
    e.on = e.on && b0 + lane < a.batch;
    return e;
  }
  static __device__ __forceinline__ uint64_t sum(uint64_t v) {  // (lanes below 2^42 each)
    return (uint64_t)(uint32_t)nlg_wave_sum_i32((int)(v & 0xffffff)) +
           ((uint64_t)(uint32_t)nlg_wave_sum_i32((int)(v >> 24)) << 24);
  }
  __device__ __forceinline__ uint32_t slots(const Kv8Attn &a, const Kv8Extent &e) const {
    return kv8_groups(e, a.grp, a.rowslog) * kv8_chunks(kv8_steps(e), per);
  }
  __device__ __forceinline__ Kv8Plan(const Kv8Attn &a, int lane) {
    mine = of(a, 0, lane);
    uint32_t g = kv8_groups(mine, a.grp, a.rowslog);
    uint64_t total = (uint64_t)g * kv8_steps(mine), pairs = g;
    for (uint32_t b0 = 64; b0 < a.batch; b0 += 64) {
      const Kv8Extent e = of(a, b0, lane);
      g = kv8_groups(e, a.grp, a.rowslog);
      total += (uint64_t)g * kv8_steps(e);
      pairs += g;
    }
    total = sum(total);
    pairs = sum(pairs);
    const Kv8Per p = kv8_per(total ? total : 1, pairs, a.want, a.least, a.unit);
    per = p.first;
    // (a better fit than the bound, for up to 64 sequences)
    for (int i = 0; i < 4 && per < p.last; i++) {
      if (a.batch > 64 || i == 3) {
        per = p.last;
        break;
      }
      const uint32_t n = (uint32_t)nlg_wave_sum_i32((int)slots(a, mine));
      if (n <= a.want) break;
      per = kv8_more(per, n, a.want, p.last, a.unit);
    }
  }
  // inclusive sums over the lanes
  static __device__ __forceinline__ uint32_t sums(uint32_t v) {
    v += (uint32_t)nlg_dpp<0x111>((int)v);       // row_shr:1
    v += (uint32_t)nlg_dpp<0x112>((int)v);       // row_shr:2
    v += (uint32_t)nlg_dpp<0x114>((int)v);       // row_shr:4
    v += (uint32_t)nlg_dpp<0x118>((int)v);       // row_shr:8
    v += (uint32_t)nlg_dpp<0x142, 0xa>((int)v);  // row_bcast:15 into rows 1, 3
    v += (uint32_t)nlg_dpp<0x143, 0xc>((int)v);  // row_bcast:31 into rows 2, 3
    return v;
  }
  // The sequence, group and chunk of slot x; false: there are fewer.
  __device__ __forceinline__ bool find(const Kv8Attn &a, uint32_t x, int lane, uint32_t &b, Kv8Extent &e, uint32_t &group,
                                       uint32_t &chunk, uint32_t &chunks) const {
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
      const Kv8Extent l = at(a, b0, lane);
      const uint32_t n = slots(a, l), to = sums(n);
      const uint64_t past = __ballot(before + to > x);
      if (past) {
        const int i = __builtin_ctzll(past);
        b = b0 + i;
        const uint32_t in = x - before - (__builtin_amdgcn_readlane(to, i) - __builtin_amdgcn_readlane(n, i));
        e.base = __builtin_amdgcn_readlane(l.base, i);
        e.end = __builtin_amdgcn_readlane(l.end, i);
        e.nodes = __builtin_amdgcn_readlane(l.nodes, i);
        e.on = true;
        chunks = kv8_chunks(kv8_steps(e), per);
        group = in / chunks;
        chunk = in - group * chunks;
        return true;
      }
      before += __builtin_amdgcn_readlane(to, 63);
    }
    return false;
  }
};

// What a workgroup does: which rows of which sequence and kv head over which positions.
struct Kv8Work {
  uint32_t b, h, row0, c0, c1, slot, chunks;
  Kv8Extent e;
  bool masked;
};
__device__ __forceinline__ bool kv8_work(const Kv8Attn &a, int lane, Kv8Work &w) {
  w.slot = kv8_quot(a.bykvheads, blockIdx.x);
  w.h = blockIdx.x - w.slot * a.pg.kvheads;
  uint32_t share, group;
  if (a.one) {
    w.b = kv8_quot(a.bygroups, w.slot);
    group = w.slot - w.b * a.groups;
    w.chunks = 1;
    w.e = kv8_of(a, w.b);
    w.c0 = 0;
    share = 0xffffffffu;
    if (group >= kv8_groups(w.e, a.grp, a.rowslog)) return false;
  } else {
    const Kv8Plan plan(a, lane);
    uint32_t chunk;
    if (!plan.find(a, w.slot, lane, w.b, w.e, group, chunk, w.chunks)) return false;
    share = kv8_share(kv8_steps(w.e), w.chunks, a.unit) * KV8_STEP;
    w.c0 = chunk * share;
    // for the launch that joins the chunks
    if (!group && !chunk && !w.h && threadIdx.x == 0) a.pfirst[w.b] = make_uint2(w.slot, w.chunks);
  }
  w.row0 = group * a.rowsper;
  w.masked = a.mask;
  // a causal group of rows ends at its last node
  const uint32_t stop = w.masked ? w.e.end : kv8_stop(w.e, kv8_quot(a.bygrp, w.row0 + a.rowsper - 1));
  w.c1 = w.c0 >= stop ? w.c0 : stop - w.c0 < share ? stop : w.c0 + share;
  return true;
}

// A row's maximum m is a reference only: it moves when a score is more than
// KV8_SLACK (in base 2) above it, so after a row's first steps its contexts are
// hardly ever rescaled; the probabilities are below 2^KV8_SLACK, and times the V
// scales in units of vref / 2^(15 - KV8_SLACK) they stay within fp16.
#define KV8_SLACK 6.0f
#define KV8_VUNIT 512.0f  // 2^(15 - KV8_SLACK)
// Products of a probability and a V scale this many binades below vref keep their
// bits (at least 1 in those units, the halves' last step is 2^-24 of it); how far a
// row is lifted at most (its sum of 2^31 times 2^(KV8_UP + KV8_SLACK) stays in 32
// bits); from this distance on a row has no product yet.
#define KV8_NEAR 8.0f
#define KV8_UP 90.0f
#define KV8_NEVER 1e6f
// The maximum of no score: below all that there are, and finite, so that no
// difference of two is a NaN.
#define KV8_FLOOR -3.4028234663852886e38f
// Queries are multiplied as numbers whose largest is 2^(KV8_QTOP - 1) or more, times
// coef (0.13, 0.18): well below fp16's end, so that elements down to 2^-14 of a row's
// largest keep 22 bits in two halves (with 2 in place of 16, down to 1).
#define KV8_QTOP 16
// K scales are multiplied as numbers up to 2^KV8_KTOP: they then keep their bits down
// to 2^-190 of the largest met (a masked row's).
#define KV8_KTOP 64

// A wave's running state over NT tiles of sixteen query rows.  A lane holds the
// query row n = lane & 15 of each tile, and of its scores the sixteen positions
// of the step's tile g = lane >> 4.
template <int HD, int NT>
struct WaveState {
  half8v qh[NT][HD / 32], ql[NT][HD / 32];
  float rs[NT];            // what the row's q was divided by (a power of two, a normal number)
  int ke;                  // no K scale so far exceeds 2^(ke + KV8_KTOP), 1 at first
  float m[NT], z[NT];      // running maximum; this lane's part of the sum
  float up[NT], far[NT];   // probabilities carry 2^up; binades from vref down to the row's largest product with a V scale
  float4v o[NT][HD / 16];  // out[dim 16 i + 4 g + r][query n], times 2^up KV8_VUNIT / vref
  float vref, vinv;        // a power of two no V scale so far exceeds, or 0; KV8_VUNIT / vref
  uint32_t node[NT];
  uint64_t word[NT];       // the node's mask

  // The rows' queries asked for, and made ready (what is loaded between the two
  // arrives while they are).
  struct Queries {
    float4 x[NT][HD / 16];
  };
  __device__ __forceinline__ void fetch(const Kv8Attn &a, const Kv8Work &k, uint32_t row0, int lane, Queries &f) {
    const int g = lane >> 4, n = lane & 15;
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const uint32_t row = row0 + i * 16 + n;
      node[i] = kv8_quot(a.bygrp, row);
      const bool on = node[i] < k.e.nodes;
      const size_t qrow = (size_t)k.b * a.tmax + (on ? node[i] : 0);
      const float *q = a.q + (qrow * a.heads + (size_t)k.h * a.grp + (on ? row - node[i] * a.grp : 0)) * HD + g * 16;
      word[i] = k.masked && on ? a.mask[qrow] : 0;
#pragma unroll
      for (int j = 0; j < HD / 16; j++) f.x[i][j] = *(const float4 *)(q + j / 4 * 64 + j % 4 * 4);
    }
  }
  __device__ __forceinline__ void begin(const Kv8Attn &a, const Kv8Work &k, const Queries &f) {
    constexpr int C = HD / 64;
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const bool on = node[i] < k.e.nodes;
      word[i] = kv8_word(word[i], k.e.nodes);
      float x[HD / 4], top = 0.0f;
#pragma unroll
      for (int j = 0; j < HD / 16; j++) {
        float *y = x + j * 4;
        y[0] = f.x[i][j].x; y[1] = f.x[i][j].y; y[2] = f.x[i][j].z; y[3] = f.x[i][j].w;
      }
#pragma unroll
      for (int j = 0; j < HD / 4; j++) {
        x[j] = on ? x[j] : 0.0f;
        top = fmaxf(top, fabsf(x[j]));
      }
      top = rows_max(top);
      const int e = top > 0.0f && top <= 3.4028234663852886e38f ? __builtin_amdgcn_frexp_expf(top) - KV8_QTOP : 0;
      const int ex = e < -126 ? -126 : e;
      rs[i] = ldexpf(1.0f, ex);
#pragma unroll
      for (int j = 0; j < HD / 4; j++) x[j] = ldexpf(x[j], -ex) * a.coef;
#pragma unroll
      for (int c = 0; c < C; c++) {
        split8(x + c * 16, qh[i][2 * c], ql[i][2 * c]);
        split8(x + c * 16 + 8, qh[i][2 * c + 1], ql[i][2 * c + 1]);
      }
      m[i] = KV8_FLOOR;
      z[i] = up[i] = 0.0f;
      far[i] = on ? KV8_NEVER : -INFINITY;  // (a row that is none: never lifted)
#pragma unroll
      for (int d = 0; d < HD / 16; d++) o[i][d] = {0.0f, 0.0f, 0.0f, 0.0f};
    }
    vref = vinv = 0.0f;
    ke = -KV8_KTOP;
  }

  // K scales in units of 2^ke: a sum of codes times queries (below 2^28) times one
  // stays within f32 where the score does.  unit: what the rows' scores are to be
  // multiplied by for it, 2^ke rs, kept where -infinity times it is that and 0 is 0 (at
  // the lower end scores are below 2^-34).
  __device__ __forceinline__ float rescale_k(float ks) {
    float u = ldexpf(ks, -ke);
    if (__any(fabsf(u) > ldexpf(1.0f, KV8_KTOP))) {
      ke = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(nlg_wave_max_f32(fabsf(ks)))) - KV8_KTOP;
      u = ldexpf(ks, -ke);
    }
    return u;
  }
  __device__ __forceinline__ float unit(int i) const {
    return __builtin_amdgcn_fmed3f(ldexpf(rs[i], ke), 1.17549435e-38f, 1.70141183e38f);
  }

  // V scales in units of vref / KV8_VUNIT: the probabilities times them, as
  // halves, then use the type's whole range.  vs: this lane's of the step; one
  // that is no number counts as 0 there and is named in `odd`, a bit for each of
  // this lane's sixteen positions (any: of the whole wave).  Returns what the
  // contexts so far are to be multiplied by.
  __device__ __forceinline__ float rescale(float &vs, uint32_t &odd, bool &any, int lane) {
    float f = 1.0f;
    const bool bad = !(fabsf(vs) <= 3.4028234663852886e38f);
    const uint64_t all = __ballot(bad);
    any = all != 0;
    odd = 0;
    if (any) {
      odd = (uint32_t)(all >> (lane & 48)) & 0xffffu;
      vs = bad ? 0.0f : vs;
    }
    if (__any(fabsf(vs) > vref)) {
      const int e = __builtin_amdgcn_frexp_expf(nlg_wave_max_f32(fabsf(vs)));
      const int ne = e < -100 ? -100 : e;
      const float nv = ldexpf(1.0f, ne);
      f = vref > 0.0f ? vref * ldexpf(1.0f, -ne) : 0.0f;
      vref = nv;
      vinv = ldexpf(KV8_VUNIT, -ne);
    }
    vs = vs * vinv;
    return f;
  }

  // vref is of all positions: of those that a row does not attend (another
  // branch's, a later token's) and of those that it gives next to no weight.  A row
  // whose own products p V are all far below it has its probabilities, sum and context
  // carry 2^up, so that no such V row, however large, takes the bits of those that
  // make its output.  s: the step's scores in units of su, top: their largest; by: how far the
  // maximum has moved.  Returns what up has grown by, as a factor.
  __device__ __forceinline__ float raise(int i, const float *s, float su, float top, const float *vb, float by, float vresc) {
    // earlier products are smaller by both
    far[i] = far[i] + (fminf(by, KV8_NEVER) + (vresc > 0.0f ? (float)(1 - __builtin_amdgcn_frexp_expf(vresc)) : KV8_NEVER));
    // most often the step's largest probability times its smallest V scale is near
    // enough, and says so without an exponential for each position
    float low = fabsf(vb[0]);
#pragma unroll
    for (int j = 1; j < 16; j++) low = fminf(low, fabsf(vb[j]));
    low = -rows_max(-low);
    float v = nlg_exp2(top - m[i]) * low;
    if (__any(far[i] > KV8_NEAR && !(v >= 1.0f))) {
      v = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; j++) v = fmaxf(v, nlg_exp2(fmaf(s[j], su, -m[i])) * fabsf(vb[j]));
      v = rows_max(v);
    }
    if (v > 0.0f) far[i] = fminf(far[i], (float)(9 - __builtin_amdgcn_frexp_expf(v)));
    const float now = far[i] > KV8_NEAR && far[i] < KV8_NEVER ? fminf(floorf(far[i]), KV8_UP) : 0.0f;
    const float lift = ldexpf(1.0f, (int)(now - up[i]));
    up[i] = now;
    return lift;
  }

  // A step's scores of tile i (products of the codes with q) made probabilities:
  // the running maximum and sum, the contexts rescaled, and the probabilities
  // times the V scales (vb, all sixteen) as halves hi + lo: the product rounded,
  // and what that left, 22 bits together.
  template <bool GEN>
  __device__ __forceinline__ void soften(int i, const float4v *acc, float ks, const float *vb, float vresc,
                                         uint32_t bits, uint32_t odd, bool any, half8v *ph, half8v *pl) {
    const float su = unit(i);
    float s[16];
    each<16>([&](auto J) {
      constexpr int j = decltype(J)::value;
      s[j] = acc[j >> 2][j & 3] * row_lane<j>(ks);
      // (the bit as a word of ones or zeros: no comparison)
      if (GEN) {
        const uint32_t on = (uint32_t)((int32_t)(bits << (31 - j)) >> 31);
        s[j] = __uint_as_float((__float_as_uint(s[j]) & on) | (0xff800000u & ~on));
      }
    });
    float top = max3(s[0], s[1], s[2]);
#pragma unroll
    for (int j = 3; j < 15; j += 2) top = max3(top, s[j], s[j + 1]);
    top = max3(top, s[15], s[15]) * su;
    if (__any(top > m[i] + KV8_SLACK || vresc != 1.0f || far[i] > KV8_NEAR)) {
      top = rows_max(top);
      const float mn = top > m[i] + KV8_SLACK ? top : m[i];
      const float by = mn - m[i], al = nlg_exp2(-by);
      m[i] = mn;
      const float lift = raise(i, s, su, top, vb, by, vresc), sc = al * (vresc * lift);
      z[i] = z[i] * (al * lift);
#pragma unroll
      for (int d = 0; d < HD / 16; d++) o[i][d] = o[i][d] * sc;
    }
    const float ms = m[i] - up[i];
    float zz[4] = {z[i], 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 16; j++) {
      s[j] = nlg_exp2(fmaf(s[j], su, -ms));
      zz[j & 3] = zz[j & 3] + s[j];
    }
    z[i] = (zz[0] + zz[1]) + (zz[2] + zz[3]);
    // a row that attends a V row which is no number is none either
    if (any) z[i] = odd & (GEN ? bits : 0xffffu) ? __uint_as_float(0x7fc00000u) : z[i];
    split_products(s, vb, ph[0], pl[0]);
    split_products(s + 8, vb + 8, ph[1], pl[1]);
  }
};

// The tiles of 1,024 positions from p0 on, one a lane.
__device__ __forceinline__ uint32_t kv8_tiles(const Kv8Attn &a, const Kv8Work &k, uint32_t p0, int lane) {
  const uint32_t mine = p0 + lane * KV8_TILE;
  return mine < k.c1 ? kv8_tile(a.pg, k.b, k.h, mine / KV8_TILE) : KV8_NONE;
}
// Which bytes of a V column's sixteen exist.
__device__ __forceinline__ uint4 kv8_keep(bool there, int left) {
  uint32_t keep[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int k = left - 4 * i;
    keep[i] = !there || k <= 0 ? 0u : k >= 4 ? 0xffffffffu : (1u << (8 * k)) - 1;
  }
  return make_uint4(keep[0], keep[1], keep[2], keep[3]);
}
__device__ __forceinline__ uint4 and4(uint4 x, uint4 m) { return make_uint4(x.x & m.x, x.y & m.y, x.z & m.z, x.w & m.w); }

#define MFMA(x, y, c) __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0)

// PAST: past the caches, for K and V that they will not hold until they are read
// again.
template <bool PAST>
__device__ __forceinline__ uint4 load16(const uint8_t *p) {
  return PAST ? nlg_ld_stream((const uint4 *)p) : *(const uint4 *)p;
}

// One step of a wave on its own: 64 positions from p on, tile `tk` holding this
// lane's K row (4 positions of each of the four tiles a time), tile `tv` its V
// columns and both scales.  GEN: some of the positions are masked or past the
// end.
template <int HD, int FMT, int NT, bool GEN, bool PAST>
__device__ __forceinline__ void kv8_step(const Kv8Attn &a, const Kv8Work &k, WaveState<HD, NT> &w, uint32_t tk,
                                         uint32_t tv, uint32_t p, int lane) {
  constexpr int C = HD / 64, D = HD / 16;
  const int g = lane >> 4, n = lane & 15;
  uint4 kr[4][C], vr[D];
  const bool hk = tk != KV8_NONE, hv = tv != KV8_NONE;
  const uint8_t *kp = a.kpool + (size_t)(hk ? tk : 0) * kv8_tile_bytes(HD) + (lane & 3) * HD + g * 16;
  const size_t vt = (size_t)(hv ? tv : 0) * kv8_tile_bytes(HD);
  const uint8_t *vp = a.vpool + vt;
  float ks = *(const float *)(a.kpool + vt + kv8_scale_byte(HD, n));
  float vs = *(const float *)(vp + kv8_scale_byte(HD, n));
#pragma unroll
  for (int t = 0; t < 4; t++)
#pragma unroll
    for (int c = 0; c < C; c++) kr[t][c] = load16<PAST>(kp + t * 4 * HD + c * 64);
#pragma unroll
  for (int i = 0; i < D; i++) vr[i] = load16<PAST>(vp + i * 256 + n * 16);
  const uint32_t q0 = p + g * KV8_TILE;  // this lane's first position
  const int left = GEN ? kv8_left(k.e, q0) : 16;
  if (__any(!hv || left < 16)) {
    // absent tiles read as zero rows; what lies past the end is not used
    if (!hk)
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int c = 0; c < C; c++) kr[t][c] = make_uint4(0, 0, 0, 0);
    const uint4 keep = kv8_keep(hv, left);
#pragma unroll
    for (int i = 0; i < D; i++) vr[i] = and4(vr[i], keep);
    if (!hv || n >= left) ks = vs = 0.0f;
  }
  ks = w.rescale_k(ks);
  uint32_t odd;
  bool any;
  const float vresc = w.rescale(vs, odd, any, lane);
  float vb[16];
  each<16>([&](auto J) { vb[decltype(J)::value] = row_lane<decltype(J)::value>(vs); });
#pragma unroll
  for (int i = 0; i < NT; i++) {
    // (four sums side by side: a product waits for the one before it on its sum)
    float4v acc[4];
    const float4v none = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < 2 * C; c++) {
      half8v f[4];
#pragma unroll
      for (int t = 0; t < 4; t++)
        f[t] = c & 1 ? kv8_half8<FMT>(kr[t][c / 2].z, kr[t][c / 2].w) : kv8_half8<FMT>(kr[t][c / 2].x, kr[t][c / 2].y);
#pragma unroll
      for (int t = 0; t < 4; t++) acc[t] = MFMA(f[t], w.ql[i][c], c ? acc[t] : none);
#pragma unroll
      for (int t = 0; t < 4; t++) acc[t] = MFMA(f[t], w.qh[i][c], acc[t]);
    }
    half8v ph[2], pl[2];
    const uint32_t bits = GEN ? kv8_bits(k.e, k.masked, w.node[i], w.word[i], q0) : 0u;
    w.template soften<GEN>(i, acc, ks, vb, vresc, bits, odd, any, ph, pl);
#pragma unroll
    for (int d = 0; d < D; d += 4)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        half8v f[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
          f[j] = u ? kv8_half8<FMT>(vr[d + j].z, vr[d + j].w) : kv8_half8<FMT>(vr[d + j].x, vr[d + j].y);
#pragma unroll
        for (int j = 0; j < 4; j++) w.o[i][d + j] = MFMA(f[j], pl[u], w.o[i][d + j]);
#pragma unroll
        for (int j = 0; j < 4; j++) w.o[i][d + j] = MFMA(f[j], ph[u], w.o[i][d + j]);
      }
  }
}

// Few rows (16 NT a group): the workgroup's W waves take its positions in turn,
// 64 at a time, straight from memory into the matrix cores' operands, and meet
// in LDS.  S^T = K q^T and O^T = V^T p^T: a lane then holds one query row and, as
// the scores come out, the very sixteen positions that the second product wants
// of it, with K's rows dealt to the first so (4 of each tile a time); nothing is
// exchanged but maxima and sums.  One pass over the cache, bound by its bytes:
// 8 sequences at 24,000-32,768, 32/8 heads of 128, 480 MB: 84 us, 5.7 TB/s; 32
// of up to 4,096, 20/5 heads, 87 MB: 21.5 us, 4.0 TB/s (25.5 with the join), chunks
// of unequal lengths and a step's loads that wait for the step before (42% of a
// wave's cycles wait for something, 27% for their turn to issue).  One sequence
// (eight waves, no second launch), 20/5 heads: 6.4 us at 64 positions, one step of
// one wave; 8.7 at 512, one of each; 9.6 at 640; 11.7 at 1,024, two: five
// workgroups, each wave's second step asked for after its first.
template <int HD, int FMT, int NT, int W, bool PAST>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2, 2)))
void k_attn_q8(Kv8Attn a) {
  constexpr int D = HD / 16;
  __shared__ float4v s_o[W][D][64];
  __shared__ float s_m[W][16], s_z[W][16];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  Kv8Work k;
  if (!kv8_work(a, lane, k)) return;
  uint32_t tid = kv8_tiles(a, k, k.c0, lane);
  WaveState<HD, NT> w;
  typename WaveState<HD, NT>::Queries qx;
  w.fetch(a, k, k.row0, lane, qx);
  w.begin(a, k, qx);
  const uint32_t whole = k.e.base < k.c1 ? k.e.base : k.c1;  // no mask below this position
  uint32_t p0 = k.c0;  // tid: the tiles from here on
  uint32_t p = k.c0 + wv * KV8_STEP;
  auto step = [&](auto GENV) {
    const uint32_t from = k.c0 + (p - k.c0) / (64 * KV8_TILE) * (64 * KV8_TILE);
    if (from != p0) {
      p0 = from;
      tid = kv8_tiles(a, k, p0, lane);
    }
    const int t0 = (int)(p - p0) / KV8_TILE;
    const uint32_t tv = __shfl(tid, t0 + g), tk = __shfl(tid, t0 + (n >> 2));
    kv8_step<HD, FMT, NT, decltype(GENV)::value != 0, PAST>(a, k, w, tk, tv, p, lane);
    p += W * KV8_STEP;
  };
  while (p + KV8_STEP <= whole) step(Int<0>{});
  while (p < k.c1) step(Int<1>{});

  // the waves' parts meet, one tile of rows at a time, as averages of V with a weight each
  const float vs = w.vref > 0.0f ? w.vref * (1.0f / KV8_VUNIT) : 0.0f;
#pragma unroll
  for (int i = 0; i < NT; i++) {
    if (i) __syncthreads();
    const float z = rows_sum(w.z[i]), inv = kv8_inverse(z);
    if (g == 0) {
      s_m[wv][n] = w.m[i];
      s_z[wv][n] = ldexpf(z, -(int)w.up[i]);
    }
#pragma unroll
    for (int d = 0; d < D; d++) s_o[wv][d][lane] = (w.o[i][d] * inv) * vs;
    __syncthreads();
    float mm = s_m[0][n];
#pragma unroll
    for (int j = 1; j < W; j++) mm = fmaxf(mm, s_m[j][n]);
    float f[W], zz = 0.0f;
#pragma unroll
    for (int j = 0; j < W; j++) {
      f[j] = s_z[j][n] * nlg_exp2(s_m[j][n] - mm);
      zz = zz + f[j];
    }
    const float share = kv8_inverse(zz);
    const uint32_t row = k.row0 + i * 16 + n;
    if (row < (uint64_t)k.e.nodes * a.grp) {
      const uint64_t part = ((uint64_t)k.slot * a.pg.kvheads + k.h) * a.rowsper + row - k.row0;
      if (k.chunks > 1 && wv == 0 && g == 0) *(float2 *)(a.pmz + part * 2) = make_float2(mm, zz);
      float *o = k.chunks > 1 ? a.pctx + part * HD
                              : a.out + (((size_t)k.b * a.tmax + w.node[i]) * a.heads + k.h * a.grp + row - w.node[i] * a.grp) * HD;
#pragma unroll
      for (int d = wv; d < D; d += W) {
        float4v t = s_o[0][d][lane] * (f[0] * share);
#pragma unroll
        for (int j = 1; j < W; j++) t = t + s_o[j][d][lane] * (f[j] * share);
        *(float4v *)(o + d * 16 + g * 4) = t;
      }
    }
  }
}

// More rows: each of the waves has 16 NT of its own, all walk the same positions,
// and K and V are made halves once for the workgroup, in LDS, in the order in
// which the waves' operands lie (a fragment's 64 lanes side by side: no bank is
// asked twice).  While a step is computed the next one's halves are written and
// the one's after it are on their way from memory.  Two chunks of 500-512 tokens
// over 1,024-2,047, 32/8 heads of 64: 60 us, 62.5 with the join, 238 TFLOP/s (each
// product counted once; it is done twice, for hi and lo), bound by issue: a wave
// issues vector arithmetic in 36% of its cycles, two waves a SIMD.  16 us are left
// without any step (the join 6, the partials' stores 4, launch, plan and queries
// 6), 25 with only the loads and the halves in LDS, 41 without the softmax, 62
// without the second product, 58 without waiting for memory.  16 trees of up to 32
// nodes over up to 4,000, 20/5 heads of 128: 32 us, 37 with the join: 15 without
// any step (the join 5, the partials 3), 22 with the loads and halves alone, 31
// without the softmax, 36 without the second product; a wave waits in 45% of its
// cycles, for memory or the other waves, and issues arithmetic in 24%.  Three waves a
// SIMD at head dim 64, with 64 rows a workgroup, took 69 us for 60; eight waves a
// workgroup 85 for 76.
template <int HD, int FMT, int NT>
__global__ __launch_bounds__(64 * KV8_WAVES) __attribute__((amdgpu_waves_per_eu(2, 2)))
void k_attn_wide_q8(Kv8Attn a) {
  constexpr int C = HD / 64, D = HD / 16, DW = D / 4;
  __shared__ half8v s_k[2][4][2 * C][64], s_v[2][D][2][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  Kv8Work k;
  if (!kv8_work(a, lane, k)) return;
  const uint32_t row0 = k.row0 + wv * (NT * 16);
  const bool rows = row0 < (uint64_t)k.e.nodes * a.grp;
  // where this wave's rows stop attending
  const uint32_t stop = k.masked ? k.e.end : kv8_stop(k.e, kv8_quot(a.bygrp, row0 + NT * 16 - 1));
  WaveState<HD, NT> w;
  const uint32_t whole = k.e.base < k.c1 ? k.e.base : k.c1;

  // this wave's share of a step: tile wv's K, DW sixteens of V's dimensions
  uint4 kr[C], vr[DW];
  float ks, vs;
  uint32_t tid = KV8_NONE, tid0 = 0xffffffffu;
  auto load = [&](uint32_t p) {
    const uint32_t p0 = k.c0 + (p - k.c0) / (64 * KV8_TILE) * (64 * KV8_TILE);
    if (p0 != tid0) {
      tid0 = p0;
      tid = kv8_tiles(a, k, p0, lane);
    }
    const int t0 = (int)(p - p0) / KV8_TILE;
    const uint32_t tv = __shfl(tid, t0 + g), tk = __shfl(tid, t0 + (n >> 2));
    const bool hk = tk != KV8_NONE, hv = tv != KV8_NONE;
    const uint8_t *kp = a.kpool + (size_t)(hk ? tk : 0) * kv8_tile_bytes(HD) + (wv * 4 + (lane & 3)) * HD + g * 16;
    const size_t vt = (size_t)(hv ? tv : 0) * kv8_tile_bytes(HD);
    const uint8_t *vp = a.vpool + vt + wv * DW * 256 + n * 16;
    ks = *(const float *)(a.kpool + vt + kv8_scale_byte(HD, n));
    vs = *(const float *)(a.vpool + vt + kv8_scale_byte(HD, n));
#pragma unroll
      for (int c = 0; c < C; c++) kr[c] = *(const uint4 *)(kp + c * 64);
#pragma unroll
      for (int d = 0; d < DW; d++) vr[d] = *(const uint4 *)(vp + d * 256);
    const int left = kv8_left(k.e, p + g * KV8_TILE);
    if (__any(!hv || left < 16)) {
      if (!hk)
#pragma unroll
        for (int c = 0; c < C; c++) kr[c] = make_uint4(0, 0, 0, 0);
      const uint4 keep = kv8_keep(hv, left);
#pragma unroll
      for (int d = 0; d < DW; d++) vr[d] = and4(vr[d], keep);
      if (!hv || n >= left) ks = vs = 0.0f;
    }
  };
  auto store = [&](int buf) {
#pragma unroll
      for (int c = 0; c < C; c++) {
        s_k[buf][wv][2 * c][lane] = kv8_half8<FMT>(kr[c].x, kr[c].y);
        s_k[buf][wv][2 * c + 1][lane] = kv8_half8<FMT>(kr[c].z, kr[c].w);
      }
#pragma unroll
      for (int d = 0; d < DW; d++) {
        s_v[buf][wv * DW + d][0][lane] = kv8_half8<FMT>(vr[d].x, vr[d].y);
        s_v[buf][wv * DW + d][1][lane] = kv8_half8<FMT>(vr[d].z, vr[d].w);
      }
  };
  auto compute = [&](auto GENV, int buf, float ksc, float vsc, uint32_t p) {
    constexpr bool GEN = decltype(GENV)::value != 0;
    ksc = w.rescale_k(ksc);
    uint32_t odd;
    bool any;
    const float vresc = w.rescale(vsc, odd, any, lane);
    float4v acc[NT][4];
    const float4v none = {0.0f, 0.0f, 0.0f, 0.0f};
    half8v f[2][4];
#pragma unroll
    for (int t = 0; t < 4; t++) f[0][t] = s_k[buf][t][0][lane];
#pragma unroll
    for (int c = 0; c < 2 * C; c++) {
#pragma unroll
      for (int t = 0; t < 4; t++)
        if (c + 1 < 2 * C) f[(c + 1) & 1][t] = s_k[buf][t][c + 1][lane];
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[i][t] = MFMA(f[c & 1][t], w.ql[i][c], c ? acc[i][t] : none);
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int t = 0; t < 4; t++) acc[i][t] = MFMA(f[c & 1][t], w.qh[i][c], acc[i][t]);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) f[0][j] = s_v[buf][j][0][lane];
    half8v ph[NT][2], pl[NT][2];
    float vb[16];
    each<16>([&](auto J) { vb[decltype(J)::value] = row_lane<decltype(J)::value>(vsc); });
#pragma unroll
    for (int i = 0; i < NT; i++) {
      const uint32_t bits = GEN ? kv8_bits(k.e, k.masked, w.node[i], w.word[i], p + g * KV8_TILE) : 0u;
      w.template soften<GEN>(i, acc[i], ksc, vb, vresc, bits, odd, any, ph[i], pl[i]);
    }
#pragma unroll
    for (int r = 0; r < D / 2; r++) {  // four sixteens of dimensions, half of the positions
      const int d = r / 2 * 4, u = r & 1;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (r + 1 < D / 2) f[(r + 1) & 1][j] = s_v[buf][(r + 1) / 2 * 4 + j][(r + 1) & 1][lane];
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) w.o[i][d + j] = MFMA(f[r & 1][j], pl[i][u], w.o[i][d + j]);
#pragma unroll
      for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) w.o[i][d + j] = MFMA(f[r & 1][j], ph[i][u], w.o[i][d + j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  typename WaveState<HD, NT>::Queries qx;
  w.fetch(a, k, row0, lane, qx);
  if (k.c0 < k.c1) load(k.c0);
  w.begin(a, k, qx);
  if (k.c0 < k.c1) {
    store(0);
    float ksc = ks, vsc = vs;
    if (k.c1 - k.c0 > KV8_STEP) load(k.c0 + KV8_STEP);
    __syncthreads();
    int buf = 0;
    uint32_t p = k.c0;
    auto turn = [&](auto &&work) {
      float ksn = 0.0f, vsn = 0.0f;
      if (k.c1 - p > KV8_STEP) {
        store(buf ^ 1);
        ksn = ks;
        vsn = vs;
        if (k.c1 - p > 2 * KV8_STEP) load(p + 2 * KV8_STEP);
      }
      work();
      __syncthreads();
      ksc = ksn;
      vsc = vsn;
      buf ^= 1;
      p += KV8_STEP;
    };
    // (loops of their own, not branches of one: where two ways meet, the contexts are copied)
    if (rows) {
      while (p + KV8_STEP <= whole) turn([&] { compute(Int<0>{}, buf, ksc, vsc, p); });
      while (p < stop && p < k.c1) turn([&] { compute(Int<1>{}, buf, ksc, vsc, p); });
    }
    while (p < k.c1) turn([] {});
  }
  if (!rows) return;
  const float vall = w.vref > 0.0f ? w.vref * (1.0f / KV8_VUNIT) : 0.0f;
#pragma unroll
  for (int i = 0; i < NT; i++) {
    const float z = rows_sum(w.z[i]), inv = kv8_inverse(z);
    const uint32_t row = row0 + i * 16 + n;
    if (row >= (uint64_t)k.e.nodes * a.grp) continue;
    const uint64_t part = ((uint64_t)k.slot * a.pg.kvheads + k.h) * a.rowsper + row - k.row0;
    if (k.chunks > 1 && g == 0) *(float2 *)(a.pmz + part * 2) = make_float2(w.m[i], ldexpf(z, -(int)w.up[i]));
    float *o = k.chunks > 1 ? a.pctx + part * HD
                            : a.out + (((size_t)k.b * a.tmax + w.node[i]) * a.heads + k.h * a.grp + row - w.node[i] * a.grp) * HD;
#pragma unroll
    for (int d = 0; d < D; d++) *(float4v *)(o + d * 16 + g * 4) = (w.o[i][d] * inv) * vall;
  }
}

// The chunks' parts of each output row, joined by their maxima and sums: SUBS
// groups of hd / 4 threads walk a row's chunks.  The sum of averages times weights is
// held in units of the weights' sum's power of two, no larger than the largest V.  A
// workgroup's rows are of one sequence.  4-6.5 us traced: eight groups where one
// each would leave the card empty and walk tens of chunks one after another.
template <int SUBS>
__global__ __launch_bounds__(256) void k_attn_q8_merge(Kv8Attn a, uint32_t hd, uint32_t blocks) {
  __shared__ float4v s_o[256];
  __shared__ float2 s_mz[256];
  const uint32_t per = hd / 4, t = threadIdx.x, b = blockIdx.x / blocks;
  const uint32_t r = blockIdx.x % blocks * (256 / per / SUBS) + t / (per * SUBS), sub = t / per % SUBS, d = t % per * 4;
  const Kv8Extent e = kv8_of(a, b);
  const uint2 f = a.pfirst[b];
  const uint32_t slot = f.x, chunks = f.y;
  if (!e.on || chunks < 2) return;  // (one: its workgroup has written the row)
  const uint32_t node = r / a.heads, head = r % a.heads;
  const bool on = node < e.nodes;
  const uint32_t h = kv8_quot(a.bygrp, head), row = node * a.grp + head - h * a.grp, group = row >> a.rowslog;
  const uint64_t p0 = ((uint64_t)(slot + group * chunks) * a.pg.kvheads + h) * a.rowsper + (row & (a.rowsper - 1));
  const uint64_t step = (uint64_t)a.pg.kvheads * a.rowsper;
  float m = KV8_FLOOR, z = 0.0f;
  float4v o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (on)
    for (uint32_t c = sub; c < chunks; c += SUBS) {
      const uint64_t p = p0 + c * step;
      const float2 x = *(const float2 *)(a.pmz + p * 2);
      const float4v y = *(const float4v *)(a.pctx + p * hd + d);
      const float mn = fmaxf(m, x.x);
      const float f = nlg_exp2(m - mn), wx = x.y * nlg_exp2(x.x - mn);
      const int e = __builtin_amdgcn_frexp_expf(z);
      m = mn;
      z = fmaf(z, f, wx);
      const int ne = __builtin_amdgcn_frexp_expf(z);
      o = o * ldexpf(f, e - ne) + y * ldexpf(wx, -ne);
    }
  if (SUBS > 1) {
    s_mz[t] = make_float2(m, z);
    s_o[t] = o;
    __syncthreads();
    if (sub) return;
    float mm = m;
#pragma unroll
    for (int i = 1; i < SUBS; i++) mm = fmaxf(mm, s_mz[t + i * per].x);
    const float f = nlg_exp2(m - mm);
    const int e = __builtin_amdgcn_frexp_expf(z);
    z = z * f;
#pragma unroll
    for (int i = 1; i < SUBS; i++) z = fmaf(s_mz[t + i * per].y, nlg_exp2(s_mz[t + i * per].x - mm), z);
    const int ne = __builtin_amdgcn_frexp_expf(z);
    o = o * ldexpf(f, e - ne);
#pragma unroll
    for (int i = 1; i < SUBS; i++) {
      const float2 x = s_mz[t + i * per];
      o = o + s_o[t + i * per] * ldexpf(nlg_exp2(x.x - mm), __builtin_amdgcn_frexp_expf(x.y) - ne);
    }
  }
  if (!on) return;
  *(float4v *)(a.out + (((size_t)b * a.tmax + node) * a.heads + head) * hd + d) =
      o * kv8_inverse(ldexpf(z, -__builtin_amdgcn_frexp_expf(z)));
}

// ------------------------------------------------------------------ commit

#define KV8_TREE 64  // most nodes of a masked tree, and of a committed path

struct CommitArgs {
  uint8_t *kpool, *vpool;
  const int32_t *base, *path, *accepted;  // [batch], [batch][tmax], [batch]
  Kv8Pages pg;
  uint32_t tmax;
};
// A workgroup moves the rows of one sequence, kv head and pool: all are read
// before the first is written.  A few kilobytes: the chain path -> block -> bytes
// -> store bounds it, 5 us for one sequence as for 64.
template <int HD>
__global__ __launch_bounds__(256) void k_commit_q8(CommitArgs a) {
  __shared__ uint32_t s_from[KV8_TREE], s_to[KV8_TREE];
  __shared__ uint8_t s_row[KV8_TREE][HD + 4];
  const uint32_t h = blockIdx.x >> 1, b = blockIdx.y;
  const bool isv = blockIdx.x & 1;
  const int32_t base = a.base[b], acc = a.accepted[b];
  if (base < 0 || acc <= 0) return;
  const uint32_t n = (uint32_t)acc < a.tmax ? (uint32_t)acc : a.tmax;
  const uint32_t i = threadIdx.x;
  if (i < n) {
    const int32_t p = a.path[(size_t)b * a.tmax + i];
    const uint32_t to = (uint32_t)base + i, from = (uint32_t)base + (uint32_t)p;
    const bool move = p >= 0 && (uint32_t)p < a.tmax && (uint32_t)p != i;
    uint32_t tf = move ? kv8_tile(a.pg, b, h, from / KV8_TILE) : KV8_NONE;
    const uint32_t tt = move ? kv8_tile(a.pg, b, h, to / KV8_TILE) : KV8_NONE;
    if (tt == KV8_NONE) tf = KV8_NONE;
    s_from[i] = tf;
    s_to[i] = tt;
  }
  __syncthreads();
  uint8_t *pool = isv ? a.vpool : a.kpool;
  for (uint32_t e = i; e < n * (HD + 4); e += 256) {
    const uint32_t r = e / (HD + 4), d = e % (HD + 4);
    if (s_from[r] == KV8_NONE) continue;
    const uint32_t at = ((uint32_t)base + (uint32_t)a.path[(size_t)b * a.tmax + r]) % KV8_TILE;
    const uint32_t off = d >= HD ? kv8_scale_byte(HD, at) + d - HD : isv ? kv8_v_byte(at, d) : kv8_k_byte(HD, at, d);
    s_row[r][d] = pool[(size_t)s_from[r] * kv8_tile_bytes(HD) + off];
  }
  __syncthreads();
  for (uint32_t e = i; e < n * (HD + 4); e += 256) {
    const uint32_t r = e / (HD + 4), d = e % (HD + 4);
    if (s_from[r] == KV8_NONE) continue;
    const uint32_t at = ((uint32_t)base + r) % KV8_TILE;
    const uint32_t off = d >= HD ? kv8_scale_byte(HD, at) + d - HD : isv ? kv8_v_byte(at, d) : kv8_k_byte(HD, at, d);
    pool[(size_t)s_to[r] * kv8_tile_bytes(HD) + off] = s_row[r][d];
  }
}

// ------------------------------------------------------------------ read-back

struct ReadArgs {
  const uint8_t *kpool, *vpool;
  const int32_t *seq, *slot;
  Kv8Pages pg;
  uint16_t *k, *v;  // [rows][kvheads][hd]
  uint64_t rows;
  uint32_t batch;
};
// Codes 2 i and 2 i + 1 of a word times their scale, rounded to fp16.  The
// products are f32 numbers: not folded with their rounding into one.
template <int FMT, int I>
__device__ __forceinline__ half2v kv8_value2(uint32_t w, float scale) {
  float x, y;
  if (FMT == NLG_KV_I8) {
    x = (float)(int8_t)(w >> 16 * I);
    y = (float)(int8_t)(w >> (16 * I + 8));
  } else {
    const half2v t = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, I != 0);
    x = (float)t[0];
    y = (float)t[1];
  }
  x = x * scale;
  y = y * scale;
  asm("" : "+v"(x), "+v"(y));
  const float2v f = {x, y};
  return __builtin_convertvector(f, half2v);
}
// Sixteen positions of two dimensions (held in 64-bit values: a choice between
// words of a struct would put it in memory).
struct Columns {
  uint64_t a0, a1, b0, b1;
};
// Byte `at` (the same for the wave) of sixteen.
__device__ __forceinline__ uint32_t kv8_pick(uint64_t lo, uint64_t hi, uint32_t at) {
  return (uint32_t)((at < 8 ? lo : hi) >> 8 * (at & 7)) & 0xffu;
}
// Rows that no cache will hold until they are read are stored past it (many rows
// only: 20,384 of 8 heads of 128 33 -> 26 us).
template <bool NT>
__device__ __forceinline__ void store16(void *p, uint4 v) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  const v4u t = {v.x, v.y, v.z, v.w};
  if (NT) __builtin_nontemporal_store(t, (v4u *)p);
  else *(v4u *)p = t;
}
// A wave reads N rows of one kv head: sixteen, or one where there are too few
// rows to fill the card.  K: HD / 8 lanes a row.  V: a lane holds the sixteen
// positions of two (HD 128) or one dimensions of a tile, and gives each of its
// rows that lie there theirs; of rows that follow each other in a sequence the
// first's and the last's tiles are all there are, and both are loaded ahead.
template <int HD, int FMT, int N>
__global__ __launch_bounds__(256) void k_read_q8(ReadArgs a) {
  constexpr int L = HD / 8, RP = 64 / L < N ? 64 / L : N, DV = HD / 64;
  const int lane = threadIdx.x & 63, m = lane % L;
  const uint64_t w = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t h = (uint32_t)(w % a.pg.kvheads);
  const uint64_t r0 = w / a.pg.kvheads * N;
  if (r0 >= a.rows) return;
  const int n = a.rows - r0 < N ? (int)(a.rows - r0) : N;
  uint32_t tile = KV8_NONE, at = 0;
  if (lane < n) {
    const int32_t slot = a.slot[r0 + lane];
    const uint32_t b = a.seq ? (uint32_t)a.seq[r0 + lane] : (uint32_t)(r0 + lane);
    if (slot >= 0 && b < a.batch) tile = kv8_tile(a.pg, b, h, (uint32_t)slot / KV8_TILE);
    at = (uint32_t)slot % KV8_TILE;
  }
  auto columns = [&](uint32_t from) {
    const uint8_t *t = a.vpool + (size_t)(from == KV8_NONE ? 0 : from) * kv8_tile_bytes(HD) + lane * DV * KV8_TILE;
    const uint4 x = *(const uint4 *)t, y = DV == 2 ? *(const uint4 *)(t + KV8_TILE) : x;
    return Columns{(uint64_t)x.y << 32 | x.x, (uint64_t)x.w << 32 | x.z, (uint64_t)y.y << 32 | y.x,
                   (uint64_t)y.w << 32 | y.z};
  };
  const uint32_t last = __builtin_amdgcn_readlane(tile, n - 1);
  uint32_t held = __builtin_amdgcn_readlane(tile, 0);
  Columns c = columns(held);
  const Columns cl = columns(last);
  // row r0 + lane's scale of V
  const float vscale =
      tile == KV8_NONE ? 0.0f : *(const float *)(a.vpool + (size_t)tile * kv8_tile_bytes(HD) + kv8_scale_byte(HD, at));
  uint2 k[N / RP];
  float ks[N / RP];
#pragma unroll
  for (int p = 0; p < N / RP; p++) {
    const int i = p * RP + lane / L;
    const uint32_t from = __shfl(tile, i), fa = __shfl(at, i);
    k[p] = make_uint2(0, 0);
    ks[p] = 0.0f;
    if (from != KV8_NONE) {
      const uint8_t *t = a.kpool + (size_t)from * kv8_tile_bytes(HD);
      k[p] = *(const uint2 *)(t + kv8_k_byte(HD, fa, m * 8));
      ks[p] = *(const float *)(t + kv8_scale_byte(HD, fa));
    }
  }
  for (int i = 0; i < n; i++) {
    const uint32_t from = __builtin_amdgcn_readlane(tile, i), fa = __builtin_amdgcn_readlane(at, i);
    if (from != held) {
      held = from;
      if (from == last) c = cl;
      else c = columns(from);
    }
    const float s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vscale), i));
    const uint64_t o = ((r0 + i) * a.pg.kvheads + h) * HD + lane * DV;
    uint32_t pair = kv8_pick(c.a0, c.a1, fa) | (DV == 2 ? kv8_pick(c.b0, c.b1, fa) << 8 : 0u);
    if (from == KV8_NONE) pair = 0;
    const half2v v = kv8_value2<FMT, 0>(pair, s);
    if (DV == 2) {
      if (N > 1) __builtin_nontemporal_store(__builtin_bit_cast(uint32_t, v), (uint32_t *)(a.v + o));
      else *(half2v *)(a.v + o) = v;
    } else {
      *(_Float16 *)(a.v + o) = v[0];
    }
  }
#pragma unroll
  for (int p = 0; p < N / RP; p++) {
    const int i = p * RP + lane / L;
    if (i >= n) continue;
    union {
      half2v h[4];
      uint4 u;
    } o;
    o.h[0] = kv8_value2<FMT, 0>(k[p].x, ks[p]);
    o.h[1] = kv8_value2<FMT, 1>(k[p].x, ks[p]);
    o.h[2] = kv8_value2<FMT, 0>(k[p].y, ks[p]);
    o.h[3] = kv8_value2<FMT, 1>(k[p].y, ks[p]);
    store16<(N > 1)>(a.k + ((r0 + i) * a.pg.kvheads + h) * HD + m * 8, o.u);
  }
}

// ------------------------------------------------------------------ host side

// What every entry point checks of the cache itself.
static int kv8_check(const char *what, const void *kpool, const void *vpool, const int32_t *table, uint32_t npool,
                     int fmt, uint32_t batch, uint32_t kvheads, uint32_t hd, uint32_t bs, uint32_t mbps, Kv8Pages &pg) {
  if (!kpool || !vpool || !table) return nlg_fail("%s: null pointer", what);
  if (((uintptr_t)kpool & 15) || ((uintptr_t)vpool & 15)) return nlg_fail("%s: pools must be 16-byte aligned", what);
  if ((uintptr_t)table & 3) return nlg_fail("%s: the block table must be 4-byte aligned", what);
  if (fmt != NLG_KV_I8 && fmt != NLG_KV_E4M3) return nlg_fail("%s: unknown cache format %d", what, fmt);
  if (hd != 64 && hd != 128) return nlg_fail("%s: head_dim %u (64 or 128)", what, hd);
  if (!kvheads) return nlg_fail("%s: kvheads must be nonzero", what);
  if (!bs || bs % KV8_TILE || !mbps || (uint64_t)bs * mbps > 0x7fffffffull)
    return nlg_fail("%s: block size %u (a multiple of %d), %u blocks a sequence (fewer than 2^31 positions)", what, bs,
                    KV8_TILE, mbps);
  if (!kv8_pool_bytes(npool, bs, kvheads, hd)) return nlg_fail("%s: bad pool of %u blocks", what, npool);
  pg.table = table; pg.npool = npool; pg.mbps = mbps; pg.bpt = kv8_div(bs / KV8_TILE);
  pg.kvheads = kvheads;
  return NLG_OK;
}
// Arrays of 32-bit numbers, those that may be null among them.
template <class... P>
static bool kv8_words(P... p) {
  return ((... | (uintptr_t)p) & 3) == 0;
}
// (after the checks of arguments: those need no device)
#define KV8_SCOPE(what)                                       \
  if (nlg_ensure_init()) return NLG_ERR;                      \
  DeviceScope scope_;                                         \
  if (!scope_.ok) return nlg_fail("%s: cannot select the library's device", what)

extern "C" size_t nlg_kv_q8_pool_bytes(uint32_t npool, uint32_t kvheads, uint32_t head_dim, uint32_t bs) {
  return (size_t)kv8_pool_bytes(npool, bs, kvheads, head_dim);
}

extern "C" int nlg_qk_norm_rope_append_paged_q8(const float *qkv, const float *qgain, const float *kgain, float eps,
                                                const float *rope_cos, const float *rope_sin, uint32_t trows,
                                                int rope_half, const int32_t *seq, const int32_t *slot,
                                                const int32_t *rpos, const int32_t *table, uint32_t npool, float *q,
                                                uint8_t *kpool, uint8_t *vpool, int fmt, uint32_t rows,
                                                uint32_t batch, uint32_t heads, uint32_t kvheads, uint32_t head_dim,
                                                uint32_t bs, uint32_t mbps, void *stream) {
  const char *what = "q8 append";
  if (!rows) return NLG_OK;
  AppendArgs a;
  if (kv8_check(what, kpool, vpool, table, npool, fmt, batch, kvheads, head_dim, bs, mbps, a.pg)) return NLG_ERR;
  if (!qkv || !rope_cos || !rope_sin || !slot || !q) return nlg_fail("%s: null pointer", what);
  if (!heads || !batch || !trows) return nlg_fail("%s: heads, batch and trows must be nonzero", what);
  if (((uintptr_t)qkv & 15) || ((uintptr_t)q & 15) || ((uintptr_t)rope_cos & 15) || ((uintptr_t)rope_sin & 15) ||
      ((uintptr_t)qgain & 15) || ((uintptr_t)kgain & 15))
    return nlg_fail("%s: qkv, q, gains and rotation tables must be 16-byte aligned", what);
  if (!kv8_words(seq, slot, rpos)) return nlg_fail("%s: seq, slot and rpos must be 4-byte aligned", what);
  if (!seq && rows > batch) return nlg_fail("%s: %u rows without a sequence each, batch %u", what, rows, batch);
  const uint64_t per = (uint64_t)heads + 2ull * kvheads;
  const uint64_t qb = ((uint64_t)rows * (heads + (uint64_t)kvheads) * (head_dim / 8) + 255) / 256;
  const uint64_t vb = (((uint64_t)rows + 15) / 16 * kvheads + 3) / 4;
  if (per > 0xffffffffull || !nlg_fits(qb + vb, 256))
    return nlg_fail("%s: too many rows and heads (%u x %llu) for one launch", what, rows, (unsigned long long)per);
  // (head rows are read by some workgroups while others store queries)
  const uintptr_t x0 = (uintptr_t)qkv, q0 = (uintptr_t)q;
  if (x0 < q0 + (uint64_t)rows * heads * head_dim * 4 && q0 < x0 + (uint64_t)rows * per * head_dim * 4)
    return nlg_fail("%s: q overlaps qkv", what);
  KV8_SCOPE(what);
  a.qkv = qkv; a.qgain = qgain; a.kgain = kgain; a.co = rope_cos; a.si = rope_sin;
  a.seq = seq; a.slot = slot; a.rpos = rpos; a.q = q; a.kpool = kpool; a.vpool = vpool;
  a.eps = eps; a.rows = rows; a.batch = batch; a.heads = heads; a.trows = trows; a.qblocks = (uint32_t)qb;
  // queries that outgrow the L2 caches are not kept in them (4,731 rows of 32 heads of 128, with
  // the codes read back: 62 -> 57 us)
  a.past = (uint64_t)rows * heads * head_dim * 4 > (32u << 20);
  const dim3 grid((uint32_t)(qb + vb)), blk(256);
  hipStream_t st = nlg_stream(stream);
#define GO(HD, F)                                                                          \
  do {                                                                                     \
    if (rope_half) hipLaunchKernelGGL((k_append_q8<HD, F, true>), grid, blk, 0, st, a);    \
    else hipLaunchKernelGGL((k_append_q8<HD, F, false>), grid, blk, 0, st, a);             \
  } while (0)
  if (head_dim == 128) {
    if (fmt == NLG_KV_I8) GO(128, NLG_KV_I8); else GO(128, NLG_KV_E4M3);
  } else {
    if (fmt == NLG_KV_I8) GO(64, NLG_KV_I8); else GO(64, NLG_KV_E4M3);
  }
#undef GO
  NLG_LAUNCHED("q8 append");
  return NLG_OK;
}

// The partials' bytes: contexts, (maximum, sum) pairs, where each sequence's are; 0 where one chunk needs none.
static uint64_t kv8_partials(const Kv8Split &s, uint32_t batch, uint32_t kvheads, uint32_t hd) {
  return s.one ? 0 : s.slots * kvheads * s.rowsper * (hd + 2) * 4 + 8ull * batch;
}
// Sizes an attention call can have at all (0: none).
static uint64_t kv8_rows(uint32_t tmax, uint32_t heads, uint32_t kvheads) {
  if (!kvheads || !heads || heads % kvheads || !tmax) return 0;
  const uint64_t rows = (uint64_t)tmax * (heads / kvheads);
  return rows <= 0x7fffffffull ? rows : 0;
}

extern "C" size_t nlg_tree_attn_paged_q8_workspace(uint32_t batch, uint32_t tmax, uint32_t heads, uint32_t kvheads,
                                                   uint32_t head_dim, uint32_t bs, uint32_t mbps) {
  const uint64_t rows = kv8_rows(tmax, heads, kvheads);
  if (!batch || !rows || !bs || bs % KV8_TILE || !mbps || (uint64_t)bs * mbps > 0x7fffffffull ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  return (size_t)kv8_partials(kv8_split(batch, (uint32_t)rows, kvheads, head_dim, (uint64_t)bs * mbps), batch, kvheads, head_dim);
}
extern "C" size_t nlg_decode_attn_paged_q8_workspace(uint32_t batch, uint32_t heads, uint32_t kvheads,
                                                     uint32_t head_dim, uint32_t bs, uint32_t mbps) {
  return nlg_tree_attn_paged_q8_workspace(batch, 1, heads, kvheads, head_dim, bs, mbps);
}

static int kv8_attend(const char *what, bool tree, const float *q, const uint8_t *kpool, const uint8_t *vpool, int fmt,
                      const int32_t *base, const int32_t *nodes, const uint64_t *mask, const int32_t *table,
                      uint32_t npool, float *out, uint32_t batch, uint32_t tmax, uint32_t heads, uint32_t kvheads,
                      uint32_t hd, uint32_t bs, uint32_t mbps, void *workspace, size_t workspace_bytes, void *stream) {
  if (!batch || !tmax) return NLG_OK;
  Kv8Attn a;
  if (kv8_check(what, kpool, vpool, table, npool, fmt, batch, kvheads, hd, bs, mbps, a.pg)) return NLG_ERR;
  if (!q || !base || !out) return nlg_fail("%s: null pointer", what);
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15)) return nlg_fail("%s: q and out must be 16-byte aligned", what);
  if (!kv8_words(base, nodes))
    return nlg_fail("%s: %s must be 4-byte aligned", what, tree ? "base and nodes" : "lens");
  const uint64_t rows = kv8_rows(tmax, heads, kvheads);
  if (!rows) return nlg_fail("%s: %u heads over %u kv heads, %u queries", what, heads, kvheads, tmax);
  if (mask && tmax > KV8_TREE) return nlg_fail("%s: %u nodes under a mask (at most %d)", what, tmax, KV8_TREE);
  if (mask && ((uintptr_t)mask & 7)) return nlg_fail("%s: the masks must be 8-byte aligned", what);
  const Kv8Split s = kv8_split(batch, (uint32_t)rows, kvheads, hd, (uint64_t)bs * mbps);
  const uint64_t need = kv8_partials(s, batch, kvheads, hd);
  // joining: eight groups of threads a row while its rows would not fill the card with one
  const uint64_t orows = (uint64_t)tmax * heads;
  const bool subs = orows * batch * (hd / 4) < 65536;
  const uint64_t oper = 256 / (hd / 4) / (subs ? 8 : 1), oblocks = (orows + oper - 1) / oper;
  if (!nlg_fits(s.blocks, 512) || !nlg_fits(oblocks * batch, 256) || orows > 0xffffffffull)
    return nlg_fail("%s: too many queries for one launch", what);
  if (need) {
    if (!workspace || workspace_bytes < need)
      return nlg_fail("%s: workspace holds %zu bytes, needs %llu", what, workspace ? workspace_bytes : 0,
                      (unsigned long long)need);
    if ((uintptr_t)workspace & 15) return nlg_fail("%s: the workspace must be 16-byte aligned", what);
  }
  KV8_SCOPE(what);
  a.q = q; a.kpool = kpool; a.vpool = vpool; a.base = base; a.nodes = nodes; a.mask = mask; a.out = out;
  a.batch = batch; a.tmax = tmax; a.heads = heads; a.grp = heads / kvheads;
  a.rowsper = s.rowsper; a.rowslog = s.rowslog; a.groups = s.groups; a.want = s.want;
  a.least = s.least; a.unit = s.unit;
  a.bygroups = kv8_div(s.groups); a.bykvheads = kv8_div(kvheads); a.bygrp = kv8_div(a.grp);
  a.tree = tree; a.one = s.one;
  a.pctx = (float *)workspace;
  a.pmz = need ? a.pctx + s.slots * kvheads * s.rowsper * hd : nullptr;
  a.pfirst = need ? (uint2 *)(a.pmz + s.slots * kvheads * s.rowsper * 2) : nullptr;
  a.coef = NLG_LOG2E / sqrtf((float)hd);
  const dim3 grid((uint32_t)s.blocks);
  hipStream_t st = nlg_stream(stream);
  // K and V of more than the 256 MB MALL are gone from it before the next call
  // reads them (eight sequences at 24,000-32,768 of 8 heads of 128, 480 MB: 94 ->
  // 88 us).  By the table's capacity: the lengths are on the device.  Where they are
  // far below it that matters little (32 at up to 4,096 of 5, 87 MB: kept and past
  // 24.9 and 25.6 us replayed alone, 25.4 and 27.1 over three layers' pools, 28.7 and
  // 28.5 over eight; at up to 600 13.8 and 14.2, 15.5 and 15.2 over forty)
  const bool past = (uint64_t)batch * mbps * bs * kvheads * 2 * (hd + 4) > (256u << 20);
#define GO(HD, F)                                                                                                 \
  do {                                                                                                            \
    if (s.rowsper == 16 && s.one) hipLaunchKernelGGL((k_attn_q8<HD, F, 1, 8, false>), grid, dim3(512), 0, st, a); \
    else if (s.rowsper == 16 && past) hipLaunchKernelGGL((k_attn_q8<HD, F, 1, 4, true>), grid, dim3(256), 0, st, a); \
    else if (s.rowsper == 16) hipLaunchKernelGGL((k_attn_q8<HD, F, 1, 4, false>), grid, dim3(256), 0, st, a);     \
    else if (s.rowsper == 32) hipLaunchKernelGGL((k_attn_q8<64, F, 2, 4, false>), grid, dim3(256), 0, st, a);     \
    else if (s.rowsper == 64) hipLaunchKernelGGL((k_attn_wide_q8<HD, F, 1>), grid, dim3(256), 0, st, a);          \
    else hipLaunchKernelGGL((k_attn_wide_q8<64, F, 2>), grid, dim3(256), 0, st, a);                               \
  } while (0)
  if (hd == 128) {
    if (fmt == NLG_KV_I8) GO(128, NLG_KV_I8); else GO(128, NLG_KV_E4M3);
  } else {
    if (fmt == NLG_KV_I8) GO(64, NLG_KV_I8); else GO(64, NLG_KV_E4M3);
  }
#undef GO
  NLG_LAUNCHED(what);
  if (need) {
    const dim3 mg((uint32_t)(oblocks * batch));
    const uint32_t ob = (uint32_t)oblocks;
    if (subs) hipLaunchKernelGGL(k_attn_q8_merge<8>, mg, dim3(256), 0, st, a, hd, ob);
    else hipLaunchKernelGGL(k_attn_q8_merge<1>, mg, dim3(256), 0, st, a, hd, ob);
    NLG_LAUNCHED(what);
  }
  return NLG_OK;
}

extern "C" int nlg_decode_attn_paged_q8(const float *q, const uint8_t *kpool, const uint8_t *vpool, int fmt,
                                        const int32_t *lens, const int32_t *table, uint32_t npool, float *out,
                                        uint32_t batch, uint32_t heads, uint32_t kvheads, uint32_t head_dim,
                                        uint32_t bs, uint32_t mbps, void *workspace, size_t workspace_bytes,
                                        void *stream) {
  return kv8_attend("q8 decode attn", false, q, kpool, vpool, fmt, lens, nullptr, nullptr, table, npool, out, batch, 1,
                    heads, kvheads, head_dim, bs, mbps, workspace, workspace_bytes, stream);
}

extern "C" int nlg_tree_attn_paged_q8(const float *q, const uint8_t *kpool, const uint8_t *vpool, int fmt,
                                      const int32_t *base, const int32_t *nodes, const uint64_t *mask,
                                      const int32_t *table, uint32_t npool, float *out, uint32_t batch, uint32_t tmax,
                                      uint32_t heads, uint32_t kvheads, uint32_t head_dim, uint32_t bs, uint32_t mbps,
                                      void *workspace, size_t workspace_bytes, void *stream) {
  return kv8_attend("q8 tree attn", true, q, kpool, vpool, fmt, base, nodes, mask, table, npool, out, batch, tmax,
                    heads, kvheads, head_dim, bs, mbps, workspace, workspace_bytes, stream);
}

extern "C" int nlg_tree_commit_paged_q8(uint8_t *kpool, uint8_t *vpool, const int32_t *base, const int32_t *path,
                                        const int32_t *accepted, const int32_t *table, uint32_t npool, uint32_t batch,
                                        uint32_t tmax, uint32_t kvheads, uint32_t head_dim, uint32_t bs, uint32_t mbps,
                                        void *stream) {
  const char *what = "q8 tree commit";
  if (!batch || !tmax) return NLG_OK;
  CommitArgs a;
  if (kv8_check(what, kpool, vpool, table, npool, NLG_KV_I8, batch, kvheads, head_dim, bs, mbps, a.pg)) return NLG_ERR;
  if (!base || !path || !accepted) return nlg_fail("%s: null pointer", what);
  if (!kv8_words(base, path, accepted)) return nlg_fail("%s: base, path and accepted must be 4-byte aligned", what);
  if (tmax > KV8_TREE) return nlg_fail("%s: paths of %u nodes (at most %d)", what, tmax, KV8_TREE);
  if (batch > 65535 || !nlg_fits(2ull * kvheads, 256)) return nlg_fail("%s: batch %u x %u kv heads", what, batch, kvheads);
  KV8_SCOPE(what);
  a.kpool = kpool; a.vpool = vpool; a.base = base; a.path = path; a.accepted = accepted; a.tmax = tmax;
  const dim3 grid(2 * kvheads, batch), blk(256);
  if (head_dim == 128) hipLaunchKernelGGL(k_commit_q8<128>, grid, blk, 0, nlg_stream(stream), a);
  else hipLaunchKernelGGL(k_commit_q8<64>, grid, blk, 0, nlg_stream(stream), a);
  NLG_LAUNCHED(what);
  return NLG_OK;
}

extern "C" int nlg_cache_read_paged_q8(const uint8_t *kpool, const uint8_t *vpool, int fmt, const int32_t *seq,
                                       const int32_t *slot, const int32_t *table, uint32_t npool, uint16_t *k,
                                       uint16_t *v, uint32_t rows, uint32_t batch, uint32_t kvheads, uint32_t head_dim,
                                       uint32_t bs, uint32_t mbps, void *stream) {
  const char *what = "q8 read";
  if (!rows) return NLG_OK;
  ReadArgs a;
  if (kv8_check(what, kpool, vpool, table, npool, fmt, batch, kvheads, head_dim, bs, mbps, a.pg)) return NLG_ERR;
  if (!slot || !k || !v) return nlg_fail("%s: null pointer", what);
  if (!batch) return nlg_fail("%s: batch must be nonzero", what);
  if (((uintptr_t)k & 15) || ((uintptr_t)v & 15)) return nlg_fail("%s: k and v must be 16-byte aligned", what);
  if (!kv8_words(seq, slot)) return nlg_fail("%s: seq and slot must be 4-byte aligned", what);
  if (!seq && rows > batch) return nlg_fail("%s: %u rows without a sequence each, batch %u", what, rows, batch);
  const bool few = (uint64_t)rows * kvheads < 16384;  // (2,000 rows of 8 heads of 128: 7.9 us, 8.1 in sixteens; 480: 4.1, 6.7; 16,000: 48, 24)
  const uint64_t per = few ? 1 : 16, blocks = (((uint64_t)rows + per - 1) / per * kvheads + 3) / 4;
  if (!nlg_fits(blocks, 256)) return nlg_fail("%s: too many rows for one launch", what);
  KV8_SCOPE(what);
  a.kpool = kpool; a.vpool = vpool; a.seq = seq; a.slot = slot; a.k = k; a.v = v; a.rows = rows; a.batch = batch;
  const dim3 grid((uint32_t)blocks), blk(256);
  hipStream_t st = nlg_stream(stream);
#define GO(HD, F)                                                                     \
  do {                                                                                \
    if (few) hipLaunchKernelGGL((k_read_q8<HD, F, 1>), grid, blk, 0, st, a);          \
    else hipLaunchKernelGGL((k_read_q8<HD, F, 16>), grid, blk, 0, st, a);             \
  } while (0)
  if (head_dim == 128) {
    if (fmt == NLG_KV_I8) GO(128, NLG_KV_I8); else GO(128, NLG_KV_E4M3);
  } else {
    if (fmt == NLG_KV_I8) GO(64, NLG_KV_I8); else GO(64, NLG_KV_E4M3);
  }
#undef GO
  NLG_LAUNCHED(what);
  return NLG_OK;
}
