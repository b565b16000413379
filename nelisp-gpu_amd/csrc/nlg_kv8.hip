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

// All in 64 bits: a code then depends on the inputs alone and not on the order
// of a sum, so a prefix cached twice holds the same bytes.  They cost little
// only where lanes share a row's root and quotients: a head row is on HD / 8
// lanes, eight values (four rotation pairs) each.  The first qblocks workgroups
// take the q and k heads; the others V, a wave sixteen rows of one head, whose
// codes pass through LDS: a position's bytes of a tile lie sixteen apart, and a
// store then runs over 64 dimensions (8 lines) instead of one byte a line.
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
    *(float4 *)(q + d0) = make_float4((float)y[0], (float)y[1], (float)y[2], (float)y[3]);
    *(float4 *)(q + d1) = make_float4((float)y[4], (float)y[5], (float)y[6], (float)y[7]);
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
  float *out, *pctx, *pmz;  // partials: [batch][kvheads][nchunk][rows][hd], [..][rows][2]
  uint32_t batch, tmax, heads, grp, rows;  // rows = tmax * grp
  uint32_t groups, chunk, nchunk;
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
  union {
    half8v v;
    half2v p[4];
  } a, b;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2v t = {w[2 * i], w[2 * i + 1]};
    a.p[i] = __builtin_convertvector(t, half2v);
    const float2v r = {fmaf((float)a.p[i][0], -1.0f, t[0]), fmaf((float)a.p[i][1], -1.0f, t[1])};
    b.p[i] = __builtin_convertvector(r, half2v);
  }
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
__device__ __forceinline__ float rows_max(float v) {  // over lanes 16, 32 and 48 apart
  float2 r = nlg_pair_f32<16>(v);
  v = fmaxf(r.x, r.y);
  r = nlg_pair_f32<32>(v);
  return fmaxf(r.x, r.y);
}
__device__ __forceinline__ float rows_sum(float v) {
  float2 r = nlg_pair_f32<16>(v);
  v = r.x + r.y;
  r = nlg_pair_f32<32>(v);
  return r.x + r.y;
}

// A wave's running state over NT tiles of sixteen query rows.  A lane holds the
// query row n = lane & 15 of each tile, and of its scores the sixteen positions
// of the step's tile g = lane >> 4.
template <int HD, int NT>
struct WaveState {
  half8v qh[NT][HD / 32], ql[NT][HD / 32];
  float rs[NT];            // what the row's q was divided by (a power of two)
  float m[NT], z[NT];      // running maximum; this lane's part of the sum
  float4v o[NT][HD / 16];  // out[dim 16 i + 4 g + r][query n], times 2^15 / vref
  float vref;              // a power of two no V scale so far exceeds, or 0
};

// One step: 64 positions, tile `tk` holding this lane's K row (4 positions of
// each of the four tiles a time), tile `tv` its V columns and both scales.
// GEN: some of the positions are masked, absent or past the end; bits[i]: which
// of this lane's sixteen the query row of tile i attends; left: how many of
// them exist.
template <int HD, int FMT, int NT, bool GEN>
__device__ __forceinline__ void kv8_step(const Kv8Attn &a, WaveState<HD, NT> &w, uint32_t tk, uint32_t tv,
                                         const uint32_t *bits, int left, int lane) {
  constexpr int C = HD / 64, D = HD / 16;
  const int g = lane >> 4, n = lane & 15;
  uint4 kr[4][C], vr[D];
  float ks, vs;
  {
    const bool hk = !GEN || tk != KV8_NONE, hv = !GEN || tv != KV8_NONE;
    const uint8_t *kp = a.kpool + (size_t)(hk ? tk : 0) * kv8_tile_bytes(HD) + (lane & 3) * HD + g * 16;
    const size_t vt = (size_t)(hv ? tv : 0) * kv8_tile_bytes(HD);
    const uint8_t *vp = a.vpool + vt;
    ks = *(const float *)(a.kpool + vt + kv8_scale_byte(HD, n));
    vs = *(const float *)(vp + kv8_scale_byte(HD, n));
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int c = 0; c < C; c++) kr[t][c] = *(const uint4 *)(kp + t * 4 * HD + c * 64);
#pragma unroll
    for (int i = 0; i < D; i++) vr[i] = *(const uint4 *)(vp + i * 256 + n * 16);
    if (GEN) {
      // absent tiles read as zero rows; what lies past the end is not used
      if (!hk)
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
          for (int c = 0; c < C; c++) kr[t][c] = make_uint4(0, 0, 0, 0);
      uint32_t keep[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int k = left - 4 * i;
        keep[i] = !hv || k <= 0 ? 0u : k >= 4 ? 0xffffffffu : (1u << (8 * k)) - 1;
      }
#pragma unroll
      for (int i = 0; i < D; i++) {
        vr[i].x &= keep[0]; vr[i].y &= keep[1]; vr[i].z &= keep[2]; vr[i].w &= keep[3];
      }
      if (!hv || n >= left) ks = vs = 0.0f;
    }
  }
  // V scales in units of vref / 2^15: the probabilities times them, as halves,
  // then use the type's whole range
  float vtop = fabsf(vs);
  vtop = vtop <= 3.4028234663852886e38f ? vtop : 0.0f;
  vtop = nlg_wave_max_f32(vtop);
  float vresc = 1.0f;
  if (vtop > w.vref) {  // the same in every lane
    const int e = __builtin_amdgcn_frexp_expf(vtop);
    const float nv = ldexpf(1.0f, e < -100 ? -100 : e);
    vresc = w.vref / nv;
    w.vref = nv;
  }
  vs = w.vref > 0.0f ? vs * (32768.0f / w.vref) : vs;
#pragma unroll
  for (int i = 0; i < NT; i++) {
    float s[16];
    float4v acc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      acc[t] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < C; c++) {
        const half8v k0 = kv8_half8<FMT>(kr[t][c].x, kr[t][c].y), k1 = kv8_half8<FMT>(kr[t][c].z, kr[t][c].w);
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, w.ql[i][2 * c], acc[t], 0, 0, 0);
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, w.ql[i][2 * c + 1], acc[t], 0, 0, 0);
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, w.qh[i][2 * c], acc[t], 0, 0, 0);
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, w.qh[i][2 * c + 1], acc[t], 0, 0, 0);
      }
    }
    each<16>([&](auto J) {
      constexpr int j = decltype(J)::value;
      s[j] = acc[j >> 2][j & 3] * row_lane<j>(ks);
      if (GEN) s[j] = bits[i] >> j & 1 ? s[j] : -INFINITY;
    });
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 16; j++) top = fmaxf(top, s[j]);
    top = rows_max(top) * w.rs[i];
    const float mn = fmaxf(w.m[i], top);
    const float ms = mn == -INFINITY ? 0.0f : mn;
    const float al = nlg_exp2(w.m[i] - ms);
    w.m[i] = mn;
    float zz = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; j++) {
      s[j] = nlg_exp2(fmaf(s[j], w.rs[i], -ms));
      zz = zz + s[j];
    }
    w.z[i] = fmaf(w.z[i], al, zz);
    const float sc = al * vresc;
    if (__any(sc != 1.0f)) {
#pragma unroll
      for (int d = 0; d < D; d++) w.o[i][d] = w.o[i][d] * sc;
    }
    each<16>([&](auto J) {
      constexpr int j = decltype(J)::value;
      s[j] = s[j] * row_lane<j>(vs);
      if (GEN) s[j] = bits[i] >> j & 1 ? s[j] : 0.0f;
    });
    half8v ph[2], pl[2];
    split8(s, ph[0], pl[0]);
    split8(s + 8, ph[1], pl[1]);
#pragma unroll
    for (int d = 0; d < D; d++) {
      const half8v v0 = kv8_half8<FMT>(vr[d].x, vr[d].y), v1 = kv8_half8<FMT>(vr[d].z, vr[d].w);
      w.o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], w.o[i][d], 0, 0, 0);
      w.o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1], w.o[i][d], 0, 0, 0);
      w.o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], w.o[i][d], 0, 0, 0);
      w.o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1], w.o[i][d], 0, 0, 0);
    }
  }
}

// The positions of sequence b.
template <bool TREE>
__device__ __forceinline__ Kv8Extent kv8_of(const Kv8Attn &a, uint32_t b) {
  return kv8_extent(TREE, a.base[b], TREE && a.nodes ? a.nodes[b] : (int32_t)a.tmax, a.tmax,
                    a.pg.mbps * a.pg.bpt * KV8_TILE);
}

template <int HD, int FMT, int NT, bool TREE>
__global__ __launch_bounds__(64 * KV8_WAVES) void k_attn_q8(Kv8Attn a) {
  constexpr int C = HD / 64, D = HD / 16;
  __shared__ float4v s_o[KV8_WAVES][D][64];
  __shared__ float s_m[KV8_WAVES][16], s_z[KV8_WAVES][16];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  uint32_t id = blockIdx.x;
  const uint32_t chunk = id % a.nchunk;
  id /= a.nchunk;
  const uint32_t grp = id % a.groups;
  id /= a.groups;
  const uint32_t h = id % a.pg.kvheads, b = id / a.pg.kvheads;
  const Kv8Extent e = kv8_of<TREE>(a, b);
  if (!e.on) return;
  const uint32_t row0 = grp * (NT * 16);
  if (row0 >= (uint64_t)e.nodes * a.grp) return;
  const uint32_t c0 = chunk * a.chunk;
  if (c0 >= e.end && chunk) return;
  const bool masked = TREE && a.mask;
  // a causal group of rows ends at its last node
  const uint32_t stop = TREE && !masked ? kv8_stop(e, (row0 + NT * 16 - 1) / a.grp) : e.end;
  const uint32_t c1 = kv8_chunk_end(c0, stop, a.chunk);

  WaveState<HD, NT> w;
  uint32_t node[NT];
  uint64_t word[NT];
#pragma unroll
  for (int i = 0; i < NT; i++) {
    const uint32_t row = row0 + i * 16 + n;
    node[i] = row / a.grp;
    const bool on = node[i] < e.nodes;
    const float *q = a.q + ((size_t)b * a.tmax + (on ? node[i] : 0)) * a.heads * HD +
                     (size_t)(h * a.grp + (on ? row % a.grp : 0)) * HD + g * 16;
    word[i] = masked && on ? kv8_word(a.mask[(size_t)b * a.tmax + node[i]], e.nodes) : 0;
    float x[HD / 4], top = 0.0f;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float4 t = *(const float4 *)(q + c * 64 + k * 4);
        float *y = x + c * 16 + k * 4;
        y[0] = t.x; y[1] = t.y; y[2] = t.z; y[3] = t.w;
      }
#pragma unroll
    for (int k = 0; k < HD / 4; k++) {
      x[k] = on ? x[k] * a.coef : 0.0f;
      top = fmaxf(top, fabsf(x[k]));
    }
    top = rows_max(top);
    const int ex = top > 0.0f && top <= 3.4028234663852886e38f ? __builtin_amdgcn_frexp_expf(top) : 0;
    w.rs[i] = ldexpf(1.0f, ex);
#pragma unroll
    for (int k = 0; k < HD / 4; k++) x[k] = ldexpf(x[k], -ex);
#pragma unroll
    for (int c = 0; c < C; c++) {
      split8(x + c * 16, w.qh[i][2 * c], w.ql[i][2 * c]);
      split8(x + c * 16 + 8, w.qh[i][2 * c + 1], w.ql[i][2 * c + 1]);
    }
    w.m[i] = -INFINITY;
    w.z[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < D; d++) w.o[i][d] = {0.0f, 0.0f, 0.0f, 0.0f};
  }
  w.vref = 0.0f;

  for (uint32_t p0 = c0; p0 < c1; p0 += 64 * KV8_TILE) {
    // the tiles of the next 1,024 positions, one a lane
    const uint32_t mine = p0 + lane * KV8_TILE;
    const uint32_t tid = mine < c1 ? kv8_tile(a.pg, b, h, mine / KV8_TILE) : KV8_NONE;
    const uint32_t p1 = c1 - p0 < 64 * KV8_TILE ? c1 : p0 + 64 * KV8_TILE;
    for (uint32_t p = p0 + wv * KV8_STEP; p < p1; p += KV8_WAVES * KV8_STEP) {
      const int t0 = (int)(p - p0) / KV8_TILE;
      const uint32_t tv = __shfl(tid, t0 + g), tk = __shfl(tid, t0 + (n >> 2));
      const bool gen = p + KV8_STEP > (e.base < stop ? e.base : stop) || __any(tv == KV8_NONE);
      if (gen) {
        uint32_t bits[NT];
        const uint32_t q0 = p + g * KV8_TILE;  // this lane's first position
        const int left = kv8_left(e, q0);
#pragma unroll
        for (int i = 0; i < NT; i++)
          bits[i] = TREE ? kv8_bits(e, masked, node[i], word[i], q0) : (1u << left) - 1;
        kv8_step<HD, FMT, NT, true>(a, w, tk, tv, bits, left, lane);
      } else {
        kv8_step<HD, FMT, NT, false>(a, w, tk, tv, nullptr, 16, lane);
      }
    }
  }

  // the waves' parts meet, one tile of rows at a time
  const float vs = w.vref > 0.0f ? w.vref * (1.0f / 32768.0f) : 0.0f;
#pragma unroll
  for (int i = 0; i < NT; i++) {
    if (i) __syncthreads();
    const float z = rows_sum(w.z[i]);
    if (g == 0) {
      s_m[wv][n] = w.m[i];
      s_z[wv][n] = z;
    }
#pragma unroll
    for (int d = 0; d < D; d++) s_o[wv][d][lane] = w.o[i][d] * vs;
    __syncthreads();
    float mm = s_m[0][n];
#pragma unroll
    for (int k = 1; k < KV8_WAVES; k++) mm = fmaxf(mm, s_m[k][n]);
    const float ms = mm == -INFINITY ? 0.0f : mm;
    float f[KV8_WAVES], zz = 0.0f;
#pragma unroll
    for (int k = 0; k < KV8_WAVES; k++) {
      f[k] = nlg_exp2(s_m[k][n] - ms);
      zz = fmaf(s_z[k][n], f[k], zz);
    }
    const uint32_t row = row0 + i * 16 + n;
    if (row < (uint64_t)e.nodes * a.grp) {
      const uint64_t part = (((uint64_t)b * a.pg.kvheads + h) * a.nchunk + chunk) * a.rows + row;
      if (a.nchunk > 1 && wv == 0 && g == 0) *(float2 *)(a.pmz + part * 2) = make_float2(mm, zz);
      const float inv = a.nchunk > 1 ? 1.0f : zz > 0.0f || zz != zz ? 1.0f / zz : 0.0f;
      float *o = a.nchunk > 1 ? a.pctx + part * HD
                              : a.out + (((size_t)b * a.tmax + row / a.grp) * a.heads + h * a.grp + row % a.grp) * HD;
  #pragma unroll
      for (int d = wv; d < D; d += KV8_WAVES) {
        float4v t = s_o[0][d][lane] * f[0];
  #pragma unroll
        for (int k = 1; k < KV8_WAVES; k++) t = t + s_o[k][d][lane] * f[k];
        *(float4v *)(o + d * 16 + g * 4) = t * inv;
      }
    }
  }
}

// The chunks' parts of each output row, joined.
template <bool TREE>
__global__ __launch_bounds__(256) void k_attn_q8_merge(Kv8Attn a, uint32_t hd, uint64_t total) {
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const uint32_t per = hd / 4, d = (uint32_t)(i % per) * 4;
  const uint64_t r = i / per;
  const uint32_t head = (uint32_t)(r % a.heads);
  const uint64_t bn = r / a.heads;
  const uint32_t node = (uint32_t)(bn % a.tmax), b = (uint32_t)(bn / a.tmax);
  const Kv8Extent e = kv8_of<TREE>(a, b);
  if (!e.on || node >= e.nodes) return;
  uint32_t live = (uint32_t)(((uint64_t)e.end + a.chunk - 1) / a.chunk);
  live = live ? live : 1;
  const uint32_t h = head / a.grp, row = node * a.grp + head % a.grp;
  const uint64_t p0 = ((uint64_t)b * a.pg.kvheads + h) * a.nchunk * a.rows + row;
  const float2 *mz = (const float2 *)a.pmz;
  float mm = -INFINITY;
  for (uint32_t c = 0; c < live; c++) mm = fmaxf(mm, mz[p0 + (uint64_t)c * a.rows].x);
  const float ms = mm == -INFINITY ? 0.0f : mm;
  float z = 0.0f;
  float4v o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t c = 0; c < live; c++) {
    const uint64_t p = p0 + (uint64_t)c * a.rows;
    const float2 t = mz[p];
    const float f = nlg_exp2(t.x - ms);
    z = fmaf(t.y, f, z);
    o = o + *(const float4v *)(a.pctx + p * hd + d) * f;
  }
  const float inv = z > 0.0f || z != z ? 1.0f / z : 0.0f;
  *(float4v *)(a.out + r * hd + d) = o * inv;
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
// before the first is written.
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
// A wave reads N rows of one kv head: sixteen, or four where there are too few
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
    if (DV == 2) *(half2v *)(a.v + o) = v;
    else *(_Float16 *)(a.v + o) = v[0];
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
    *(uint4 *)(a.k + ((r0 + i) * a.pg.kvheads + h) * HD + m * 8) = o.u;
  }
}

// ------------------------------------------------------------------ host side

// What every entry point checks of the cache itself.
static int kv8_check(const char *what, const void *kpool, const void *vpool, const int32_t *table, uint32_t npool,
                     int fmt, uint32_t batch, uint32_t kvheads, uint32_t hd, uint32_t bs, uint32_t mbps, Kv8Pages &pg) {
  if (!kpool || !vpool || !table) return nlg_fail("%s: null pointer", what);
  if (((uintptr_t)kpool & 15) || ((uintptr_t)vpool & 15)) return nlg_fail("%s: pools must be 16-byte aligned", what);
  if (((uintptr_t)table & 3)) return nlg_fail("%s: the block table must be 4-byte aligned", what);
  if (fmt != NLG_KV_I8 && fmt != NLG_KV_E4M3) return nlg_fail("%s: unknown cache format %d", what, fmt);
  if (hd != 64 && hd != 128) return nlg_fail("%s: head_dim %u (64 or 128)", what, hd);
  if (!kvheads) return nlg_fail("%s: kvheads must be nonzero", what);
  if (!bs || bs % KV8_TILE || !mbps || (uint64_t)bs * mbps > 0x7fffffffull)
    return nlg_fail("%s: block size %u (a multiple of %d), %u blocks a sequence (fewer than 2^31 positions)", what, bs,
                    KV8_TILE, mbps);
  if (!kv8_pool_bytes(npool, bs, kvheads, hd)) return nlg_fail("%s: bad pool of %u blocks", what, npool);
  pg.table = table; pg.npool = npool; pg.mbps = mbps; pg.bpt = bs / KV8_TILE; pg.kvheads = kvheads;
  return NLG_OK;
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
  if (!seq && rows > batch) return nlg_fail("%s: %u rows without a sequence each, batch %u", what, rows, batch);
  const uint64_t per = (uint64_t)heads + 2ull * kvheads;
  const uint64_t qb = ((uint64_t)rows * (heads + (uint64_t)kvheads) * (head_dim / 8) + 255) / 256;
  const uint64_t vb = (((uint64_t)rows + 15) / 16 * kvheads + 3) / 4;
  if (per > 0xffffffffull || !nlg_fits(qb + vb, 256))
    return nlg_fail("%s: too many rows and heads (%u x %llu) for one launch", what, rows, (unsigned long long)per);
  KV8_SCOPE(what);
  a.qkv = qkv; a.qgain = qgain; a.kgain = kgain; a.co = rope_cos; a.si = rope_sin;
  a.seq = seq; a.slot = slot; a.rpos = rpos; a.q = q; a.kpool = kpool; a.vpool = vpool;
  a.eps = eps; a.rows = rows; a.batch = batch; a.heads = heads; a.trows = trows; a.qblocks = (uint32_t)qb;
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

// The partials' bytes: contexts, then (maximum, sum) pairs; 0 where one chunk needs none.
static uint64_t kv8_partials(const Kv8Split &s, uint32_t batch, uint64_t rows, uint32_t kvheads, uint32_t hd) {
  return s.nchunk < 2 ? 0 : (uint64_t)batch * kvheads * s.nchunk * rows * (hd + 2) * 4;
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
  return (size_t)kv8_partials(kv8_split(batch, (uint32_t)rows, kvheads, (uint64_t)bs * mbps), batch, rows, kvheads,
                              head_dim);
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
  const uint64_t rows = kv8_rows(tmax, heads, kvheads);
  if (!rows) return nlg_fail("%s: %u heads over %u kv heads, %u queries", what, heads, kvheads, tmax);
  if (mask && tmax > KV8_TREE) return nlg_fail("%s: %u nodes under a mask (at most %d)", what, tmax, KV8_TREE);
  if (mask && ((uintptr_t)mask & 7)) return nlg_fail("%s: the masks must be 8-byte aligned", what);
  const Kv8Split s = kv8_split(batch, (uint32_t)rows, kvheads, (uint64_t)bs * mbps);
  const uint64_t need = kv8_partials(s, batch, rows, kvheads, hd);
  const uint64_t total = (uint64_t)batch * tmax * heads * (hd / 4);
  if (!nlg_fits(s.blocks, 64 * KV8_WAVES) || !nlg_fits((total + 255) / 256, 256))
    return nlg_fail("%s: too many queries for one launch", what);
  if (need) {
    if (!workspace || workspace_bytes < need)
      return nlg_fail("%s: workspace holds %zu bytes, needs %llu", what, workspace ? workspace_bytes : 0,
                      (unsigned long long)need);
    if ((uintptr_t)workspace & 15) return nlg_fail("%s: the workspace must be 16-byte aligned", what);
  }
  KV8_SCOPE(what);
  a.q = q; a.kpool = kpool; a.vpool = vpool; a.base = base; a.nodes = nodes; a.mask = mask; a.out = out;
  a.batch = batch; a.tmax = tmax; a.heads = heads; a.grp = heads / kvheads; a.rows = (uint32_t)rows;
  a.groups = s.groups; a.chunk = s.chunk; a.nchunk = s.nchunk;
  a.pctx = (float *)workspace;
  a.pmz = need ? a.pctx + (uint64_t)batch * kvheads * s.nchunk * rows * hd : nullptr;
  a.coef = NLG_LOG2E / sqrtf((float)hd);
  const dim3 grid((uint32_t)s.blocks), blk(64 * KV8_WAVES);
  hipStream_t st = nlg_stream(stream);
#define GO(HD, F)                                                                               \
  do {                                                                                          \
    if (!tree && s.rowsper == 16) hipLaunchKernelGGL((k_attn_q8<HD, F, 1, false>), grid, blk, 0, st, a); \
    else if (!tree) hipLaunchKernelGGL((k_attn_q8<HD, F, 2, false>), grid, blk, 0, st, a);      \
    else if (s.rowsper == 16) hipLaunchKernelGGL((k_attn_q8<HD, F, 1, true>), grid, blk, 0, st, a); \
    else hipLaunchKernelGGL((k_attn_q8<HD, F, 2, true>), grid, blk, 0, st, a);                  \
  } while (0)
  if (hd == 128) {
    if (fmt == NLG_KV_I8) GO(128, NLG_KV_I8); else GO(128, NLG_KV_E4M3);
  } else {
    if (fmt == NLG_KV_I8) GO(64, NLG_KV_I8); else GO(64, NLG_KV_E4M3);
  }
#undef GO
  NLG_LAUNCHED(what);
  if (need) {
    const dim3 mg((uint32_t)((total + 255) / 256));
    if (tree) hipLaunchKernelGGL(k_attn_q8_merge<true>, mg, dim3(256), 0, st, a, hd, total);
    else hipLaunchKernelGGL(k_attn_q8_merge<false>, mg, dim3(256), 0, st, a, hd, total);
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
