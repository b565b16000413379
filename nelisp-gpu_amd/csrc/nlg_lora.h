// nlg_lora.h -- what kernels that add low-rank adapters share: which adapter a
// row has, the 16-bit formats, and 32-bit values as the parts that the bf16
// matrix cores take.
#pragma once

#include "nlg_internal.h"

typedef float v4f __attribute__((ext_vector_type(4)));

struct LoraArgs {
  const int32_t *start;     // [requests + 1] or null: request i is row i
  const int32_t *adapter;   // [requests]
  const int32_t *rank;      // [adapters] or null
  const float *scale;       // [adapters]
  const uint16_t *a, *b;    // [adapters][rmax][cols], [adapters][out][rmax]
  uint32_t requests, adapters, rmax, seq;
};

__device__ __forceinline__ uint32_t lora_rank(const LoraArgs &l, int32_t ad) {
  if (!l.rank) return l.rmax;
  const int32_t r = l.rank[ad];
  return r < 0 ? 0u : min((uint32_t)r, l.rmax);
}

// A wave finds the adapters of rows row0 .. row0 + n - 1 (n <= 64), lane i
// row0 + i's; -1: none.  A row that two requests name belongs to the first.
__device__ __forceinline__ int32_t lora_rows(const LoraArgs &l, uint32_t row0, uint32_t n, int lane) {
  int32_t got = -1;
  const uint32_t row = row0 + lane;
  if (!l.start) {
    if ((uint32_t)lane < n && row < l.seq && row < l.requests) got = l.adapter[row];
  } else {
    bool found = false;
    for (uint32_t i0 = 0; i0 < l.requests; i0 += 64) {
      const uint32_t i = i0 + lane;
      const bool in = i < l.requests;
      const int32_t s = in ? l.start[i] : 0, e = in ? l.start[i + 1] : 0, ad = in ? l.adapter[i] : -1;
      // requests of this block that touch the rows, in order
      uint64_t hit = __ballot(in && s < e && (int64_t)s < (int64_t)row0 + n && (int64_t)e > (int64_t)row0);
      while (hit) {
        const int k = __builtin_ctzll(hit);
        hit &= hit - 1;
        const int64_t ks = __builtin_amdgcn_readlane(s, k), ke = __builtin_amdgcn_readlane(e, k);
        const int32_t ka = __builtin_amdgcn_readlane(ad, k);
        if (!found && (int64_t)row >= ks && (int64_t)row < ke) {
          got = ka;
          found = true;
        }
      }
      if (__all(found || (uint32_t)lane >= n || row >= l.seq)) break;
    }
    if ((uint32_t)lane >= n || row >= l.seq) got = -1;
  }
  return got >= 0 && (uint32_t)got < l.adapters ? got : -1;
}

template <bool BF>
__device__ __forceinline__ float wide(uint32_t h) {  // a 16-bit value (low half)
  return BF ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
union Bf8 {
  uint32_t u[4];
  uint4 q;
  bf8v v;
};
// Two f32 as the pairs of bf16 that add up to them, largest first (what is
// left after each is exact).
__device__ __forceinline__ void split3(float a, float b, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
  const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
  p0 = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
  const float ra = a - __uint_as_float(ua & 0xffff0000u), rb = b - __uint_as_float(ub & 0xffff0000u);
  const uint32_t va = __float_as_uint(ra), vb = __float_as_uint(rb);
  p1 = __builtin_amdgcn_perm(vb, va, 0x07060302u);
  const float sa = ra - __uint_as_float(va & 0xffff0000u), sb = rb - __uint_as_float(vb & 0xffff0000u);
  p2 = __builtin_amdgcn_perm(__float_as_uint(sb), __float_as_uint(sa), 0x07060302u);
}
// A pair of f16 as two pairs of bf16.
__device__ __forceinline__ void split_f16(uint32_t h, uint32_t &p0, uint32_t &p1) {
  const float a = wide<false>(h & 0xffff), b = wide<false>(h >> 16);
  const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
  p0 = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
  const float ra = a - __uint_as_float(ua & 0xffff0000u), rb = b - __uint_as_float(ub & 0xffff0000u);
  p1 = __builtin_amdgcn_perm(__float_as_uint(rb), __float_as_uint(ra), 0x07060302u);
}

// Whether the call below (and nlg_batched_gemm with NLG_EPI_STORE) takes rows of so many columns: also multiples of 64
// that nlg_batched leaves to the kernels of few tokens.
bool nlg_batched_lora(uint32_t seq, uint32_t cols);
// The shared projection on the matrix cores with the adapters added to it
// (nlg_batched_gemm otherwise, split as there); *done: whether the form that
// this size takes adds them, or only the projection was run.  u [seq][rmax].
int nlg_batched_gemm_lora(const FusedArgs &f, const uint8_t *xq, const float *gamma, const LoraArgs &l, const float *u,
                          bool bf, uint32_t *split, bool *done, hipStream_t st);
