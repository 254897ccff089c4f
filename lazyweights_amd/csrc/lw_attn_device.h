// Device helpers shared by the attention kernels (lw_attn_decode.hip, lw_attn_prompt.hip).
//
// Both kernels form the scores transposed, S^T = K Q^T: a lane of the product holds several keys of one row (a row is a
// new token's query head; the heads that share a key-value head are rows of the same tile), so the maximum, the sum and
// the rescaling of a row are per-lane scalars, and the weights P^T lie in a lane as the second product's operand
// O^T = V^T P^T takes them. The contraction runs over keys in whatever order the score product left them; V^T's operand,
// read transposed from LDS (ds_read_b64_tr_b16: 16 lanes give 4 keys x 16 dims and get 4 keys of one dim each), follows
// that order.
#pragma once
#include <cmath>

#include "lw_attention.h"
#include "lw_device.h"

namespace lw {

namespace {

typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v LdsS4;
typedef __attribute__((address_space(3))) const u32x4 LdsU4;
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }

// 16-bit conversions, rounded to nearest even
template <bool BF>
__device__ __forceinline__ float wide(uint16_t h) {
  if (BF) return __uint_as_float((uint32_t)h << 16);
  return (float)__builtin_bit_cast(_Float16, h);
}
template <bool BF>
__device__ __forceinline__ uint32_t narrow2(float x, float y) {  // x in the low half
  if (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v){x, y}, b2v));
  return __builtin_bit_cast(uint32_t, (h2v){(_Float16)x, (_Float16)y});
}

template <bool BF>
__device__ __forceinline__ f4v mfma16(u32x4 a, u32x4 b, f4v c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f16x16 mfma32(u32x4 a, u32x4 b, f16x16 c) {
  if (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}

// 4 keys x 16 dims of 16 lanes, transposed: lane l of the 16 gets dim l of the 4 keys
__device__ __forceinline__ uint2 read_tr(const uint16_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)p));
}

// 16 bytes per lane from src to LDS, lane l's at dst + 16 l (dst the same in every lane)
__device__ __forceinline__ void copy_lds16(const uint16_t* src, uint16_t* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                   (__attribute__((address_space(3))) uint32_t*)dst, 16, 0, 0);
}

// v combined with lane ^ 32's (and ^ 16's)
__device__ __forceinline__ uint2 swap32(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return make_uint2(r[0], r[1]);
}
__device__ __forceinline__ uint2 swap16(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return make_uint2(r[0], r[1]);
}
__device__ __forceinline__ float max32(float v) {
  const uint2 r = swap32(__float_as_uint(v));
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float max16(float v) {
  const uint2 r = swap16(__float_as_uint(v));
  return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float add32(float v) {
  const uint2 r = swap32(__float_as_uint(v));
  return __uint_as_float(r.x) + __uint_as_float(r.y);
}
__device__ __forceinline__ float add16(float v) {
  const uint2 r = swap16(__float_as_uint(v));
  return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// 2^v by the hardware's instruction (results below 2^-126 are 0: weights are at most 1 and sums at least that of a row's
// largest)
__device__ __forceinline__ float pow2(float v) { return __builtin_amdgcn_exp2f(v); }

__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) < INFINITY; }

// The last s in [0, n) with first(s) <= x, first non-decreasing (0 if there is none): 64 candidates at a time.
template <class F>
__device__ __forceinline__ int last_at_most(int n, int x, F first) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = lane * step;
    const int c = __popcll(__ballot(at < n && first(lo + at) <= x));
    const int skip = max(c - 1, 0) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// sum += x, with what rounding has added to the sum so far taken off x first (W. Kahan, 1965)
__device__ __forceinline__ void add_exactly(float& sum, float& lost, float x) {
  const float y = x - lost, t = sum + y;
  lost = (t - sum) - y;
  sum = t;
}

// a sequence's rows and keys, whatever the arrays hold: rows lie in [0, tokens), keys in the page table
struct Seq {
  int row0, rows, len;
};
__device__ __forceinline__ Seq sequence(const KvView& c, int s) {
  Seq q;
  q.row0 = clampi(c.q_start[s], 0, c.tokens);
  q.rows = clampi(c.q_start[s + 1], q.row0, c.tokens) - q.row0;
  q.len = clampi(c.kv_len[s], 0, c.table_pages << c.page_shift);  // (the host keeps that within 2^30)
  return q;
}

// element offset of key `key` of the sequence whose table row is `table`, and whether it is there
__device__ __forceinline__ int64_t key_offset(const KvView& c, uint32_t page, int key, bool& there) {
  there = page < c.pages;
  return (there ? (int64_t)page * c.pstride : 0) + (int64_t)(key & ((1 << c.page_shift) - 1)) * c.rstride;
}

template <int OUT>
__device__ __forceinline__ void store4(void* out, int64_t i, f4v v) {
  if (OUT == 0)
    *reinterpret_cast<f4v*>(static_cast<float*>(out) + i) = v;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) =
        make_uint2(narrow2<OUT == 2>(v[0], v[1]), narrow2<OUT == 2>(v[2], v[3]));
}
__device__ __forceinline__ void store4(int type, void* out, int64_t i, f4v v) {
  if (type == 0) store4<0>(out, i, v);
  else if (type == 1) store4<1>(out, i, v);
  else store4<2>(out, i, v);
}

// v / sum, zeros for a row that has seen nothing
__device__ __forceinline__ f4v normal(f4v v, float sum) { return sum == 0.f ? (f4v)0.f : v * (1.f / sum); }

// two values stored to, and read from, where every XCD sees them
__device__ __forceinline__ void put2(float* p, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ f2v get2(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return (f2v){__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}

// Weights are 2^(score - m + lift), m the row's largest score or less by `ahead` at most; numerators and sums carry the same
// factor. The least step of fp16 is 2^-24, in a second part too, so what rounding takes from a weight is up to 2^-25 of the unit.
// Lifted so that the largest is 2^15 (65504 is the last number), or 2^(15 - ahead) at least, that is 2^-40, or 2^(ahead - 40), of
// the row's largest weight; not lifted, a weight e^-17.4 of the largest would be lost whole, while the row's sum counts it.
// bf16 has the range of fp32.
template <bool BF>
constexpr float lift(float ahead) {
  return BF ? 0.f : 15.f - ahead;
}

// weights p as the operand of the second product, in NP 16-bit parts that add up to p (two of fp16: 22 bits, three of
// bf16: 24; one: rounded)
template <bool BF, int NP>
__device__ __forceinline__ void split8(const float* p, u32x4* part) {
  float r[8], minus = -1.f;
  if (!BF) asm("" : "+s"(minus));  // (not seen as -1, so that a conversion and a difference are one instruction)
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = p[i];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w = narrow2<BF>(r[2 * i], r[2 * i + 1]);
      part[n][i] = w;
      if (n + 1 < NP) {
        if (!BF) asm("" : "+v"(w));  // (what was rounded is read from the part: the compiler would round each value once more)
        r[2 * i] = __builtin_fmaf(wide<BF>((uint16_t)w), minus, r[2 * i]);
        r[2 * i + 1] = __builtin_fmaf(wide<BF>((uint16_t)(w >> 16)), minus, r[2 * i + 1]);
      }
    }
  }
}

}  // namespace

}  // namespace lw
