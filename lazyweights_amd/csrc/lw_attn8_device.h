// Device helpers of the kernels over a cache held in 8 bits (lw_kv8_append.hip, lw_attn8_decode.hip, lw_attn8_prompt.hip): numbers of 1
// sign, 4 exponent and 3 mantissa bits (up to 448; 0x7F and 0xFF are NaN), and a power of two for the 16 rows of a block.
#pragma once
#include "lw_attn_device.h"

namespace lw {

namespace {

typedef int i2v __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i2v LdsI2;

__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// four numbers, the lowest byte first
__device__ __forceinline__ f4v from8(uint32_t w) {
  const f2v a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return (f4v){a[0], a[1], b[0], b[1]};
}

// eight numbers as fp16 or bf16, which hold them exactly: the products' operand
template <bool BF>
__device__ __forceinline__ u32x4 widen8(uint32_t x, uint32_t y) {
  if (BF)
    return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, true))};
  return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.f, true))};
}

// 8 keys x 16 dims of 16 lanes (lane l gives dims 8 (l & 1) .. of key l >> 1), transposed: lane l gets dim l of the 8 keys
__device__ __forceinline__ uint2 read_tr8(const uint8_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsI2*)p));
}

}  // namespace

}  // namespace lw
