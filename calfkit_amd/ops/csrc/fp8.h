// e4m3fn codes with power-of-two row scales (gfx950 conversions).
#pragma once

#include "common.h"

#include <torch/types.h>

using bf16x2v = __attribute__((ext_vector_type(2))) __bf16;

// Least e in [-127, 127] with a * 2^-e <= 448 = 0.875 * 2^9; 0 for a = 0.
// (a finite and >= 0; the largest finite a gives 120.)
__device__ __forceinline__ int e4m3_row_exponent(const float a) {
  int e;
  const float m = frexpf(a, &e);  // a = m * 2^e, 0.5 <= m < 1
  e -= (m > 0.875f) ? 8 : 9;
  return (a > 0.f) ? max(e, -127) : 0;
}

// Four values of magnitude <= 448 (or NaN) -> four codes, half to even.
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c,
                                              float d) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}

// The conversion below uses the scale's exponent field alone, so byte 0 is
// 2^-127 although these float bits are those of 0.
__device__ __forceinline__ float e8m0_scale(const int byte) {
  return __int_as_float(byte << 23);
}

// Two of a word's four codes times 2^e as a pair of bf16: exact (4
// significant bits), but for results below bf16's least normal value.
template <bool HIGH>
__device__ __forceinline__ unsigned e4m3_to_bf16x2(const unsigned codes,
                                                   const float scale) {
  const bf16x2v r =
      __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH);
  return __builtin_bit_cast(unsigned, r);
}

inline void check_fp8_cache(const torch::Tensor& kcache,
                            const torch::Tensor& vcache,
                            const torch::Tensor& kscale,
                            const torch::Tensor& vscale,
                            const torch::Device dev) {
  for (const auto* c : {&kcache, &vcache}) {
    TORCH_CHECK(c->device() == dev, "the cache is on another device");
    TORCH_CHECK(c->scalar_type() == torch::kFloat8_e4m3fn,
                "the cache must be float8_e4m3fn");
    TORCH_CHECK(c->dim() == 4 && c->size(2) == 64 && c->size(3) == 128 &&
                    c->size(1) > 0 && c->is_contiguous() &&
                    c->sizes() == kcache.sizes(),
                "the caches must be contiguous [P, Hkv, 64, 128]");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(c->data_ptr()) % 16 == 0,
                "the caches must start on 16 bytes");
  }
  for (const auto* c : {&kscale, &vscale}) {
    TORCH_CHECK(c->device() == dev, "the scales are on another device");
    TORCH_CHECK(c->scalar_type() == torch::kUInt8, "the scales must be uint8");
    TORCH_CHECK(c->dim() == 3 && c->size(0) == kcache.size(0) &&
                    c->size(1) == kcache.size(1) && c->size(2) == 64 &&
                    c->is_contiguous(),
                "the scales must be contiguous [P, Hkv, 64]");
  }
}
