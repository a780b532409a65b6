// cache_format.cuh -- the row formats of a key/value cache (include/wfattn.h)
// as the kernels see them.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/wfattn.h"
#include "sm100_ptx.cuh"
#include "wfattn_internal.h"

namespace wfattn {

// Bytes of a row of D values.
template <int kFmt, int D>
struct CacheRow {
  static constexpr int kBytes = kFmt == WFATTN_CACHE_F32    ? 4 * D
                                : kFmt == WFATTN_CACHE_BF16 ? 2 * D
                                : kFmt == WFATTN_CACHE_E4M3 ? D
                                                            : D / 2;
  static constexpr bool kScaled = kFmt == WFATTN_CACHE_E4M3 || kFmt == WFATTN_CACHE_INT4;
};

namespace ptx {

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Two e4m3 codes (the low 16 bits of w) as f16x2: exact, NaN codes stay NaN.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)w));
  return r;
}

// Two f32 as e4m3 codes (nearest even; |x| <= 448 here), lo in the low byte.
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float2 f16x2_to_f32(uint32_t w) {
  float2 f;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(f.x), "=f"(f.y)
      : "r"(w));
  return f;
}

}  // namespace ptx

// Eight consecutive values of a row as f32, from the row's eight codes (32, 16,
// 8 or 4 bytes) and its scale word.
template <int kFmt>
__device__ __forceinline__ void cache_values8(const uint32_t *w, uint32_t scale, float (&f)[8]) {
  if constexpr (kFmt == WFATTN_CACHE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  } else if constexpr (kFmt == WFATTN_CACHE_BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = ptx::bf16_lo(w[i]), f[2 * i + 1] = ptx::bf16_hi(w[i]);
  } else if constexpr (kFmt == WFATTN_CACHE_E4M3) {
    const float s = __uint_as_float(scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = ptx::f16x2_to_f32(ptx::e4m3x2_to_f16x2(w[i / 2] >> (16 * (i & 1))));
      f[2 * i] = x.x * s, f[2 * i + 1] = x.y * s;
    }
  } else {
    const float s = ptx::bf16_lo(scale), m = ptx::bf16_hi(scale);
    // A code left where it is in its half of the word, under 2^23, is 16^i u;
    // s 16^-i is exact (for s >= 2^-130), as is s u (8 and 4 bits): one rounding
    // is left.
    const float s1 = s * 0x1p-4f, s2 = s * 0x1p-8f, s3 = s * 0x1p-12f;
    const uint64_t s01 = ptx::f2_pack(s, s1), s23 = ptx::f2_pack(s2, s3);
    const uint64_t m2 = ptx::f2_pack(m, m), less = ptx::f2_pack(-8388608.f, -8388608.f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t h = i ? w[0] >> 16 : w[0];
      const uint64_t a = ptx::f2_pack(__uint_as_float((h & 0xfu) | 0x4b000000u),
                                      __uint_as_float((h & 0xf0u) | 0x4b000000u));
      const uint64_t b = ptx::f2_pack(__uint_as_float((h & 0xf00u) | 0x4b000000u),
                                      __uint_as_float((h & 0xf000u) | 0x4b000000u));
      ptx::f2_unpack(ptx::f2_fma(s01, ptx::f2_add(a, less), m2), f[4 * i], f[4 * i + 1]);
      ptx::f2_unpack(ptx::f2_fma(s23, ptx::f2_add(b, less), m2), f[4 * i + 2], f[4 * i + 3]);
    }
  }
}

}  // namespace wfattn
