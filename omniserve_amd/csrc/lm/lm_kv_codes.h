// A cache row (one token's key or value of one kv head) as 8-bit floats under a power of two: value = e4m3(code) * 2^(byte - 127).
// 2^(byte - 127) is the least power that brings the row's largest finite magnitude to 448, the format's largest: dividing by it is
// exact, so a code is the one nearest to its value whatever the arithmetic around it, and a float format loses nothing by the power
// of two (its step is relative).  NaN and infinities become NaN codes.
#pragma once
#include "lm_common.h"

namespace lm {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int LOW_EXP = -100, HIGH_EXP = 120;      // of a row's scale: smaller rows lose bits, larger ones do not exist
constexpr float BIGGEST = 448.f;

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }        // 2^(byte - 127)

// top: largest finite magnitude of the row
__device__ __forceinline__ int row_exponent(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = (int)(u >> 23) - 135 + ((u & 0x7fffffu) > 0x600000u);      // top = 1.f * 2^(E - 127), 448 = 1.75 * 2^8
  return min(max(e, LOW_EXP), HIGH_EXP);
}

// Four codes of values under the row's exponent
__device__ __forceinline__ uint32_t encode4(const float* x, int e) {
  const float f = pow2(-e), lim = e == HIGH_EXP ? 240.f : BIGGEST;      // (256 * 2^120 would be read back as infinity)
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float z = x[i] * f;
    y[i] = fabsf(x[i]) < __builtin_inff() ? fminf(fmaxf(z, -lim), lim) : __builtin_nanf("");
  }
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
}

// Four values of codes
__device__ __forceinline__ quad_t decode4(uint32_t w, float scale) {
#if LM_ELEM == 0
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
#else
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
#endif
  return (quad_t){a[0], a[1], b[0], b[1]};
}

// i / d for i * d < 2^32
struct Divisor {
  uint32_t d, m;
  Divisor(uint32_t n = 1) : d(n), m(n > 1 ? (uint32_t)((0x100000000ull + n - 1) / n) : 0) {}
  __device__ __forceinline__ uint32_t quotient(uint32_t i) const { return d > 1 ? __umulhi(i, m) : i; }
};

}  // namespace lm
