// Codes and exponents of the cache of 8-bit floats: what its writers share.
#pragma once
#include "atf_common.h"

namespace atf {

constexpr float kQ8Max = 448.f;
constexpr uint32_t kInfBits = 0x7f800000u;

// The exponent of a half whose largest finite magnitude has these bits.
__device__ __forceinline__ int q8_exponent(uint32_t top) {
  // 448 2^e = 1.75 2^(e + 8): with top = 1.f 2^E, e = E - 8 where 1.f <= 1.75, else E - 7
  const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kQ8MinExp), kQ8MaxExp);  // (top 0 or subnormal: the least)
}
__device__ __forceinline__ float exp2_int(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Eight values times `inv` as codes.  odd: some value of the page is not finite, or
// the exponent was cut at its limit.
__device__ __forceinline__ u32x2 q8_codes(const float (&x)[8], float inv, bool odd) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = (__float_as_uint(x[i]) & 0x7fffffffu) >= kInfBits ? __uint_as_float(0x7fc00000u)
                                                                : fminf(fmaxf(y[i], -kQ8Max), kQ8Max);
  }
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
    w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], p, true));
  }
  return w;
}

// Four codes of a half moved up by d exponents (scale = 2^-d).
__device__ __forceinline__ uint32_t q8_shift(uint32_t w, float scale) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
  const int p = __builtin_amdgcn_cvt_pk_fp8_f32(a[0], a[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(b[0], b[1], p, true));
}
__device__ __forceinline__ float shift_scale(int from, int to) { return exp2_int(max(from - to, -126)); }

// Bits of |x| for the page's maximum; a value that is not finite counts for nothing and is noted.
__device__ __forceinline__ void note(float x, uint32_t& top, uint32_t& odd) {
  const uint32_t m = __float_as_uint(x) & 0x7fffffffu;
  odd |= m >= kInfBits ? 1u : 0u;
  top = max(top, m >= kInfBits ? 0u : m);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), m)));
  return x;
}

// 4 x 4 bytes transposed: word i of the result holds byte i of the four words.
__device__ __forceinline__ u32x4 transpose4(const u32x4& w) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  return u32x4{__builtin_amdgcn_perm(b, a, 0x05040100u), __builtin_amdgcn_perm(b, a, 0x07060302u),
               __builtin_amdgcn_perm(d, c, 0x05040100u), __builtin_amdgcn_perm(d, c, 0x07060302u)};
}

}  // namespace atf
