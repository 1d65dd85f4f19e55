// 8-bit floats with block scales: e4m3 codes (largest 448, no infinities, NaN 0x7f), and for each block a byte s that
// stands for 2^(s - 127): the smallest power of two (2^-126 at least) with which the block's largest finite value a is
// at most 448.  With a = m 2^E, 1 <= m < 2, that is 2^(E - 8) for m <= 1.75 and 2^(E - 7) above.  Scaling by it is exact,
// so a code is rounded once (to the nearest, ties to even, by the conversion instruction); what is not finite has the
// code of NaN and no part in its block's scale.  Powers of two, because the matrix instructions apply them for nothing:
// a scale with a mantissa would cost a multiplication of every accumulator for every 128 products.
#pragma once
#include "common.h"

namespace e2v2 {

constexpr int kBlock8 = 128;                 // values that share a scale

// The bits of |v|: compared as integers they order as the values do, what is not finite from kInfBits on.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
// The same where v is finite, else 0.
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t u = abs_bits(v);
  return u < kInfBits ? u : 0u;
}
// f(bits), f being the largest of these bits over some of the wavefront's values, in every lane that shares it: over all
// values first, and where that finds one that is not finite once more without those (a test of each cost as much as the
// rest of quantising it).
template <typename F>
__device__ __forceinline__ uint32_t top_bits(F&& f) {
  const uint32_t m = f([](float v) { return abs_bits(v); });
  if (!__any(m >= kInfBits)) return m;
  return f([](float v) { return finite_bits(v); });
}
// The scale byte of a block whose largest finite value has these bits: 1 to 247.
__device__ __forceinline__ int scale_byte(uint32_t top) { return max((int)((top + 0x1fffffu) >> 23) - 8, 1); }
// 2^(127 - s)
__device__ __forceinline__ float scale_up(int s) { return __builtin_bit_cast(float, (254 - s) << 23); }
// 2^(s - 127), also for s = 0 (2^-127, a subnormal number) and s = 255 (NaN), which other writers of such bytes may use
__device__ __forceinline__ float scale_value(int s) {
  return __builtin_bit_cast(float, s == 0 ? 0x00400000 : s == 255 ? 0x7fc00000 : s << 23);
}

// Four codes in a dword; the conversion makes NaN of what is not finite.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, false));
}
// Largest value over aligned groups of G lanes (1 to 64), in every lane.
template <int G>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (G >= 2) v = dpp_max<0xB1>(v);
  if constexpr (G >= 4) v = dpp_max<0x4E>(v);
  if constexpr (G >= 8) v = dpp_max<0x141>(v);
  if constexpr (G >= 16) v = dpp_max<0x140>(v);
  if constexpr (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  if constexpr (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  return v;
}

}  // namespace e2v2
