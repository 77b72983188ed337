// The 4-bit paged KV cache: its layout in memory and the arithmetic of a row.
//
// A cached head row of D values is held as D / 2 bytes of codes (value 2j in the low half of
// byte j) and two bf16 numbers, scale and zero; value = zero + code * scale. zero is the row's
// minimum (a bf16 value, so exact) and scale the smallest bf16 with 15 * scale >= maximum -
// minimum, so every value lies within half a step of what it is held as. One pair per row
// lets attention multiply codes: a score is scale * (q . c) + zero * sum(q), and the V scale
// goes into the probability. A row narrower than 2^-100 is held as its minimum (scale 0); a
// row with an infinity or a NaN, or a range past the largest 32-bit number, reads as NaN.
#pragma once

#include "common.cuh"

namespace b200asr {

// The caller's description, checked: rows of codes 16-byte, parameter rows 8-byte aligned.
inline bool kv4_cache_ok(const b200asr_kv4 &c) {
  return c.num_blocks >= 1 && c.block_size >= 1 && c.num_kv_heads >= 1 && aligned16(c.k_codes) &&
         aligned16(c.v_codes) && (reinterpret_cast<uintptr_t>(c.params) & 7) == 0 &&
         c.code_stride[0] % 16 == 0 && c.code_stride[1] % 16 == 0 && c.code_stride[2] % 16 == 0 &&
         c.param_stride[0] % 4 == 0 && c.param_stride[1] % 4 == 0 && c.param_stride[2] % 4 == 0;
}

// One head row, 2 W consecutive values (bf16 pairs) per lane of a LANES-wide group: this lane's
// codes, eight to a word, and the row's (scale, zero) as a bf16 pair.
template <int LANES, int W>
__device__ __forceinline__ void kv4_quantise(const uint32_t (&x)[W], uint32_t (&codes)[W / 4],
                                             uint32_t &scale_zero) {
  // (minimum, -maximum) of the row in one pair, NaN once a value is
  auto as_pair = [](uint32_t v) { return *reinterpret_cast<const __nv_bfloat162 *>(&v); };
  __nv_bfloat162 lo2 = as_pair(x[0]), hi2 = lo2;
#pragma unroll
  for (int i = 1; i < W; ++i) {
    lo2 = __hmin2_nan(lo2, as_pair(x[i]));
    hi2 = __hmax2_nan(hi2, as_pair(x[i]));
  }
  __nv_bfloat162 ends = __halves2bfloat162(__hmin_nan(__low2bfloat16(lo2), __high2bfloat16(lo2)),
                                           __hneg(__hmax_nan(__low2bfloat16(hi2), __high2bfloat16(hi2))));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) ends = __hmin2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, o));
  const float lo = bf2f(__low2bfloat16(ends)), hi = -bf2f(__high2bfloat16(ends));
  const float wide = __fsub_rn(hi, lo);
  // the bf16 next to wide / 15, then one step up or down until it is the smallest that reaches
  uint32_t s16 = __float_as_uint(wide * (1.f / 15.f));
  s16 = (s16 + 0x7fffu + ((s16 >> 16) & 1u)) >> 16;
  if (15.f * __uint_as_float(s16 << 16) < wide) ++s16;
  else if (s16 > 0 && 15.f * __uint_as_float((s16 - 1) << 16) >= wide) --s16;
  if (wide < 0x1p-100f) s16 = 0;
  const float scale = __uint_as_float(s16 << 16);
  const float inv = s16 ? __frcp_rn(scale) : 0.f;
  const bool ok = wide < INFINITY;
#pragma unroll
  for (int i = 0; i < W / 4; ++i) {
    // rounding by adding 1.5 * 2^23: the sum's low bits are the code (0 to 15, as 15 * scale
    // reaches the maximum); the constant's own bits, shifted along with them, come off at the end
    uint32_t w = 0u - (0x4b400000u + (0x4b400000u << 4) + (0x4b400000u << 8));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // the correctly rounded quotient d / scale from the correctly rounded reciprocal
      // (Markstein 1990: quotient estimate, its exact remainder, one correction)
      const float2 v = unpack2(x[4 * i + e / 2]);
      const float d = __fsub_rn(e & 1 ? v.y : v.x, lo);
      const float q0 = __fmul_rn(d, inv);
      const float q = __fmaf_rn(__fmaf_rn(-q0, scale, d), inv, q0);
      w += __float_as_uint(__fadd_rn(q, 12582912.f)) << (4 * e);
    }
    codes[i] = ok ? w : 0u;
  }
  scale_zero = ok ? (s16 | (__float_as_uint(lo) & 0xffff0000u)) : 0x7fc07fc0u;
}

}  // namespace b200asr
