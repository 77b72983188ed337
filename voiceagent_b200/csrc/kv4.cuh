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

// One head row, 8 consecutive values per lane of a LANES-wide group (LANES = D / 8): this
// lane's 8 codes and the row's (scale, zero) as a bf16 pair.
template <int LANES>
__device__ __forceinline__ void kv4_quantise(const float (&x)[8], uint32_t &codes,
                                             uint32_t &scale_zero) {
  float lo = x[0], hi = x[0];
  uint32_t top = 0;  // the largest magnitude's bits: 0x7f800000 and up is not finite
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const float wide = __fsub_rn(hi, lo);
  // the bf16 next to wide / 15, then one step up or down until it is the smallest that reaches
  uint32_t s16 = __float_as_uint(wide * (1.f / 15.f));
  s16 = (s16 + 0x7fffu + ((s16 >> 16) & 1u)) >> 16;
  if (15.f * __uint_as_float(s16 << 16) < wide) ++s16;
  else if (s16 > 0 && 15.f * __uint_as_float((s16 - 1) << 16) >= wide) --s16;
  if (wide < 0x1p-100f) s16 = 0;
  const float scale = __uint_as_float(s16 << 16);
  const float inv = s16 ? __frcp_rn(scale) : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // the correctly rounded quotient d / scale from the correctly rounded reciprocal
    // (Markstein 1990: quotient estimate, its exact remainder, one correction)
    const float d = __fsub_rn(x[e], lo);
    const float q0 = __fmul_rn(d, inv);
    const float q = __fmaf_rn(__fmaf_rn(-q0, scale, d), inv, q0);
    w |= static_cast<uint32_t>(min(15, max(0, __float2int_rn(q)))) << (4 * e);
  }
  const bool ok = top < 0x7f800000u && wide < INFINITY;
  codes = ok ? w : 0u;
  scale_zero = ok ? (s16 | (__float_as_uint(lo) & 0xffff0000u)) : 0x7fc07fc0u;
}

}  // namespace b200asr
