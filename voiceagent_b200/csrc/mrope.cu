// q/k RMSNorm + rotary positions with several axes + the paged KV store.
//
// The several-axes form of qk_norm_rope_store (models/qwen3.py:43-48, attention.py:90): the
// upstream model's positions are rows of [axes, T] (time, height, width), each of the D / 2
// frequencies turning by the position of its own axis. For a head vector x and frequency j,
//   y = x * rsqrt(mean(x^2) + eps) * w,      a = positions[axis[j]][t],
//   (y_j, y_{j + D/2}) -> (y_j cos - y_{j + D/2} sin, y_{j + D/2} cos + y_j sin) at (a, j),
// in 32 bits and rounded to bf16 once. K and V go to the token's slot of a bf16 cache, or of a
// 4-bit one (kv4.cuh), quantised from the rounded K.
//
// Bound by memory (the projection in, q and the cache out) and, for a decode step, by latency.
// A CTA takes whole tokens: D / 2 threads per token turn the axes into cos and sin once, in
// shared memory, while every warp's head vectors are already on their way; a vector is D / 8
// lanes of 8 consecutive dims, one 16-byte load, and a lane's rotation partner is the lane
// half a vector away.
#include "kv4.cuh"

namespace b200asr {

struct MropeArgs {
  const __nv_bfloat16 *qkv;
  int64_t qkv_stride;
  const int64_t *positions;  // [axes, T], row stride pos_stride
  int64_t pos_stride;
  int axes;
  const int32_t *axis;       // [D / 2]
  int num_tokens, num_heads, num_kv_heads;
  const __nv_bfloat16 *qw, *kw;
  float eps;
  const float *cos_sin;      // [max_position, D]: cos | sin
  int max_position;
  __nv_bfloat16 *q_out;
  int64_t q_out_stride;
  const int32_t *slots;      // null: no store
  __nv_bfloat16 *k_cache, *v_cache;  // bf16 cache, or null with c set
  b200asr_kv4 c;
  int64_t num_slots;
  int32_t *error_flag;
};

constexpr int kMrWarps = 8;

// TOK tokens per CTA; a warp's step is 32 / LANES head vectors of one token, STEPS at a time.
template <int LANES, int TOK, int STEPS, bool KV4>
__global__ void __launch_bounds__(kMrWarps * 32) qk_norm_mrope_store_kernel(const MropeArgs a) {
  constexpr int D = LANES * 8, PER = 32 / LANES;
  __shared__ float cs[TOK][D];  // cos | sin of each frequency at its own position
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gl = lane & (LANES - 1);
  const int t0 = blockIdx.x * TOK;
  const int heads = a.num_heads + 2 * a.num_kv_heads;
  const int steps = (heads + PER - 1) / PER;  // of one token
  const int total = min(TOK, a.num_tokens - t0) * steps;
  pdl_wait();
  bool ready = false;
  for (int first = warp * STEPS; first < total || !ready; first += kMrWarps * STEPS) {
    uint4 raw[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int s = first + i, tk = s / steps, head = (s - tk * steps) * PER + lane / LANES;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (s < total && head < heads)
        raw[i] = *reinterpret_cast<const uint4 *>(a.qkv + (t0 + tk) * a.qkv_stride +
                                                  static_cast<int64_t>(head) * D + gl * 8);
    }
    if (!ready) {
      for (int i = tid; i < TOK * (D / 2); i += kMrWarps * 32) {
        const int tk = i / (D / 2), j = i - tk * (D / 2);
        if (t0 + tk < a.num_tokens) {
          const int ax = a.axis[j];
          const bool ax_ok = ax >= 0 && ax < a.axes;
          int64_t p = ax_ok ? a.positions[ax * a.pos_stride + t0 + tk] : -1;
          if (p < 0 || p >= a.max_position) {
            raise_flag(a.error_flag, B200ASR_DEVERR_POSITION);
            p = 0;
          }
          cs[tk][j] = a.cos_sin[p * D + j];
          cs[tk][D / 2 + j] = a.cos_sin[p * D + D / 2 + j];
        }
      }
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int s = first + i;
      if (s >= total) break;
      const int tk = s / steps, head = (s - tk * steps) * PER + lane / LANES;
      const int64_t t = t0 + tk;
      const bool is_q = head < a.num_heads, is_v = head >= a.num_heads + a.num_kv_heads;
      float x[8];
      unpack8(raw[i], x);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.f / D) + a.eps);
      float w[8];
      unpack8(*reinterpret_cast<const uint4 *>((is_q ? a.qw : a.kw) + gl * 8), w);
      const float *row = cs[tk] + (gl & (LANES / 2 - 1)) * 8;
      const bool low = gl < LANES / 2;
      uint32_t y[4];
      float out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= r * w[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_xor_sync(0xffffffffu, x[e], LANES / 2);
        out[e] = fmaf(x[e], row[e], (low ? -other : other) * row[D / 2 + e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = pack2(out[2 * e], out[2 * e + 1]);
      const uint4 v = is_v ? raw[i] : make_uint4(y[0], y[1], y[2], y[3]);
      if (is_q) *reinterpret_cast<uint4 *>(a.q_out + t * a.q_out_stride + static_cast<int64_t>(head) * D + gl * 8) = v;
      int64_t slot = -1;
      if (!is_q && head < heads && a.slots != nullptr) {
        slot = a.slots[t];
        if (slot != -1 && (slot < 0 || slot >= a.num_slots)) {
          if (gl == 0) raise_flag(a.error_flag, B200ASR_DEVERR_SLOT);
          slot = -1;
        }
      }
      const int h = is_v ? head - a.num_heads - a.num_kv_heads : head - a.num_heads;
      if (!KV4) {
        if (slot >= 0)
          *reinterpret_cast<uint4 *>((is_v ? a.v_cache : a.k_cache) + (slot * a.num_kv_heads + h) * D + gl * 8) = v;
      } else if (__any_sync(0xffffffffu, slot >= 0)) {  // the reductions below need every lane
        const uint32_t rows[4] = {v.x, v.y, v.z, v.w};
        uint32_t codes[1], sz;
        kv4_quantise<LANES, 4>(rows, codes, sz);
        if (slot >= 0) {
          const int64_t block = slot / a.c.block_size, at = slot - block * a.c.block_size;
          reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(is_v ? a.c.v_codes : a.c.k_codes) +
                                       block * a.c.code_stride[0] + at * a.c.code_stride[1] +
                                       h * a.c.code_stride[2])[gl] = codes[0];
          if (gl == 0)
            reinterpret_cast<uint32_t *>(static_cast<__nv_bfloat16 *>(a.c.params) +
                                         block * a.c.param_stride[0] + at * a.c.param_stride[1] +
                                         h * a.c.param_stride[2])[is_v ? 1 : 0] = sz;
        }
      }
    }
  }
}

template <int LANES, bool KV4>
int launch_mrope(const MropeArgs &a, cudaStream_t stream) {
  // One token per CTA while that leaves SMs idle; two, with two steps in flight per warp, from
  // there on.
  const bool wide = a.num_tokens > 2 * num_sms();
  auto kfn = wide ? qk_norm_mrope_store_kernel<LANES, 2, 2, KV4> : qk_norm_mrope_store_kernel<LANES, 1, 1, KV4>;
  const unsigned grid = wide ? (a.num_tokens + 1) / 2 : a.num_tokens;
  B200_LAUNCH_CHECK_ERR(launch_kernel(kfn, dim3(grid), dim3(kMrWarps * 32), 0, stream, true, 1, a),
                        "qk_norm_mrope_store");
  return B200ASR_OK;
}

}  // namespace b200asr

using namespace b200asr;

extern "C" int b200asr_qk_norm_mrope_store(
    const void *qkv, int64_t qkv_row_stride, const int64_t *positions, int64_t position_stride,
    int32_t axes, const int32_t *freq_axis, int32_t num_tokens, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, const void *q_norm_weight, const void *k_norm_weight,
    float eps, const float *cos_sin_cache, int32_t max_position, void *q_out,
    int64_t q_out_row_stride, const int32_t *slot_mapping, void *k_cache, void *v_cache,
    int64_t num_slots, const b200asr_kv4 *cache4, int32_t *error_flag, b200asr_stream_t stream) {
  B200_REQUIRE(num_tokens >= 0 && num_heads >= 1 && num_kv_heads >= 1 && max_position >= 1 && axes >= 1,
               "qk_norm_mrope_store: bad sizes");
  B200_REQUIRE(head_dim == 64 || head_dim == 128, "qk_norm_mrope_store: head_dim %d unsupported (64 or 128)",
               head_dim);
  if (num_tokens == 0) return B200ASR_OK;
  B200_REQUIRE(qkv && positions && freq_axis && q_norm_weight && k_norm_weight && cos_sin_cache && q_out,
               "qk_norm_mrope_store: null pointer");
  B200_REQUIRE(slot_mapping == nullptr || ((k_cache && v_cache && num_slots >= 1) != (cache4 != nullptr)),
               "qk_norm_mrope_store: slot_mapping needs a bf16 cache or a 4-bit one");
  B200_REQUIRE(qkv_row_stride % 8 == 0 && q_out_row_stride % 8 == 0 && aligned16(qkv) && aligned16(q_out) &&
                   aligned16(q_norm_weight) && aligned16(k_norm_weight) && aligned16(k_cache) &&
                   aligned16(v_cache),
               "qk_norm_mrope_store: rows must be 16-byte aligned");
  MropeArgs a{};
  if (slot_mapping != nullptr && cache4 != nullptr) {
    B200_REQUIRE(cache4->k_codes && cache4->v_codes && cache4->params, "qk_norm_mrope_store: null pointer");
    B200_REQUIRE(kv4_cache_ok(*cache4) && cache4->head_dim == head_dim && cache4->num_kv_heads == num_kv_heads,
                 "qk_norm_mrope_store: cache sizes, or rows not 16-byte (codes) and 8-byte (parameters) aligned");
    a.c = *cache4;
    num_slots = static_cast<int64_t>(cache4->num_blocks) * cache4->block_size;
  }
  a.qkv = static_cast<const __nv_bfloat16 *>(qkv);
  a.qkv_stride = qkv_row_stride;
  a.positions = positions;
  a.pos_stride = position_stride;
  a.axes = axes;
  a.axis = freq_axis;
  a.num_tokens = num_tokens;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.qw = static_cast<const __nv_bfloat16 *>(q_norm_weight);
  a.kw = static_cast<const __nv_bfloat16 *>(k_norm_weight);
  a.eps = eps;
  a.cos_sin = cos_sin_cache;
  a.max_position = max_position;
  a.q_out = static_cast<__nv_bfloat16 *>(q_out);
  a.q_out_stride = q_out_row_stride;
  a.slots = slot_mapping;
  a.k_cache = static_cast<__nv_bfloat16 *>(k_cache);
  a.v_cache = static_cast<__nv_bfloat16 *>(v_cache);
  a.num_slots = num_slots;
  a.error_flag = error_flag;
  const bool kv4 = slot_mapping != nullptr && cache4 != nullptr;
  auto fn = head_dim == 128 ? (kv4 ? launch_mrope<16, true> : launch_mrope<16, false>)
                            : (kv4 ? launch_mrope<8, true> : launch_mrope<8, false>);
  return fn(a, stream);
}
