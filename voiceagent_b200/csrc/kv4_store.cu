// Rows into and out of the 4-bit paged KV cache (kv4.cuh has the format).
//
// store_kvcache4 <- store_kvcache (layers/attention.py:52-67), quantising on the way
// load_kvcache4     its inverse: cached rows gathered by slot as bf16
//
// Both are bound by memory: a row is read once and written once. A group of D / 8 lanes takes
// one (token, head, K or V) row, 16 bytes of bf16 and 4 bytes of codes per lane, so every
// access of a group is one contiguous run; the row's extremes are a shuffle reduction.
#include "kv4.cuh"

namespace b200asr {

template <int LANES, bool STORE>
__global__ void kv4_rows_kernel(const b200asr_kv4 c, __nv_bfloat16 *key, int64_t k_token,
                                int64_t k_head, __nv_bfloat16 *value, int64_t v_token,
                                int64_t v_head, const int32_t *__restrict__ slots,
                                int64_t num_tokens, int32_t *error_flag) {
  pdl_trigger();
  pdl_wait();
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / LANES;
  const int lane = threadIdx.x & (LANES - 1);
  const int per_token = 2 * c.num_kv_heads;
  const int64_t t = row / per_token;
  const bool in = t < num_tokens;  // whole groups: the shuffles below need every lane
  const int j = static_cast<int>(row - t * per_token);
  const bool is_v = j >= c.num_kv_heads;
  const int h = is_v ? j - c.num_kv_heads : j;
  int64_t slot = in ? slots[t] : -1;
  if (slot != -1 && (slot < 0 || slot >= static_cast<int64_t>(c.num_blocks) * c.block_size)) {
    if (lane == 0) raise_flag(error_flag, B200ASR_DEVERR_SLOT);
    slot = -1;
  }
  const int64_t block = slot >= 0 ? slot / c.block_size : 0;
  const int64_t at = slot >= 0 ? slot - block * c.block_size : 0;
  uint32_t *codes = reinterpret_cast<uint32_t *>(
      static_cast<uint8_t *>(is_v ? c.v_codes : c.k_codes) + block * c.code_stride[0] +
      at * c.code_stride[1] + h * c.code_stride[2]);
  uint32_t *params = reinterpret_cast<uint32_t *>(
                         static_cast<__nv_bfloat16 *>(c.params) + block * c.param_stride[0] +
                         at * c.param_stride[1] + h * c.param_stride[2]) + (is_v ? 1 : 0);
  __nv_bfloat16 *x = (is_v ? value + t * v_token + h * v_head : key + t * k_token + h * k_head) + lane * 8;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (STORE) {
    if (slot >= 0) unpack8(*reinterpret_cast<const uint4 *>(x), v);
    uint32_t w, sz;
    kv4_quantise<LANES>(v, w, sz);
    if (slot >= 0) {
      codes[lane] = w;
      if (lane == 0) *params = sz;
    }
  } else {
    if (!in) return;
    if (slot >= 0) {
      const uint32_t w = codes[lane];
      const float2 sz = unpack2(*params);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = fmaf(static_cast<float>((w >> (4 * e)) & 15u), sz.x, sz.y);
    }
    *reinterpret_cast<uint4 *>(x) =
        make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
  }
}

template <bool STORE>
int kv4_rows(const char *what, const b200asr_kv4 &c, void *key, int64_t k_token,
             int64_t k_head, void *value, int64_t v_token, int64_t v_head, const int32_t *slots,
             int num_tokens, int32_t *error_flag, cudaStream_t stream) {
  B200_REQUIRE(num_tokens >= 0, "%s: bad token count", what);
  B200_REQUIRE(c.head_dim == 64 || c.head_dim == 128, "%s: head_dim %d unsupported (64 or 128)",
               what, c.head_dim);
  if (num_tokens == 0) return B200ASR_OK;
  B200_REQUIRE(key && value && slots && c.k_codes && c.v_codes && c.params, "%s: null pointer", what);
  B200_REQUIRE(kv4_cache_ok(c), "%s: cache sizes, or rows not 16-byte (codes) and "
               "8-byte (parameters) aligned", what);
  B200_REQUIRE(aligned16(key) && aligned16(value) && k_token % 8 == 0 && k_head % 8 == 0 &&
                   v_token % 8 == 0 && v_head % 8 == 0,
               "%s: key and value rows must be 16-byte aligned", what);
  const int lanes = c.head_dim / 8;
  const int64_t threads = 2ll * num_tokens * c.num_kv_heads * lanes;
  const int64_t grid = (threads + 255) / 256;
  B200_REQUIRE(grid <= 0x7fffffffll, "%s: too many rows", what);
  auto kfn = lanes == 16 ? kv4_rows_kernel<16, STORE> : kv4_rows_kernel<8, STORE>;
  B200_LAUNCH_CHECK_ERR(
      launch_kernel(kfn, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, true, 1, c,
                    static_cast<__nv_bfloat16 *>(key), k_token, k_head,
                    static_cast<__nv_bfloat16 *>(value), v_token, v_head, slots,
                    static_cast<int64_t>(num_tokens), error_flag),
      what);
  return B200ASR_OK;
}

}  // namespace b200asr

using namespace b200asr;

extern "C" int b200asr_store_kvcache4(const void *key, int64_t key_token_stride,
                                      int64_t key_head_stride, const void *value,
                                      int64_t value_token_stride, int64_t value_head_stride,
                                      const b200asr_kv4 *cache, const int32_t *slot_mapping,
                                      int32_t num_tokens, int32_t *error_flag,
                                      b200asr_stream_t stream) {
  B200_REQUIRE(cache != nullptr, "store_kvcache4: null cache");
  return kv4_rows<true>("store_kvcache4", *cache, const_cast<void *>(key),
                        key_token_stride, key_head_stride, const_cast<void *>(value),
                        value_token_stride, value_head_stride, slot_mapping, num_tokens,
                        error_flag, stream);
}

extern "C" int b200asr_load_kvcache4(const b200asr_kv4 *cache, const int32_t *slots,
                                     int32_t num_tokens, void *key,
                                     int64_t key_token_stride, int64_t key_head_stride, void *value,
                                     int64_t value_token_stride, int64_t value_head_stride,
                                     int32_t *error_flag, b200asr_stream_t stream) {
  B200_REQUIRE(cache != nullptr, "load_kvcache4: null cache");
  return kv4_rows<false>("load_kvcache4", *cache, key, key_token_stride,
                         key_head_stride, value, value_token_stride, value_head_stride, slots,
                         num_tokens, error_flag, stream);
}
