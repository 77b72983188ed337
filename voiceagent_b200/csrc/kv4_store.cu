// Rows into and out of the 4-bit paged KV cache (kv4.cuh has the format).
//
// store_kvcache4 <- store_kvcache (layers/attention.py:52-67), quantising on the way
// load_kvcache4     its inverse: cached rows gathered by slot as bf16
//
// Both are bound by memory: a row is read once and written once. A group of D / 16 lanes takes
// one (token, head, K or V) row, 32 bytes of bf16 and 8 bytes of codes per lane, so every access
// of a group is one contiguous run; the row's extremes are a shuffle reduction. 16 values per
// lane, not 8, halve what a row costs beside its values (the scale, the addresses). 8192 rows of
// 8 heads of 128, stored and read back: 23.4 us, 3.6 TB/s of the 13.2 us that the bytes alone would
// take; the extremes, the exact quotients and the addresses fill the issue slots of the first half.
#include "kv4.cuh"

namespace b200asr {

template <int LANES, bool STORE>
__global__ void __launch_bounds__(256) kv4_rows_kernel(
    const b200asr_kv4 c, int bs_shift, __nv_bfloat16 *key, int64_t k_token, int64_t k_head,
    __nv_bfloat16 *value, int64_t v_token, int64_t v_head, const int32_t *__restrict__ slots,
    int num_tokens, int32_t *error_flag) {
  pdl_trigger();
  pdl_wait();
  const unsigned row = (blockIdx.x * 256u + threadIdx.x) / LANES;
  const int lane = threadIdx.x & (LANES - 1);
  const unsigned per_token = 2u * c.num_kv_heads;
  const int t = static_cast<int>(row / per_token);
  const bool in = t < num_tokens;  // whole groups: the shuffles below need every lane
  int h = static_cast<int>(row - t * per_token);
  const bool is_v = h >= c.num_kv_heads;
  if (is_v) h -= c.num_kv_heads;
  int slot = in ? slots[t] : -1;
  __nv_bfloat16 *x = (is_v ? value + t * v_token + h * v_head : key + t * k_token + h * k_head) + lane * 16;
  uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (STORE && in) {
    v[0] = *reinterpret_cast<const uint4 *>(x);
    v[1] = *reinterpret_cast<const uint4 *>(x + 8);
  }
  const int block = slot < 0 ? 0 : bs_shift >= 0 ? slot >> bs_shift : slot / c.block_size;
  if (slot != -1 && (slot < 0 || block >= c.num_blocks)) {
    if (lane == 0) raise_flag(error_flag, B200ASR_DEVERR_SLOT);
    slot = -1;
  }
  const int at = slot < 0 ? 0 : slot - block * c.block_size;
  const int64_t code_off = block * c.code_stride[0] + at * c.code_stride[1] + h * c.code_stride[2];
  uint2 *codes = reinterpret_cast<uint2 *>(static_cast<uint8_t *>(is_v ? c.v_codes : c.k_codes) + code_off);
  uint32_t *params = reinterpret_cast<uint32_t *>(
                         static_cast<__nv_bfloat16 *>(c.params) + block * c.param_stride[0] +
                         at * c.param_stride[1] + h * c.param_stride[2]) + (is_v ? 1 : 0);
  if (STORE) {
    const uint32_t words[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
    uint32_t w[2], sz;
    kv4_quantise<LANES, 8>(words, w, sz);
    if (slot >= 0) {
      codes[lane] = make_uint2(w[0], w[1]);
      if (lane == 0) *params = sz;
    }
  } else {
    if (!in) return;
    if (slot >= 0) {
      const uint2 w = codes[lane];
      const float2 sz = unpack2(*params);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t word = i ? w.y : w.x;
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)  // whole numbers below 16 by the low bits of 2^23
          y[e] = pack2(fmaf(__uint_as_float(0x4b000000u | ((word >> (8 * e)) & 15u)) - 8388608.f, sz.x, sz.y),
                       fmaf(__uint_as_float(0x4b000000u | ((word >> (8 * e + 4)) & 15u)) - 8388608.f, sz.x, sz.y));
        v[i] = make_uint4(y[0], y[1], y[2], y[3]);
      }
    }
    *reinterpret_cast<uint4 *>(x) = v[0];
    *reinterpret_cast<uint4 *>(x + 8) = v[1];
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
  const int lanes = c.head_dim / 16;
  const int64_t threads = 2ll * num_tokens * c.num_kv_heads * lanes;
  const int64_t grid = (threads + 255) / 256;
  B200_REQUIRE(grid < (1ll << 24), "%s: too many rows", what);  // row indices stay in 32 bits
  const int bs = c.block_size, bs_shift = (bs & (bs - 1)) == 0 ? __builtin_ctz(bs) : -1;
  auto kfn = lanes == 8 ? kv4_rows_kernel<8, STORE> : kv4_rows_kernel<4, STORE>;
  B200_LAUNCH_CHECK_ERR(
      launch_kernel(kfn, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, true, 1, c, bs_shift,
                    static_cast<__nv_bfloat16 *>(key), k_token, k_head,
                    static_cast<__nv_bfloat16 *>(value), v_token, v_head, slots,
                    num_tokens, error_flag),
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
