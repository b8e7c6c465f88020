// extern "C" entry points of the 8-bit paged KV cache (include/b200ep.h): argument checks, then the
// launchers of kernels/paged_q8.cu (write, read) and kernels/paged_q8_attn.cu (attention).  No counterpart
// in the reference, whose caches hold the I/O type.
#include <cmath>
#include <cstring>
#include <string>

#include "kernels/paged_q8.cuh"

namespace b200ep {
namespace {

constexpr size_t kCounterBytes = 8192;  // arrival counters at the front of the workspace

int check_geometry(const b200ep_paged_q8_params* p, int dtype, const char* op) {
  const std::string n = op;
  B200EP_CHECK_ARG(p != nullptr, n + ": params is null");
  B200EP_CHECK_ARG(is_float_dtype(dtype), n + ": dtype must be float32, float16 or bfloat16");
  B200EP_CHECK_ARG(p->cache_type == kI8 || p->cache_type == kE4M3, n + ": cache_type must be 3 (int8) or 17 (float8e4m3fn)");
  B200EP_CHECK_ARG(p->head_size == 32 || p->head_size == 64 || p->head_size == 128 || p->head_size == 256,
                   n + ": head_size must be 32, 64, 128 or 256");
  B200EP_CHECK_ARG(p->batch >= 0 && p->num_tokens >= 0 && p->kv_heads > 0 && p->kv_heads <= 65535,
                   n + ": batch, num_tokens >= 0 and 0 < kv_heads < 65536 required");
  B200EP_CHECK_ARG((int64_t)p->num_tokens * 2 * p->kv_heads < (1ll << 31),
                   n + ": num_tokens * kv_heads must be below 2^30");
  B200EP_CHECK_ARG(p->num_tokens == 0 || p->batch > 0, n + ": packed rows need a sequence to belong to");
  B200EP_CHECK_ARG(p->num_blocks > 0 && p->block_size > 0 && p->max_blocks > 0 &&
                       (int64_t)p->num_blocks * p->block_size < (1ll << 31) &&
                       (int64_t)p->num_blocks * p->block_size * p->kv_heads < (1ll << 31),
                   n + ": bad cache / block-table geometry (num_blocks * block_size * kv_heads must be < 2^31)");
  B200EP_CHECK_ARG(!p->do_rotary || (p->rotary_half > 0 && 2 * (int64_t)p->rotary_half <= p->head_size && p->max_seq > 0),
                   n + ": do_rotary needs cos/sin caches of [max_seq, rotary_half <= head_size / 2]");
  return B200EP_OK;
}

bool aligned(const void* a, const void* b, size_t n) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % n == 0;
}

PagedQ8 common(const b200ep_paged_q8_params* p, void* kc, void* vc, float* ks, float* vs, const int32_t* cum,
               const int32_t* past, const int32_t* bt, const void* cos_c, const void* sin_c, int dtype) {
  PagedQ8 a{};
  a.kc = static_cast<uint8_t*>(kc), a.vc = static_cast<uint8_t*>(vc), a.kscale = ks, a.vscale = vs;
  a.cum = cum, a.past = past, a.bt = bt, a.cos_c = cos_c, a.sin_c = sin_c, a.err = device_error_slot();
  a.batch = p->batch, a.ntok = p->num_tokens, a.H = p->num_heads, a.HK = p->kv_heads, a.D = p->head_size;
  a.nblocks = p->num_blocks, a.bs = p->block_size, a.maxb = p->max_blocks, a.max_seq = p->max_seq;
  a.bs_shift = -1;
  for (int t = 0; t < 31; ++t)
    if (a.bs == 1 << t) a.bs_shift = t;
  a.half = p->rotary_half, a.rot = p->do_rotary ? 1 : 0, a.inter = p->interleaved ? 1 : 0;
  a.dtype = dtype, a.ctype = p->cache_type;
  a.ks = p->key_stride ? p->key_stride : (int64_t)p->kv_heads * p->head_size;
  a.vs = p->value_stride ? p->value_stride : (int64_t)p->kv_heads * p->head_size;
  a.qs = p->query_stride ? p->query_stride : (int64_t)p->num_heads * p->head_size;
  return a;
}

}  // namespace
}  // namespace b200ep

using namespace b200ep;

extern "C" B200EP_API int b200ep_paged_kv_quantize(const b200ep_paged_q8_params* p, const void* key, const void* value,
                                                   void* key_cache, void* value_cache, float* key_scales,
                                                   float* value_scales, const int32_t* cumulative_seqlens,
                                                   const int32_t* past_seqlens, const int32_t* block_table,
                                                   const void* cos_cache, const void* sin_cache, int dtype,
                                                   void* stream) {
  try {
    if (int rc = check_geometry(p, dtype, "PagedKvQuantize")) return rc;
    if (p->num_tokens == 0) return B200EP_OK;
    B200EP_CHECK_ARG(key && value && key_cache && value_cache && key_scales && value_scales && cumulative_seqlens &&
                         past_seqlens && block_table && (!p->do_rotary || (cos_cache && sin_cache)),
                     "PagedKvQuantize: null pointer");
    B200EP_CHECK_ARG(aligned(key_cache, value_cache, 16) && aligned(key_scales, value_scales, 4),
                     "PagedKvQuantize: key / value caches must be 16-byte aligned");
    const int64_t dense = (int64_t)p->kv_heads * p->head_size;
    B200EP_CHECK_ARG((!p->key_stride || p->key_stride >= dense) && (!p->value_stride || p->value_stride >= dense),
                     "PagedKvQuantize: row strides must be at least kv_heads * head_size");
    PagedQ8 a = common(p, key_cache, value_cache, key_scales, value_scales, cumulative_seqlens, past_seqlens,
                       block_table, cos_cache, sin_cache, dtype);
    a.k = key, a.v = value;
    return cuda_status(launch_paged_q8_write(a, static_cast<cudaStream_t>(stream)), "PagedKvQuantize launch");
  } catch (const std::exception& e) {
    return set_error(B200EP_EINTERNAL, std::string("exception: ") + e.what());
  }
}

extern "C" B200EP_API int b200ep_paged_kv_dequantize(const b200ep_paged_q8_params* p, const void* key_cache,
                                                     const void* value_cache, const float* key_scales,
                                                     const float* value_scales, const int32_t* seqlens,
                                                     const int32_t* block_table, void* key, void* value, int64_t cap,
                                                     int dtype, void* stream) {
  try {
    if (int rc = check_geometry(p, dtype, "PagedKvDequantize")) return rc;
    B200EP_CHECK_ARG(p->batch <= 65535, "PagedKvDequantize: at most 65535 sequences");
    B200EP_CHECK_ARG(cap >= 0 && cap < (1ll << 31), "PagedKvDequantize: cap must lie in [0, 2^31)");
    if (p->batch == 0 || cap == 0) return B200EP_OK;
    B200EP_CHECK_ARG(key_cache && value_cache && key_scales && value_scales && seqlens && block_table && key && value,
                     "PagedKvDequantize: null pointer");
    B200EP_CHECK_ARG(aligned(key_cache, value_cache, 16) && aligned(key, value, 16),
                     "PagedKvDequantize: caches and outputs must be 16-byte aligned");
    PagedQ8Read a{};
    a.kc = static_cast<const uint8_t*>(key_cache), a.vc = static_cast<const uint8_t*>(value_cache);
    a.kscale = key_scales, a.vscale = value_scales, a.lens = seqlens, a.bt = block_table;
    a.k = key, a.v = value, a.err = device_error_slot();
    a.batch = p->batch, a.HK = p->kv_heads, a.D = p->head_size, a.nblocks = p->num_blocks, a.bs = p->block_size;
    a.maxb = p->max_blocks, a.dtype = dtype, a.ctype = p->cache_type, a.cap = cap;
    return cuda_status(launch_paged_q8_read(a, static_cast<cudaStream_t>(stream)), "PagedKvDequantize launch");
  } catch (const std::exception& e) {
    return set_error(B200EP_EINTERNAL, std::string("exception: ") + e.what());
  }
}

extern "C" B200EP_API size_t b200ep_paged_attention_quantized_workspace_size(const b200ep_paged_q8_params* p) {
  if (!p || p->kv_heads <= 0 || p->num_heads <= 0 || p->num_heads % p->kv_heads || p->head_size <= 0) return 0;
  const int heads = paged_q8_heads_per_cta(p->head_size, p->num_heads / p->kv_heads);
  return kCounterBytes + (size_t)2 * paged_q8_max_ctas() * heads * (p->head_size + 2) * sizeof(float);
}

extern "C" B200EP_API int b200ep_paged_attention_quantized(
    const b200ep_paged_q8_params* p, const void* query, const void* key, const void* value, void* key_cache,
    void* value_cache, float* key_scales, float* value_scales, const int32_t* cumulative_seqlens,
    const int32_t* past_seqlens, const int32_t* block_table, const void* cos_cache, const void* sin_cache, void* out,
    int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  try {
    if (int rc = check_geometry(p, dtype, "PagedAttentionQuantized")) return rc;
    B200EP_CHECK_ARG(p->num_heads > 0 && p->num_heads % p->kv_heads == 0,
                     "PagedAttentionQuantized: num_heads must be a positive multiple of kv_heads");
    B200EP_CHECK_ARG((key == nullptr) == (value == nullptr),
                     "PagedAttentionQuantized: key and value come together, or neither (rows already written)");
    if (p->num_tokens == 0) return B200EP_OK;
    B200EP_CHECK_ARG(query && key_cache && value_cache && key_scales && value_scales && cumulative_seqlens &&
                         past_seqlens && block_table && out && (!p->do_rotary || (cos_cache && sin_cache)),
                     "PagedAttentionQuantized: null pointer");
    B200EP_CHECK_ARG(aligned(key_cache, value_cache, 16) && aligned(key_scales, value_scales, 4),
                     "PagedAttentionQuantized: key / value caches must be 16-byte aligned");
    const int64_t dense = (int64_t)p->kv_heads * p->head_size;
    B200EP_CHECK_ARG((!p->query_stride || p->query_stride >= (int64_t)p->num_heads * p->head_size) &&
                         (!p->key_stride || p->key_stride >= dense) && (!p->value_stride || p->value_stride >= dense),
                     "PagedAttentionQuantized: row strides must be at least heads * head_size");
    B200EP_CHECK_ARG(aligned(out, nullptr, 16), "PagedAttentionQuantized: out must be 16-byte aligned");
    const size_t need = b200ep_paged_attention_quantized_workspace_size(p);
    B200EP_CHECK_ARG(workspace && workspace_bytes >= need && aligned(workspace, nullptr, 16),
                     "PagedAttentionQuantized: a 16-byte aligned workspace of " + std::to_string(need) +
                         " bytes is needed");
    PagedQ8 a = common(p, key_cache, value_cache, key_scales, value_scales, cumulative_seqlens, past_seqlens,
                       block_table, cos_cache, sin_cache, dtype);
    a.q = query, a.k = key, a.v = value, a.out = out;
    a.G = p->num_heads / p->kv_heads;
    a.scale = p->scale != 0.f ? p->scale : 1.f / std::sqrt((float)p->head_size);
    a.ctas = paged_q8_max_ctas();
    B200EP_CHECK_ARG((size_t)a.ctas * sizeof(int) <= kCounterBytes, "PagedAttentionQuantized: device has too many SMs");
    a.counters = static_cast<int*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (key)
      if (cudaError_t e = launch_paged_q8_write(a, st)) return cuda_status(e, "PagedAttentionQuantized write");
    return cuda_status(launch_paged_q8_attn(a, key != nullptr, st), "PagedAttentionQuantized launch");
  } catch (const std::exception& e) {
    return set_error(B200EP_EINTERNAL, std::string("exception: ") + e.what());
  }
}
