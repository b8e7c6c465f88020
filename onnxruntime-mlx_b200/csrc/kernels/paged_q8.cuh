// Shared pieces of the 8-bit paged KV cache: its geometry, the control-tensor lookups and the
// internal launchers (csrc/paged_q8.cu validates and calls them).
//
// Layout: codes [num_blocks, kv_heads, block_size, head_size] (1 byte each), scales fp32
// [num_blocks, kv_heads, block_size]; value = code * scale.  The rows of one kv head within a page
// are contiguous (unlike the 16-bit PagedAttention cache), so a CTA that attends for one kv head
// reads block_size * head_size contiguous bytes per page.
#pragma once

#include <cstring>

#include "../common.cuh"

namespace b200ep {

// a position or page outside the tables (detail: packed row or sequence); a bounded wait that ran out
enum { kErrPagedQ8 = 122, kErrPagedQ8Timeout = 123 };
enum { kI8 = 3, kE4M3 = 17 };  // cache_type: ONNX TensorProto INT8 / FLOAT8E4M3FN

struct PagedQ8 {
  const void *q, *k, *v;  // packed rows, strides in elements
  int64_t qs, ks, vs;
  uint8_t *kc, *vc;
  float *kscale, *vscale;
  const int32_t *cum, *past, *bt;
  const void *cos_c, *sin_c;
  void* out;
  DeviceErrorSlot* err;
  int batch, ntok, H, HK, D, G, nblocks, bs, bs_shift, maxb, max_seq, half, rot, inter;
  int dtype, ctype;
  float scale;
  // attention work split (see paged_q8_attn.cu)
  float* part;      // [2 * ctas][heads per CTA][D + 2]
  int* counters;    // [ctas], zero before the attention launch
  int ctas;
};

struct PagedQ8Read {
  const uint8_t *kc, *vc;
  const float *kscale, *vscale;
  const int32_t *lens, *bt;
  void *k, *v;
  DeviceErrorSlot* err;
  int batch, HK, D, nblocks, bs, maxb, dtype, ctype;
  int64_t cap;
};

// The sequence of packed row i (cum[b] <= i < cum[b + 1]), or -1.  One new token per sequence (row i
// is sequence i) is the usual call and needs no search.
__device__ __forceinline__ int q8_seq(const int32_t* cum, int batch, int i) {
  if (i < batch && __ldg(cum + i) == i && __ldg(cum + i + 1) == i + 1) return i;
  int lo = 0, hi = batch;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(cum + mid) <= i) lo = mid;
    else hi = mid - 1;
  }
  if (lo >= batch || __ldg(cum + lo) > i || i >= __ldg(cum + lo + 1)) return -1;
  return lo;
}

// Row (of block_size-row pages of one kv head) of position pos of sequence b for kv head h, or -1.  shift: log2 of
// the block size where that is a power of two, else -1.
__device__ __forceinline__ int q8_row(const int32_t* bt, int maxb, int nblocks, int bs, int HK, int b, int h, int pos,
                                      int shift = -1) {
  const int blk = shift >= 0 ? pos >> shift : pos / bs;
  if (pos < 0 || blk >= maxb) return -1;
  const int phys = __ldg(bt + (size_t)b * maxb + blk);
  return phys < 0 || phys >= nblocks ? -1 : (phys * HK + h) * bs + (pos - blk * bs);
}

// The bits of two fp16 numbers, and back.
__device__ __forceinline__ uint32_t word_of(__half2 h) {
  uint32_t w;
  memcpy(&w, &h, 4);
  return w;
}
__device__ __forceinline__ __half2 half2_of(uint32_t w) {
  __half2 h;
  memcpy(&h, &w, 4);
  return h;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// The four codes of a word as two f16x2 (codes 0, 1 and 2, 3).
template <int CT>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& h01, uint32_t& h23) {
  if constexpr (CT == kI8) {
    // 0x6400 | (code + 128) is 1024 + 128 + code in fp16
    const uint32_t x = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    h01 = word_of(__hsub2(half2_of(prmt(x, 0x64646464u, 0x4140)), bias));
    h23 = word_of(__hsub2(half2_of(prmt(x, 0x64646464u, 0x4342)), bias));
  } else {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(h01), "=r"(h23) : "r"(w));
  }
}

int paged_q8_max_ctas();                                 // upper bound of the attention grid
int paged_q8_heads_per_cta(int D, int G);                // query heads that share one K / V stream
cudaError_t launch_paged_q8_write(const PagedQ8& a, cudaStream_t st);
cudaError_t launch_paged_q8_read(const PagedQ8Read& a, cudaStream_t st);
cudaError_t launch_paged_q8_attn(const PagedQ8& a, bool appended, cudaStream_t st);

}  // namespace b200ep
