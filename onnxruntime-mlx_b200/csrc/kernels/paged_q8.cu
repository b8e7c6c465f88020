// Writing and reading the 8-bit paged KV cache (layout: paged_q8.cuh).
//
// paged_q8_write_kernel — new key / value rows into their pages.  For a row x of one kv head (the key
//   row after RoPE at its position, in fp32), with F = 127 (int8) or 448 (e4m3):
//     a = max |x|,  scale = a / F,  code = round_to_nearest_even(x F / a).
//   For fp16 / bf16 rows without RoPE, x F is exact in fp32 (11 + 7 bits; 448 = 7 * 2^6) and a / x are
//   integers of at most 11 bits times a power of two, so the quotient is either a rounding point of
//   the code or further from it than fp32's rounding: the codes are those of the formula in exact
//   arithmetic.  a = 0 gives code 0 and scale 0; a row that holds an infinity or a NaN gets scale NaN
//   and reads back as NaN.
//   D / 8 lanes hold one row, 8 elements each: one 16-byte load (16-bit types), an xor-shuffle maximum,
//   one 8-byte store.  Keys and values of a token are handled by one CTA.
// paged_q8_read_kernel — sequences gathered into [B, HK, cap, D] rows of a float type (the layout of
//   GroupQueryAttention's shared buffers); rows at and past a sequence's length are zeros.
// Both are bound by HBM: 2 B + 1 B (+ 4 / D) per element each way for 16-bit types.
#include "paged_q8.cuh"

#include <cuda_fp8.h>

#include <type_traits>

namespace b200ep {
namespace {

__device__ __forceinline__ void store_bytes8(uint8_t* dst, uint32_t a, uint32_t b) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(a, b);
}

// 8 consecutive elements to fp32; `vec`: the address is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    uint4 w[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    const T* h = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f<T>(h[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f<T>(p[e]);
  }
}

// RoPE of the 8 elements [d0, d0 + 8) of a row held 8 per lane by D / 8 lanes; every lane of the row
// takes part.  Products and sums are rounded one by one (no fused multiply-add), as PagedAttention
// rounds them.
template <typename T, int D>
__device__ __forceinline__ void rope8(float (&x)[8], const T* row, int d0, const PagedQ8& kp, int pos, bool cvec) {
  const T* C = static_cast<const T*>(kp.cos_c) + (size_t)pos * kp.half;
  const T* S = static_cast<const T*>(kp.sin_c) + (size_t)pos * kp.half;
  if (kp.inter) {  // pairs (2i, 2i + 1) lie in one lane
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int i = (d0 + e) >> 1;
      if (i >= kp.half) break;
      const float c = to_f<T>(C[i]), s = to_f<T>(S[i]), a = x[e], b = x[e + 1];
      x[e] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
      x[e + 1] = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
    }
    return;
  }
  if (kp.half % 8 == 0) {  // the partner's 8 elements are another lane's
    const bool in = d0 < 2 * kp.half, first = d0 < kp.half;
    const int step = kp.half / 8, lane = threadIdx.x & (D / 8 - 1);
    const int src = !in ? lane : first ? lane + step : lane - step;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], src, D / 8);
    if (!in) return;
    float c[8], s[8];
    const int i0 = first ? d0 : d0 - kp.half;
    load8<T>(C + i0, cvec, c);
    load8<T>(S + i0, cvec, s);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = first ? __fsub_rn(__fmul_rn(x[e], c[e]), __fmul_rn(y[e], s[e]))
                   : __fadd_rn(__fmul_rn(x[e], c[e]), __fmul_rn(y[e], s[e]));
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {  // any other half: the partner is read again
    const int i = d0 + e;
    if (i >= 2 * kp.half) break;
    const bool first = i < kp.half;
    const int pi = first ? i : i - kp.half;
    const float y = to_f<T>(row[first ? i + kp.half : pi]), c = to_f<T>(C[pi]), s = to_f<T>(S[pi]);
    x[e] = first ? __fsub_rn(__fmul_rn(x[e], c), __fmul_rn(y, s)) : __fadd_rn(__fmul_rn(x[e], c), __fmul_rn(y, s));
  }
}

template <int CT>
__device__ __forceinline__ uint32_t code_of(float x, float amax) {
  if constexpr (CT == kI8) {
    return (uint32_t)__float2int_rn(__fdiv_rn(__fmul_rn(x, 127.f), amax)) & 0xffu;
  } else {
    return __nv_cvt_float_to_fp8(__fdiv_rn(__fmul_rn(x, 448.f), amax), __NV_SATFINITE, __NV_E4M3);
  }
}

constexpr int kWriteThreads = 128;

template <typename T, int D, int CT>
__global__ void __launch_bounds__(kWriteThreads) paged_q8_write_kernel(PagedQ8 kp, int vec) {
  constexpr int L = D / 8;  // lanes of a row
  constexpr float F = CT == kI8 ? 127.f : 448.f;
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x;
  if (kp.counters && i == 0)  // the attention launch that follows counts arrivals from zero
    for (int t = threadIdx.x; t < kp.ctas; t += kWriteThreads) kp.counters[t] = 0;
  const int b = q8_seq(kp.cum, kp.batch, i);
  const int pos = b >= 0 ? __ldg(kp.past + b) + (i - __ldg(kp.cum + b)) : -1;
  const bool pos_ok = pos >= 0 && !(kp.rot && pos >= kp.max_seq);
  const int row0 = pos_ok ? q8_row(kp.bt, kp.maxb, kp.nblocks, kp.bs, kp.HK, b, 0, pos) : -1;
  if (row0 < 0) {
    if (threadIdx.x == 0) report_device_error(kp.err, kErrPagedQ8, i);
    return;
  }
  const int lane = threadIdx.x & (L - 1), d0 = lane * 8;
  // row r < HK: the key row of kv head r; then the value rows.  All lanes of a warp stay in the loop
  // (the shuffles name the full warp).
  const int rows = 2 * kp.HK, per = kWriteThreads / L;
  for (int r0 = 0; r0 < rows; r0 += per) {
    const int r = r0 + (int)threadIdx.x / L;
    const bool live = r < rows, is_k = r < kp.HK;
    const int h = !live ? 0 : is_k ? r : r - kp.HK;
    const T* src = (is_k || !live ? static_cast<const T*>(kp.k) + (size_t)i * kp.ks
                                  : static_cast<const T*>(kp.v) + (size_t)i * kp.vs) + (size_t)h * D;
    float x[8];
    load8<T>(src + d0, vec & 1, x);
    if (kp.rot) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[e];
      rope8<T, D>(y, src, d0, kp, pos, vec & 2);
      if (is_k)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e];
    }
    uint32_t m = 0;  // |x| as bits: ordered like the values, a NaN above all
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!live) continue;
    float amax = __uint_as_float(m), scale = __fdiv_rn(amax, F);
    if (m >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);
    if (amax > 1e30f) {  // x F stays finite (a power of two: exact)
      amax *= 0x1p-32f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= 0x1p-32f;
    }
    uint32_t w[2] = {0, 0};
    if (m)
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e >> 2] |= code_of<CT>(x[e], amax) << (8 * (e & 3));
    const int64_t row = row0 + (int64_t)h * kp.bs;
    store_bytes8((is_k ? kp.kc : kp.vc) + row * D + d0, w[0], w[1]);
    if (lane == 0) (is_k ? kp.kscale : kp.vscale)[row] = scale;
  }
}

// one code to its value (before the scale)
template <int CT>
__device__ __forceinline__ float value_of(uint32_t byte) {
  if constexpr (CT == kI8) {
    return (float)(int8_t)byte;
  } else {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
  }
}

constexpr int kReadThreads = 256;
constexpr int kReadRows = 64;  // positions of one CTA

template <typename T, int D, int CT>
__global__ void __launch_bounds__(kReadThreads) paged_q8_read_kernel(PagedQ8Read kp) {
  constexpr int L = D / 8, PER = kReadThreads / L;  // lanes of a row; rows of a pass
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t t0 = (int64_t)blockIdx.x * kReadRows;
  const int n = __ldg(kp.lens + b), lane = threadIdx.x & (L - 1);
  if (threadIdx.x == 0 && t0 == 0 && h == 0 && (n < 0 || n > kp.cap)) report_device_error(kp.err, kErrPagedQ8, b);
  bool bad = false;
  for (int64_t t = t0 + threadIdx.x / L; t < t0 + kReadRows && t < kp.cap; t += PER) {
    const int row = t < n ? q8_row(kp.bt, kp.maxb, kp.nblocks, kp.bs, kp.HK, b, h, (int)t) : -1;
    bad |= t < n && row < 0;
    const size_t o = (((size_t)b * kp.HK + h) * kp.cap + t) * D + lane * 8;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      alignas(16) T y[8];
      uint2 w = make_uint2(0, 0);
      float scale = 0.f;
      if (row >= 0) {
        w = __ldg(reinterpret_cast<const uint2*>((s ? kp.vc : kp.kc) + (size_t)row * D) + lane);
        scale = __ldg((s ? kp.vscale : kp.kscale) + row);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        y[e] = from_f<T>(row >= 0 ? value_of<CT>(((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 0xffu) * scale : 0.f);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(s ? kp.v : kp.k) + o);
#pragma unroll
      for (int u = 0; u < (int)sizeof(T) / 2; ++u) dst[u] = reinterpret_cast<const uint4*>(y)[u];
    }
  }
  if (bad && lane == 0) report_device_error(kp.err, kErrPagedQ8, b);
}

bool aligned16(const void* p, int64_t stride_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
}

template <typename T, int D, int CT>
cudaError_t write_t(const PagedQ8& a, cudaStream_t st) {
  const int es = (int)sizeof(T);
  int vec = aligned16(a.k, a.ks * es) && aligned16(a.v, a.vs * es) ? 1 : 0;
  if (a.rot && aligned16(a.cos_c, (int64_t)a.half * es) && aligned16(a.sin_c, (int64_t)a.half * es)) vec |= 2;
  return launch_k(paged_q8_write_kernel<T, D, CT>, dim3((unsigned)a.ntok), dim3(kWriteThreads), 0, st, a, vec);
}

template <typename T, int D, int CT>
cudaError_t read_t(const PagedQ8Read& a, cudaStream_t st) {
  return launch_k(paged_q8_read_kernel<T, D, CT>,
                  dim3((unsigned)div_up(a.cap, kReadRows), (unsigned)a.HK, (unsigned)a.batch), dim3(kReadThreads), 0,
                  st, a);
}

template <typename T, int CT, typename A>
cudaError_t by_head(const A& a, cudaStream_t st) {
  constexpr bool write = std::is_same<A, PagedQ8>::value;
#define B200EP_Q8_HEAD(DD)                                  \
  case DD:                                                  \
    if constexpr (write) return write_t<T, DD, CT>(a, st);  \
    else return read_t<T, DD, CT>(a, st);
  switch (a.D) {
    B200EP_Q8_HEAD(32)
    B200EP_Q8_HEAD(64)
    B200EP_Q8_HEAD(128)
    B200EP_Q8_HEAD(256)
  }
#undef B200EP_Q8_HEAD
  return cudaErrorInvalidValue;
}

template <typename A>
cudaError_t by_type(const A& a, cudaStream_t st) {
  const bool i8 = a.ctype == kI8;
  switch (a.dtype) {
    case kF32: return i8 ? by_head<float, kI8>(a, st) : by_head<float, kE4M3>(a, st);
    case kF16: return i8 ? by_head<__half, kI8>(a, st) : by_head<__half, kE4M3>(a, st);
    case kBF16: return i8 ? by_head<__nv_bfloat16, kI8>(a, st) : by_head<__nv_bfloat16, kE4M3>(a, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_paged_q8_write(const PagedQ8& a, cudaStream_t st) { return by_type(a, st); }
cudaError_t launch_paged_q8_read(const PagedQ8Read& a, cudaStream_t st) { return by_type(a, st); }

}  // namespace b200ep
