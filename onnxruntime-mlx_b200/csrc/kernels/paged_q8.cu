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
//   one 8-byte store.
// paged_q8_read_kernel — sequences gathered into [B, HK, cap, D] rows of a float type (the layout of
//   GroupQueryAttention's shared buffers); rows at and past a sequence's length are zeros.  A CTA looks its 64
//   positions up once and has all its 16-byte loads on their way before the first is used: 16 sequences of 8192
//   tokens (8 kv heads, head size 128) to bf16 in 143 us, 87 % of the copy rate.
// Bytes of both: 2 B + 1 B (+ 4 / D) per element each way for 16-bit types.  Reading is bound by HBM; writing by
// its instructions (90 us for 32768 tokens of that shape, 35 %).
#include "paged_q8.cuh"

#include <cuda_fp8.h>

#include <cstring>
#include <type_traits>

namespace b200ep {
namespace {

// 8 consecutive elements to fp32; `vec`: the address is 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    uint4 w[sizeof(T) / 2];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    T h[8];
    memcpy(h, w, sizeof(h));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f<T>(h[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f<T>(p[e]);
  }
}

// RoPE of the 8 elements [d0, d0 + 8) of a row, in pairs (2i, 2i + 1) or from halves of any length.  Products and
// sums are rounded one by one (no fused multiply-add), as PagedAttention rounds them.
template <typename T, int D>
__device__ __forceinline__ void rope8(float (&x)[8], const T* row, int d0, const PagedQ8& kp, int pos) {
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

// The larger of two numbers, a NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// x F / amax to codes, 8 of them.  With r = F / amax to two last places, x r is within 2^-21 of the true quotient:
// where that cannot move any of them over a rounding point it decides, else the division does.  Adding 1.5 2^23
// rounds to a whole number whose low byte is the code (the conversion instructions run at an eighth of the rate).
template <int CT>
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float amax) {
  uint32_t w[2];
  bool near_tie = false;
  const float r = __fdividef(CT == kI8 ? 127.f : 448.f, amax);
  if constexpr (CT == kI8) {
    constexpr float kMagic = 12582912.f;
    float y[8], off = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = fmaf(x[e], r, kMagic);
      off = fmaxf(off, fabsf(fmaf(x[e], r, kMagic - y[e])));
    }
    near_tie = !(off < 0.4999f);
    if (near_tie)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __fadd_rn(__fdiv_rn(__fmul_rn(x[e], 127.f), amax), kMagic);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      w[q] = prmt(prmt(__float_as_uint(y[4 * q]), __float_as_uint(y[4 * q + 1]), 0x0040),
                  prmt(__float_as_uint(y[4 * q + 2]), __float_as_uint(y[4 * q + 3]), 0x0040), 0x5410);
    }
  } else {
    const float lo = r * 0.9999995f, hi = r * 1.0000005f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(x[e] * lo, x[e + 1] * lo), __NV_SATFINITE, __NV_E4M3);
      const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(x[e] * hi, x[e + 1] * hi), __NV_SATFINITE, __NV_E4M3);
      near_tie |= a != b;
      w[e >> 2] = e & 2 ? prmt(w[e >> 2], a, 0x5410) : a;
    }
    if (near_tie)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(__fmul_rn(x[e], 448.f), amax),
                                                                __fdiv_rn(__fmul_rn(x[e + 1], 448.f), amax)),
                                                    __NV_SATFINITE, __NV_E4M3);
        w[e >> 2] = e & 2 ? prmt(w[e >> 2], c, 0x5410) : c;
      }
  }
  return make_uint2(w[0], w[1]);
}

constexpr int kWriteThreads = 256;

// The rows of all tokens as one list (the HK key rows of a token, then its HK value rows), one to D / 8 lanes.  The
// page rows of a CTA's tokens are looked up once, while its loads are on their way.  Instructions bound it (about 30
// an element: two kinds of row, RoPE, the maximum, the rounding), so more rows a thread (2 or 4, measured) only
// cost occupancy: 32768 tokens of 8 kv heads, head size 128, fp16: 91 us with one, 99 and 103 us with two and four.
template <typename T, int D, int CT>
__global__ void __launch_bounds__(kWriteThreads, sizeof(T) == 2 ? 8 : 6) paged_q8_write_kernel(PagedQ8 kp, int vec) {
  constexpr int L = D / 8, ROWS = kWriteThreads / L;  // lanes of a row; rows
  constexpr float F = CT == kI8 ? 127.f : 448.f;
  __shared__ int2 tok_s[ROWS];  // a token's page row (-1: none) and position
  pdl_wait();
  pdl_trigger();
  if (kp.counters && blockIdx.x == 0)  // the attention launch that follows counts arrivals from zero
    for (int t = threadIdx.x; t < kp.ctas; t += kWriteThreads) kp.counters[t] = 0;
  const uint32_t r0 = blockIdx.x * ROWS, total = (uint32_t)kp.ntok * 2 * kp.HK, hk2 = 2 * kp.HK;  // (below 2^31)
  const int first = (int)(r0 / hk2), ntok = (int)((min(total, r0 + ROWS) - 1) / hk2) - first + 1;
  const int lane = threadIdx.x & (L - 1), d0 = lane * 8;
  const uint32_t r = r0 + threadIdx.x / L;
  const bool live = r < total;
  const int i = (int)((live ? r : r0) / hk2), hd = (int)((live ? r : r0) - i * hk2);
  const bool is_k = hd < kp.HK;
  const int h = is_k ? hd : hd - kp.HK;
  const T* src = (is_k ? static_cast<const T*>(kp.k) + (size_t)i * kp.ks : static_cast<const T*>(kp.v) + (size_t)i * kp.vs) +
                 (size_t)h * D;
  uint4 raw[sizeof(T) / 2];
  if (vec & 1) {
#pragma unroll
    for (int w = 0; w < (int)sizeof(T) / 2; ++w) raw[w] = __ldg(reinterpret_cast<const uint4*>(src + d0) + w);
  } else {
    T one[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) one[e] = src[d0 + e];
    memcpy(raw, one, sizeof(one));
  }
  // a warp a token: the sequence is the number of sequences that end at or before the row (one look at 32 ends at once,
  // where a search would wait for each of its steps)
  for (int q = threadIdx.x >> 5; q < ntok; q += kWriteThreads / 32) {
    const int t = first + q, ln = threadIdx.x & 31;
    int b = 0;
    for (int b0 = 0; b0 < kp.batch; b0 += 32) {
      const bool ends = b0 + ln < kp.batch && __ldg(kp.cum + b0 + ln + 1) <= t;
      const int n = __popc(__ballot_sync(0xffffffffu, ends));
      b += n;
      if (n < 32) break;
    }
    if (ln) continue;
    int pos = -1, row = -1;
    if (b < kp.batch) pos = __ldg(kp.past + b) + (t - __ldg(kp.cum + b));
    if (t >= __ldg(kp.cum) && pos >= 0 && !(kp.rot && pos >= kp.max_seq))
      row = q8_row(kp.bt, kp.maxb, kp.nblocks, kp.bs, kp.HK, b, 0, pos);
    if (row < 0) report_device_error(kp.err, kErrPagedQ8, t);
    tok_s[q] = make_int2(row, pos);
  }
  __syncthreads();
  const int2 at = live ? tok_s[i - first] : make_int2(-1, 0);
  const bool turn = kp.rot && is_k && at.x >= 0;
  float x[8];
  {
    T one[8];
    memcpy(one, raw, sizeof(one));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f<T>(one[e]);
  }
  if ((vec & 2) && __any_sync(0xffffffffu, turn)) {  // halves of whole 8-element chunks, aligned rows: the partner's elements are another lane's
    const bool turned = d0 < 2 * kp.half, lower = d0 < kp.half;
    const int step = kp.half / 8, from = !turned ? lane : lower ? lane + step : lane - step;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], from, L);
    if (turn && turned) {
      const size_t o = (size_t)at.y * kp.half + (lower ? d0 : d0 - kp.half);
      float c[8], s[8];
      load8<T>(static_cast<const T*>(kp.cos_c) + o, true, c);
      load8<T>(static_cast<const T*>(kp.sin_c) + o, true, s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = __fmul_rn(x[e], c[e]), b = __fmul_rn(y[e], s[e]);
        x[e] = __fadd_rn(a, lower ? -b : b);
      }
    }
  } else if (turn) {
    rope8<T, D>(x, src, d0, kp, at.y);
  }
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = max_nan(amax, fabsf(x[e]));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (at.x < 0) return;
  float scale = __fdiv_rn(amax, F);
  uint2 w = make_uint2(0, 0);
  if (amax > 1e-30f && amax < 1e30f) {
    w = codes_of<CT>(x, amax);
  } else if (!(amax < INFINITY)) {
    scale = __uint_as_float(0x7fc00000u);
  } else if (amax > 0.f) {  // x F and F / amax stay in range (a power of two: exact)
    const float s = amax > 1.f ? 0x1p-32f : 0x1p64f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= s;
    w = codes_of<CT>(x, amax * s);
  }
  const int64_t row = at.x + (int64_t)h * kp.bs;
  *reinterpret_cast<uint2*>((is_k ? kp.kc : kp.vc) + row * D + d0) = w;
  if (lane == 0) (is_k ? kp.kscale : kp.vscale)[row] = scale;
}

constexpr int kReadThreads = 256;
constexpr int kReadRows = 64;  // positions of one CTA

template <typename T, int D, int CT>
__global__ void __launch_bounds__(kReadThreads) paged_q8_read_kernel(PagedQ8Read kp) {
  // 16 codes a load; K and V of a position are two rows of the list
  constexpr int L = D / 16, PER = kReadThreads / L, N = 2 * kReadRows / PER;
  __shared__ int row_s[kReadRows];
  __shared__ float scale_s[2][kReadRows];
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t t0 = (int64_t)blockIdx.x * kReadRows;
  const int n = __ldg(kp.lens + b);
  if ((int)threadIdx.x < kReadRows) {
    const int64_t t = t0 + threadIdx.x;
    if (t == 0 && h == 0 && (n < 0 || n > kp.cap)) report_device_error(kp.err, kErrPagedQ8, b);
    const bool in = t < n && t < kp.cap;
    const int row = in ? q8_row(kp.bt, kp.maxb, kp.nblocks, kp.bs, kp.HK, b, h, (int)t) : -1;
    if (in && row < 0) report_device_error(kp.err, kErrPagedQ8, b);
    row_s[threadIdx.x] = row;
    scale_s[0][threadIdx.x] = row < 0 ? 0.f : __ldg(kp.kscale + row);
    scale_s[1][threadIdx.x] = row < 0 ? 0.f : __ldg(kp.vscale + row);
  }
  __syncthreads();
  const int lane = threadIdx.x & (L - 1);
  uint4 w[N];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int r = u * PER + (int)threadIdx.x / L, s = r / kReadRows, row = row_s[r % kReadRows];
    w[u] = row < 0 ? make_uint4(0, 0, 0, 0)
                   : ld_stream_u4((s ? kp.vc : kp.kc) + (size_t)row * D + lane * 16);
  }
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const int r = u * PER + (int)threadIdx.x / L, s = r / kReadRows, i = r % kReadRows;
    if (t0 + i >= kp.cap) continue;
    const float scale = scale_s[s][i];
    const bool zero = row_s[i] < 0;
    alignas(16) T y[16];
    const uint32_t c[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t h01, h23;
      widen<CT>(c[q], h01, h23);
      const float2 a = __half22float2(half2_of(h01));
      const float2 d = __half22float2(half2_of(h23));
      y[4 * q] = from_f<T>(zero ? 0.f : a.x * scale), y[4 * q + 1] = from_f<T>(zero ? 0.f : a.y * scale);
      y[4 * q + 2] = from_f<T>(zero ? 0.f : d.x * scale), y[4 * q + 3] = from_f<T>(zero ? 0.f : d.y * scale);
    }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(s ? kp.v : kp.k) +
                                          (((size_t)b * kp.HK + h) * kp.cap + t0 + i) * D + lane * 16);
#pragma unroll
    for (int q = 0; q < (int)sizeof(T); ++q) {
      uint4 b;
      memcpy(&b, y + q * (16 / sizeof(T)), 16);
      dst[q] = b;
    }
  }
}

bool aligned16(const void* p, int64_t stride_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
}

template <typename T, int D, int CT>
cudaError_t write_t(const PagedQ8& a, cudaStream_t st) {
  const int es = (int)sizeof(T);
  int vec = aligned16(a.k, a.ks * es) && aligned16(a.v, a.vs * es) ? 1 : 0;
  if (a.rot && !a.inter && a.half % 8 == 0 && aligned16(a.cos_c, (int64_t)a.half * es) && aligned16(a.sin_c, 0)) vec |= 2;
  constexpr int rows = kWriteThreads / (D / 8);
  return launch_k(paged_q8_write_kernel<T, D, CT>, dim3((unsigned)div_up((int64_t)a.ntok * 2 * a.HK, rows)),
                  dim3(kWriteThreads), 0, st, a, vec);
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
