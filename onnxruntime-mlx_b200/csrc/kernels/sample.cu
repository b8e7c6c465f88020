// Token sampling with temperature, top-k, top-p and min-p from given noise.
//
// Row of logits x, M = max x, w_j = exp((x_j - M) / T).  Tokens are ordered by (logit descending, index
// ascending).  Kept are the first top_k; of these, those with less than top_p of the top_k's mass before
// them; of these, those with w_j >= min_p.  The token is the kept j with the largest w_j / e_j (lowest index
// on a tie), e_j the given noise: for independent standard exponentials the winner of that race is token j
// with probability w_j / sum of the kept w.  T = 0 takes the first token of the order.  logprob = x_j - M -
// log sum exp(x - M), of the logits as given.
//   A race is used rather than one uniform number per row because its answer is well conditioned: a relative
// error of 1e-7 in w changes the token with a probability near 1e-7, while a search in a running sum over
// 10^5 tokens is sensitive to every rounding of that sum.
//
// One cluster of C CTAs per row; each CTA keeps its slice of the row in shared memory and every pass runs on
// that copy: HBM sees the logits once, and the noise of kept tokens only.
//   * The last kept token of top-k, and of top-p, is found by radix descent over the composite key
//     (logit as an ordered integer, inverted index): 11 bits a round, counts (top-k) or masses (top-p) per
//     digit summed over the cluster, until the digit's bucket is taken whole or holds one token.  The
//     inverted index in the low bits settles ties.
//   * Masses are summed as fixed-point integers, w 2^32 in two 16-bit halves: integer sums do not depend on
//     the order of the atomics, so equal inputs give equal tokens.  Rounding is at most 2^-33 of the largest
//     weight per token.
#include <cooperative_groups.h>

#include <cmath>

#include "../common.cuh"
#include "sample.h"

namespace cg = cooperative_groups;

namespace b200ep {
namespace {

constexpr int kThreads = 512;
constexpr int kWarpsS = kThreads / 32;
constexpr int kDigit = 11, kBins = 1 << kDigit;
constexpr int kMaxCluster = 8;

struct Red {  // what CTAs of a cluster exchange; one slot per use, so that no barrier is needed before reuse
  float maxv, sum;
  unsigned long long mass, best;
};

template <typename T>
__device__ __forceinline__ float logit(const T* p, int i) {
  const float x = to_f<T>(p[i]);
  return x == x ? x + 0.f : -INFINITY;  // NaN: never sampled; -0 and 0 are one value
}

// Ordered integer of a logit: 16 bits for 16-bit types, 32 for float.
template <typename T>
__device__ __forceinline__ uint32_t ordered(float x) {
  uint32_t u;
  if constexpr (sizeof(T) == 2) {
    T t = from_f<T>(x);
    uint16_t h;
    memcpy(&h, &t, 2);
    u = (h & 0x8000u) ? (uint16_t)~h : (h | 0x8000u);
  } else {
    const uint32_t h = __float_as_uint(x);
    u = (h & 0x80000000u) ? ~h : (h | 0x80000000u);
  }
  return u;
}

__device__ __forceinline__ unsigned long long fixed32(float w) {  // w in [0, 1] times 2^32, rounded
  const float h = w * 65536.f, hi = truncf(h);
  return ((unsigned long long)(uint32_t)hi << 16) + (unsigned long long)__float2uint_rn((h - hi) * 65536.f);
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, F f, V* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = scratch[0];
  for (int w = 1; w < kWarpsS; ++w) v = f(v, scratch[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a, int slice) {
  extern __shared__ __align__(16) uint8_t sm[];
  uint32_t* cnt = reinterpret_cast<uint32_t*>(sm);  // [kBins]
  uint32_t* mlo = cnt + kBins;
  uint32_t* mhi = mlo + kBins;
  T* stage = reinterpret_cast<T*>(mhi + kBins);
  __shared__ Red red[2];
  __shared__ unsigned long long seg_s[2][2];   // this CTA's share of a round: count, mass
  __shared__ unsigned long long found_s[2][4]; // the digit found: flag, digit, above, within
  __shared__ unsigned long long scratch[kWarpsS];
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int lo = min(a.vocab, rank * slice), n = min(a.vocab, lo + slice) - lo;
  const T* g = static_cast<const T*>(a.logits) + (size_t)row * a.logits_stride + lo;
  // ---- the slice, kept at the same 16-byte phase as in global memory
  constexpr int VE = 16 / sizeof(T);
  const int phase = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T));
  T* x = stage + phase;
  {
    const int head = min(n, (VE - phase) % VE), body = (n - head) / VE;
    for (int i = tid; i < head; i += kThreads) x[i] = g[i];
    for (int i = tid; i < body; i += kThreads)
      reinterpret_cast<uint4*>(x + head)[i] = ld_stream_u4(g + head + i * VE);
    for (int i = head + body * VE + tid; i < n; i += kThreads) x[i] = g[i];
  }
  __syncthreads();
  float t = a.temperature ? __ldg(a.temperature + row) : 1.f;
  int k = a.top_k ? __ldg(a.top_k + row) : 0;
  float tp = a.top_p ? __ldg(a.top_p + row) : 1.f;
  const float mp = a.min_p ? __ldg(a.min_p + row) : 0.f;
  if (!(t > 0.f)) t = 1.f, k = 1;
  if (k <= 0 || k > a.vocab) k = a.vocab;
  const bool use_p = tp < 1.f;  // (false for NaN)

  // ---- maximum and normaliser
  float m = -INFINITY;
  for (int i = tid; i < n; i += kThreads) m = fmaxf(m, logit(x, i));
  m = block_reduce(m, [](float p, float q) { return fmaxf(p, q); }, reinterpret_cast<float*>(scratch));
  if (tid == 0) red[0].maxv = m;
  cluster.sync();
  for (int r = 0; r < C; ++r) m = fmaxf(m, cluster.map_shared_rank(red, r)[0].maxv);
  if (m == -INFINITY) {  // nothing to choose from
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    cluster.sync();
    return;
  }
  float z = 0.f;
  for (int i = tid; i < n; i += kThreads) {
    const float v = logit(x, i);
    z += v == m ? 1.f : expf(v - m);  // (m may be infinite)
  }
  z = block_reduce(z, [](float p, float q) { return p + q; }, reinterpret_cast<float*>(scratch));
  if (tid == 0) red[0].sum = z;

  const float rt = 1.f / t;
  auto weight = [&](float v) { return v == m ? 1.f : expf((v - m) * rt); };
  constexpr int KB = sizeof(T) * 8;
  const int ib = 32 - __clz(a.vocab - 1 > 0 ? a.vocab - 1 : 1);  // bits of an index
  auto key_of = [&](int i, float v) {
    return ((unsigned long long)ordered<T>(v) << ib) | (unsigned)(a.vocab - 1 - (lo + i));
  };
  int round = 0;
  // The composite key of the last token of the order such that `want` (tokens, or mass) is reached, among
  // tokens with key >= floor_key.  `all`: what those hold together (want <= all).
  auto descend = [&](bool by_mass, unsigned long long want, unsigned long long floor_key) {
    unsigned long long prefix = 0, above = 0;  // key bits fixed so far; count or mass of larger prefixes
    int left = KB + ib;                        // key bits not fixed yet
    while (left > 0) {
      const int d = min(kDigit, left), shift = left - d;
      for (int b = tid; b < kBins; b += kThreads) cnt[b] = mlo[b] = mhi[b] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const float v = logit(x, i);
        const unsigned long long key = key_of(i, v);
        if (key < floor_key || (left < KB + ib && (key >> left) != prefix)) continue;
        const int b = (int)((key >> shift) & ((1u << d) - 1));
        atomicAdd(cnt + b, 1u);
        if (by_mass) {
          const unsigned long long f = fixed32(weight(v));
          if (f) {
            atomicAdd(mlo + b, (uint32_t)(f & 0xffffu));
            atomicAdd(mhi + b, (uint32_t)(f >> 16));
          }
        }
      }
      cluster.sync();
      // this CTA sums its share of the digits, the highest ones in rank 0: thread q the digits
      // [top - q * per - per, top - q * per) of the share
      const int share = kBins / C, per = (share + kThreads - 1) / kThreads;
      const int hi_digit = kBins - rank * share;  // exclusive
      unsigned long long tc[kBins / kThreads], tm[kBins / kThreads], c0 = 0, m0 = 0;
#pragma unroll
      for (int q = 0; q < kBins / kThreads; ++q) {
        tc[q] = tm[q] = 0;
        const int off = tid * per + q;
        if (q < per && off < share) {
          const int b = hi_digit - 1 - off;
          for (int r = 0; r < C; ++r) {
            tc[q] += cluster.map_shared_rank(cnt, r)[b];
            if (by_mass)
              tm[q] += ((unsigned long long)cluster.map_shared_rank(mhi, r)[b] << 16) + cluster.map_shared_rank(mlo, r)[b];
          }
          c0 += tc[q], m0 += tm[q];
        }
      }
      unsigned long long val = by_mass ? m0 : c0, inc = val;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      __syncthreads();
      if (lane == 31) scratch[warp] = inc;
      __syncthreads();
      unsigned long long before = inc - val, total = 0;
      for (int w = 0; w < kWarpsS; ++w) {
        if (w < warp) before += scratch[w];
        total += scratch[w];
      }
      const int par = round & 1;
      if (tid == 0) seg_s[par][0] = total, found_s[par][0] = 0;
      cluster.sync();
      for (int r = 0; r < rank; ++r) before += cluster.map_shared_rank(seg_s, r)[par][0];
      before += above;
#pragma unroll
      for (int q = 0; q < kBins / kThreads; ++q) {
        const unsigned long long w = by_mass ? tm[q] : tc[q];
        if (before < want && want <= before + w) {
          for (int r = 0; r < C; ++r) {
            auto* f = cluster.map_shared_rank(found_s, r)[par];
            f[1] = (unsigned)(hi_digit - 1 - (tid * per + q));
            f[2] = before;
            f[3] = tc[q];
            f[0] = 1 + (!by_mass && before + w == want ? 1 : 0);  // 2: the bucket is taken whole
          }
        }
        before += w;
      }
      cluster.sync();
      const unsigned long long flag = found_s[par][0], digit = found_s[par][1];
      ++round;
      above = found_s[par][2];
      prefix = (prefix << d) | digit;
      left = shift;
      if (flag == 2) break;
      if (flag == 0) return floor_key;                       // (cannot happen: want <= all)
      if (found_s[par][3] == 1) break;                       // one token: it is the last one
    }
    return max(prefix << left, floor_key);  // every token of the bucket is kept, or its only one
  };

  unsigned long long cut = 0;
  if (k < a.vocab) cut = descend(false, (unsigned long long)k, 0);
  if (use_p) {
    unsigned long long mass = 0;
    for (int i = tid; i < n; i += kThreads) {
      const float v = logit(x, i);
      if (key_of(i, v) >= cut) mass += fixed32(weight(v));
    }
    mass = block_reduce(mass, [](unsigned long long p, unsigned long long q) { return p + q; }, scratch);
    if (tid == 0) red[0].mass = mass;
    cluster.sync();
    mass = 0;
    for (int r = 0; r < C; ++r) mass += cluster.map_shared_rank(red, r)[0].mass;
    unsigned long long want = (unsigned long long)ceil((double)fmaxf(tp, 0.f) * (double)mass);
    want = min(max(want, 1ull), mass);
    cut = descend(true, want, cut);
  }

  // ---- the race
  const float* e = a.noise + (size_t)row * a.noise_stride + lo;
  unsigned long long best = 0;
  for (int i = tid; i < n; i += kThreads) {
    const float v = logit(x, i);
    if (v == -INFINITY || key_of(i, v) < cut) continue;
    const float w = weight(v);
    if (mp > 0.f && w < fminf(mp, 1.f)) continue;
    const float q = __fdiv_rn(w, __ldg(e + i));
    const uint32_t bits = q >= 0.f ? __float_as_uint(q) : 0u;  // (noise that is negative or NaN never wins)
    const unsigned long long cand = ((unsigned long long)(bits & 0x7fffffffu) << 32) | (0xffffffffu - (unsigned)(lo + i));
    best = max(best, cand);
  }
  best = block_reduce(best, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; }, scratch);
  if (tid == 0) red[0].best = best;
  cluster.sync();
  if (rank == 0 && tid == 0) {
    float zs = 0.f;
    for (int r = 0; r < C; ++r) {
      const Red* o = cluster.map_shared_rank(red, r);
      best = max(best, o->best);
      zs += o->sum;
    }
    const unsigned token = 0xffffffffu - (unsigned)(best & 0xffffffffu);
    a.tokens[row] = token;
    if (a.logprobs) {
      const float v = logit(static_cast<const T*>(a.logits) + (size_t)row * a.logits_stride, (int)token);
      a.logprobs[row] = (v == m ? 0.f : v - m) - logf(zs);
    }
  }
  cluster.sync();  // the others' shared memory stays until rank 0 has read it
}

template <typename T>
cudaError_t launch_t(const SampleArgs& a, cudaStream_t st) {
  // CTAs of a row: enough that a slice fits in 64 KB (three CTAs an SM), and as many as keep one wave
  int C = 1;
  while (C < kMaxCluster && ((int64_t)a.vocab * (int64_t)sizeof(T) > C * 65536ll || (int64_t)a.rows * C * 2 <= num_sms()))
    C *= 2;
  const int slice = (div_up(a.vocab, C) + 7) / 8 * 8;
  const size_t smem = 3 * kBins * sizeof(uint32_t) + (size_t)slice * sizeof(T) + 16;
  auto kern = sample_kernel<T>;
  if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, a, slice);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  switch (a.dtype) {
    case kF32: return launch_t<float>(a, st);
    case kF16: return launch_t<__half>(a, st);
    case kBF16: return launch_t<__nv_bfloat16>(a, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace b200ep
