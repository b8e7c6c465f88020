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
//   * top-k: the k-th largest of the threads' own maxima is a lower bound of the k-th largest logit, and a close
//     one.  A histogram of one value per thread gives it; the few tokens above go to the first CTA (at most
//     kCap), which finishes the row alone: the rank and the mass before each token by comparison with every
//     other, then top-k, top-p, min-p and the race.
//   * top-p (and a top-k too large for that): tokens are split by d = M - x into 16 bins, then those of the bin
//     that holds the border into 512.  In the first split every thread adds its elements to bins of its own (a
//     column of shared memory): no atomics, and fp32 sums that always add in the same order.  The tokens of the
//     last bin, or all up to it where those are few, go to the first CTA, which finds the border; all CTAs race.
//   * Rows that stay crowded (hundreds of equal logits at the border) go through radix descent over the composite
//     key (logit as an ordered integer, inverted index), 9 bits a round, with integer atomics.
//   * Masses of single tokens are summed as fixed-point integers (w 2^32 rounded, at most 2^-33 of the largest
//     weight off per token), so no sum depends on the order of atomics: equal inputs give equal tokens.
// Bound by the latency of its passes and cluster barriers, not by bytes: 64 rows of 128256 fp16 logits take 16 us
// with min-p, 21 us with top-k 50 and top-p 0.9, 23 us unfiltered (the noise's 33 MB among it) and 54 us with top-p
// 0.95 alone on flat logits (tens of thousands of tokens kept); one row takes 15 us.
#include <cooperative_groups.h>

#include <cmath>
#include <cstring>

#include "../common.cuh"
#include "sample.h"

namespace cg = cooperative_groups;

namespace b200ep {
namespace {

constexpr int kThreads = 512;
constexpr int kWarpsS = kThreads / 32;
constexpr int kDigit = 9, kBins = 1 << kDigit;  // a thread sums one bin at most
constexpr int kMaxCluster = 8;

constexpr int kSplit = 16;   // bins of the first split: one warp adds up each
constexpr int kCap = kThreads;  // tokens that one CTA finishes alone, one per thread
constexpr int kTop = 128;    // bins of the threads' maxima
constexpr int kNear = 1024;  // tokens of the border's bin that a warp lists
static_assert(kSplit == kWarpsS && kCap <= kThreads && kBins <= kThreads, "one warp a bin, one thread a token");

struct __align__(8) Token {
  float x;
  int index;
};
__device__ __forceinline__ bool before(Token a, Token b) { return a.x > b.x || (a.x == b.x && a.index < b.index); }

struct __align__(8) Red {  // what CTAs of a cluster exchange; one slot per use, so that no barrier is needed before reuse
  float maxv, sum;
  unsigned long long mass, best;
  float bin[2][kSplit];  // of the first split, by count and by mass
  int top[kTop];
  Token cut;             // written by the first CTA
  int got;               // tokens collected
  Token list[kCap];
};

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

// The logit with that ordered integer (below -infinity: -infinity).
template <typename T>
__device__ __forceinline__ float from_ordered(uint32_t u) {
  float x;
  if constexpr (sizeof(T) == 2) {
    const uint16_t h = (uint16_t)((u & 0x8000u) ? u & 0x7fffu : ~u);
    T t;
    memcpy(&t, &h, 2);
    x = to_f<T>(t);
  } else {
    x = __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
  }
  return x == x ? x : -INFINITY;
}

__device__ __forceinline__ unsigned long long fixed32(float w) {  // w in [0, 1] times 2^32, rounded
  const float h = w * 65536.f, hi = truncf(h);
  return ((unsigned long long)(uint32_t)hi << 16) + (unsigned long long)__float2uint_rn((h - hi) * 65536.f);
}

// 16 bytes of the slice, at a 16-byte boundary.
template <typename T>
__device__ __forceinline__ uint4 get16(const T* p) {
  uint4 w;
  memcpy(&w, __builtin_assume_aligned(p, 16), 16);
  return w;
}
template <typename T>
__device__ __forceinline__ void put16(T* p, const uint4& w) {
  memcpy(__builtin_assume_aligned(p, 16), &w, 16);
}

// 16 bytes of logits: NaN to -infinity, and the largest.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static __device__ __forceinline__ float clean(uint4& w) {
    float f[4];
    memcpy(f, &w, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = fmaxf(f[j], -INFINITY);
    memcpy(&w, f, 16);
    return largest(w);
  }
  static __device__ __forceinline__ float largest(const uint4& w) {
    float f[4];
    memcpy(f, &w, 16);
    return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
  }
};
template <typename T2>
__device__ __forceinline__ T2 both(float v);
template <>
__device__ __forceinline__ __half2 both<__half2>(float v) { return __float2half2_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat162 both<__nv_bfloat162>(float v) { return __float2bfloat162_rn(v); }
template <typename T2>
struct Vec16 {
  static __device__ __forceinline__ float clean(uint4& w) {
    T2 h[4];
    memcpy(h, &w, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __hmax2(h[j], both<T2>(-INFINITY));  // (the operand that is a number)
    memcpy(&w, h, 16);
    return largest(w);
  }
  static __device__ __forceinline__ float largest(const uint4& w) {
    T2 h[4];
    memcpy(h, &w, 16);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(to_f(m.x), to_f(m.y));
  }
};
template <> struct Vec<__half> : Vec16<__half2> {};
template <> struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat162> {};

// Reads and writes of the same variable in CTA r of the cluster.  (As instructions of their own: addresses that the
// compiler could share over the whole kernel would take up its registers.)
template <typename V>
__device__ __forceinline__ V peer(const V* p, int r) {
  V v;
  if constexpr (sizeof(V) == 8) {
    unsigned long long u;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.b64 %0, [a];\n\t}"
                 : "=l"(u) : "r"(smem_u32(p)), "r"(r) : "memory");
    memcpy(&v, &u, 8);
  } else {
    uint32_t u;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.b32 %0, [a];\n\t}"
                 : "=r"(u) : "r"(smem_u32(p)), "r"(r) : "memory");
    memcpy(&v, &u, 4);
  }
  return v;
}
__device__ __forceinline__ void peer_set(unsigned long long* p, int r, unsigned long long v) {
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.b64 [a], %2;\n\t}" ::"r"(
                   smem_u32(p)), "r"(r), "l"(v)
               : "memory");
}
__device__ __forceinline__ unsigned long long bits_of(Token t) {
  unsigned long long u;
  memcpy(&u, &t, 8);
  return u;
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
#pragma unroll
  for (int w = 1; w < kWarpsS; ++w) v = f(v, scratch[w]);
  return v;
}

__device__ __forceinline__ float exp2a(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a, int slice) {
  extern __shared__ __align__(16) uint8_t sm[];
  float* col = reinterpret_cast<float*>(sm);        // first split: [kSplit][kThreads]
  uint16_t* near = reinterpret_cast<uint16_t*>(sm) + (threadIdx.x >> 5) * kNear;  // a warp's tokens of one bin
  Token* all = reinterpret_cast<Token*>(sm);        // the first CTA's list of a row: [kCap] tokens,
  unsigned long long* wall = reinterpret_cast<unsigned long long*>(all + kCap);  // and their weights
  constexpr int kScratch = kSplit * kThreads * 4;   // the union of these
  static_assert(kWarpsS * kNear * 2 <= kScratch && kCap * 16 <= kScratch, "scratch");
  uint32_t* cnt = reinterpret_cast<uint32_t*>(sm + kScratch);  // histograms: [kBins] counts, masses (low, high half)
  uint32_t* mlo = cnt + kBins;
  uint32_t* mhi = mlo + kBins;
  T* stage = reinterpret_cast<T*>(mhi + kBins);
  __shared__ Red red;
  __shared__ unsigned long long seg_s[2];       // histograms: this CTA's share
  __shared__ unsigned long long found_s[2][4];  // the bin found: flag, bin, before it, its count
  __shared__ unsigned long long scratch[kWarpsS];
  __shared__ int top_s, lead_s;
  __shared__ unsigned long long best_s;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int lo = min(a.vocab, rank * slice), n = min(a.vocab, lo + slice) - lo;
  const T* g = static_cast<const T*>(a.logits) + (size_t)row * a.logits_stride + lo;
  // ---- the slice, padded to whole 16 bytes with tokens of -infinity.  A thread's elements (and so the order of
  // every sum) do not depend on the row's address: a row that starts off a 16-byte boundary is shifted here.
  constexpr int VE = 16 / sizeof(T);
  const int phase = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T)), nvec = (n + VE - 1) / VE;
  float mine = -INFINITY;  // this thread's largest
  if (!phase) {
#pragma unroll 4
    for (int i = tid; i < n / VE; i += kThreads) {
      uint4 w = ld_stream_u4(g + i * VE);
      mine = fmaxf(mine, Vec<T>::clean(w));
      put16(stage + i * VE, w);
    }
  }
#pragma unroll 1
  for (int i = (phase ? 0 : n / VE * VE) + tid; i < nvec * VE; i += kThreads) {
    const float f = i < n ? fmaxf(to_f<T>(g[i]), -INFINITY) : -INFINITY;
    mine = fmaxf(mine, f);
    stage[i] = from_f<T>(f);
  }
  __syncthreads();
  // f(logit, index in the slice) for every element of a thread in 16 bytes whose largest is at least `least`
  auto each = [&](float least, auto f) {
#pragma unroll 1
    for (int i = tid; i < nvec; i += kThreads) {
      const uint4 w = get16(stage + i * VE);
      if (Vec<T>::largest(w) < least) continue;
      T v[VE];
      memcpy(v, &w, 16);
#pragma unroll
      for (int j = 0; j < VE; ++j) f(to_f<T>(v[j]) + 0.f, i * VE + j);  // (-0 and 0 are one value)
    }
  };
  const float t0 = a.temperature ? __ldg(a.temperature + row) : 1.f;
  int k = a.top_k ? __ldg(a.top_k + row) : 0;
  float tp = a.top_p ? __ldg(a.top_p + row) : 1.f;
  float mp = a.min_p ? fminf(__ldg(a.min_p + row), 1.f) : 0.f;
  const bool greedy = !(t0 > 0.f);
  const float t = greedy ? 1.f : fminf(fmaxf(t0, 1e-38f), 3.4e38f);  // (1 / t stays finite, and above 0)
  if (greedy) k = 0, tp = 1.f, mp = 0.f;
  if (k <= 0 || k > a.vocab) k = a.vocab;
  const bool use_p = tp < 1.f;  // (false for NaN)
  tp = fmaxf(tp, 0.f);

  // ---- maximum
  float m = block_reduce(mine, [](float p, float q) { return fmaxf(p, q); }, reinterpret_cast<float*>(scratch));
  if (tid == 0) red.maxv = m;
  for (int i = tid; i < kTop; i += kThreads) red.top[i] = 0;
  cluster.sync();
#pragma unroll
  for (int r = 0; r < kMaxCluster; ++r)
    if (r < C) m = fmaxf(m, peer(&red.maxv, r));
  m += 0.f;
  if (m == -INFINITY) {  // nothing to choose from
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
    }
    cluster.sync();
    return;
  }
  if (m == INFINITY) {  // the infinite logits share everything: zeros among tokens of -infinity
    for (int i = tid; i < nvec * VE; i += kThreads) stage[i] = from_f<T>(to_f<T>(stage[i]) == m ? 0.f : -INFINITY);
    mine = mine == m ? 0.f : -INFINITY;
    m = 0.f;
    __syncthreads();
  }
  const float c2 = 1.4426950408889634f / t;
  auto weight = [&](float v) { return exp2a((v - m) * c2); };
  if (a.logprobs) {
    float z = 0.f;
    each(-INFINITY, [&](float v, int) { z += exp2a((v - m) * 1.4426950408889634f); });
    z = block_reduce(z, [](float p, float q) { return p + q; }, reinterpret_cast<float*>(scratch));
    if (tid == 0) red.sum = z;
  }
  // the race's result; called by one thread of the first CTA, after a barrier that follows red.sum
  auto finish = [&](unsigned long long best) {
    if (best == 0) {  // (no row comes here: its largest logit is always kept)
      a.tokens[row] = -1;
      if (a.logprobs) a.logprobs[row] = -INFINITY;
      return;
    }
    const int token = (int)(0xffffffffu - (unsigned)(best & 0xffffffffu));
    a.tokens[row] = token;
    if (a.logprobs) {
      float zs = 0.f;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < C) zs += peer(&red.sum, r);
      const float v = to_f<T>(static_cast<const T*>(a.logits)[(size_t)row * a.logits_stride + token]);
      a.logprobs[row] = (v == INFINITY ? 0.f : v - m) - logf(zs);
    }
  };
  const float* noise = a.noise + (size_t)row * a.noise_stride;
  auto ticket = [&](float w, float e, int token) {  // larger for a larger w / e, then for a lower index
    const float q = __fdiv_rn(w, e);
    return ((unsigned long long)(q >= 0.f ? __float_as_uint(q) & 0x7fffffffu : 0u) << 32) |  // (bad noise never wins)
           (0xffffffffu - (unsigned)token);
  };
  auto max64 = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
  auto add64 = [](unsigned long long p, unsigned long long q) { return p + q; };

  Token cut{-INFINITY, a.vocab};  // tokens up to this one in the order are kept
  auto put = [&](float v, int i) {
    const int p = atomicAdd(&red.got, 1);
    if (p < kCap) red.list[p] = Token{v, lo + i};
  };
  auto gather = [&]() {  // the CTAs' lists, where they fit, into the first CTA's; the number of their tokens
    cluster.sync();
    int c[kMaxCluster], got = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) c[r] = r < C ? peer(&red.got, r) : 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      if (rank == 0 && tid < c[r] && got + c[r] <= kCap) all[got + tid] = peer(&red.list[tid], r);
      got += c[r];
    }
    __syncthreads();
    return got;
  };
  // Collects the tokens that in(v) holds for in the CTAs' lists (all of them have values of `least` and more), and,
  // where they fit, all of them in the first CTA's.  Returns their number.
  auto collect = [&](float least, auto in) {
    if (tid == 0) red.got = 0;
    __syncthreads();
    each(least, [&](float v, int i) {
      if (in(v)) put(v, i);
    });
    return gather();
  };
  // This thread's token of the first CTA's list, the number of tokens before it and their mass
  Token me;
  float wt;
  int place;
  unsigned long long ahead;
  auto rank_all = [&](int got) {
    me = tid < got ? all[tid] : Token{-INFINITY, a.vocab};
    wt = tid < got ? weight(me.x) : 0.f;
    if (tid < got) wall[tid] = fixed32(wt);
    __syncthreads();
    place = 0, ahead = 0;
    if (tid < got) {
#pragma unroll 4
      for (int j = 0; j < got; ++j)
        if (before(all[j], me)) ++place, ahead += wall[j];
    }
  };
  // The rest of a row whose kept tokens are all in the list; `need`: the mass that top-p asks for, 0: the share
  // of the first k tokens'
  auto conclude = [&](int got, unsigned long long need) {
    rank_all(got);
    bool keep = tid < got && place < k;
    if (use_p) {
      if (!need) {
        const unsigned long long kept = block_reduce(keep ? wall[tid] : 0ull, add64, scratch);
        need = (unsigned long long)ceil((double)tp * (double)kept);
      }
      keep = keep && (ahead < need || place == 0);
    }
    keep = keep && wt >= mp;
    const unsigned long long best = block_reduce(keep ? ticket(wt, __ldg(noise + me.index), me.index) : 0ull, max64, scratch);
    if (tid == 0) finish(best);
  };

  // ---- top-k from the threads' maxima
  if (k <= kCap && k < a.vocab) {
    auto bin_of = [&](float v) { return (int)fminf(fmaxf((m - v) * 8.f, 0.f), (float)(kTop - 1)); };
    if (mine > -INFINITY) atomicAdd(&red.top[bin_of(mine)], 1);
    cluster.sync();
    if (warp == 0) {
      int own[kTop / 32], sum = 0;
#pragma unroll
      for (int q = 0; q < kTop / 32; ++q) {
        own[q] = 0;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < C) own[q] += peer(&red.top[lane * (kTop / 32) + q], r);
        sum += own[q];
      }
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      int at = kTop - 1, run = inc - sum;
#pragma unroll
      for (int q = kTop / 32 - 1; q >= 0; --q) {
        int upto = run;
#pragma unroll
        for (int u = 0; u <= q; ++u) upto += own[u];
        if (upto >= k) at = lane * (kTop / 32) + q;
      }
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0) top_s = at;
    }
    __syncthreads();
    const int at = top_s;
    if (at < kTop - 1) {
      const int got = collect(m - (float)(at + 2) * 0.125f, [&](float v) { return bin_of(v) <= at; });
      if (got <= kCap) {
        if (rank == 0) conclude(got, 0);
        cluster.sync();  // the others' shared memory stays until rank 0 has read it
        return;
      }
      cluster.sync();  // (before the lists are used again)
    }
  }

  // ---- the border, by count (top-k) and by mass (top-p)
  int round = 0;
  // After every CTA has filled its histogram: the bin, from the highest one down, with which `goal` is reached (or
  // all there is, if that is less).  Leaves it in found_s of the round's parity.
  auto find = [&](bool by_mass, unsigned long long goal) {
    cluster.sync();
    // this CTA sums its share of the bins, the highest ones in rank 0, one a thread
    const int share = kBins / C, bin = kBins - 1 - rank * share - tid;
    unsigned long long own = 0, val = 0;
    if (tid < share) {
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < C) {
          own += peer(cnt + bin, r);
          if (by_mass)
            val += ((unsigned long long)peer(mhi + bin, r) << 16) + peer(mlo + bin, r);
        }
      if (!by_mass) val = own;
    }
    unsigned long long inc = val;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    unsigned long long ahead_ = inc - val, total = 0;
    for (int w = 0; w < kWarpsS; ++w) {
      if (w < warp) ahead_ += scratch[w];
      total += scratch[w];
    }
    const int par = round++ & 1;
    if (tid == 0) seg_s[par] = total, found_s[par][0] = 0;
    cluster.sync();
    unsigned long long sum = 0;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      const unsigned long long v = r < C ? peer(&seg_s[par], r) : 0;
      if (r < rank) ahead_ += v;
      sum += v;
    }
    goal = min(goal, sum);
    if (ahead_ < goal && goal <= ahead_ + val)
      for (int r = 0; r < C; ++r) {
        unsigned long long* f = found_s[par];
        peer_set(f + 1, r, (unsigned long long)(unsigned)bin);
        peer_set(f + 2, r, ahead_);
        peer_set(f + 3, r, own);
        peer_set(f, r, !by_mass && ahead_ + val == goal ? 2ull : 1ull);  // 2: the bin is taken whole
      }
    cluster.sync();
    return par;
  };
  auto erase = [&]() {  // what lies behind `cut` leaves the slice
    each(-INFINITY, [&](float v, int i) {
      if (before(cut, Token{v, lo + i})) stage[i] = from_f<T>(-INFINITY);
    });
    __syncthreads();
  };
  auto clear = [&]() {
    for (int b = tid; b < 3 * kBins; b += kThreads) cnt[b] = 0;
    __syncthreads();
  };
  auto count_in = [&](int b, bool by_mass, float v) {
    atomicAdd(cnt + b, 1u);
    if (by_mass) {
      const unsigned long long f = fixed32(weight(v));
      if (f) {
        atomicAdd(mlo + b, (uint32_t)(f & 0xffffu));
        atomicAdd(mhi + b, (uint32_t)(f >> 16));
      }
    }
  };
#pragma unroll 1
  for (int by_mass = 0; by_mass < 2; ++by_mass) {
    if (by_mass ? !use_p : k >= a.vocab) continue;
    // ---- 16 bins of d = m - v, the last one without an end
    const float w = by_mass ? fminf(fmaxf(1.0397208f * t, 1e-3f), 64.f) : 1.f, rw = 1.f / w;
    constexpr float kMagic = 8388608.f;  // + 2^23 rounds to a whole number, in the low bits
    auto spot = [&](float v) { return fmaf(m - v, rw, kMagic); };  // 2^23 + the bin
#pragma unroll
    for (int b = 0; b < kSplit; ++b) col[b * kThreads + tid] = 0.f;
    {
      uint8_t* mine_col = reinterpret_cast<uint8_t*>(col + tid);
      auto slot = [&](float v) {
        const uint32_t bin = __float_as_uint(fminf(spot(v), kMagic + (float)(kSplit - 1))) & (kSplit - 1);
        return reinterpret_cast<float*>(mine_col + bin * (kThreads * 4));
      };
      if (by_mass)
        each(-INFINITY, [&](float v, int) { *slot(v) += weight(v); });
      else
        each(-INFINITY, [&](float v, int) { *slot(v) += v > -INFINITY ? 1.f : 0.f; });
    }
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < kThreads / 32; ++q) s += col[warp * kThreads + q * 32 + lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red.bin[by_mass][warp] = s;
    cluster.sync();
    // every warp: one lane a bin, the same order of additions everywhere
    float upto = 0.f, above, total, want;
    int at;
    bool whole;
    {
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < C) upto += peer(&red.bin[by_mass][lane & (kSplit - 1)], r);
      // at least so many tokens are in the bin: none of them weighs more than its first
      float few = !by_mass || upto == 0.f ? upto : upto / exp2a(-fmaxf((float)(lane & (kSplit - 1)) - 0.5f, 0.f) * w * c2);
#pragma unroll
      for (int o = 1; o < kSplit; o <<= 1) {
        const float u = __shfl_up_sync(0xffffffffu, upto, o, kSplit), f = __shfl_up_sync(0xffffffffu, few, o, kSplit);
        if ((lane & (kSplit - 1)) >= o) upto += u, few += f;
      }
      total = __shfl_sync(0xffffffffu, upto, kSplit - 1);
      want = by_mass ? tp * total : (float)k;
      at = __ffs((int)(__ballot_sync(0xffffffffu, upto >= want) | 1u << (kSplit - 1))) - 1;
      above = __shfl_sync(0xffffffffu, upto, max(at - 1, 0));
      if (at == 0) above = 0.f;
      whole = __shfl_sync(0xffffffffu, few, at) <= (float)kCap;
    }
    if (!by_mass && total <= (float)k) continue;  // (tokens of -infinity are never kept)
    const float rest = want - above;
    const unsigned long long need = by_mass ? (unsigned long long)((double)want * 4294967296.0) : 0;
    const float least = at == kSplit - 1 ? -INFINITY : m - ((float)at + 0.501f) * w;  // no token of the bins is smaller
    // what spot() gives for the tokens of bin `at` (-infinity gives infinity)
    const float spot0 = kMagic + (float)at, spot1 = at == kSplit - 1 ? 3e38f : spot0;
    int got = kCap + 1;
    if (whole) {
      got = collect(least, [&](float v) { return spot(v) <= spot1; });
      if (got > kCap) cluster.sync();  // (before the lists are used again)
    }
    if (got > kCap) {
      // ---- the tokens of that bin in 512, the largest ones in the highest
      whole = false;
      const float from = fmaxf((float)at - 0.5f, 0.f);
      auto fine = [&](float v) {
        const float h = fmaxf((m - v) * rw - from, 0.f);
        // (the last bin has no end: a rising function of it that does)
        const float q = at == kSplit - 1 ? 1.f - __fdiv_rn(16.f, h + 16.f) : h;
        return kBins - 1 - (int)fminf(q * (float)kBins, (float)(kBins - 1));
      };
      // each warp lists its tokens of the bin (indices within the slice), then works on them with all lanes
      int mine_n = 0;
#pragma unroll 1
      for (int i0 = warp * 32; i0 < nvec; i0 += kThreads) {
        const int i = i0 + lane;
        const uint4 w4 = i < nvec ? get16(stage + i * VE) : uint4{};
        T v[VE];
        memcpy(v, &w4, 16);
        uint32_t in = 0;  // which of the thread's VE tokens
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float sp = spot(to_f<T>(v[j]));
          if (sp >= spot0 && sp <= spot1) in |= 1u << j;
        }
        if (i >= nvec) in = 0;
        const int own = __popc(in);
        int to = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, to, o);
          if (lane >= o) to += u;
        }
        const int all_n = __shfl_sync(0xffffffffu, to, 31);
        to += mine_n - own;
        for (; in && to < kNear; in &= in - 1) near[to++] = (uint16_t)(i * VE + __ffs((int)in) - 1);
        mine_n += all_n;
      }
      clear();
      auto visit = [&](auto f) {
        if (mine_n <= kNear) {
#pragma unroll 1
          for (int q = lane; q < mine_n; q += 32) f(to_f<T>(stage[near[q]]) + 0.f, (int)near[q]);
        } else {  // too many: from the slice (a warp's vectors are the ones it listed)
          each(least, [&](float v, int i) {
            if (spot(v) >= spot0 && spot(v) <= spot1) f(v, i);
          });
        }
      };
      visit([&](float v, int) { count_in(fine(v), by_mass, v); });
      const int par = find(by_mass, max(1ull, by_mass ? (unsigned long long)((double)rest * 4294967296.0)
                                                      : (unsigned long long)rest));
      const int bin = (int)found_s[par][1];
      const unsigned long long over = found_s[par][2];
      if (found_s[par][0] && found_s[par][3] <= kCap) {
        if (tid == 0) red.got = 0;
        __syncthreads();
        visit([&](float v, int i) {
          if (fine(v) == bin) put(v, i);
        });
        got = gather();
        if (rank == 0) {
          rank_all(got);
          const double goal = by_mass ? (double)rest * 4294967296.0 - (double)over : (double)rest - (double)over;
          const int last = max(1, __syncthreads_count(tid < got && (by_mass ? (double)ahead : (double)place) < goal)) - 1;
          if (tid < got && place == last)
            for (int r = 0; r < C; ++r) peer_set(reinterpret_cast<unsigned long long*>(&red.cut), r, bits_of(me));
        }
        cluster.sync();
        cut = red.cut;
        if (!by_mass && use_p) erase();
        continue;
      }
    } else {
      if (rank == 0) conclude(got, by_mass ? max(need, 1ull) : 0);
      cluster.sync();
      return;
    }
    // ---- crowded: radix descent to the last token such that `goal` tokens, or that much mass, is reached
    constexpr int KB = sizeof(T) * 8;
    const int ib = 32 - __clz(a.vocab - 1 > 0 ? a.vocab - 1 : 1);  // bits of an index
    unsigned long long prefix = 0, over = 0;  // key bits fixed so far; count or mass of larger prefixes
    unsigned long long goal = (unsigned long long)k;
    if (by_mass) {
      unsigned long long mass = 0;
      each(-INFINITY, [&](float v, int i) {
        if (v > -INFINITY) mass += fixed32(weight(v));
      });
      mass = block_reduce(mass, add64, scratch);
      if (tid == 0) red.mass = mass;
      cluster.sync();
      mass = 0;
      for (int r = 0; r < C; ++r) mass += peer(&red.mass, r);
      goal = min(max((unsigned long long)ceil((double)tp * (double)mass), 1ull), mass);
    }
    int left = KB + ib;  // key bits not fixed yet
    while (left > 0) {
      const int d = min(kDigit, left), shift = left - d;
      clear();
      each(-INFINITY, [&](float v, int i) {
        if (i >= n) return;
        const unsigned long long key = ((unsigned long long)ordered<T>(v) << ib) | (unsigned)(a.vocab - 1 - (lo + i));
        if (left < KB + ib && (key >> left) != prefix) return;
        count_in((int)((key >> shift) & ((1u << d) - 1)), by_mass, v);
      });
      const int par = find(by_mass, goal - over);
      over += found_s[par][2];
      prefix = (prefix << d) | found_s[par][1];
      left = shift;
      // taken whole, or its one token is the last: all with keys from prefix << left on
      if (found_s[par][0] != 1 || found_s[par][3] == 1) break;
    }
    const unsigned long long bound = prefix << left;
    const Token b{from_ordered<T>((uint32_t)(bound >> ib)), a.vocab - 1 - (int)(bound & ((1ull << ib) - 1))};
    if (before(b, cut)) cut = b;
    if (!by_mass && use_p) erase();
  }

  // ---- the race
  unsigned long long best = 0;
  // min-p as a bound of the logit (a little low: the weight itself decides)
  const float least = greedy ? m : fmaxf(cut.x, mp > 0.f ? m + (log2f(mp) * 1.0001f - 1e-3f) / c2 : -INFINITY);
  auto kept = [&](float v, int i) { return v > -INFINITY && !before(cut, Token{v, lo + i}) && weight(v) >= mp; };
  if (greedy) {
    each(m, [&](float v, int i) {
      if (v == m) best = max64(best, (1ull << 32) | (0xffffffffu - (unsigned)(lo + i)));
    });
  } else {
    // All threads share the best quotient so far, a little lowered (lead_s): few tokens come near it, so the
    // division that decides, and the tests of what is kept, run for those only.
    const float* e = noise + lo;
    const bool vec = (reinterpret_cast<uintptr_t>(e) & 15) == 0;
    auto load_noise = [&](int i, float (&en)[VE]) {
      if (vec && (i + 1) * VE <= n) {
#pragma unroll
        for (int q = 0; q < VE / 4; ++q) {
          const uint4 b = ld_stream_u4(e + i * VE + 4 * q);
          en[4 * q] = __uint_as_float(b.x), en[4 * q + 1] = __uint_as_float(b.y);
          en[4 * q + 2] = __uint_as_float(b.z), en[4 * q + 3] = __uint_as_float(b.w);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) en[j] = i * VE + j < n ? __ldg(e + i * VE + j) : 1.f;
      }
    };
    float first = 0.f;  // from each thread's first tokens
    if (tid < nvec) {
      const uint4 w = get16(stage + tid * VE);
      if (Vec<T>::largest(w) >= least) {
        T v[VE];
        float en[VE];
        memcpy(v, &w, 16);
        load_noise(tid, en);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float x = to_f<T>(v[j]) + 0.f, q = __fdividef(weight(x), en[j]);
          if (kept(x, tid * VE + j) && q < 3e38f) first = fmaxf(first, q);
        }
      }
    }
    first = block_reduce(first, [](float p, float q) { return fmaxf(p, q); }, reinterpret_cast<float*>(scratch));
    if (tid == 0) best_s = 0, lead_s = __float_as_int(first * 0.9999f);
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < nvec; i += kThreads) {
      const uint4 w = get16(stage + i * VE);
      if (Vec<T>::largest(w) < least) continue;
      T v[VE];
      memcpy(v, &w, 16);
      float en[VE];
      load_noise(i, en);
      const float lead = __int_as_float(*reinterpret_cast<volatile int*>(&lead_s));
      bool near_lead = false;  // (w / e > lead; a negative or NaN e is no matter here)
#pragma unroll
      for (int j = 0; j < VE; ++j) near_lead |= weight(to_f<T>(v[j])) > lead * en[j];
      if (!near_lead) continue;
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float x = to_f<T>(v[j]) + 0.f;
        const int at = i * VE + j;
        if (!(weight(x) > lead * en[j]) || at >= n || !kept(x, at)) continue;
        const unsigned long long cand = ticket(weight(x), en[j], lo + at);
        if (cand >> 32 == 0) continue;
        atomicMax(&best_s, cand);
        atomicMax(&lead_s, __float_as_int(fminf(__uint_as_float((uint32_t)(cand >> 32)) * 0.9999f, 3e38f)));
      }
    }
    __syncthreads();
    best = best_s;
  }
  best = block_reduce(best, max64, scratch);
  if (tid == 0) red.best = best;
  cluster.sync();
#pragma unroll 1
  for (int r = 0; r < C; ++r) best = max64(best, peer(&red.best, r));
  if (best == 0) {  // every kept token's quotient is 0 (its noise infinite, negative or NaN): the first of them
    each(least, [&](float v, int i) {
      if (kept(v, i)) best = max64(best, 0xffffffffu - (unsigned)(lo + i));
    });
    best = block_reduce(best, max64, scratch);
    cluster.sync();
    if (tid == 0) red.best = best;
    cluster.sync();
#pragma unroll 1
    for (int r = 0; r < C; ++r) best = max64(best, peer(&red.best, r));
  }
  if (rank == 0 && tid == 0) finish(best);
  cluster.sync();  // the others' shared memory stays until rank 0 has read it
}

template <typename T>
cudaError_t launch_t(const SampleArgs& a, cudaStream_t st) {
  // CTAs of a row: enough that a slice fits in 64 KB (two CTAs an SM), more while all rows fit in one wave
  int C = 1;
  while (C < kMaxCluster && ((int64_t)a.vocab * (int64_t)sizeof(T) > C * 65536ll || (int64_t)a.rows * C * 2 <= num_sms()))
    C *= 2;
  const int slice = (div_up(a.vocab, C) + 7) / 8 * 8;
  constexpr int kFixed = kSplit * kThreads * 4 + 3 * kBins * 4 + 16;
  const size_t smem = kFixed + (size_t)slice * sizeof(T);
  auto kern = sample_kernel<T>;
  static std::atomic<bool> allowed[kMaxSmemDevices];
  constexpr int kMost = kFixed + (int)(kMaxVocab / kMaxCluster * sizeof(T));
  if (cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed, kMost)) return e;
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
