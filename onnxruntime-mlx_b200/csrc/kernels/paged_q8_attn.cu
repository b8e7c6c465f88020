// Attention of packed query rows over the 8-bit paged KV cache (layout: paged_q8.cuh).
//
// For row i of sequence b at position p: s_j = scale <q, K_j> ks_j (q after RoPE, K_j the codes, ks_j
// their scale), o = sum_j softmax(s)_j vs_j V_j over j = 0 .. p.  Every code is exact in fp16, so both
// products run on mma.sync.m16n8k16 with fp32 accumulation; ks multiplies the finished score and vs
// the probability.  With G query heads per kv head a cache byte feeds 2 G multiply-adds, so HBM bounds
// the kernel while the head group fits one matrix tile.
//
//   * Keys are the 16 rows of the tile and the query heads its 8 columns (S^T = K Q^T, O^T = V^T P^T):
//     groups of up to 8 heads fill the tile, where heads as rows would leave half of it empty.  The
//     score tile becomes the operand of the second product by movmatrix (an 8x8 transpose).
//   * The contraction order is free, so each thread takes D / 4 consecutive bytes of a key row (and
//     D / 8 of a value row) with wide shared-memory loads; the query is laid out to match.  No
//     ldmatrix, which moves 16-bit elements.
//   * q is divided by a power of two so that its largest element lies in [1, 2) (any input range fits
//     fp16); P vs is divided by a running power of two of vs and lifted by 2^14 (fp16 keeps 11 bits
//     down to 2^-28 of the largest).  SPLIT carries q and P as the sum of two fp16 numbers (22 bits),
//     for fp32 rows.
//   * Work is cut evenly: the (row, kv head, head chunk, 32-key unit) list of the whole batch, in that
//     order, is divided into equal runs, one per CTA, so ragged lengths cost nothing.  The 4 warps of a
//     CTA take its units in turn; each streams its own through kStages shared-memory buffers (16-byte
//     cp.async, swizzled) and runs ahead over the run's segment borders.
//   * A segment (the part of one (row, head chunk) within a run) is merged over the warps; a segment
//     that is not the whole of its row goes to the workspace, and the last CTA to arrive joins the
//     parts in the order of the keys, so results do not depend on timing.
// A row whose position lies outside the block table or the cos / sin rows, or that no sequence owns, gives zeros; a key
// whose page lies outside the tables is skipped; both set the device error word.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "paged_q8.cuh"

namespace b200ep {
namespace {

constexpr int kWarps = 4;
constexpr int kUnit = 32;  // keys of a unit
constexpr int kLift = 14;  // P vs is held times 2^kLift

template <int D, int NT>
struct Cfg {
  static constexpr int kStages = D >= 256 ? 3 : D == 128 ? 3 : 4;
  static constexpr int kCtasPerSm = D >= 256 || (D == 128 && NT == 2) ? 1 : 2;
  static constexpr int kHeads = 8 * NT;
  static constexpr int kData = kUnit * D;                          // K (or V) codes of a unit
  static constexpr int kStageBytes = 2 * kData + 2 * kUnit * 4;    // K, V, ks, vs
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kMerge = kRing;                             // [2][kHeads][D + 4] fp32 (two warps at a time)
  static constexpr int kMl = kMerge + 2 * kHeads * (D + 4) * 4;    // [kWarps][kHeads][2] fp32
  static constexpr int kMeta = kMl + kWarps * kHeads * 2 * 4;      // [kWarps][kStages] Meta
  static constexpr int kTotal = kMeta + kWarps * kStages * 32;
};

struct Meta {  // what a streamed unit is
  int row, hc, u, n;
  uint32_t valid;
  int pad[3];
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Byte offset of 16-byte chunk ch of key r in a unit, chosen so that the loads of both products touch
// all banks: rows 2c of four threads, and rows g of eight, land on different chunks.
template <int D>
__device__ __forceinline__ int swz(int r, int ch) {
  if constexpr (D >= 128) return r * D + ((ch ^ (r & 7)) << 4);
  if constexpr (D == 64) return (r >> 1) * 128 + (((r ^ (r >> 1)) & 1) << 6) + ((ch ^ ((r >> 1) & 2)) << 4);
  return (r >> 2) * 128 + (((r + (r >> 2)) & 3) << 5) + (ch << 4);
}

// Byte offset within a row of the w-th 4-byte word that thread c of a quad takes of a key (D / 16 words).
template <int D>
__host__ __device__ __forceinline__ constexpr int kbyte(int c, int w) {
  if (D >= 128) return ((w >> 3) * 8 + 2 * c + ((w >> 2) & 1)) * 16 + (w & 3) * 4;
  return c * (D / 4) + w * 4;
}
// ... and of the first of the D / 8 value bytes (two runs of 16 for D = 256) of thread row g.
template <int D>
__host__ __device__ __forceinline__ constexpr int vbyte(int g, int w) {
  if (D == 256) return (w >> 2) * 128 + g * 16 + (w & 3) * 4;
  return g * (D / 8) + w * 4;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// The four codes of a word as two f16x2 (codes 0, 1 and 2, 3); e4m3 values come out times 2^-8.
template <int CT>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& h01, uint32_t& h23) {
  if constexpr (CT == kI8) {
    // 0x6400 | (code + 128) is 1024 + 128 + code in fp16
    const uint32_t x = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    uint32_t a = prmt(x, 0x64646464u, 0x4140), b = prmt(x, 0x64646464u, 0x4342);
    __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), bias), hb = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    h01 = *reinterpret_cast<uint32_t*>(&ha), h23 = *reinterpret_cast<uint32_t*>(&hb);
  } else {
    // sign to bit 15, exponent and mantissa to bits 13..7: the same number with fp16's bias, 2^8 lower
    const uint32_t a = prmt(w, 0, 0x1404), b = prmt(w, 0, 0x3424);
    h01 = ((a >> 1) & 0x3f803f80u) | (a & 0x80008000u);
    h23 = ((b >> 1) & 0x3f803f80u) | (b & 0x80008000u);
  }
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t* r) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(addr));
}
__device__ __forceinline__ float lds_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Element d of query row x after RoPE at position pos, in fp32.
template <typename T>
__device__ __forceinline__ float q_at(const T* x, int d, const PagedQ8& kp, int pos) {
  const float v = to_f<T>(x[d]);
  if (!kp.rot || d >= 2 * kp.half) return v;
  int pi, o;
  bool first;
  if (kp.inter) {
    first = !(d & 1), pi = d >> 1, o = d ^ 1;
  } else {
    first = d < kp.half, pi = first ? d : d - kp.half, o = first ? d + kp.half : pi;
  }
  const float c = to_f<T>(static_cast<const T*>(kp.cos_c)[(size_t)pos * kp.half + pi]);
  const float s = to_f<T>(static_cast<const T*>(kp.sin_c)[(size_t)pos * kp.half + pi]);
  const float y = to_f<T>(x[o]);
  return first ? __fsub_rn(__fmul_rn(v, c), __fmul_rn(y, s)) : __fadd_rn(__fmul_rn(v, c), __fmul_rn(y, s));
}

// Keys that row i sees (0: none, an invalid row) and its sequence.
__device__ __forceinline__ int row_keys(const PagedQ8& kp, int i, int& seq) {
  seq = i < kp.ntok ? q8_seq(kp.cum, kp.batch, i) : -1;
  if (seq < 0) return 0;
  const int pos = __ldg(kp.past + seq) + (i - __ldg(kp.cum + seq));
  return pos < 0 || pos >= (int64_t)kp.maxb * kp.bs || (kp.rot && pos >= kp.max_seq) ? 0 : pos + 1;
}

__global__ void paged_q8_reset_kernel(int* counters, int n) {
  pdl_wait();
  pdl_trigger();
  for (int t = threadIdx.x; t < n; t += blockDim.x) counters[t] = 0;
}

template <typename T, int D, int CT, int NT>
__global__ void __launch_bounds__(kWarps * 32, (Cfg<D, NT>::kCtasPerSm))
paged_q8_attn_kernel(PagedQ8 kp, int hchunks, int appended) {
  using C = Cfg<D, NT>;
  constexpr bool SPLIT = std::is_same<T, float>::value;
  constexpr int NS = SPLIT ? 2 : 1;   // fp16 terms of q and of P
  constexpr int KW = D / 16;          // 4-byte words of a key per thread = k-steps of q.k
  constexpr int VW = D / 32;          // 4-byte words of a value row per thread
  constexpr int MT = D / 16;          // 16-dim tiles of the output
  constexpr int KV = KW >= 4 ? 4 : KW;   // words of one load
  constexpr int VV = VW >= 4 ? 4 : VW;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ long long plan_s[3];
  __shared__ int scan_s[kWarps], plan_i[3], flag_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const uint32_t sbase = smem_u32(sm);
  const uint32_t ring = sbase + warp * C::kStages * C::kStageBytes;
  Meta* meta = reinterpret_cast<Meta*>(sm + C::kMeta) + warp * C::kStages;
  float* mls = reinterpret_cast<float*>(sm + C::kMl);
  const int HC = kp.HK * hchunks;
  bool waited = false;
  if (appended) {  // the launch before this one wrote rows that are read here
    pdl_wait();
    waited = true;
  }

  // ---- this CTA's run [w0, w1) of the unit list, and the row that w0 lies in
  long long total = 0;
  for (int i0 = 0; i0 < kp.ntok; i0 += kWarps * 32) {
    int seq, i = i0 + tid, n = row_keys(kp, i, seq);
    if (i < kp.ntok && n == 0 && i % (int)gridDim.x == (int)blockIdx.x) {
      T* o = static_cast<T*>(kp.out) + (size_t)i * kp.H * D;
      // (no launch before this one reads `out` unless it already completed or is waited for here)
      if (!waited) pdl_wait();
      for (int e = 0; e < kp.H * D; ++e) o[e] = from_f<T>(0.f);
      report_device_error(kp.err, kErrPagedQ8, i);
    }
    int s = (n + kUnit - 1) / kUnit;
    s = __reduce_add_sync(0xffffffffu, s);
    if (lane == 0) scan_s[warp] = s;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) total += scan_s[w];
    __syncthreads();
  }
  const long long W = total * HC;
  const long long ctas = max(1ll, min((long long)gridDim.x, (W + kWarps - 1) / kWarps));
  const int cta = blockIdx.x;
  if (W == 0 || cta >= ctas) {
    if (!waited) pdl_wait();
    pdl_trigger();
    return;
  }
  const long long w0 = W * cta / ctas, w1 = W * (cta + 1) / ctas;
  {
    long long base = 0;
    for (int i0 = 0; i0 < kp.ntok; i0 += kWarps * 32) {
      int seq, i = i0 + tid, n = row_keys(kp, i, seq);
      const int nu = (n + kUnit - 1) / kUnit;
      int inc = nu;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
      }
      if (lane == 31) scan_s[warp] = inc;
      __syncthreads();
      long long pre = base;
      int all = 0;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) pre += scan_s[w];
        all += scan_s[w];
      }
      pre += inc - nu;
      if (nu && pre * HC <= w0 && w0 < (pre + nu) * HC) {
        plan_i[0] = i;
        plan_s[0] = pre * HC;
      }
      base += all;
      const bool found = base * HC > w0;
      __syncthreads();
      if (found) break;
    }
  }
  // a position in the unit list: unit u of head chunk hc of row `row`
  struct Pos {
    int row, seq, n, nu, hc, u;
  };
  auto settle = [&](Pos& p) {  // carries u past the head chunks and rows that it has left
    while (p.u >= p.nu) {
      p.u -= p.nu;
      if (++p.hc == HC) {
        p.hc = 0;
        do {
          ++p.row;
          p.n = row_keys(kp, p.row, p.seq);
        } while (p.n == 0 && p.row < kp.ntok);
        p.nu = (p.n + kUnit - 1) / kUnit;
        if (p.row >= kp.ntok) {  // past the end: nothing is issued from here
          p.nu = 0x7fffffff;
        }
      }
    }
  };
  Pos at;  // the segment in work
  at.row = plan_i[0];
  at.n = row_keys(kp, at.row, at.seq);
  at.nu = (at.n + kUnit - 1) / kUnit;
  {
    const long long off = w0 - plan_s[0];
    at.hc = (int)(off / at.nu);
    at.u = (int)(off % at.nu);
  }

  // ---- the warp's stream: units x = warp, warp + 4, ... of the run
  Pos is = at;
  is.u += warp;
  settle(is);
  long long ix = warp;             // of the next unit to issue
  const long long run = w1 - w0;
  auto lookup = [&]() -> int {     // page row of key `lane` of the next unit, or -1
    if (ix >= run) return -1;
    const int key = is.u * kUnit + lane;
    return key < is.n ? q8_row(kp.bt, kp.maxb, kp.nblocks, kp.bs, kp.HK, is.seq, is.hc / hchunks, key) : -1;
  };
  int next_row = lookup();
  bool bad = false;
  auto issue = [&](int stage) {
    if (ix < run) {
      const int row = next_row, key = is.u * kUnit + lane;
      bad |= row < 0 && key < is.n;
      const uint32_t dst = ring + stage * C::kStageBytes;
      constexpr int CH = D / 16;  // chunks of a row
#pragma unroll
      for (int t = 0; t < CH; ++t) {
        const int idx = t * 32 + lane, r = idx / CH, ch = idx % CH;
        const int src = __shfl_sync(0xffffffffu, row, r);
        const size_t o = (size_t)(src < 0 ? 0 : src) * D + ch * 16;
        const uint32_t d = dst + swz<D>(r, ch);
        cp16(d, kp.kc + o, src >= 0);
        cp16(d + C::kData, kp.vc + o, src >= 0);
      }
      cp4(dst + 2 * C::kData + lane * 4, kp.kscale + (row < 0 ? 0 : row), row >= 0);
      cp4(dst + 2 * C::kData + kUnit * 4 + lane * 4, kp.vscale + (row < 0 ? 0 : row), row >= 0);
      const uint32_t valid = __ballot_sync(0xffffffffu, row >= 0);
      if (lane == 0) {
        Meta m;
        m.row = is.row, m.hc = is.hc, m.u = is.u, m.n = is.n, m.valid = valid;
        meta[stage] = m;
      }
      ix += kWarps;
      is.u += kWarps;
      if (ix < run) settle(is);
      next_row = lookup();
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) issue(s);

  int stage = 0;
  long long x = 0;  // first unit of the segment, within the run
  long long mine = warp;  // the warp's next unit
  while (x < run) {
    const int nseg = (int)min((long long)(at.nu - at.u), run - x);  // units of this segment
    const int kvh = at.hc / hchunks, h0 = kvh * kp.G + (at.hc % hchunks) * C::kHeads;  // first query head
    const int heads = min(C::kHeads, kp.G - (at.hc % hchunks) * C::kHeads);
    // q as the second operand: thread (g, c) holds head g, the dims of its key bytes
    uint32_t qf[NS][NT][KW][2];
    float qs[NT][2];  // per owned score column (heads 2c, 2c + 1): what turns a score into base-2 logits
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int hq = nt * 8 + g;
      const T* qrow = static_cast<const T*>(kp.q) + (size_t)at.row * kp.qs + (size_t)(h0 + hq) * D;
      float qv[KW * 4];
      float amax = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          qv[w * 4 + e] = hq < heads ? q_at<T>(qrow, kbyte<D>(c, w) + e, kp, at.n - 1) : 0.f;
          amax = fmaxf(amax, fabsf(qv[w * 4 + e]));
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int ex = min(max((int)(__float_as_uint(amax) >> 23), 1), 253);  // biased exponent
      const float down = __uint_as_float((uint32_t)(254 - ex) << 23), up = __uint_as_float((uint32_t)ex << 23);
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a = qv[w * 4 + 2 * e] * down, b = qv[w * 4 + 2 * e + 1] * down;
          const __half2 hi = __floats2half2_rn(a, b);
          qf[0][nt][w][e] = *reinterpret_cast<const uint32_t*>(&hi);
          if constexpr (SPLIT) qf[1][nt][w][e] = half2_bits(a - __low2float(hi), b - __high2float(hi));
        }
      const float f = up * kp.scale * (CT == kE4M3 ? 256.f : 1.f) * 1.4426950408889634f;
      qs[nt][0] = __shfl_sync(0xffffffffu, f, 8 * c);
      qs[nt][1] = __shfl_sync(0xffffffffu, f, 8 * c + 4);
    }

    float o[MT][NT][4], m[NT][2], l[NT][2];
    int E = kLift + 1;  // biased exponent that P vs is relative to
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int t = 0; t < MT; ++t) o[t][nt][0] = o[t][nt][1] = o[t][nt][2] = o[t][nt][3] = 0.f;
    }

    for (; mine < x + nseg; mine += kWarps) {
      cp_wait<C::kStages - 2>();
      __syncwarp();
      const int ahead = stage == 0 ? C::kStages - 1 : stage - 1;  // the buffer that was consumed last
      issue(ahead);
      const uint32_t buf = ring + stage * C::kStageBytes;
      const uint32_t valid = meta[stage].valid;
      const uint32_t sks = buf + 2 * C::kData, svs = sks + kUnit * 4;
      // S^T: two 16-key tiles
      float s[2][NT][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[kt][nt][0] = s[kt][nt][1] = s[kt][nt][2] = s[kt][nt][3] = 0.f;
#pragma unroll
        for (int w0_ = 0; w0_ < KW; w0_ += KV) {
          uint32_t ka[KV], kb[KV];
          const int r0 = kt * 16 + g, byte = kbyte<D>(c, w0_);
          lds<KV * 4>(buf + swz<D>(r0, byte >> 4) + (byte & 15), ka);
          lds<KV * 4>(buf + swz<D>(r0 + 8, byte >> 4) + (byte & 15), kb);
#pragma unroll
          for (int w = 0; w < KV; ++w) {
            uint32_t a[4];
            widen<CT>(ka[w], a[0], a[2]);
            widen<CT>(kb[w], a[1], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int t = 0; t < NS; ++t) mma(s[kt][nt], a, qf[t][nt][w0_ + w][0], qf[t][nt][w0_ + w][1]);
          }
        }
      }
      // scores in base 2; keys g and g + 8 of each tile
      float vsk[2][2];
      float mx[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mx[nt][0] = m[nt][0], mx[nt][1] = m[nt][1];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = kt * 16 + r * 8 + g;
          const float ks = lds_f(sks + key * 4);
          const bool on = (valid >> key) & 1u;
          vsk[kt][r] = lds_f(svs + key * 4);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float v = on ? s[kt][nt][r * 2 + h] * (ks * qs[nt][h]) : -INFINITY;
              s[kt][nt][r * 2 + h] = v;
              mx[nt][h] = fmaxf(mx[nt][h], v);
            }
        }
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) mx[nt][h] = fmaxf(mx[nt][h], __shfl_xor_sync(0xffffffffu, mx[nt][h], d));
          moved |= mx[nt][h] > m[nt][h];
        }
      // the running power of two of the value scales
      const int eu = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(lds_f(svs + lane * 4))) >> 23);
      const int En = min(max(E, eu), 253);
      if (En != E || __any_sync(0xffffffffu, moved)) {
        const float back = __uint_as_float((uint32_t)max(127 + E - En, 0) << 23);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float a = m[nt][h] == -INFINITY ? 0.f : ex2(m[nt][h] - mx[nt][h]);
            l[nt][h] *= a;
            m[nt][h] = mx[nt][h];
#pragma unroll
            for (int t = 0; t < MT; ++t) o[t][nt][h] *= a * back, o[t][nt][2 + h] *= a * back;
          }
        E = En;
      }
      const float down = __uint_as_float((uint32_t)(254 + kLift - E) << 23);  // 2^(127 + kLift - E)
      // P^T into the second operand
      uint32_t pf[NS][2][NT][2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float vs = vsk[kt][r] * down;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float p[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float v = s[kt][nt][r * 2 + h];
              p[h] = v == -INFINITY ? 0.f : ex2(v - m[nt][h]);
              l[nt][h] += p[h];
              p[h] *= vs;
            }
            const __half2 hi = __floats2half2_rn(p[0], p[1]);
            pf[0][kt][nt][r] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hi));
            if constexpr (SPLIT)
              pf[1][kt][nt][r] = transpose8x8(half2_bits(p[0] - __low2float(hi), p[1] - __high2float(hi)));
          }
        }
      // O^T += V^T P^T
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int w0_ = 0; w0_ < VW; w0_ += VV) {
          uint32_t v[4][VV];  // value rows 2c, 2c + 1, 2c + 8, 2c + 9
          const int byte = vbyte<D>(g, w0_);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = kt * 16 + 2 * c + (r & 1) + (r >> 1) * 8;
            lds<VV * 4>(buf + C::kData + swz<D>(key, byte >> 4) + (byte & 15), v[r]);
          }
#pragma unroll
          for (int w = 0; w < VV; ++w) {
            // codes of two keys side by side, dim by dim
            uint32_t d01[2], d23[2], d[2][4];
            d01[0] = prmt(v[0][w], v[1][w], 0x5140), d23[0] = prmt(v[0][w], v[1][w], 0x7362);
            d01[1] = prmt(v[2][w], v[3][w], 0x5140), d23[1] = prmt(v[2][w], v[3][w], 0x7362);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              widen<CT>(d01[r], d[r][0], d[r][1]);
              widen<CT>(d23[r], d[r][2], d[r][3]);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t a[4] = {d[0][2 * t], d[0][2 * t + 1], d[1][2 * t], d[1][2 * t + 1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < NS; ++u) mma(o[(w0_ + w) * 2 + t][nt], a, pf[u][kt][nt][0], pf[u][kt][nt][1]);
            }
          }
        }
      __syncwarp();
      stage = stage + 1 == C::kStages ? 0 : stage + 1;
    }

    // ---- the segment's end: join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], d);
    if (g == 0)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int hd = nt * 8 + 2 * c + h;
          mls[(warp * C::kHeads + hd) * 2] = m[nt][h];
          mls[(warp * C::kHeads + hd) * 2 + 1] = l[nt][h];
        }
    __syncthreads();
    float mt_[NT][2], lt[NT][2];
    {
      const float unscale = __uint_as_float((uint32_t)min(E, 253) << 23) * (CT == kE4M3 ? 0x1p-6f : 0x1p-14f);
      static_assert(kLift == 14, "the power above");
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int hd = nt * 8 + 2 * c + h;
          float mm = -INFINITY, ll = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, mls[(w * C::kHeads + hd) * 2]);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float lw = mls[(w * C::kHeads + hd) * 2 + 1];
            if (lw != 0.f) ll += lw * ex2(mls[(w * C::kHeads + hd) * 2] - mm);  // (a NaN stays one)
          }
          mt_[nt][h] = mm, lt[nt][h] = ll;
          const float f = l[nt][h] == 0.f ? 0.f : ex2(m[nt][h] - mm) * unscale;  // 0: the warp saw no key, o = 0
#pragma unroll
          for (int t = 0; t < MT; ++t) o[t][nt][h] *= f, o[t][nt][2 + h] *= f;
        }
    }
    // warps 2, 3 hand theirs to 0, 1, then 1 to 0 (always the same order of additions)
    float* mg = reinterpret_cast<float*>(sm + C::kMerge);
    constexpr int MS = D + 4;
    auto put = [&](int slot) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < MT; ++t)
            *reinterpret_cast<float2*>(mg + (slot * C::kHeads + nt * 8 + 2 * c + h) * MS + vbyte<D>(g, t >> 1) + (t & 1) * 2) =
                make_float2(o[t][nt][h], o[t][nt][2 + h]);
    };
    auto add = [&](int slot) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const float2 v = *reinterpret_cast<const float2*>(
                mg + (slot * C::kHeads + nt * 8 + 2 * c + h) * MS + vbyte<D>(g, t >> 1) + (t & 1) * 2);
            o[t][nt][h] += v.x, o[t][nt][2 + h] += v.y;
          }
    };
    if (warp >= 2) put(warp - 2);
    __syncthreads();
    if (warp < 2) add(warp);
    __syncthreads();
    if (warp == 1) put(0);
    __syncthreads();
    if (warp == 0) {
      add(0);
      put(1);
      if (g == 0)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int hd = nt * 8 + 2 * c + h;
            mls[hd * 2] = mt_[nt][h];  // (every warp has read the others' by now)
            mls[hd * 2 + 1] = lt[nt][h];
          }
    }
    __syncthreads();
    const float* res = mg + C::kHeads * MS;
    const bool whole = nseg == at.nu;
    if (!waited) {  // before anything is written
      pdl_wait();
      waited = true;
    }
    T* out = static_cast<T*>(kp.out) + (size_t)at.row * kp.H * D + (size_t)h0 * D;
    if (whole) {
      for (int e = tid; e < heads * D; e += kWarps * 32) {
        const int hd = e / D;
        const float ll = mls[hd * 2 + 1];
        out[e] = from_f<T>(ll == 0.f ? 0.f : res[hd * MS + e % D] / ll);
      }
    } else {
      const int slot = 2 * cta + (at.u > 0 ? 0 : 1);
      float* part = kp.part + (size_t)slot * C::kHeads * (D + 2);
      for (int e = tid; e < heads * D; e += kWarps * 32) part[(e / D) * (D + 2) + e % D] = res[(e / D) * MS + e % D];
      if (tid < 2 * heads) part[(tid >> 1) * (D + 2) + D + (tid & 1)] = mls[tid];
      __threadfence();
      __syncthreads();
      // the runs that hold units of this (row, head chunk)
      const long long a = w0 + x - at.u, z = a + at.nu;
      const int kf = (int)(((a + 1) * ctas - 1) / W), kl = (int)((z * ctas - 1) / W);
      if (tid == 0) flag_s = atomicAdd(kp.counters + kf, 1) == kl - kf;
      __syncthreads();
      if (flag_s) {  // the last to arrive joins the parts
        __threadfence();
        for (int e = tid; e < heads * D; e += kWarps * 32) {
          const int hd = e / D;
          float mm = -INFINITY, ll = 0.f, acc = 0.f;
          for (int k = kf; k <= kl; ++k) {
            const long long k0 = W * k / ctas;
            const float* pp = kp.part + ((size_t)(2 * k + (k0 > a ? 0 : 1)) * C::kHeads + hd) * (D + 2);
            const float mk = __ldcg(pp + D), lk = __ldcg(pp + D + 1), ok = __ldcg(pp + e % D);
            if (lk == 0.f) continue;
            const float mn = fmaxf(mm, mk);
            const float fa = mm == -INFINITY ? 0.f : ex2(mm - mn), fb = ex2(mk - mn);
            ll = ll * fa + lk * fb;
            acc = acc * fa + ok * fb;
            mm = mn;
          }
          out[e] = from_f<T>(ll == 0.f ? 0.f : acc / ll);
        }
      }
    }
    __syncthreads();  // the merge buffers and mls are free again
    x += nseg;
    at.u += nseg;
    if (x < run) settle(at);
  }
  cp_wait<0>();
  if (__any_sync(0xffffffffu, bad) && lane == 0) report_device_error(kp.err, kErrPagedQ8, at.row);
  pdl_trigger();
}

template <typename T, int D, int CT, int NT>
cudaError_t launch_t(const PagedQ8& a, bool appended, cudaStream_t st) {
  using C = Cfg<D, NT>;
  auto kern = paged_q8_attn_kernel<T, D, CT, NT>;
  if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal)) return e;
  if (!appended)
    if (cudaError_t e = launch_k(paged_q8_reset_kernel, dim3(1), dim3(256), 0, st, a.counters, a.ctas)) return e;
  const int hchunks = (a.G + C::kHeads - 1) / C::kHeads;
  const int grid = std::min(a.ctas, num_sms() * C::kCtasPerSm);
  return launch_k(kern, dim3((unsigned)grid), dim3(kWarps * 32), C::kTotal, st, a, hchunks, appended ? 1 : 0);
}

template <typename T, int D, int CT>
cudaError_t by_group(const PagedQ8& a, bool appended, cudaStream_t st) {
  if constexpr (D <= 128)
    if (paged_q8_heads_per_cta(D, a.G) == 16) return launch_t<T, D, CT, 2>(a, appended, st);
  return launch_t<T, D, CT, 1>(a, appended, st);
}

template <typename T, int CT>
cudaError_t by_head(const PagedQ8& a, bool appended, cudaStream_t st) {
  switch (a.D) {
    case 32: return by_group<T, 32, CT>(a, appended, st);
    case 64: return by_group<T, 64, CT>(a, appended, st);
    case 128: return by_group<T, 128, CT>(a, appended, st);
    case 256: return by_group<T, 256, CT>(a, appended, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

int paged_q8_max_ctas() { return 2 * num_sms(); }
// more than 8 query heads per kv head: 16 to a CTA (two column tiles share each widened code), except
// at head size 256, whose output tile would not fit the registers
int paged_q8_heads_per_cta(int D, int G) { return G > 8 && D <= 128 ? 16 : 8; }

cudaError_t launch_paged_q8_attn(const PagedQ8& a, bool appended, cudaStream_t st) {
  const bool i8 = a.ctype == kI8;
  switch (a.dtype) {
    case kF32: return i8 ? by_head<float, kI8>(a, appended, st) : by_head<float, kE4M3>(a, appended, st);
    case kF16: return i8 ? by_head<__half, kI8>(a, appended, st) : by_head<__half, kE4M3>(a, appended, st);
    case kBF16:
      return i8 ? by_head<__nv_bfloat16, kI8>(a, appended, st) : by_head<__nv_bfloat16, kE4M3>(a, appended, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace b200ep
