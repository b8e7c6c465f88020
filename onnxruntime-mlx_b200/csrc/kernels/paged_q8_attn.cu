// Attention of packed query rows over the 8-bit paged KV cache (layout: paged_q8.cuh).
//
// For row i of sequence b at position p: s_j = scale <q, K_j> ks_j (q after RoPE, K_j the codes, ks_j
// their scale), o = sum_j softmax(s)_j vs_j V_j over j = 0 .. p.  With G query heads per kv head a cache
// byte feeds 2 G multiply-adds, so HBM should bound it at long contexts: 64 sequences of 8192 keys (32 / 8
// heads, head size 128, fp16) take 207 us on int8 and 202 us on e4m3 codes, 82 and 84 % of the copy
// rate in cache bytes, at 1965 MHz; its instructions are as near a bound: back to back for longer the power cap holds
// 1.69 GHz, and the time follows the clock (230 us).  Short ragged contexts are bound by what a segment costs to start
// and end (256 rows of 1 to 500 keys: 52 us), one sequence alone by latency (1024 keys: 12.4 us).
//
//   * Products on mma.sync with keys as the 16 rows and the query heads as the 8 columns of a tile
//     (S^T = K Q^T, O^T = V^T P^T): groups of up to 8 heads fill it, where heads as rows would leave half
//     of it empty.  The score tile becomes the operand of the second product by movmatrix.  tcgen05 has
//     64 or 128 rows for these 4 to 16 heads, and takes no operand with a scale per key.
//   * int8: K Q^T on integer products (m16n8k32), q as three bytes of a fixed-point number,
//     exact but for q's last place; the codes go from shared memory straight into the tile.  (Widening
//     them to fp16 and splitting q in two there: 212 us instead of 197 at that step.)  e4m3: codes widened to fp16 by
//     the conversion instruction (193 us where bit shifts took 280 at that step; mma on the e4m3 codes themselves, q as
//     four e4m3 numbers: 244 us), q as two fp16 numbers over a power of two that brings its
//     largest element into [1, 2).
//   * V widens to fp16 (both kinds of code are exact there).  P vs is held times a power of two, each head's own, that
//     brings the largest product of a warp's keys so far into [2^kLift, kFull), as two fp16 numbers: 22 bits, and a
//     smallest step of 2^-31 of that product.  (Of the products, and for each head: a value row of a huge scale takes no
//     bits from the heads that give its key no weight; with one power for all heads, of the scales alone, the int8 case
//     took 203 us.)  One adds as much error again as an fp16 output's own rounding
//     (1.4 times plain fp32's against 64 bits, 1.0 times with two; 194 us against 203).  RoPE leaves q with more bits than
//     the rows' type, and an output that averages many values is far smaller than they are, so bf16 rows need the same: q
//     and P in one fp16 number (q in two bytes) moved 9 to 14 % of their outputs to a neighbouring number, none with two
//     (64 x 8192: 187 us against 205).
//     ks multiplies the finished score.  Sums and statistics are fp32.
//   * The running maximum and the power of two move only when a sum or a product passes its limit: most units cost
//     one vote instead of the shuffles of exact maxima.
//   * The contraction order is free, so each thread takes D / 4 consecutive bytes of a key row (and
//     D / 8 of a value row) with wide shared-memory loads; the query is laid out to match.  No
//     ldmatrix, which moves 16-bit elements.
//   * Work is cut evenly: the list of (row, kv head, head chunk, unit of 16 or 32 keys) of the whole batch
//     is divided into runs of equal weight, one per CTA, so ragged lengths cost nothing; a segment's start
//     weighs kOver units (without that the CTAs with many short segments ended last: 256 short rows 74 us
//     instead of 51).  The 4 warps of a CTA take its units in turn; each streams its own through kStages
//     shared-memory buffers (16-byte cp.async, swizzled; a unit lies in one page where the block size
//     allows) and runs ahead over the run's segment borders.  Four CTAs an SM (16 warps): instruction
//     latency, not bytes in flight, is what they hide (two CTAs of twice the unit: 235 us).
//   * A segment (the part of one (row, head chunk) within a run) is merged over the warps; a segment
//     that is not the whole of its row goes to the workspace, and the last CTA to arrive joins the
//     parts in the order of the keys, so results do not depend on timing.
// A row whose position lies outside the block table or the cos / sin rows, or that no sequence owns, gives zeros; a key
// whose page lies outside the tables is skipped; both set the device error word.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "paged_q8.cuh"

namespace b200ep {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRowTab = 48;
constexpr int kLift = 6;       // P vs is held times 2^kLift
constexpr float kLow = -1e30f;  // the running maximum before the first key: far below any, and finite
constexpr float kSlack = 0x1p64f;  // the sum of exp(score - running maximum) may reach this before the maximum moves,
constexpr float kFull = 16384.f;   // and a product with the value's scale, as it is held, this

template <typename T, int D, int CT, int NT>
struct Cfg {
  static constexpr bool kInt = CT == kI8;  // K Q^T on 8-bit integers: q as kNQ bytes; else q as kNQ fp16 terms
  static constexpr int kNQ = kInt ? 3 : 2;
  static constexpr int kNP = 2;  // fp16 terms of P
  static constexpr int kUnit = 16 * NT;  // keys of a unit
  static constexpr int kOver = 8 / NT;   // units that a segment's start and end are counted as
  static constexpr int kHeads = 8 * NT;  // query heads of a CTA
  static constexpr int kStages = D >= 128 ? 3 : D == 64 ? 5 : 8;
  static constexpr int kCtasPerSm = D == 256 || NT == 2 ? 2 : std::is_same<T, float>::value ? 3 : 4;
  static constexpr int kData = kUnit * D;                         // K (or V) codes of a unit
  static constexpr int kStageBytes = 2 * kData + 2 * kUnit * 4;   // K, V, ks, vs; holds [kHeads][D] fp32 at a merge
  static constexpr int kQ = kWarps * kStages * kStageBytes;       // the query operand
  static constexpr int kQBytes = kNQ * NT * (D / 16) * 32 * (kInt ? 4 : 8);
  static constexpr int kMl = kQ + kQBytes;                        // [kWarps][kHeads] (m, l)
  static constexpr int kScale = kMl + kWarps * kHeads * 8;        // [kHeads] score factor
  static constexpr int kMisc = kScale + kHeads * 4;               // [kWarps][kHeads] output factor, [kWarps] buffer
  static constexpr int kRaw = kMisc + kWarps * (kHeads + 1) * 4;  // the next segment's q rows, cos and sin row
  static constexpr int kStatic = 768;                             // (bound on the static shared memory)
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
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

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  return word_of(__floats2half2_rn(lo, hi));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t* r) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float lds_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Element d of query row x after RoPE by the row (cs, sn), in fp32.
template <typename T>
__device__ __forceinline__ float q_at(const T* x, int d, const PagedQ8& kp, const T* cs, const T* sn) {
  const float v = to_f<T>(x[d]);
  if (!kp.rot || d >= 2 * kp.half) return v;
  const bool first = kp.inter ? !(d & 1) : d < kp.half;
  const int pi = kp.inter ? d >> 1 : first ? d : d - kp.half;
  const float y = to_f<T>(x[kp.inter ? d ^ 1 : first ? d + kp.half : pi]), c = to_f<T>(cs[pi]), s = to_f<T>(sn[pi]);
  const float a = __fmul_rn(v, c), b = __fmul_rn(y, s);
  return first ? __fsub_rn(a, b) : __fadd_rn(a, b);
}

// Keys that row i sees (0: none, an invalid row) and its sequence.  Out of line: it is needed in many places, and
// what runs once per CTA costs instruction fetches.
__device__ __noinline__ int2 row_keys(const int32_t* cum, const int32_t* past_, int ntok, int batch, int most, int i) {
  if (i >= ntok) return make_int2(0, -1);
  int seq = i, past = i < batch ? __ldg(past_ + i) : 0, first = i;  // (one new token per sequence: row i is sequence i)
  if (!(i < batch && __ldg(cum + i) == i && __ldg(cum + i + 1) == i + 1)) {
    seq = q8_seq(cum, batch, i);
    if (seq < 0) return make_int2(0, -1);
    past = __ldg(past_ + seq), first = __ldg(cum + seq);
  }
  const int pos = past + (i - first);
  return make_int2(pos < 0 || pos >= most ? 0 : pos + 1, seq);
}

// a / b for a >= 0, b > 0: almost always of 32-bit numbers
__device__ __forceinline__ long long div64(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (uint32_t)a / (uint32_t)b : a / b;
}

__global__ void paged_q8_reset_kernel(int* counters, int n) {
  pdl_wait();
  pdl_trigger();
  for (int t = threadIdx.x; t < n; t += blockDim.x) counters[t] = 0;
}

// Pair p (dims 2p, 2p + 1) of head h in a warp's [kHeads][D] merge buffer: the 16 lanes that store at
// once (4 g x 4 c) land on different 8-byte banks.
template <int D>
__device__ __forceinline__ int merge_at(int h, int p) {
  const int c = (h >> 1) & 3;
  const int f = D >= 128 ? ((p >> 4) & 1) | (c << 1) : D == 64 ? c : (c & 1) | ((c >> 1) << 3);
  return h * (D / 2) + (p ^ f);
}

// acc / l to four elements of the output (0 where no key was seen)
template <typename T>
__device__ __forceinline__ void store4(T* dst, float4 a, float l) {
  const float r = l == 0.f ? 0.f : __frcp_rn(l);
  alignas(4 * sizeof(T)) T v[4] = {from_f<T>(a.x * r), from_f<T>(a.y * r), from_f<T>(a.z * r), from_f<T>(a.w * r)};
  using W = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
  W w;
  memcpy(&w, v, sizeof(w));
  *reinterpret_cast<W*>(dst) = w;
}

template <typename T, int D, int CT, int NT>
__global__ void __launch_bounds__(kThreads, (Cfg<T, D, CT, NT>::kCtasPerSm))
paged_q8_attn_kernel(PagedQ8 kp, int hchunks, int appended, int vec) {
  using C = Cfg<T, D, CT, NT>;
  constexpr int NQ = C::kNQ, NP = C::kNP, S = C::kStages, U = C::kUnit;
  constexpr int KW = D / 16;  // 4-byte words of a key per thread = k-steps of q.k
  constexpr int VW = D / 32;  // 4-byte words of a value row per thread
  constexpr int MT = D / 16;  // 16-dim tiles of the output
  constexpr int KV = KW >= 4 ? 4 : KW, VV = VW >= 4 ? 4 : VW;  // words of one load
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ uint64_t qbar;
  __shared__ long long plan_s, real0_s, real1_s, per_s, rem_s, scan_s[kWarps];
  __shared__ int plan_i, flag_s, tab0_s, tab_n_s, most_s;
  __shared__ int2 row_s[kRowTab];  // (keys, sequence) of the rows from the run's first on
  __shared__ int4 seg_s[2];        // (row, keys, head chunk, first unit) of this segment and the next
  __shared__ uint32_t valid_s[kWarps][S];  // keys of the units in flight, a bit each
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(sm) + warp * S * C::kStageBytes;
  float2* mls = reinterpret_cast<float2*>(sm + C::kMl);
  float* qscale = reinterpret_cast<float*>(sm + C::kScale);
  float* factor = reinterpret_cast<float*>(sm + C::kMisc);
  int* buffer = reinterpret_cast<int*>(factor + kWarps * C::kHeads);
  const int HC = kp.HK * hchunks;
  if (tid == 0) {
    mbar_init(&qbar, 1);
    fence_mbarrier_init();
  }
  if (appended) pdl_wait();  // the launch before this one wrote rows that are read here

  // positions that a row may have: inside the block table, and inside the cos / sin rows
  if (tid == 0) most_s = (int)min((int64_t)kp.maxb * kp.bs, (int64_t)(kp.rot ? kp.max_seq : 0x7fffffff));
  __syncthreads();
  auto keys_at = [&](int i) { return row_keys(kp.cum, kp.past, kp.ntok, kp.batch, most_s, i); };
  for (int i = tid; i < (C::kQBytes + 4 * C::kHeads) / 4; i += kThreads)  // heads that a group lacks: q = 0
    (i < C::kQBytes / 4 ? reinterpret_cast<uint32_t*>(sm + C::kQ)[i]
                        : reinterpret_cast<uint32_t*>(sm + C::kScale)[i - C::kQBytes / 4]) = 0;

  // ---- this CTA's run of the unit list.  A (row, head chunk) of nu units weighs nu + kOver, the first kOver
  // of which stand for its start; all CTAs get the same weight.  Every CTA adds up all rows, then looks for the
  // two ends of its run.
  constexpr int OV = C::kOver;
  constexpr long long kUnits = (1ll << 40) - 1;  // sums hold units and, above them, rows with keys
  long long W = 0, w0 = 0, w1 = 0, per = 0, rem = 0, pre = 0;
  int ctas = 1, tab_n = 0;
  const int cta = blockIdx.x;
  const bool once = kp.ntok <= kThreads;  // one row per thread: the second pass has all it needs
  int2 r = keys_at(tid);
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    long long base = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < kp.ntok; i0 += kThreads) {
      const int i = i0 + tid;
      if (!once) r = keys_at(i);
      const int nu = (r.x + U - 1) / U;
      if (!(pass && once)) {
        const long long own = nu ? nu + (1ll << 40) : 0;
        long long inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long t = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += t;
        }
        __syncthreads();
        if (lane == 31) scan_s[warp] = inc;
        __syncthreads();
        pre = base + inc - own;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) pre += scan_s[w];
          base += scan_s[w];
        }
      }
      if (!pass) {
        if (i < kp.ntok && r.x == 0 && i % (int)gridDim.x == cta) {  // an invalid row
          pdl_wait();  // an earlier launch may still use `out`
#pragma unroll 1
          for (int e = 0; e < kp.H * D; ++e) static_cast<T*>(kp.out)[(size_t)i * kp.H * D + e] = from_f<T>(0.f);
          report_device_error(kp.err, kErrPagedQ8, i);
        }
        continue;
      }
      if (nu) {
        const long long units = (pre & kUnits) * HC, v = units + (pre >> 40) * OV * HC;  // before this row
        const int nv = nu + OV;
        auto real = [&](long long w) {  // units before weight w of this row
          const int hc = (int)div64(w - v, nv), off = (int)(w - v - (long long)hc * nv);
          return units + (long long)hc * nu + max(0, off - OV);
        };
        const long long end = v + (long long)nv * HC;
        if (v <= w0 && w0 < end) plan_i = i, plan_s = v, real0_s = real(w0);
        if (v < w1 && w1 <= end) real1_s = real(w1);
      }
      __syncthreads();
      const long long done = once ? W : ((base & kUnits) + (base >> 40) * OV) * HC;
      if (done > w0 && !tab_n) {
        const int j = i - plan_i;
        if (j >= 0 && j < kRowTab) row_s[j] = r;
        tab_n = min(kRowTab, i0 + kThreads - plan_i);
      }
      if (done >= w1) break;
    }
    if (!pass) {
      W = ((base & kUnits) + (base >> 40) * OV) * HC;
      // (a run of more than kOver holds at least one unit)
      ctas = (int)max(1ll, min((long long)gridDim.x, div64(W, OV + kWarps)));
      if (W == 0 || cta >= ctas) {
        pdl_wait();
        pdl_trigger();
        return;
      }
      per = div64(W, ctas), rem = W - per * ctas;  // the first rem runs weigh one more
      w0 = cta * per + min((long long)cta, rem);
      w1 = w0 + per + (cta < rem);
    }
  }
  if (tid == 0) per_s = per, rem_s = rem, tab0_s = plan_i, tab_n_s = tab_n;
  __syncthreads();
  const int run = (int)(real1_s - real0_s);
  // a position in the unit list: unit u of head chunk hc of row `row`, which has n keys
  struct Pos {
    int row, seq, n, hc, u;
  };
  auto settle = [&](Pos& p) {  // carries u past the head chunks and rows that it has left
    int nu = (p.n + U - 1) / U;
    while (p.u >= nu) {
      p.u -= nu;
      if (++p.hc == HC) {
        p.hc = 0;
        int2 r;
        do {
          ++p.row;
          r = p.row - tab0_s < tab_n_s ? row_s[p.row - tab0_s] : keys_at(p.row);
        } while (r.x == 0 && p.row < kp.ntok);
        p.n = r.x, p.seq = r.y;
        nu = p.row < kp.ntok ? (p.n + U - 1) / U : 0x7fffffff;  // (past the last row: nothing is issued)
      }
    }
  };
  Pos is;  // of the warp's next unit to issue; first the run's first unit
  is.row = tab0_s;
  is.n = row_s[0].x, is.seq = row_s[0].y;
  {
    const int nv = (is.n + U - 1) / U + OV;
    const long long off = w0 - plan_s;  // < nv HC
    is.hc = (int)div64(off, nv);
    is.u = max(0, (int)(off - (long long)is.hc * nv) - OV);
    __syncthreads();
    if (tid == 0) {
      seg_s[0] = make_int4(is.row, is.n, is.hc, is.u);
      plan_s += (long long)is.hc * nv;  // from here: the weight before the segment's (row, head chunk)
    }
  }

  // ---- q rows of a segment, and the cos / sin row of its position, on their way to shared memory (one
  // thread; aligned rows only)
  T* raw = reinterpret_cast<T*>(sm + C::kRaw);
  auto fetch_q = [&](const Pos& p) {
    const int ck = hchunks == 1 ? 0 : p.hc % hchunks, nh = min(C::kHeads, kp.G - ck * C::kHeads);
    const int first = (hchunks == 1 ? p.hc : p.hc / hchunks) * kp.G + ck * C::kHeads;
    const uint32_t qb = nh * D * sizeof(T), cb = kp.rot ? kp.half * sizeof(T) : 0;
    mbar_arrive_expect_tx(&qbar, qb + 2 * cb);
    bulk_g2s(raw, static_cast<const T*>(kp.q) + (size_t)p.row * kp.qs + (size_t)first * D, qb, &qbar);
    if (cb) {
      T* cs = raw + min(C::kHeads, kp.G) * D;
      bulk_g2s(cs, static_cast<const T*>(kp.cos_c) + (size_t)(p.n - 1) * kp.half, cb, &qbar);
      bulk_g2s(cs + kp.half, static_cast<const T*>(kp.sin_c) + (size_t)(p.n - 1) * kp.half, cb, &qbar);
    }
  };
  if ((vec & 1) && tid == 0) fetch_q(is);
  uint32_t qphase = 0;

  // ---- the warp's stream: units warp, warp + 4, ... of the run, S - 1 ahead of their use
  is.u += warp;
  settle(is);
  // whole units lie in one page (16-row aligned): one lookup a unit, else one a key
  const bool paged = kp.bs % U == 0 && (vec & 2);
  auto lookup = [&](int ix) -> int {
    if (ix >= run) return -1;
    const int key = is.u * U + (paged ? 0 : lane);
    return key < is.n && (paged || lane < U)
               ? q8_row(kp.bt, kp.maxb, kp.nblocks, kp.bs, kp.HK, is.seq, hchunks == 1 ? is.hc : is.hc / hchunks, key,
                        kp.bs_shift)
               : -1;
  };
  int next_row = lookup(warp);
  constexpr int CH = D / 16, PER = U * CH / 32;  // 16-byte chunks of a row; of a unit's K per lane
  auto issue = [&](int stage, int ix) {  // unit ix of the run into buffer `stage`
    uint32_t valid = 0;
    if (ix < run) {
      const int row = next_row, left = is.n - is.u * U;  // keys from this unit's first on
      const uint32_t dst = ring + stage * C::kStageBytes;
      const uint32_t inside = left >= U ? (U == 32 ? 0xffffffffu : 0xffffu) : (1u << left) - 1u;
      if (paged) {
        if (row < 0 && lane == 0) report_device_error(kp.err, kErrPagedQ8, is.row);
        if (row >= 0) {
          valid = inside;
          const size_t o = (size_t)row * D + lane * 16;
          const uint8_t *ks = kp.kc + o, *vs = kp.vc + o;
#pragma unroll
          for (int t = 0; t < PER; ++t) {
            const uint32_t d = dst + swz<D>((t * 32 + lane) / CH, (t * 32 + lane) % CH);
            cp16(d, ks + t * 512);
            cp16(d + C::kData, vs + t * 512);
          }
          if (lane < U / 4) cp16(dst + 2 * C::kData + lane * 16, kp.kscale + row + lane * 4);
          else if (lane < U / 2) cp16(dst + 2 * C::kData + lane * 16, kp.vscale + row + (lane - U / 4) * 4);
        }
      } else {
        if (row < 0 && lane < U && lane < left) report_device_error(kp.err, kErrPagedQ8, is.row);
        valid = __ballot_sync(0xffffffffu, row >= 0);
#pragma unroll 1
        for (int t = 0; t < PER; ++t) {
          const int r = (t * 32 + lane) / CH, ch = (t * 32 + lane) % CH;
          const int src = __shfl_sync(0xffffffffu, row, r);
          if (src >= 0) {
            const size_t o = (size_t)src * D + ch * 16;
            const uint32_t d = dst + swz<D>(r, ch);
            cp16(d, kp.kc + o);
            cp16(d + C::kData, kp.vc + o);
          }
        }
        if (row >= 0) {
          cp4(dst + 2 * C::kData + lane * 4, kp.kscale + row);
          cp4(dst + 2 * C::kData + U * 4 + lane * 4, kp.vscale + row);
        }
      }
      is.u += kWarps;
      if (ix + kWarps < run) settle(is);
      next_row = lookup(ix + kWarps);
    }
    cp_commit();
    if (lane == 0) valid_s[warp][stage] = valid;
  };
#pragma unroll 1
  for (int i = 0; i < S - 1; ++i) issue(i, warp + i * kWarps);

  int stage = 0;
  int x = 0;        // first unit of the segment, within the run
  int mine = warp;  // the warp's next unit
  int par = 0;  // which of seg_s
  while (x < run) {
    const int4 sg = seg_s[par];  // row, keys, head chunk, first unit
    const int nseg = min((sg.y + U - 1) / U - sg.w, run - x);  // units of this segment
    const int chunk = hchunks == 1 ? 0 : sg.z % hchunks;
    const int h0 = (hchunks == 1 ? sg.z : sg.z / hchunks) * kp.G + chunk * C::kHeads;  // first query head
    const int heads = min(C::kHeads, kp.G - chunk * C::kHeads);
    if (vec & 1) {
      if (!mbar_wait(&qbar, qphase) && tid == 0) report_device_error(kp.err, kErrPagedQ8Timeout, sg.x);
      qphase ^= 1;
    }
    else {
      const T* src = static_cast<const T*>(kp.q) + (size_t)sg.x * kp.qs + (size_t)h0 * D;
#pragma unroll 1
      for (int e = tid; e < heads * D; e += kThreads) raw[e] = src[e];
      if (kp.rot)
#pragma unroll 1
        for (int e = tid; e < 2 * kp.half; e += kThreads)
          raw[min(C::kHeads, kp.G) * D + e] =
              (e < kp.half ? static_cast<const T*>(kp.cos_c) + e : static_cast<const T*>(kp.sin_c) + e - kp.half)
                  [(size_t)(sg.y - 1) * kp.half];
      __syncthreads();
    }
    // ---- q as the second operand, in shared memory: a head per LPH lanes
    constexpr int LPH = D / 4 < 32 ? D / 4 : 32, EPL = D / LPH, HPW = 32 / LPH;
#pragma unroll 1
    for (int hb = warp * HPW; hb < heads; hb += kWarps * HPW) {
      const int h = hb + lane / LPH, d0 = (lane % LPH) * EPL;
      const bool on = h < heads;
      const T* cs = raw + min(C::kHeads, kp.G) * D;
      float q[EPL];
      uint32_t amax = 0;
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        q[e] = on ? q_at<T>(raw + h * D, d0 + e, kp, cs, cs + kp.half) : 0.f;
        amax = max(amax, __float_as_uint(q[e]) & 0x7fffffffu);
      }
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (!on) continue;
      const float base = kp.scale * 1.4426950408889634f;
      uint32_t* dst = reinterpret_cast<uint32_t*>(sm + C::kQ);
      const bool finite = amax < 0x7f800000u;
      float mul;  // what q is multiplied by
      if constexpr (C::kInt) {
        // q / amax as an integer of kNQ bytes, each in [-128, 127]
        constexpr float M = 127.f * 65536.f;
        const float top = fmaxf(__uint_as_float(amax), 1e-30f);  // (all below: q rounds to 0, as its scores would)
        mul = __fdiv_rn(M, top);
        if (lane % LPH == 0)  // what the sum, in units of the upper two bytes' last place, stands for
          qscale[h] = finite ? top * base * (256.f / M) : __uint_as_float(0x7fc00000u);
      } else {
        const int ex = min(max((int)(amax >> 23), 1), 253);  // biased exponent
        mul = __uint_as_float((uint32_t)(254 - ex) << 23);
        if (lane % LPH == 0) qscale[h] = __uint_as_float((uint32_t)ex << 23) * base;
      }
#pragma unroll
      for (int j = 0; j < EPL / 4; ++j) {  // 4 dims: word w of thread (h % 8, qc)
        const int ch = (d0 + 4 * j) >> 4, w4 = ((d0 + 4 * j) >> 2) & 3;
        const int qc = D >= 128 ? (ch & 7) >> 1 : D == 64 ? ch : 2 * ch + (w4 >> 1);
        const int w = D >= 128 ? (ch >> 3) * 8 + (ch & 1) * 4 + w4 : D == 64 ? w4 : w4 & 1;
        const int to = (h & 7) * 4 + qc;
        if constexpr (C::kInt) {
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)  // every byte lifted by 128: no carries between them
            u[e] = (uint32_t)__float2int_rn(finite ? q[4 * j + e] * mul : 0.f) + 0x808080u;
#pragma unroll
          for (int t = 0; t < NQ; ++t) {
            const int bi = NQ - 1 - t;  // the most significant byte first
            const uint32_t a = prmt(u[0], u[1], (4 + bi) << 4 | bi), b = prmt(u[2], u[3], (4 + bi) << 4 | bi);
            dst[((((h >> 3) * (KW / 2) + (w >> 1)) * NQ + t) * 32 + to) * 2 + (w & 1)] = prmt(a, b, 0x5410) ^ 0x80808080u;
          }
        } else {
          const float a0 = q[4 * j] * mul, a1 = q[4 * j + 1] * mul, a2 = q[4 * j + 2] * mul, a3 = q[4 * j + 3] * mul;
          const __half2 p0 = __floats2half2_rn(a0, a1), p1 = __floats2half2_rn(a2, a3);
          uint32_t* o = dst + (((h >> 3) * KW + w) * 32 + to) * (2 * NQ);
          o[0] = word_of(p0), o[1] = word_of(p1);
          o[2] = half2_bits(a0 - __low2float(p0), a1 - __high2float(p0));
          o[3] = half2_bits(a2 - __low2float(p1), a3 - __high2float(p1));
        }
      }
    }
    __syncthreads();  // q is there; the merge buffers of the segment before, and the raw rows, are free
    if (tid == 0 && x + nseg < run) {
      Pos nx{sg.x, 0, sg.y, sg.z, sg.w + nseg};
      settle(nx);
      seg_s[par ^ 1] = make_int4(nx.row, nx.n, nx.hc, nx.u);
      if (vec & 1) fetch_q(nx);
    }

    float qs[NT][2];  // what turns a score's sum into base-2 logits, but for the key's scale
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) qs[nt][0] = qscale[nt * 8 + 2 * c], qs[nt][1] = qscale[nt * 8 + 2 * c + 1];
    float o[MT][NT][4], m[NT][2], l[NT][2];
    float dn[NT][2];  // the power of two that a head's P vs is multiplied by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = kLow, l[nt][0] = l[nt][1] = 0.f, dn[nt][0] = dn[nt][1] = 0x1p126f;
#pragma unroll
      for (int t = 0; t < MT; ++t) o[t][nt][0] = o[t][nt][1] = o[t][nt][2] = o[t][nt][3] = 0.f;
    }

#pragma unroll 1
    for (; mine < x + nseg; mine += kWarps) {
      cp_wait<S - 2>();
      __syncwarp();
      const uint32_t valid_u = valid_s[warp][stage];
      issue(stage == 0 ? S - 1 : stage - 1, mine + (S - 1) * kWarps);  // into the buffer that was consumed last
      const uint32_t buf = ring + stage * C::kStageBytes;
      if constexpr (CT == kE4M3)
        if (valid_u != (U == 32 ? 0xffffffffu : 0xffffu)) {  // what lies in rows without a key may be NaN codes: P = 0 times 0
#pragma unroll
          for (int t = 0; t < PER; ++t) {
            const int r = (t * 32 + lane) / CH, ch = (t * 32 + lane) % CH;
            if (!((valid_u >> r) & 1u))
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(buf + C::kData + swz<D>(r, ch)), "r"(0) : "memory");
          }
          __syncwarp();
        }
#pragma unroll 1
      for (int kt = 0; kt < NT; ++kt) {  // 16 keys
        const uint32_t valid = valid_u >> (kt * 16);
        const uint32_t sks = buf + 2 * C::kData + kt * 64, svs = sks + U * 4;
        float s[NT][4];
        if constexpr (C::kInt) {
          int si[NT][NQ][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int t = 0; t < NQ; ++t) si[nt][t][0] = si[nt][t][1] = si[nt][t][2] = si[nt][t][3] = 0;
#pragma unroll
          for (int wb = 0; wb < KW; wb += KV) {
            uint32_t ka[KV], kb[KV];
            const int r0 = kt * 16 + g, byte = kbyte<D>(c, wb);
            lds<KV * 4>(buf + swz<D>(r0, byte >> 4) + (byte & 15), ka);
            lds<KV * 4>(buf + swz<D>(r0 + 8, byte >> 4) + (byte & 15), kb);
#pragma unroll
            for (int w = 0; w < KV; w += 2)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < NQ; ++t) {
                  uint32_t b[2];
                  lds<8>(smem_u32(sm) + C::kQ + (((nt * (KW / 2) + (wb + w) / 2) * NQ + t) * 32 + lane) * 8, b);
                  mma_s8(si[nt][t], ka[w], kb[w], ka[w + 1], kb[w + 1], b[0], b[1]);
                }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // |sums| <= D 127 128: 2^22 at D = 256, 2^30 after the shift
              const int v = si[nt][0][e] * 256 + si[nt][1][e] + ((si[nt][2][e] + 128) >> 8);
              s[nt][e] = (float)v;
            }
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
          for (int wb = 0; wb < KW; wb += KV) {
            uint32_t ka[KV], kb[KV];
            const int r0 = kt * 16 + g, byte = kbyte<D>(c, wb);
            lds<KV * 4>(buf + swz<D>(r0, byte >> 4) + (byte & 15), ka);
            lds<KV * 4>(buf + swz<D>(r0 + 8, byte >> 4) + (byte & 15), kb);
#pragma unroll
            for (int w = 0; w < KV; ++w) {
              uint32_t a[4];
              widen<CT>(ka[w], a[0], a[2]);
              widen<CT>(kb[w], a[1], a[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                uint32_t b[2 * NQ];
                lds<8 * NQ>(smem_u32(sm) + C::kQ + ((nt * KW + wb + w) * 32 + lane) * (8 * NQ), b);
#pragma unroll
                for (int t = 0; t < NQ; ++t) mma(s[nt], a, b[2 * t], b[2 * t + 1]);
              }
            }
          }
        }
        // scores in base 2, key g (r = 0) and g + 8 (r = 1), heads 2c and 2c + 1
        float vs[2], p[NT][4], pv[NT][4], ln[NT][2];
        bool move = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const bool on = (valid >> (g + r * 8)) & 1u;
          const float ks = lds_f(sks + (g + r * 8) * 4);
          vs[r] = on ? lds_f(svs + (g + r * 8) * 4) : 0.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int e = r * 2 + h;
              s[nt][e] = on ? s[nt][e] * (ks * qs[nt][h]) : -INFINITY;
              p[nt][e] = ex2(s[nt][e] - m[nt][h]);
              pv[nt][e] = p[nt][e] * (vs[r] * dn[nt][h]);
              move |= !(pv[nt][e] < kFull);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ln[nt][h] = l[nt][h] + p[nt][h] + p[nt][2 + h];
            move |= !(ln[nt][h] <= kSlack);
          }
        if (__any_sync(0xffffffffu, move)) {  // a larger score, or a larger product: rescale what there is
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float mx = fmaxf(m[nt][h], fmaxf(s[nt][h], s[nt][2 + h]));
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
              const float a = ex2(m[nt][h] - mx);
              m[nt][h] = mx;
              // the head's largest product, those of the keys before at their present weight (a NaN is passed over)
              float most = a * __uint_as_float(((uint32_t)(254 + kLift) << 23) - __float_as_uint(dn[nt][h]));
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                p[nt][r * 2 + h] = ex2(s[nt][r * 2 + h] - mx);
                most = fmaxf(most, p[nt][r * 2 + h] * vs[r]);
              }
              ln[nt][h] = l[nt][h] * a + p[nt][h] + p[nt][2 + h];
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
              const int ex = min(max((int)(__float_as_uint(most) >> 23), kLift + 1), 253);
              const float to = __uint_as_float((uint32_t)(254 + kLift - ex) << 23);  // brings it into [1, 2) 2^kLift
              // to / dn (where a is not 0, `to` is 2^127 dn at most)
              const int by = (int)(__float_as_uint(to) - __float_as_uint(dn[nt][h])) + (127 << 23);
              const float back = a == 0.f ? 0.f : a * __int_as_float(max(by, 0));
              dn[nt][h] = to;
#pragma unroll
              for (int t = 0; t < MT; ++t) o[t][nt][h] *= back, o[t][nt][2 + h] *= back;
#pragma unroll
              for (int r = 0; r < 2; ++r) pv[nt][r * 2 + h] = p[nt][r * 2 + h] * vs[r] * to;
            }
        }
        // P^T as the second operand
        uint32_t pf[NP][NT][2];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float* x = pv[nt] + r * 2;
            l[nt][r] = ln[nt][r];  // (r: a head, here)
            const __half2 hi = __floats2half2_rn(x[0], x[1]);
            pf[0][nt][r] = transpose8x8(word_of(hi));
            pf[1][nt][r] = transpose8x8(half2_bits(x[0] - __low2float(hi), x[1] - __high2float(hi)));
          }
        // O^T += V^T P^T
#pragma unroll
        for (int wb = 0; wb < VW; wb += VV) {
          uint32_t v[4][VV];  // value rows 2c, 2c + 1, 2c + 8, 2c + 9
          const int byte = vbyte<D>(g, wb);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = kt * 16 + 2 * c + (r & 1) + (r >> 1) * 8;
            lds<VV * 4>(buf + C::kData + swz<D>(key, byte >> 4) + (byte & 15), v[r]);
          }
#pragma unroll
          for (int w = 0; w < VV; ++w) {
            uint32_t d[2][4];  // two keys side by side, dim by dim
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              widen<CT>(prmt(v[2 * r][w], v[2 * r + 1][w], 0x5140), d[r][0], d[r][1]);
              widen<CT>(prmt(v[2 * r][w], v[2 * r + 1][w], 0x7362), d[r][2], d[r][3]);
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t a[4] = {d[0][2 * t], d[0][2 * t + 1], d[1][2 * t], d[1][2 * t + 1]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < NP; ++u) mma(o[(wb + w) * 2 + t][nt], a, pf[u][nt][0], pf[u][nt][1]);
            }
          }
        }
      }
      __syncwarp();
      stage = stage + 1 == S ? 0 : stage + 1;
    }

    // ---- the segment's end: each warp leaves (m, l, o) in its one buffer that no copy is in flight to
    const int freeb = stage == 0 ? S - 1 : stage - 1;
    {
      float2* mg = reinterpret_cast<float2*>(sm + (warp * S + freeb) * C::kStageBytes);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], d);
          const int hd = nt * 8 + 2 * c + h;
          if (g == 0) {
            mls[warp * C::kHeads + hd] = make_float2(m[nt][h], l[nt][h]);
            factor[warp * C::kHeads + hd] = __uint_as_float((254u << 23) - __float_as_uint(dn[nt][h]));  // 1 / dn
          }
          if (hd < heads)
#pragma unroll
            for (int t = 0; t < MT; ++t)
              mg[merge_at<D>(hd, (vbyte<D>(g, t >> 1) >> 1) + (t & 1))] = make_float2(o[t][nt][h], o[t][nt][2 + h]);
        }
      if (lane == 0) buffer[warp] = freeb;
    }
    __syncthreads();
    pdl_wait();  // before anything is written
    const int4 sw = seg_s[par];
    const int nu = (sw.y + U - 1) / U;
    const bool whole = nseg == nu;
    T* out = static_cast<T*>(kp.out) + (size_t)sw.x * kp.H * D + (size_t)h0 * D;
    const int slot = 2 * cta + (sw.w > 0 ? 0 : 1);
    float* part = kp.part + (size_t)slot * C::kHeads * (D + 2);
#pragma unroll 1
    for (int e = tid; e < heads * (D / 4); e += kThreads) {  // 4 dims of a head
      const int hd = e / (D / 4), d = (e % (D / 4)) * 4;
      float mm = -INFINITY, ll = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, mls[w * C::kHeads + hd].x);
      const int at2 = merge_at<D>(hd, d / 2), at3 = merge_at<D>(hd, d / 2 + 1);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = mls[w * C::kHeads + hd];
        const float f = ml.y == 0.f ? 0.f : ex2(ml.x - mm);  // 0: the warp saw no key of this segment (a NaN is not 0)
        const float2* mg = reinterpret_cast<const float2*>(sm + (w * S + buffer[w]) * C::kStageBytes);
        ll += ml.y * f;
        if (f != 0.f) {  // (else the buffer holds something else)
          const float2 a = mg[at2], b = mg[at3];
          const float ff = f * factor[w * C::kHeads + hd];
          acc.x += a.x * ff, acc.y += a.y * ff, acc.z += b.x * ff, acc.w += b.y * ff;
        }
      }
      if (whole) {
        store4<T>(out + hd * D + d, acc, ll);
      } else {
        *reinterpret_cast<float4*>(part + hd * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(part + C::kHeads * D + hd * 2) = make_float2(mm, ll);
      }
    }
    if (!whole) {
      // the runs that hold units of this (row, head chunk); in the first of them it is the last segment
      auto run_of = [&](long long w) {
        const long long n = per_s, m = rem_s, big = m * (n + 1);
        return (int)(w < big ? div64(w, n + 1) : m + div64(w - big, n));
      };
      __syncthreads();
      if (tid == 0) {
        const long long a = plan_s + OV;  // weight before the first unit
        const int kf = run_of(a), parts = run_of(a + nu - 1) - kf + 1;
        __threadfence();  // (orders what the whole CTA wrote before the barrier)
        flag_s = atomicAdd(kp.counters + kf, 1) == parts - 1 ? parts : 0;
        __threadfence();
        plan_i = kf;
      }
      __syncthreads();
      const int parts = flag_s, kf = plan_i;
      if (parts) {  // the last to arrive joins the parts, in the order of the keys
        constexpr int step = 2 * C::kHeads * (D + 2);  // from one run's first part to the next one's
        const float* first = kp.part + kf * step;
        auto part_at = [&](int k) { return first + (k ? k * step : step / 2); };
        constexpr int KC = D / 2;  // parts at a time: their (m, l) fit a merge buffer
        float2* mlb = reinterpret_cast<float2*>(sm + buffer[0] * C::kStageBytes);
#pragma unroll 1
        for (int e0 = 0; e0 < heads * (D / 4); e0 += kThreads) {
          const int e = e0 + tid;
          const bool on = e < heads * (D / 4);
          const int hd = on ? e / (D / 4) : 0, d = (e % (D / 4)) * 4;
          float mm = -INFINITY, ll = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
          for (int k0 = 0; k0 < parts; k0 += KC) {
            const int nk = min(KC, parts - k0);
            __syncthreads();
#pragma unroll 1
            for (int i = tid; i < nk * C::kHeads; i += kThreads)
              if (i % C::kHeads < heads)
                mlb[i] = __ldcg(reinterpret_cast<const float2*>(part_at(k0 + i / C::kHeads) + C::kHeads * D) + i % C::kHeads);
            __syncthreads();
            float mn = mm;
#pragma unroll 4
            for (int k = 0; k < nk; ++k) mn = fmaxf(mn, mlb[k * C::kHeads + hd].x);
            const float a0 = ll == 0.f ? 0.f : ex2(mm - mn);
            mm = mn, ll *= a0;
            acc.x *= a0, acc.y *= a0, acc.z *= a0, acc.w *= a0;
            auto take = [&](const float4& v, int k) {
              const float2 ml = mlb[k * C::kHeads + hd];
              const float f = ml.y == 0.f ? 0.f : ex2(ml.x - mn);
              ll += ml.y * f;
              acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
            };
            int k = 0;
            if (k0 == 0) take(__ldcg(reinterpret_cast<const float4*>(part_at(0) + hd * D + d)), k++);
            const float* pk = first + (k0 + k) * step + hd * D + d;
            if (x + nseg >= run) {
              // the run's last segment: the buffers of warps 1 to 3 are free and take many parts at once (74 parts
              // of one long sequence: 13 us by registers alone)
              constexpr int room = (kWarps - 1) * S * C::kStageBytes / (kThreads * 16), NB = room < 32 ? room : 32;
              const uint32_t slot_ = smem_u32(sm) + S * C::kStageBytes + tid * 16;
#pragma unroll 1
              for (; k < nk; k += NB, pk += NB * step) {
                const int n = min(NB, nk - k);
#pragma unroll 4
                for (int j = 0; j < n; ++j) cp16(slot_ + j * (kThreads * 16), pk + j * step);
                cp_commit();
                cp_wait<0>();
#pragma unroll 4
                for (int j = 0; j < n; ++j) {
                  uint32_t u[4];
                  lds<16>(slot_ + j * (kThreads * 16), u);
                  take(make_float4(__uint_as_float(u[0]), __uint_as_float(u[1]), __uint_as_float(u[2]),
                                   __uint_as_float(u[3])), k + j);
                }
              }
            }
            constexpr int MLP = 6;  // else by registers: parts on their way at once
#pragma unroll 1
            for (; k < nk; k += MLP, pk += MLP * step) {
              float4 v[MLP];
#pragma unroll
              for (int j = 0; j < MLP; ++j)
                if (k + j < nk) v[j] = __ldcg(reinterpret_cast<const float4*>(pk + j * step));
#pragma unroll
              for (int j = 0; j < MLP; ++j)
                if (k + j < nk) take(v[j], k + j);
            }
          }
          if (on) store4<T>(out + hd * D + d, acc, ll);
        }
      }
    }
    if (tid == 0 && sw.w + nseg == nu) plan_s += nu + OV;
    x += nseg;
    par ^= 1;
  }
  cp_wait<0>();
  pdl_trigger();
}

template <typename T, int D, int CT, int NT>
cudaError_t launch_t(const PagedQ8& a, bool appended, cudaStream_t st) {
  using C = Cfg<T, D, CT, NT>;
  auto kern = paged_q8_attn_kernel<T, D, CT, NT>;
  const int smem = C::kRaw + (std::min(a.G, C::kHeads) * D + (a.rot ? 2 * a.half : 0)) * (int)sizeof(T);
  static std::atomic<bool> allowed[kMaxSmemDevices];
  const int most = C::kRaw + (C::kHeads * D + D) * (int)sizeof(T);
  if (cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), allowed, most)) return e;
  // one wave: the CTAs that the SM's 228 KB hold (1 KB of each is the system's)
  const int per_sm = std::min<int>(C::kCtasPerSm, 228 * 1024 / (smem + C::kStatic + 1024));
  const int grid = std::min(a.ctas, num_sms() * per_sm);
  if (!appended)
    if (cudaError_t e = launch_k(paged_q8_reset_kernel, dim3(1), dim3(256), 0, st, a.counters, grid)) return e;
  const int hchunks = (a.G + C::kHeads - 1) / C::kHeads;
  auto al = [](const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && bytes % 16 == 0; };
  const int es = (int)sizeof(T);
  int vec = al(a.q, a.qs * es) &&
            (!a.rot || (al(a.cos_c, (int64_t)a.half * es) && al(a.sin_c, 0)));
  if (al(a.kscale, 0) && al(a.vscale, 0)) vec |= 2;
  return launch_k(kern, dim3((unsigned)grid), dim3(kThreads), smem, st, a, hchunks, appended ? 1 : 0, vec);
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

int paged_q8_max_ctas() { return 4 * num_sms(); }
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
