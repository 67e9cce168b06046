// kv4_attention.cu — attention of one query row per sequence over the 4-bit KV cache
// (rrr_attention_kv4): the decode step's `attention` dispatch (src/model/phi4.rs:1680-1688)
// for a batch of sequences of different lengths on pages.
//
// Mathematics. A key is k = d_j code + m_j in groups j of 32 values, so q . k = sum_j d_j (q_j .
// code_j) + m_j (sum q_j). The products with the codes run on mma.m16n8k16
// (f16 in, f32 accumulate): 16 rows of codes are the A operand, and the B operand's eight columns
// are four query heads as (hi, lo) pairs: the f16 part of the (power-of-two scaled) query and
// the remainder (q - hi) * 2^11, so a score carries 22 bits of the query. A code shifted into the
// top of an f16's mantissa is 1 + code / 16 (a shift and an AND-OR for two operands); sum q_j is
// taken off the products (as the accumulators' start it cost two moves per subtraction), the power
// of two leaves with the scales and d_j multiplies them in f32. One more product takes the m_j.
// (The code in the low bits would be the subnormal code * 2^-24 for fewer instructions, but the
// tensor core aligns a subnormal's products as if they were normal: they lost 6 bits, an error of
// 1e-6 in the scores.) The second product is alike: A holds V's codes, B the weights p_i d_ij of
// group j as (hi, lo), and the sums of p_i (m_ij + 8 d_ij) run beside it in f32. V's codes are
// centred, code - 8: over a long context the weighted values nearly cancel, and sums of the codes
// themselves would be hundreds of times the result (measured: an error of 1.2e-3 at 131,000 rows).
// (8 rather than 7.5 because both nibbles of a byte can then be centred where they stand.) A weight
// is 2^(s - ref) with ref below the running maximum by as much as brings the largest weight times the
// largest step so far to 2^-1 (for larger steps ref is the maximum): a p d keeps 22 bits down to 2^-13
// of that, and 2^-35 of it below, where f16 has no normal numbers. (Relative to the maximum, values of
// 1e-4 behind a first row that draws the weight, as texts have, came out with 8 bits.) The
// tensor core truncates its sums, so they are moved to shared memory, rounded, every kFlush pages.
// The softmax runs online in base 2, with 32-bit maxima and sums: a slice of rows without a new
// maximum, as most of a long run are, skips the exchange of maxima and the rescaling. Scores,
// weights and sums keep f32 accuracy throughout.
//
// Bound by instructions and their latency: about 500 per warp for 16 rows of 4 heads x 128, where
// the issue slots are 60 % taken by 12 warps (131,000 rows of 8 heads: 59 us, 2.8 TB/s of codes; 64
// sequences, 261,424 rows: 110 us, 3.0 TB/s; the memory alone would take 26 and 51 us). A fourth CTA
// per SM leaves 96 registers, some of which spilt: 8 % slower.
//
// Work. A unit is one page (64 rows) of one (sequence, KV head), and each of those has kStart units
// more in front, which is what beginning and ending one costs. The CTAs share all U units of the
// batch evenly, in order, whatever the lengths are (read on the device): CTA c of G takes the
// pages in [c U / G, (c+1) U / G). (Without the units in front, the CTA with the most short
// sequences took 137 us of the batch of 64, the middle one 103; with them all took 118.) One
// producer warp streams the pages' blocks, each one contiguous, with bulk copies into a ring of
// stages, the segment's query row with its first page; four consumer warps take 16 rows of a page
// each and keep their own softmax state. At the end of a (sequence, head) segment the warps' states
// are joined in order; a segment that other CTAs share goes to the workspace, and a second small
// kernel joins the parts in order. (The CTA that finishes last did that first, found by a counter:
// 6 of 14 us at one short sequence, most of it instructions that no SM had executed before, by one
// CTA per head.)
#include <math.h>

#include "kv4.cuh"

namespace rrr {
namespace {

constexpr int kConsumers = 4;  // warps
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kMaxStages = 16;
constexpr int kMaxHpk = 8;
constexpr float kLo = 1.f / 2048.f;
constexpr float kNone = -3e38f;  // the maximum of no rows: finite, so that it may be subtracted from -inf
constexpr int kStart = 2;   // units in front of a (sequence, head)'s pages
constexpr int kFlush = 16;  // pages whose products one set of accumulators takes
constexpr int kWeightBits = -1;  // weights times V's steps stay below 2^kWeightBits, if the steps do

struct Kv4Params {
  const uint8_t* pages;
  int64_t n_pages, table_stride;
  const int* table;
  int n_seqs, max_pages;
  int nkv, hpk;   // heads that CTAs take apart, and query heads of each: KV heads, or `split` parts of them
  int split;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  const int* lens;
  float scale;  // with log2(e)
  int2* runs;    // [seq][head]: first CTA and CTAs of its pages
  float* parts;  // [CTA][2][hpk * (HD + 2)]: sums, references, weights' sums
  int stages, stage_bytes;
  int ctas;      // of the first kernel
  int* err;
};

struct Segment {  // beside each stage: this CTA's run of pages of one (sequence, head)
  long long base;  // unit of the (sequence, head)'s first page
  int seq, head, pages;
  int more;        // whether another run follows
  int valid;       // rows of this page that count
  int first_page;  // of the run
  int first, left; // whether this page is the run's first; its pages from this one on
};

// CTAs of an SM by what its registers hold: HD/4 accumulators and HD/8 of the query per column tile
// (NT = 1: up to four query heads per KV head, 2: up to eight).
template <int HD, int NT>
constexpr int ctas_per_sm() { return HD * NT >= 512 ? 1 : HD * NT >= 256 ? 2 : 3; }

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t* a, uint32_t b0, uint32_t b1,
                                        const float (&c)[4]) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a, b as f16 pairs hi and lo = (x - hi) * 2^11
__device__ __forceinline__ float from_half(__half h, float x) {  // h - x
  float r;
  asm("sub.rn.f32.f16 %0, %1, %2;" : "=f"(r) : "h"(__half_as_ushort(h)), "f"(x));
  return r;
}
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 rest = __fmul2_rn(make_float2(from_half(__low2half(h), a), from_half(__high2half(h), b)),
                                 make_float2(-2048.f, -2048.f));
  const __half2 l = __floats2half2_rn(rest.x, rest.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ float half_of(uint32_t w, int i) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return i ? __high2float(h) : __low2float(h);
}

// (w & mask) | bits in one instruction: `bits` comes in a register, an instruction has room for
// one constant (with both as constants each pair of operands cost two)
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t x;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w), "r"(mask), "r"(bits));
  return x;
}
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
  asm volatile("" : "+r"(v));
  return v;
}
// 1 + code / 16 of the four bits at 6..9 of both halves of w (one: 0x3C003C00)
__device__ __forceinline__ uint32_t from_one(uint32_t w, uint32_t one) { return and_or(w, 0x03C003C0u, one); }
// 16 (code - 8) of the four bits at 4..7 and at 0..3 of both halves of w, exact: 1024 + 16 code
// - 1152, and 16 (1024 + code) - 16512 (big: 0x64006400)
__device__ __forceinline__ uint32_t centred(uint32_t w, uint32_t big) {
  const uint32_t x = and_or(w, 0x00F000F0u, big);
  const __half2 y = __hadd2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0xe480)));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t centred_low(uint32_t w, uint32_t big) {
  const uint32_t x = and_or(w, 0x000F000Fu, big);
  const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x4c00)),
                            __half2half2(__ushort_as_half(0xf408)));
  return *reinterpret_cast<const uint32_t*>(&y);
}
// N words at p (N a power of two; p aligned to min(16, 4 N))
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
      w[i + 2] = v.z;
      w[i + 3] = v.w;
    }
  }
}

// The consumer warps' barrier, bounded.
struct ConsumerSync {
  uint64_t* bar;
  uint32_t phase;
  int* err;
  __device__ __forceinline__ bool operator()() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
    const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase, err, kDevErrFullTimeout));
    phase ^= 1;
    return ok;
  }
};

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<HD, NT>())
    kv4_attention_kernel(const __grid_constant__ Kv4Params p) {
  using B = Kv4Block<HD>;
  constexpr int G = B::kGroups, J = B::kJ;
  constexpr int PITCH = HD + 8;  // floats between the heads of a warp's sums
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], cons_bar;
  __shared__ Segment seg[kMaxStages];
  __shared__ float wm[kConsumers][kMaxHpk], wl[kConsumers][kMaxHpk];
  __shared__ long long warp_units[kConsumers + 1];
  __shared__ long long first_base;  // unit of the first sequence's first page
  __shared__ int first_seq;
  float* wo = reinterpret_cast<float*>(smem + (size_t)p.stages * p.stage_bytes);  // [warp][hpk][PITCH]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kConsumers);
    }
    mbar_init(&cons_bar, kConsumers);
    fence_mbarrier_init();
  }
  pdl_launch_dependents();
  pdl_wait();

  // pages of sequence s; one unit (without rows) for a sequence without any
  auto seq_len = [&](int s) {
    const int n = p.lens[s];
    if (n < 0 || n > (int64_t)p.max_pages * kPageRows) {
      flag_position(p.err);
      return 0;
    }
    return n;
  };
  auto pages_of = [](int len) { return len > 0 ? (len + kPageRows - 1) / kPageRows : 1; };
  const int per = (p.n_seqs + kThreads - 1) / kThreads;
  const int my0 = min(p.n_seqs, (int)threadIdx.x * per), my1 = min(p.n_seqs, my0 + per);
  long long mine = 0;
  for (int s = my0; s < my1; ++s) mine += (long long)(pages_of(seq_len(s)) + kStart) * p.nkv;
  long long upto = mine;  // units of this warp's threads up to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_units[warp] = upto;
  __syncthreads();
  long long before = upto - mine, U = 0;
#pragma unroll
  for (int w = 0; w <= kConsumers; ++w) {
    if (w < warp) before += warp_units[w];
    U += warp_units[w];
  }
  const long long grid = U < (long long)gridDim.x ? U : (long long)gridDim.x;  // CTAs with units
  if ((long long)blockIdx.x >= grid) return;
  const long long u0 = blockIdx.x * U / grid, u1 = (blockIdx.x + 1) * U / grid;
  if (u0 >= before && u0 < before + mine) {
    int s = my0;
    long long base = before;
    for (;; ++s) {
      const long long n = (long long)(pages_of(seq_len(s)) + kStart) * p.nkv;
      if (u0 < base + n || s + 1 >= my1) break;
      base += n;
    }
    first_seq = s;
    first_base = base;
  }
  __syncthreads();
  // the first page: its sequence, the sequence's first unit, its head and number
  int s0 = first_seq;
  const long long base0 = first_base;
  int len0 = seq_len(s0), np0 = pages_of(len0);
  const int head0 = (int)((u0 - base0) / (np0 + kStart));
  const int page0 = max(0, (int)((u0 - base0) % (np0 + kStart)) - kStart);
  if (base0 + (long long)head0 * (np0 + kStart) + kStart + page0 >= u1) return;  // units without a page

  if (warp == kConsumers) {
    // ---------------- producer
    int s = s0, len = len0, np = np0, head = head0, page = page0;
    long long base = base0;
    int first_page = page, ids_at = -1, id = 0;
    int it = 0, st = 0;
    uint32_t phase = 1;  // of the wait for a free stage: the first round finds them free
    bool ok = true;
    const uint32_t q_bytes = (uint32_t)(p.hpk * HD * sizeof(T));
    for (;; ++it) {
      if (page >= np) {
        page = 0;
        if (++head >= p.nkv) {
          head = 0;
          base += (long long)(np + kStart) * p.nkv;
          if (base + kStart >= u1) break;
          ++s;
          len = seq_len(s);
          np = pages_of(len);
        }
        first_page = 0;
        ids_at = -1;
      }
      const long long at = base + (long long)head * (np + kStart) + kStart;  // unit of page 0
      if (at + page >= u1) break;
      if (ids_at < 0 || page >= ids_at + 32) {  // the numbers of the next 32 pages, one per lane
        ids_at = page;
        id = len > 0 && page + lane < np ? p.table[(int64_t)s * p.table_stride + page + lane] : 0;
      }
      const int pid = __shfl_sync(0xffffffffu, id, page - ids_at);
      int valid = min(kPageRows, len - page * kPageRows);
      if (valid < 0) valid = 0;
      if (valid > 0 && (pid < 0 || pid >= p.n_pages)) {
        if (lane == 0) flag_position(p.err);
        valid = 0;
      }
      ok = __shfl_sync(0xffffffffu, lane == 0 ? (int)mbar_wait_bounded(&empty[st], phase, p.err, kDevErrEmptyTimeout) : 0, 0);
      if (!ok) break;
      if (lane == 0) {
        const bool first = it == 0 || page == 0;
        const int left = (int)(u1 - (at + page) < np - page ? u1 - (at + page) : np - page);
        seg[st] = Segment{at, s, head, np, at + np + kStart < u1, valid, first_page, first ? 1 : 0, left};
        uint8_t* dst = smem + (size_t)st * p.stage_bytes;
        mbar_arrive_expect_tx(&full[st], (valid ? (uint32_t)B::kBytes : 0u) + (first ? q_bytes : 0u));
        if (first)
          bulk_g2s(dst + B::kBytes,
                   static_cast<const T*>(p.q) + s * p.q_stride + (int64_t)head * p.hpk * HD, q_bytes, &full[st]);
        if (valid) bulk_g2s(dst, p.pages + ((int64_t)pid * (p.nkv / p.split) + head / p.split) * B::kBytes, B::kBytes, &full[st]);
      }
      __syncwarp();
      ++page;
      if (++st == p.stages) {
        st = 0;
        phase ^= 1;
      }
    }
    // after a wait that gave up, the copies in flight land before the CTA leaves
    if (!ok)
      for (int i = 0; i < p.stages && i < it; ++i) {
        const int uses = (it - i + p.stages - 1) / p.stages;
        mbar_wait_bounded(&full[i], (uint32_t)(uses - 1) & 1u, p.err, kDevErrDrainTimeout);
      }
    return;
  }

  // ---------------- consumers: warp w takes rows 16w .. 16w + 15 of every page
  // Fragments of lane (g, t): A rows g and g + 8, k slots 2t, + 1 and 2t + 8, + 9; B the same
  // slots of column g, that is of head g / 2's hi (g even) or lo part; C rows g, g + 8 of columns
  // 2t, 2t + 1, that is of head t. Tile n holds the heads 4n .. 4n + 3.
  const int g = lane >> 2, t = lane & 3;
  const bool odd = g & 1;
  const uint32_t one = opaque(0x3C003C00u), big = opaque(0x64006400u);
  ConsumerSync sync{&cons_bar, 0, p.err};
  uint32_t qb[NT][G][4], qm[NT];  // B: two k steps per group; the groups' sums of q
  float qs[NT][G];                // head t: the groups' sums of q
  // head t: what weights are relative to (2^(s - ref), at most 2^lift), their sum, and the reference
  // of what shared memory holds
  float kscale[NT], ref[NT], l[NT], ref_held[NT];
  uint32_t cap;  // the power of two that V's steps d stay below, as a pair of f16, each with bit 15 set
  float lift;    // how far below the maximum a reference lies
  float o[NT][2 * G][4];          // values: [16 u + (g, g + 8)] of group j, head t
  float2 om[NT][G];               // middles of group j, head g / 2, this lane's even and odd rows
  bool held = false;
  int since = 0;

  // adds this warp's accumulators to its sums in shared memory, and clears them
  auto flush = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float keep = ex2(ref_held[n] - ref[n]);
      const int h = 4 * n + t;
      float* dst = wo + ((size_t)warp * p.hpk + h) * PITCH;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        float mid = om[n][j].x + om[n][j].y;
        mid += __shfl_xor_sync(0xffffffffu, mid, 1);
        mid += __shfl_xor_sync(0xffffffffu, mid, 2);
        mid += __shfl_xor_sync(0xffffffffu, mid, 4);
        mid = __shfl_sync(0xffffffffu, mid, 8 * t);
        if (h < p.hpk) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float* c = o[n][2 * j + u] + 2 * r;
              float* d = dst + 32 * j + 16 * u + 8 * r + g;
              const float v = fmaf(fmaf(c[1], kLo, c[0]), 0.0625f, mid);
              *d = held ? fmaf(*d, keep, v) : v;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][2 * j][i] = o[n][2 * j + 1][i] = 0.f;
        om[n][j] = make_float2(0.f, 0.f);
      }
      ref_held[n] = ref[n];
    }
    held = true;
    since = 0;
  };

  // hi and lo of the weights (a, b) of this lane's head g / 2 to the lanes of B's columns
  auto columns = [&](float a, float b, uint32_t& b0, uint32_t& b1) {
    uint32_t hi, lo;
    split2(a, b, hi, lo);
    const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? hi : lo, 4);
    b0 = odd ? got : hi;
    b1 = odd ? lo : got;
  };

  // this warp's rows of a page (two pages at a time, for more independent work, measured 7 %
  // slower: the loop outgrows the instruction cache)
  auto rows = [&](const uint8_t* blk, int valid) {
    const int r0 = 16 * warp;
    const uint8_t* vb = blk + B::kHalf;
    // ---- V's steps, of a row (64 values) or half a row to each lane
    constexpr int W = G / 4 < 1 ? 1 : G / 4, kLanes = 8 * G / W;
    uint32_t steps[W];
    lds_words<W>(vb + B::kCodes + 2 * B::scale(r0, 0) + 4 * W * (lane % kLanes), steps);
    // ---- scores of rows r0 + g, r0 + 8 + g for head t of every tile
    float s[NT][2];
    {
      const int ra = r0 + g, rb = ra + 8;
      uint32_t da[G / 2], db[G / 2];  // f16 pairs of groups
      lds_words<G / 2>(blk + B::kCodes + 2 * B::scale(ra, 0), da);
      lds_words<G / 2>(blk + B::kCodes + 2 * B::scale(rb, 0), db);
      uint32_t ma[4] = {0u, 0u, 0u, 0u};
      if (2 * t < G) {
        ma[0] = *reinterpret_cast<const uint32_t*>(blk + B::kCodes + B::kScales + 2 * B::scale(ra, 2 * t));
        ma[1] = *reinterpret_cast<const uint32_t*>(blk + B::kCodes + B::kScales + 2 * B::scale(rb, 2 * t));
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = 0.f;
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int P = 0; P < B::kPlanes; ++P) {
        uint32_t wa[J], wb[J];
        lds_words<J>(blk + 4 * B::k_word(ra, P * J, t), wa);
        lds_words<J>(blk + 4 * B::k_word(rb, P * J, t), wb);
#pragma unroll
        for (int i = 0; i < J; ++i) {
          const int j = P * J + i;
          const uint32_t a0[4] = {from_one(wa[i] << 6, one), from_one(wb[i] << 6, one), from_one(wa[i] << 2, one),
                                  from_one(wb[i] << 2, one)};
          const uint32_t a1[4] = {from_one(wa[i] >> 2, one), from_one(wb[i] >> 2, one), from_one(wa[i] >> 6, one),
                                  from_one(wb[i] >> 6, one)};
          const float d0 = half_of(da[j / 2], j & 1), d1 = half_of(db[j / 2], j & 1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float c[4];
            mma_f16(c, a0, qb[n][j][0], qb[n][j][1], zero);
            mma_f16(c, a1, qb[n][j][2], qb[n][j][3]);
            s[n][0] = fmaf(d0, fmaf(c[1], kLo, c[0] - qs[n][j]), s[n][0]);
            s[n][1] = fmaf(d1, fmaf(c[3], kLo, c[2] - qs[n][j]), s[n][1]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float c[4];
        mma_f16(c, ma, qm[n], 0u, zero);
        s[n][0] = fmaf(s[n][0], 16.f, fmaf(c[1], kLo, c[0])) * kscale[n];
        s[n][1] = fmaf(s[n][1], 16.f, fmaf(c[3], kLo, c[2])) * kscale[n];
      }
      if (r0 + 16 > valid) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (r0 + 8 * i + g >= valid) s[n][i] = -INFINITY;
        if (r0 + lane % kLanes * 16 / kLanes >= valid)
#pragma unroll
          for (int i = 0; i < W; ++i) steps[i] = 0u;
      }
    }
    // ---- online softmax; then the weights in B's order: lane (g, t) takes of head g / 2 the
    // rows 2t, 2t + 1 of the first (g even) or second eight rows
    float2 pw[NT];
    float x[NT][2];
    bool above = false;  // a step above cap (a borrow from bit 15; steps are not negative)
#pragma unroll
    for (int i = 0; i < W; ++i) above |= (~(cap - steps[i]) & 0x80008000u) != 0u;
    bool grow = above;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      x[n][0] = s[n][0] - ref[n];
      x[n][1] = s[n][1] - ref[n];
      grow |= !(fmaxf(x[n][0], x[n][1]) <= lift);
    }
    if (__any_sync(0xffffffffu, grow)) {  // (rare after the first pages)
      const float lift_before = lift;
      if (__any_sync(0xffffffffu, above)) {
        uint32_t top_step = 0u;
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
          for (int k = 0; k < 32; k += 16) {
            const uint32_t d = steps[i] >> k & 0xffffu;
            if (d < 0x7c00u) top_step = max(top_step, d);  // (the NaN of a group that is not finite has no size)
          }
        top_step = __reduce_max_sync(0xffffffffu, top_step);
        if (top_step > (cap & 0x7fffu)) {  // steps are below 2^e now
          const int e = ((int)__float_as_uint(__half2float(__ushort_as_half((unsigned short)top_step))) >> 23) - 126;
          const __half to = __float2half_rn(fminf(__uint_as_float((uint32_t)(e + 127) << 23), 65504.f));
          cap = 0x80008000u | __half_as_ushort(to) * 0x10001u;
          lift = fmaxf((float)(kWeightBits - e), 0.f);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top = fmaxf(s[n][0], s[n][1]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        // (from 2^24 on a difference is rounded, to or fro between two neighbours at the worst; the
        // lift of up to 22 becomes 32 at the most, and of over 2^29 nothing)
        top = fmaxf(top, ref[n] + lift_before) - lift;
        const float alpha = ex2(ref[n] - top);
        ref[n] = top;
        x[n][0] = s[n][0] - top;
        x[n][1] = s[n][1] - top;
        l[n] *= alpha;
#pragma unroll
        for (int i = 0; i < 2 * G; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[n][i][k] *= alpha;
        const float al = __shfl_sync(0xffffffffu, alpha, g >> 1);
#pragma unroll
        for (int j = 0; j < G; ++j) om[n][j] = __fmul2_rn(om[n][j], make_float2(al, al));
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float p0 = ex2(x[n][0]), p1 = ex2(x[n][1]);
      l[n] += p0 + p1;
      const int from = 8 * t + (g >> 1);
      const float a0 = __shfl_sync(0xffffffffu, p0, from), a1 = __shfl_sync(0xffffffffu, p1, from);
      const float b0 = __shfl_sync(0xffffffffu, p0, from + 4), b1 = __shfl_sync(0xffffffffu, p1, from + 4);
      pw[n] = odd ? make_float2(a1, b1) : make_float2(a0, b0);
    }
    // ---- weighted rows
    {
      const int rw = r0 + 2 * t + (odd ? 8 : 0);  // rows of pa, pb
      uint32_t dw[G], mw[G];                      // f16 d [row][group]; m [group][row]
      lds_words<G>(vb + B::kCodes + 2 * B::scale(rw, 0), dw);
      lds_words<G>(vb + B::kCodes + B::kScales + 2 * B::v_min(rw, 0), mw);
      if (r0 + 16 > valid) {  // rows that hold nothing yet: what their d and m are does not count
        const int n = valid - rw;
#pragma unroll
        for (int i = 0; i < G; ++i) {
          if (n < (i < G / 2 ? 1 : 2)) dw[i] = 0u;
          mw[i] &= n >= 2 ? 0xffffffffu : n == 1 ? 0xffffu : 0u;
        }
      }
#pragma unroll
      for (int P = 0; P < B::kPlanes; ++P) {
        uint32_t w0[J], w1[J];
        lds_words<J>(vb + 2 * B::v_half(r0 + 2 * t, P * J, g), w0);
        lds_words<J>(vb + 2 * B::v_half(r0 + 8 + 2 * t, P * J, g), w1);
#pragma unroll
        for (int i = 0; i < J; ++i) {
          const int j = P * J + i;
          const uint32_t h0 = w0[i] >> 8, h1 = w1[i] >> 8;
          const uint32_t a0[4] = {centred_low(w0[i], big), centred(w0[i], big), centred_low(w1[i], big),
                                  centred(w1[i], big)};
          const uint32_t a1[4] = {centred_low(h0, big), centred(h0, big), centred_low(h1, big), centred(h1, big)};
          const float2 d = make_float2(half_of(dw[j / 2], j & 1), half_of(dw[(G + j) / 2], j & 1));
          const float2 c = __ffma2_rn(make_float2(8.f, 8.f), d, make_float2(half_of(mw[j], 0), half_of(mw[j], 1)));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 w = __fmul2_rn(pw[n], d);
            uint32_t b0, b1;
            columns(w.x, w.y, b0, b1);
            mma_f16(o[n][2 * j], a0, b0, b1);
            mma_f16(o[n][2 * j + 1], a1, b0, b1);
            om[n][j] = __ffma2_rn(pw[n], c, om[n][j]);
          }
        }
      }
    }
  };

  int st = 0;
  uint32_t phase = 0;
  auto landed = [&]() {
    return __all_sync(0xffffffffu, mbar_wait_bounded(&full[st], phase, p.err, kDevErrFullTimeout));
  };
  auto next = [&]() {
    if (++st == p.stages) {
      st = 0;
      phase ^= 1;
    }
  };
  for (;;) {
    if (!landed()) return;
    const Segment sg = seg[st];
    const uint8_t* blk = smem + (size_t)st * p.stage_bytes;
    if (sg.first) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        // head g / 2 of the tile, scaled by a power of two to below 2^10, and its group sums
        const int h = 4 * n + (g >> 1);
        float x[G][8];
        float top = 0.f;
        const T* q = reinterpret_cast<const T*>(blk + B::kBytes) + h * HD + 8 * t;
#pragma unroll
        for (int j = 0; j < G; ++j) {
          if (h < p.hpk) {
            load_vec<T, 8>(q + 32 * j, x[j]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int sh = min(120, 9 - ((int)(__float_as_uint(top) >> 23) - 127));
        const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
        // head t's numbers lie in the lanes of g = 2t
        kscale[n] = p.scale * __uint_as_float((uint32_t)(127 - __shfl_sync(0xffffffffu, sh, 8 * t)) << 23);
        float s0 = 0.f, s1 = 0.f;  // sums of groups 2t, 2t + 1
#pragma unroll
        for (int j = 0; j < G; ++j) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[j][i] *= up;
          float sum_hi = 0.f, sum_lo = 0.f;
          // k slots of a lane: elements 0, 4 | 1, 5 and 2, 6 | 3, 7
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t hi, lo;
            split2(x[j][i], x[j][i + 4], hi, lo);
            qb[n][j][i] = odd ? lo : hi;
            sum_hi += half_of(hi, 0) + half_of(hi, 1);
            sum_lo += half_of(lo, 0) + half_of(lo, 1);
          }
          sum_hi += __shfl_xor_sync(0xffffffffu, sum_hi, 1);
          sum_lo += __shfl_xor_sync(0xffffffffu, sum_lo, 1);
          sum_hi += __shfl_xor_sync(0xffffffffu, sum_hi, 2);
          sum_lo += __shfl_xor_sync(0xffffffffu, sum_lo, 2);
          const float sum = fmaf(sum_lo, kLo, sum_hi);
          if (j == 2 * t) s0 = sum;
          if (j == 2 * t + 1) s1 = sum;
          qs[n][j] = __shfl_sync(0xffffffffu, sum, 8 * t);
          om[n][j] = make_float2(0.f, 0.f);
        }
        uint32_t hi, lo;
        split2(s0, s1, hi, lo);
        qm[n] = odd ? lo : hi;
        ref[n] = ref_held[n] = kNone;
        l[n] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * G; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[n][i][k] = 0.f;
      }
      held = false;
      since = 0;
      cap = 0x80008000u;
      lift = 0.f;
    }
    if (16 * warp < sg.valid) rows(blk, sg.valid);
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
    next();
    const bool last = sg.left <= 1;
    if (last) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 4);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 8);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 16);
        if (g == 0 && 4 * n + t < p.hpk) {
          wm[warp][4 * n + t] = ref[n];
          wl[warp][4 * n + t] = l[n];
        }
      }
    }
    if (last || ++since == kFlush) flush();  // (in one place: with two the loop was 2 to 5 % slower)
    if (!last) continue;

    // ---------------- end of the segment: join the warps in order
    if (!sync()) return;
    // the CTAs of this (sequence, head)
    const long long last_unit = sg.base + sg.pages - 1;
    const int c0 = (int)(((sg.base + 1) * grid - 1) / U), c1 = (int)(((last_unit + 1) * grid - 1) / U);
    if (sg.first_page == 0 && threadIdx.x == 0) p.runs[(size_t)sg.seq * p.nkv + sg.head] = make_int2(c0, c1 - c0 + 1);
    const bool alone = c0 == c1;
    const size_t part_floats = (size_t)p.hpk * (HD + 2);
    float* part = p.parts + (size_t)(2 * blockIdx.x + (sg.first_page == 0 ? 1 : 0)) * part_floats;
    T* out = static_cast<T*>(p.out) + sg.seq * p.out_stride + (int64_t)sg.head * p.hpk * HD;
    for (int i = threadIdx.x; i < p.hpk * HD; i += 32 * kConsumers) {
      const int h = i / HD;
      float M = kNone;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) M = fmaxf(M, wm[w][h]);
      float v = 0.f, L = 0.f;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) {
        const float e = ex2(wm[w][h] - M);
        v = fmaf(e, wo[((size_t)w * p.hpk + h) * PITCH + i % HD], v);
        L = fmaf(e, wl[w][h], L);
      }
      if (alone) {
        out[i] = from_f32<T>(L == 0.f ? 0.f : v / L);
      } else {
        part[i] = v;
        if (i % HD == 0) {
          part[p.hpk * HD + h] = M;
          part[p.hpk * HD + p.hpk + h] = L;
        }
      }
    }
    if (!sg.more) return;
    if (!sync()) return;  // the joined states are read: the next segment may write its own
  }
}

// Joins the parts of one (sequence, head). Of a CTA's warps `across` lie side by side, four values a
// lane, and the rest are groups that take every `groups`-th part each, kAtOnce of them in flight;
// the groups' sums are added in order. Few heads: one warp across, and CTAs for the other columns,
// as each has many parts; many heads: four across, as most have one or two. Every thread takes its
// head's references and weights' sums along with the values. (A pass for them first, by one warp per
// query head, and four across always: one sequence of 1,023 rows 11.6 us instead of 10.4, of
// 131,000 66.7 instead of 59.4. One across always: 64 sequences 116 us instead of 111.)
constexpr int kJoinWarps = 16, kAtOnce = 4;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps)
    kv4_join_kernel(const __grid_constant__ Kv4Params p, int hd, int across) {
  __shared__ float4 sums[kJoinWarps][32];
  __shared__ float2 stats[kJoinWarps][32];
  pdl_launch_dependents();
  pdl_wait();
  const int2 run = p.runs[blockIdx.x];
  const int n = run.y, width = p.hpk * hd;
  if (n < 2 || run.x < 0 || n > p.ctas - run.x) return;  // (nothing written where a wait gave up)
  const size_t part_floats = (size_t)p.hpk * (hd + 2);
  // the part that starts the (sequence, head) is its CTA's slot 1, the others slot 0
  const float* base = p.parts + (size_t)2 * run.x * part_floats;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp / across, groups = kJoinWarps / across;
  const int seq = blockIdx.x / p.nkv, head = blockIdx.x % p.nkv;
  T* out = static_cast<T*>(p.out) + seq * p.out_stride + (int64_t)head * width;
  for (int e0 = 128 * across * blockIdx.y; e0 < width; e0 += 128 * across * gridDim.y) {
    const int e = e0 + 128 * (warp % across) + 4 * lane, h = e / hd;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, M = kNone, L = 0.f;
    if (e < width) {
      for (int i0 = group; i0 < n; i0 += groups * kAtOnce) {
        float m[kAtOnce], l[kAtOnce];
        float2 x[kAtOnce], y[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const int i = i0 + u * groups;
          m[u] = kNone;
          l[u] = 0.f;
          x[u] = y[u] = make_float2(0.f, 0.f);
          if (i < n) {
            const float* q = base + (size_t)(2 * i + (i == 0 ? 1 : 0)) * part_floats;
            m[u] = __ldcg(q + width + h);
            l[u] = __ldcg(q + width + p.hpk + h);
            x[u] = __ldcg(reinterpret_cast<const float2*>(q + e));
            y[u] = __ldcg(reinterpret_cast<const float2*>(q + e + 2));
          }
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) top = fmaxf(top, m[u]);
        const float keep = ex2(M - top);
        M = top;
        L *= keep;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] *= keep;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const float w = ex2(m[u] - top);
          L = fmaf(w, l[u], L);
          v[0] = fmaf(w, x[u].x, v[0]);
          v[1] = fmaf(w, x[u].y, v[1]);
          v[2] = fmaf(w, y[u].x, v[2]);
          v[3] = fmaf(w, y[u].y, v[3]);
        }
      }
      sums[warp][lane] = make_float4(v[0], v[1], v[2], v[3]);
      stats[warp][lane] = make_float2(M, L);
    }
    __syncthreads();
    if (group == 0 && e < width) {
      float top = M;
      for (int k = 1; k < groups; ++k) top = fmaxf(top, stats[k * across + warp][lane].x);
      const float keep = ex2(M - top);
      L *= keep;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] *= keep;
      for (int k = 1; k < groups; ++k) {
        const float4 x = sums[k * across + warp][lane];
        const float2 st = stats[k * across + warp][lane];
        const float w = ex2(st.x - top);
        L = fmaf(w, st.y, L);
        v[0] = fmaf(w, x.x, v[0]);
        v[1] = fmaf(w, x.y, v[1]);
        v[2] = fmaf(w, x.z, v[2]);
        v[3] = fmaf(w, x.w, v[3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = L == 0.f ? 0.f : v[i] / L;
      store_vec<T, 4>(out + e, v);
    }
    __syncthreads();
  }
}

template <int HD, int NT, typename T>
cudaError_t launch(const LaunchEnv& env, Kv4Params p) {
  constexpr int kCtas = ctas_per_sm<HD, NT>();
  constexpr int kBudget = 227 * 1024 / kCtas - 1024 - 2560;  // the system's and the static shared memory
  p.stage_bytes = Kv4Block<HD>::kBytes + p.hpk * HD * (int)sizeof(T);
  const int join = kConsumers * p.hpk * (HD + 8) * 4;
  p.stages = (kBudget - join) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const int smem = p.stages * p.stage_bytes + join;
  auto kern = kv4_attention_kernel<HD, NT, T>;
  // The attribute is the function's on the device, whatever context or thread calls: one value for
  // every number of query heads, so that no call takes back what another is about to launch with
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kBudget);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)p.n_seqs * p.nkv * ((p.max_pages > 0 ? p.max_pages : 1) + kStart);
  const int ctas = env.sm_count * kCtas;
  const int grid = (int)(units < ctas ? units : ctas);
  p.ctas = grid;
  e = rrr_launch_pdl(kern, dim3(grid), dim3(kThreads), (size_t)smem, env.stream, env.pdl, p);
  if (e != cudaSuccess || p.max_pages < 2) return e;  // a single page is one CTA's
  const int64_t heads = (int64_t)p.n_seqs * p.nkv;
  const bool few = heads <= 2 * env.sm_count;
  return rrr_launch_pdl(kv4_join_kernel<T>, dim3((unsigned)heads, few ? (p.hpk * HD + 127) / 128 : 1),
                        dim3(32 * kJoinWarps), 0, env.stream, env.pdl, p, HD, few ? 1 : 4);
}
template <int HD, typename T>
cudaError_t launch_tiles(const LaunchEnv& env, Kv4Params p) {
  // Six and eight queries per KV head of 128 or 256 values are taken as two heads of half as many,
  // which read the pages twice but keep more warps on an SM. (Eight queries on 4 KV heads, 10 x
  // 20,000 rows and 1 x 2,000: 209 -> 166 us and 29.5 -> 19.7 us with 256 values, 82 -> 84 and 18.1
  // -> 13.5 with 128. With 64 values the second tile of columns costs less than the unpacking that
  // it saves: 45 us against 59.)
  if (HD >= 128 && p.hpk > 4 && p.hpk % 2 == 0 && (int64_t)p.n_seqs * p.nkv <= INT32_MAX / 2) {
    p.split = 2;
    p.nkv *= 2;
    p.hpk /= 2;
  }
  return p.hpk <= 4 ? launch<HD, 1, T>(env, p) : launch<HD, 2, T>(env, p);
}
template <int HD>
cudaError_t launch_type(const LaunchEnv& env, int type, const Kv4Params& p) {
  switch (type) {
    case RRR_F32: return launch_tiles<HD, float>(env, p);
    case RRR_F16: return launch_tiles<HD, __half>(env, p);
    default: return launch_tiles<HD, __nv_bfloat16>(env, p);
  }
}

int64_t run_bytes(const rrr_kv4_cache* c) { return ((int64_t)c->n_seqs * c->n_kv_heads * 2 * 8 + 255) / 256 * 256; }

int check_heads(rrr_ctx* ctx, const rrr_kv4_cache* c, int n_heads, const char* fn) {
  if (n_heads < 1 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > kMaxHpk)
    return set_error(ctx, RRR_ERR_BAD_SHAPE,
                     "%s: n_heads must be a multiple of n_kv_heads, at most 8 query heads per KV head", fn);
  return RRR_OK;
}

}  // namespace
}  // namespace rrr

using namespace rrr;

extern "C" {

int rrr_kv4_workspace(rrr_ctx* ctx, const rrr_kv4_cache* c, int n_heads, int64_t* bytes) {
  const char* fn = "rrr_kv4_workspace";
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  int rc = check_kv4_cache(ctx, c, fn);
  if (rc || (rc = check_heads(ctx, c, n_heads, fn))) return rc;
  if (!bytes) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int64_t parts = 2 * 3 * (int64_t)ctx->sm_count;  // two per CTA, at most three CTAs per SM
  *bytes = run_bytes(c) + parts * (n_heads / c->n_kv_heads) * (c->head_dim + 2) * 4;
  return RRR_OK;
}

int rrr_attention_kv4(rrr_ctx* ctx, const rrr_kv4_cache* c, int n_heads, int type, const void* q,
                      int64_t q_stride, const int32_t* kv_lens, float scale, void* out,
                      int64_t out_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "rrr_attention_kv4";
  int64_t need = 0;
  int rc = rrr_kv4_workspace(ctx, c, n_heads, &need);
  if (rc) return rc;
  if (!row_type(type)) return set_error(ctx, RRR_ERR_BAD_QTYPE, "%s: type must be 0 (F32), 1 (F16) or 30 (BF16)", fn);
  if (!workspace || (c->n_seqs > 0 && (!q || !kv_lens || !out))) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int64_t width = (int64_t)n_heads * c->head_dim;
  if (!stride_fits(q_stride, width) || !stride_fits(out_stride, width))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: strides of n_heads * head_dim to 2^38", fn);
  if (!(scale >= 0.f) || scale > 3.4e38f) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: scale must be finite, not negative", fn);
  if (!aligned_to(q, 16) || !aligned_to(out, 16) || q_stride % 8 || out_stride % 8 || !aligned_to(kv_lens, 4) ||
      !aligned_to(workspace, 16))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: rows must be 16-byte aligned, strides multiples of 8 elements", fn);
  if (workspace_bytes < need)
    return set_error(ctx, RRR_ERR_BUFFER_TOO_SMALL, "%s: the workspace needs %lld bytes", fn, (long long)need);
  const int es = elem_bytes(type);
  const int64_t page_bytes = c->n_pages * c->n_kv_heads * 80 * c->head_dim;
  const RowSet qs{q, q_stride * es, width * es, c->n_seqs}, os{out, out_stride * es, width * es, c->n_seqs};
  const RowSet pages{c->pages, page_bytes, page_bytes, page_bytes ? 1 : 0}, ws{workspace, need, need, 1};
  if (!rows_disjoint(qs, os) || !rows_disjoint(os, pages) || !rows_disjoint(os, ws) || !rows_disjoint(ws, qs) ||
      !rows_disjoint(ws, pages))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: out and the workspace must overlap nothing", fn);
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  if (c->n_seqs == 0) return RRR_OK;
  const LaunchEnv env = make_env(ctx, stream);
  Kv4Params p{};
  p.pages = static_cast<const uint8_t*>(c->pages);
  p.n_pages = c->n_pages;
  p.table_stride = c->table_stride;
  p.table = c->page_table;
  p.n_seqs = c->n_seqs;
  p.max_pages = c->max_pages;
  p.nkv = c->n_kv_heads;
  p.hpk = n_heads / c->n_kv_heads;
  p.split = 1;
  p.q = q;
  p.out = out;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.lens = kv_lens;
  p.scale = (scale == 0.f ? 1.f / sqrtf((float)c->head_dim) : scale) * 1.4426950408889634f;
  p.runs = static_cast<int2*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + run_bytes(c));
  p.err = env.d_err;
  cudaError_t e;
  switch (c->head_dim) {
    case 64: e = launch_type<64>(env, type, p); break;
    case 128: e = launch_type<128>(env, type, p); break;
    default: e = launch_type<256>(env, type, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_attention_kv4 launch");
}

}  // extern "C"
