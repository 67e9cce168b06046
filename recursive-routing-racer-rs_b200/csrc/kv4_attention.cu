// kv4_attention.cu — attention of one query row per sequence over the 4-bit KV cache
// (rrr_attention_kv4): the decode step's `attention` dispatch (src/model/phi4.rs:1680-1688)
// for a batch of sequences of different lengths on pages.
//
// Mathematics. A key is k = d_j code + m_j in groups j of 32 values, so q . k = sum_j d_j (q_j .
// code_j) + m_j (sum q_j): the products with the codes run on mma.m16n8k16 (f16 in, f32
// accumulate) with the codes themselves as the B operand, and d_j multiplies each group's
// accumulator in f32. A 4-bit code in the low bits of an f16 is the subnormal code * 2^-24 (four
// bits further up, code * 2^-20), so one AND makes two operands out of a word and the powers of
// two leave with the scales. The A operand has 16 rows for at most 8 query heads: rows 0-7 hold
// the f16 part hi of the (power-of-two scaled) query, rows 8-15 the remainder (q - hi) * 2^11, so
// a score carries 22 bits of the query at no further instruction. The second product is alike: A
// holds p_i d_ij (one rescaled row set per group j, split hi and lo), B the V codes, and one
// more product of p itself with the m_ij. The softmax runs online in base 2, with 32-bit maxima and
// sums; scores, weights and sums keep f32 accuracy throughout.
//
// Work. A unit is one page (64 rows) of one (sequence, KV head). The CTAs share all units of the
// batch evenly, in order, whatever the lengths are (read on the device): CTA c of G takes the
// units [c U / G, (c+1) U / G). One producer warp streams the pages' blocks, each one
// contiguous, with bulk copies into a ring of stages, the segment's query row with its first
// page; four consumer warps take 16 rows of a page each and keep their own softmax state. At
// the end of a (sequence, head) segment the warps' states are joined in order; a segment that
// other CTAs share goes to the workspace, and the CTA that finishes last joins the parts in
// order (so results do not depend on which one that is) and leaves the counter at zero.
#include <math.h>

#include "kv4.cuh"

namespace rrr {
namespace {

constexpr int kConsumers = 4;  // warps
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr int kMaxStages = 16;
constexpr int kMaxHpk = 8;
constexpr float kLo = 1.f / 2048.f;

struct Kv4Params {
  const uint8_t* pages;
  int64_t n_pages, table_stride;
  const int* table;
  int n_seqs, max_pages, nkv, hpk;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  const int* lens;
  float scale;  // with log2(e)
  unsigned* counters;
  float* parts;
  int stages, stage_bytes;
  int* err;
};

struct Segment {  // beside each stage
  long long base;  // unit of the (sequence, head)'s first page
  int seq, head, pages;
  int valid;       // rows of this page that count
  int flags;       // 1: first page of this CTA's segment, 2: last
  int first_page;  // of this CTA's segment
};

template <int HD>
constexpr int ctas_per_sm() { return HD == 256 ? 1 : 2; }

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
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn((a - f.x) * 2048.f, (b - f.y) * 2048.f);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ float half_of(uint32_t w, int i) {
  return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w & 0xffffu)));
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

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<HD>())
    kv4_attention_kernel(const __grid_constant__ Kv4Params p) {
  using B = Kv4Block<HD>;
  constexpr int G = B::kGroups, J = B::kJ;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], cons_bar;
  __shared__ Segment seg[kMaxStages];
  __shared__ float wm[kConsumers][kMaxHpk], wl[kConsumers][kMaxHpk];
  __shared__ long long prefix[kThreads];
  __shared__ long long first_base;  // unit of the first sequence's first page
  __shared__ int first_seq, is_last;
  float* wo = reinterpret_cast<float*>(smem + (size_t)p.stages * p.stage_bytes);  // [warp][hpk][HD]

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
  for (int s = my0; s < my1; ++s) mine += (long long)pages_of(seq_len(s)) * p.nkv;
  prefix[threadIdx.x] = mine;
  __syncthreads();
  long long before = 0, U = 0;
  for (int i = 0; i < kThreads; ++i) {
    if (i == (int)threadIdx.x) before = U;
    U += prefix[i];
  }
  const long long grid = U < (long long)gridDim.x ? U : (long long)gridDim.x;  // CTAs with units
  if ((long long)blockIdx.x >= grid) return;
  const long long u0 = blockIdx.x * U / grid, u1 = (blockIdx.x + 1) * U / grid;
  if (u0 >= before && u0 < before + mine) {
    int s = my0;
    long long base = before;
    for (;; ++s) {
      const long long n = (long long)pages_of(seq_len(s)) * p.nkv;
      if (u0 < base + n || s + 1 >= my1) break;
      base += n;
    }
    first_seq = s;
    first_base = base;
  }
  __syncthreads();

  if (warp == kConsumers) {
    // ---------------- producer
    int s = first_seq;
    long long base = first_base;
    int len = seq_len(s), np = pages_of(len);
    int head = (int)((u0 - base) / np), page = (int)((u0 - base) % np);
    int first_page = page, ids_at = -1, id = 0;
    int it = 0;
    bool ok = true;
    const uint32_t q_bytes = (uint32_t)(p.hpk * HD * sizeof(T));
    for (long long u = u0; u < u1; ++u, ++it) {
      if (page >= np) {
        page = 0;
        if (++head >= p.nkv) {
          head = 0;
          base += (long long)np * p.nkv;
          ++s;
          len = seq_len(s);
          np = pages_of(len);
        }
        first_page = 0;
        ids_at = -1;
      }
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
      const int st = it % p.stages;
      if (it >= p.stages) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[st], (uint32_t)(it / p.stages - 1) & 1u, p.err,
                                                       kDevErrEmptyTimeout));
        if (!ok) break;
      }
      if (lane == 0) {
        const bool first = u == u0 || page == 0, last = u + 1 == u1 || page + 1 == np;
        seg[st] = Segment{base + (long long)head * np, s, head, np, valid, (first ? 1 : 0) | (last ? 2 : 0), first_page};
        uint8_t* dst = smem + (size_t)st * p.stage_bytes;
        mbar_arrive_expect_tx(&full[st], (valid ? (uint32_t)B::kBytes : 0u) + (first ? q_bytes : 0u));
        if (first)
          bulk_g2s(dst + B::kBytes,
                   static_cast<const T*>(p.q) + s * p.q_stride + (int64_t)head * p.hpk * HD, q_bytes, &full[st]);
        if (valid) bulk_g2s(dst, p.pages + ((int64_t)pid * p.nkv + head) * B::kBytes, B::kBytes, &full[st]);
      }
      __syncwarp();
      ++page;
    }
    // after a wait that gave up, the copies in flight land before the CTA leaves
    if (!ok)
      for (int st = 0; st < p.stages && st < it; ++st) {
        const int uses = (it - st + p.stages - 1) / p.stages;
        mbar_wait_bounded(&full[st], (uint32_t)(uses - 1) & 1u, p.err, kDevErrDrainTimeout);
      }
    return;
  }

  // ---------------- consumers
  const int g = lane >> 2, t = lane & 3;
  ConsumerSync sync{&cons_bar, 0, p.err};
  uint32_t qa[G][8], qm[4];  // A fragments: two k steps per group; the groups' sums
  float kscale = 0.f;
  float m = -INFINITY, l = 0.f;
  float o[4 * G][4], om[4];
  int it = 0;
  for (long long u = u0; u < u1; ++u, ++it) {
    const int st = it % p.stages;
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[st], (uint32_t)(it / p.stages) & 1u, p.err, kDevErrFullTimeout)))
      return;
    const uint8_t* blk = smem + (size_t)st * p.stage_bytes;
    const Segment sg = seg[st];
    if (sg.flags & 1) {
      // the query of head row g: scaled by a power of two to below 2^10, split, its group sums
      float x[G][8];
      float top = 0.f;
      const T* q = reinterpret_cast<const T*>(blk + B::kBytes) + g * HD + 8 * t;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        if (g < p.hpk) {
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
      kscale = p.scale * __uint_as_float((uint32_t)(127 - sh) << 23);
      float sum[G];
#pragma unroll
      for (int j = 0; j < G; ++j) {
        sum[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[j][i] *= up;
          sum[j] += x[j][i];
        }
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
        sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
        // k slots of a lane: elements 0, 4 | 1, 5 (codes times 16) and 2, 6 | 3, 7 (times 16)
        split2(x[j][0], x[j][4], qa[j][0], qa[j][1]);
        split2(x[j][1] * 0.0625f, x[j][5] * 0.0625f, qa[j][2], qa[j][3]);
        split2(x[j][2], x[j][6], qa[j][4], qa[j][5]);
        split2(x[j][3] * 0.0625f, x[j][7] * 0.0625f, qa[j][6], qa[j][7]);
      }
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int j = 0; j < G; j += 2)
        if (j == 2 * t) {
          s0 = sum[j];
          s1 = sum[j + 1];
        }
      split2(s0, s1, qm[0], qm[1]);
      qm[2] = qm[3] = 0;
      m = -INFINITY;
      l = 0.f;
#pragma unroll
      for (int n = 0; n < 4 * G; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) om[i] = 0.f;
    }
    const int r0 = 16 * warp;
    if (r0 < sg.valid) {
      // ---- scores of rows r0 + 8n + 2t, + 1 for head row g
      float s[2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int rg = r0 + 8 * n + g, rt = r0 + 8 * n + 2 * t;
        float cm[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t mins =
            2 * t < G ? *reinterpret_cast<const uint32_t*>(blk + B::kCodes + B::kScales + 2 * B::scale(rg, 2 * t)) : 0u;
        mma_f16(cm, qm, mins, 0u);
        uint32_t d[G];  // f16 d of rows rt, rt + 1: [row][group]
        lds_words<G>(blk + B::kCodes + 2 * B::scale(rt, 0), d);
        float a0 = 0.f, a1 = 0.f;
#pragma unroll
        for (int P = 0; P < B::kPlanes; ++P) {
          uint32_t w[J];
          lds_words<J>(blk + 4 * B::k_word(rg, P * J, t), w);
#pragma unroll
          for (int i = 0; i < J; ++i) {
            const int j = P * J + i;
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(c, &qa[j][0], w[i] & 0x000F000Fu, w[i] & 0x00F000F0u);
            const uint32_t w8 = w[i] >> 8;
            mma_f16(c, &qa[j][4], w8 & 0x000F000Fu, w8 & 0x00F000F0u);
            a0 = fmaf(half_of(d[j / 2], j & 1), fmaf(c[2], kLo, c[0]), a0);
            a1 = fmaf(half_of(d[(G + j) / 2], j & 1), fmaf(c[3], kLo, c[1]), a1);
          }
        }
        s[n][0] = fmaf(a0, 16777216.f, fmaf(cm[2], kLo, cm[0])) * kscale;
        s[n][1] = fmaf(a1, 16777216.f, fmaf(cm[3], kLo, cm[1])) * kscale;
      }
      const bool whole = r0 + 16 <= sg.valid;
      if (!whole) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (r0 + 8 * n + 2 * t + i >= sg.valid) s[n][i] = -INFINITY;
      }
      // ---- online softmax
      float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float m_new = fmaxf(m, top);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      if (__any_sync(0xffffffffu, m_new > m)) {
        const float alpha = ex2(m - m_use);
        l *= alpha;
#pragma unroll
        for (int n = 0; n < 4 * G; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][i] *= alpha;
#pragma unroll
        for (int i = 0; i < 4; ++i) om[i] *= alpha;
        m = m_new;
      }
      float pr[2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) pr[n][i] = ex2(s[n][i] - m_use);
      l += (pr[0][0] + pr[0][1]) + (pr[1][0] + pr[1][1]);
      // ---- weighted rows
      const uint8_t* vb = blk + B::kHalf;
      uint32_t d0[G], d1[G];  // f16 d of rows r0 + 2t, + 1 and r0 + 8 + 2t, + 1
      lds_words<G>(vb + B::kCodes + 2 * B::scale(r0 + 2 * t, 0), d0);
      lds_words<G>(vb + B::kCodes + 2 * B::scale(r0 + 8 + 2 * t, 0), d1);
      uint32_t pa[4];
      split2(pr[0][0], pr[0][1], pa[0], pa[1]);
      split2(pr[1][0], pr[1][1], pa[2], pa[3]);
      uint32_t v0 = 0, v1 = 0;
      if (g < G) {
        v0 = *reinterpret_cast<const uint32_t*>(vb + B::kCodes + B::kScales + 2 * B::v_min(r0 + 2 * t, g));
        v1 = *reinterpret_cast<const uint32_t*>(vb + B::kCodes + B::kScales + 2 * B::v_min(r0 + 8 + 2 * t, g));
      }
      if (!whole) {  // rows that hold nothing yet: what their d and m are does not count
        const int n0 = sg.valid - (r0 + 2 * t), n1 = n0 - 8;
        const uint32_t k0 = n0 >= 2 ? 0xffffffffu : n0 == 1 ? 0xffffu : 0u;
        const uint32_t k1 = n1 >= 2 ? 0xffffffffu : n1 == 1 ? 0xffffu : 0u;
        v0 &= k0;
        v1 &= k1;
#pragma unroll
        for (int i = 0; i < G; ++i) {
          if (i < G / 2 ? n0 < 1 : n0 < 2) d0[i] = 0u;
          if (i < G / 2 ? n1 < 1 : n1 < 2) d1[i] = 0u;
        }
      }
      mma_f16(om, pa, v0, v1);
#pragma unroll
      for (int P = 0; P < B::kPlanes; ++P) {
        uint32_t w0[J], w1[J];
        lds_words<J>(vb + 2 * B::v_half(r0 + 2 * t, P * J, g), w0);
        lds_words<J>(vb + 2 * B::v_half(r0 + 8 + 2 * t, P * J, g), w1);
#pragma unroll
        for (int i = 0; i < J; ++i) {
          const int j = P * J + i;
          uint32_t a[4];
          split2(pr[0][0] * half_of(d0[j / 2], j & 1), pr[0][1] * half_of(d0[(G + j) / 2], j & 1), a[0], a[1]);
          split2(pr[1][0] * half_of(d1[j / 2], j & 1), pr[1][1] * half_of(d1[(G + j) / 2], j & 1), a[2], a[3]);
          mma_f16(o[4 * j], a, w0[i] & 0x000F000Fu, w1[i] & 0x000F000Fu);
          mma_f16(o[4 * j + 1], a, w0[i] & 0x00F000F0u, w1[i] & 0x00F000F0u);
          const uint32_t x0 = w0[i] >> 8, x1 = w1[i] >> 8;
          mma_f16(o[4 * j + 2], a, x0 & 0x000F000Fu, x1 & 0x000F000Fu);
          mma_f16(o[4 * j + 3], a, x0 & 0x00F000F0u, x1 & 0x00F000F0u);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
    if (!(sg.flags & 2)) continue;

    // ---------------- end of the segment: join the warps in order
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0 && g < p.hpk) {
      wm[warp][g] = m;
      wl[warp][g] = l;
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      // group j's sum of p m sits in lane t = j / 2 (columns 2t, 2t + 1)
      const float mine_m = j & 1 ? fmaf(om[3], kLo, om[1]) : fmaf(om[2], kLo, om[0]);
      const float mins = __shfl_sync(0xffffffffu, mine_m, (lane & ~3) | (j / 2));
      if (g < p.hpk) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float f = r & 1 ? 1048576.f : 16777216.f;
          const float* c = o[4 * j + r];
          float2 v;
          v.x = fmaf(fmaf(c[2], kLo, c[0]), f, mins);
          v.y = fmaf(fmaf(c[3], kLo, c[1]), f, mins);
          *reinterpret_cast<float2*>(wo + ((size_t)warp * p.hpk + g) * HD + 32 * j + 8 * r + 2 * t) = v;
        }
      }
    }
    if (!sync()) return;
    // participants of this (sequence, head)
    const long long last_unit = sg.base + sg.pages - 1;
    const int c0 = (int)(((sg.base + 1) * grid - 1) / U), c1 = (int)(((last_unit + 1) * grid - 1) / U);
    const bool alone = c0 == c1;
    const size_t part_floats = (size_t)p.hpk * (HD + 2);
    float* part = p.parts + (size_t)(2 * blockIdx.x + (sg.first_page == 0 ? 1 : 0)) * part_floats;
    T* out = static_cast<T*>(p.out) + sg.seq * p.out_stride + (int64_t)sg.head * p.hpk * HD;
    for (int i = threadIdx.x; i < p.hpk * HD; i += 32 * kConsumers) {
      const int h = i / HD;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) M = fmaxf(M, wm[w][h]);
      const float Mu = M == -INFINITY ? 0.f : M;
      float v = 0.f, L = 0.f;
#pragma unroll
      for (int w = 0; w < kConsumers; ++w) {
        const float e = ex2(wm[w][h] - Mu);
        v = fmaf(e, wo[(size_t)w * p.hpk * HD + i], v);
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
    if (!alone) {
      __threadfence();
      if (!sync()) return;
      if (threadIdx.x == 0) {
        const unsigned n = (unsigned)(c1 - c0);
        is_last = atomicInc(&p.counters[(size_t)sg.seq * p.nkv + sg.head], n) == n;
        __threadfence();
      }
      if (!sync()) return;
      if (is_last) {
        for (int i = threadIdx.x; i < p.hpk * HD; i += 32 * kConsumers) {
          const int h = i / HD;
          float M = -INFINITY, v = 0.f, L = 0.f;
          for (int c = c0; c <= c1; ++c) {
            // the part that starts the (sequence, head) is its CTA's slot 1, the others slot 0
            const float* q = p.parts + (size_t)(2 * c + (c == c0 ? 1 : 0)) * part_floats;
            const float pm = __ldcg(q + p.hpk * HD + h), pl = __ldcg(q + p.hpk * HD + p.hpk + h);
            const float pv = __ldcg(q + i);
            const float Mn = fmaxf(M, pm), Mu = Mn == -INFINITY ? 0.f : Mn;
            const float e0 = ex2(M - Mu), e1 = ex2(pm - Mu);
            v = fmaf(v, e0, pv * e1);
            L = fmaf(L, e0, pl * e1);
            M = Mn;
          }
          out[i] = from_f32<T>(L == 0.f ? 0.f : v / L);
        }
      }
    }
    if (!sync()) return;  // the joined states are read: the next segment may write its own
  }
}

template <int HD, typename T>
cudaError_t launch(const LaunchEnv& env, Kv4Params p, int max_ctas) {
  constexpr int kBudget = (ctas_per_sm<HD>() == 2 ? 113 : 226) * 1024 - 6144;  // static and reserved shared memory
  p.stage_bytes = Kv4Block<HD>::kBytes + p.hpk * HD * (int)sizeof(T);
  const int join = kConsumers * p.hpk * HD * 4;
  p.stages = (kBudget - join) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const int smem = p.stages * p.stage_bytes + join;
  auto kern = kv4_attention_kernel<HD, T>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int64_t units = (int64_t)p.n_seqs * p.nkv * (p.max_pages > 0 ? p.max_pages : 1);
  const int grid = (int)(units < max_ctas ? units : max_ctas);
  return rrr_launch_pdl(kern, dim3(grid), dim3(kThreads), (size_t)smem, env.stream, env.pdl, p);
}
template <int HD>
cudaError_t launch_type(const LaunchEnv& env, int type, const Kv4Params& p) {
  const int ctas = env.sm_count * ctas_per_sm<HD>();
  switch (type) {
    case RRR_F32: return launch<HD, float>(env, p, ctas);
    case RRR_F16: return launch<HD, __half>(env, p, ctas);
    default: return launch<HD, __nv_bfloat16>(env, p, ctas);
  }
}

int64_t counter_bytes(const rrr_kv4_cache* c) { return ((int64_t)c->n_seqs * c->n_kv_heads * 4 + 255) / 256 * 256; }

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
  const int64_t parts = 2 * 2 * (int64_t)ctx->sm_count;  // two per CTA, at most two CTAs per SM
  *bytes = counter_bytes(c) + parts * (n_heads / c->n_kv_heads) * (c->head_dim + 2) * 4;
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
  if (!q || !kv_lens || !out || !workspace) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int64_t width = (int64_t)n_heads * c->head_dim;
  if (q_stride < width || out_stride < width)
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: strides of at least n_heads * head_dim", fn);
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
  p.q = q;
  p.out = out;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.lens = kv_lens;
  p.scale = (scale == 0.f ? 1.f / sqrtf((float)c->head_dim) : scale) * 1.4426950408889634f;
  p.counters = static_cast<unsigned*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + counter_bytes(c));
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
