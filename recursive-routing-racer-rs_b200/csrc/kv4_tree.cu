// kv4_tree.cu — attention of drafted rows over the 4-bit KV cache (rrr_attention_tree_kv4): the
// `attention` dispatch (src/model/phi4.rs:1284-1309, 1680-1688) for the rows of a tree of drafted
// tokens per sequence, which see the sequence's cached rows and their own ancestors.
#include <math.h>

#include <type_traits>

#include "kv4.cuh"
#include "tile_common.cuh"

namespace rrr {
namespace {

constexpr int kMaxHpk = 8, kMaxNodes = 128;
constexpr float kNone = -3e38f;  // the maximum of no rows: finite, so that it may be subtracted from -inf
constexpr int kRows = 128;       // KV rows of a block: two pages, or the drafted rows
constexpr int kStart = 2;        // units in front of a segment's blocks
constexpr int kThreads = 640;
constexpr int kInfos = 16;
constexpr float kBias = 10.f;    // weights are 2^(s - m + kBias), at most 2^(kBias + kLazy)
constexpr float kLazy = 5.f;

struct TreeParams {
  const uint8_t* pages;
  int64_t n_pages, table_stride;
  const int* table;
  int n_seqs, max_pages, nh, nkv, hpk;
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  const int* cu;
  const int* parents;
  const int* lens;
  int rows;
  float scale;   // with log2(e)
  int* err;
  // workspace
  int4* runs;     // [seq][KV head][tile]: first CTA, CTAs, whether to compute again
  float2* stats;  // [slot][column]: maximum, sum
  int* again;     // [slot]
  float* parts;   // [slot][column][value]
  int most_tiles, ctas;
};

// ---- what the sequences are
struct Shape {
  int r0, nodes, len, blocks, tiles, per;  // per: columns of a tile
};
template <int NT>
__device__ __forceinline__ Shape shape_of(const TreeParams& p, int seq) {
  Shape s;
  s.r0 = p.cu[seq];
  const int r1 = p.cu[seq + 1];
  s.nodes = r1 - s.r0;
  s.len = p.lens[seq];
  if (s.r0 < 0 || r1 < s.r0 || r1 > p.rows || s.nodes > kMaxNodes) {
    flag_position(p.err);
    s.nodes = 0;
  }
  if (s.nodes && (s.len < 0 || s.len > p.max_pages * kPageRows)) {
    flag_position(p.err);
    s.len = 0;
  }
  const int cols = s.nodes * p.hpk;
  s.tiles = (cols + NT - 1) / NT;
  s.per = s.tiles ? ((cols + s.tiles - 1) / s.tiles + 15) / 16 * 16 : 0;
  s.blocks = s.nodes ? (s.len + kRows - 1) / kRows + 1 : 0;
  return s;
}
__device__ __forceinline__ long long units_of(const TreeParams& p, const Shape& s) {
  return s.nodes ? (long long)s.tiles * p.nkv * (s.blocks + kStart) : 0;
}

enum { kDraft = 1, kFirst = 2, kLast = 4, kAlone = 8, kStop = 16, kOpens = 32 };
struct Info {  // of a block
  int flags, seq, kv, seg;    // seg: index in runs
  int r0, nodes, c0, cols, n; // the tile's columns c0 .. c0 + cols - 1 of the sequence's (row, head) pairs; n: with the padding
  int valid[2];               // rows of each page that count
  int slot, count, run;       // where a shared segment's part goes, the segment's number in this CTA, its CTAs
  int first_cta;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// Bounded wait of a warp. The limit lies in memory: it is looked up only where a few tries of some microseconds each were
// in vain.
__device__ __forceinline__ bool quick_wait(uint64_t* bar, uint32_t parity, int* err) {
  bool ok = false;
#pragma unroll 1
  for (int k = 0; k < 32 && !ok; ++k) ok = mbar_try_wait(bar, parity);
  if (__all_sync(0xffffffffu, ok)) return true;
  return warp_wait(bar, parity, err);
}

// Bounded barrier of four warps; `any`: which also tells whether one of their lanes says yes.
struct Quartet {
  uint64_t* bar;
  volatile int* votes;  // [2][4]
  uint32_t phase;
  int* err;
  __device__ __forceinline__ bool operator()() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
    const bool ok = quick_wait(bar, phase, err);
    phase ^= 1;
    return ok;
  }
  __device__ __forceinline__ bool any(bool yes, bool& ok) {
    volatile int* v = votes + 4 * phase;
    yes = __any_sync(0xffffffffu, yes);
    if ((threadIdx.x & 31) == 0) v[(threadIdx.x >> 5) & 3] = yes;
    ok = (*this)();
    return (v[0] | v[1] | v[2] | v[3]) != 0;
  }
};
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t x;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w), "r"(mask), "r"(bits));
  return x;
}
// d c + m of four pairs of codes, nibbles s and s + 4 of w for s = 0 .. 3. A code in an f16's low bits
// is 1024 + c, four bits further up 1024 + 16 c: c is exact either way, and the product is
// rounded once.
__device__ __forceinline__ void values_of(uint32_t w, __half2 d, __half2 m, uint32_t (&x)[4]) {
  const uint32_t big = 0x64006400u;
  const __half2 less = as_half2(0xe400e400u), sixteenth = as_half2(0x2c002c00u), less64 = as_half2(0xd400d400u);
  const uint32_t v = w >> 8;
  x[0] = as_u32(__hfma2(__hadd2(as_half2(and_or(w, 0x000f000fu, big)), less), d, m));
  x[1] = as_u32(__hfma2(__hfma2(as_half2(and_or(w, 0x00f000f0u, big)), sixteenth, less64), d, m));
  x[2] = as_u32(__hfma2(__hadd2(as_half2(and_or(v, 0x000f000fu, big)), less), d, m));
  x[3] = as_u32(__hfma2(__hfma2(as_half2(and_or(v, 0x00f000f0u, big)), sixteenth, less64), d, m));
}
// 128-byte swizzle of an offset from a 1024-byte border
__device__ __forceinline__ uint32_t swizzled(uint32_t off) { return off ^ (((off >> 7) & 7u) << 4); }
template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) return __half22float2(as_half2(w));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
// |values| of eight as bits, whose order is that of the values (NaN last)
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const uint4& w) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = pair_of<T>((&w.x)[i]);
    t = max(t, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
  }
  return t;
}
// The power of two that brings values of at most `top` (finite, not zero) into [1, 2)
__device__ __forceinline__ float to_one(uint32_t top, bool& fine) {
  fine = top < 0x7f800000u;
  const int e = (int)(top >> 23);  // (a subnormal top counts as 2^-126)
  return !fine || top == 0 ? 1.f : __uint_as_float((uint32_t)min(max(254 - e, 1), 254) << 23);
}
constexpr uint32_t kHalfMax = 0x477fe000u;  // 65504
// What drafted values of at most `top` are multiplied by, 2^-e, so that f16 holds them with all their bits
__device__ __forceinline__ float lift_of(uint32_t top) {
  return top >= 0x3b000000u /* 2^-9 */ ? 1.f : top >= 0x37000000u /* 2^-17 */ ? 256.f : 65536.f;
}
// Eight 16-bit values times s as f16, in the order (0,4) (1,5) (2,6) (3,7) in which a word of K's codes comes apart
template <typename T>
__device__ __forceinline__ void scaled_pairs(const uint4& w, float s, uint32_t (&x)[4]) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = pair_of<T>((&w.x)[i]);
    v[2 * i] = f.x * s;
    v[2 * i + 1] = f.y * s;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = as_u32(__floats2half2_rn(v[i], v[i + 4]));
}

// The sum over the warp's lanes of each of N values; lane l gets that of column_of<N>(l).
template <int N>
__device__ __forceinline__ int column_of(int lane) { return N >= 32 ? lane : lane % N; }
template <int N>
__device__ __forceinline__ float transposed_sum(float (&v)[N]) {
  static_assert(N == 32 || N == 16, "");
  const int lane = threadIdx.x & 31;
  int n = N;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int k = 0; k < N / 2; ++k)
      if (k < o) {
        const float give = up ? v[k] : v[k + o], keep = up ? v[k + o] : v[k];
        v[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
  }
  (void)n;
  if constexpr (N == 16) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 16);
  return v[0];
}

template <int HD, int NT>
struct Sizes {
  static constexpr int kPage = 80 * HD;             // bytes of a page's block of one head
  static constexpr int kStage = 2 * kPage;
  static constexpr int kKCols = HD / 2;             // TMEM columns of a block of keys
  static constexpr int kQ = HD / 64 * NT * 128;     // the tile's queries
  static constexpr int kERows = HD < 128 ? HD : 128;
  static constexpr int kHalves = HD > 128 ? 2 : 1;  // of V's values, 128 each
  static constexpr int kV = kHalves * 2 * kERows * 128;
  static constexpr int kVs = HD > 128 ? 1 : 2;      // places for V
  static constexpr int kP = (NT + 63) / 64 * kRows * 128;
  static constexpr int kFixed = kQ + kVs * kV + 2 * kP;
  static constexpr int kStatic = 17 * 1024;         // more than the static shared memory
  static constexpr int kFit = (227 * 1024 - kStatic - 1024 - kFixed) / kStage;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kFixed + kStages * kStage + 1024;
  static constexpr int kSCol = 2 * kKCols, kOCol = kSCol + 2 * NT;
  static_assert(kStages >= 2 && kOCol + kHalves * NT <= 512, "");
};

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    tree_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ TreeParams p) {
  using S = Sizes<HD, NT>;
  constexpr int G = HD / 32, J = G < 4 ? G : 4, PL = G / J;  // groups, groups per plane, planes
  constexpr int kHalfCols = NT / 2;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], k_full[2], s_full[2], v_full[S::kVs], p_full[2], p_empty[2], o_empty, fin;
  __shared__ Info infos[kInfos];
  __shared__ uint4 seen[4][kMaxNodes];            // of a tree's row: the rows that it sees, as bits
  __shared__ int up[kMaxNodes];
  __shared__ float q_scale[4][NT], k_scale[4][kRows], v_lift[4];
  __shared__ int k_again[4], v_again[4];
  __shared__ uint32_t k_tops[4], v_tops[4];
  __shared__ __align__(16) float2 line[NT];       // of a column: s = score * x, argument = s + y
  __shared__ float quad[2][4][kHalfCols], change[2][kHalfCols];
  __shared__ long long warp_units[kThreads / 32], first_base;
  __shared__ int first_seq;
  __shared__ uint32_t tmem_slot;
  __shared__ uint64_t teams[4];   // of the softmax's halves, K's and V's warps
  __shared__ int votes[2][2][4];
  uint8_t* smem = smem_dyn + ((1024u - (smem_addr(smem_dyn) & 1023u)) & 1023u);
  uint8_t* const qs = smem;
  uint8_t* const vs = qs + S::kQ;
  uint8_t* const ps = vs + S::kVs * S::kV;  // (behind V, whose operand of 64 values reads 8 KB further)
  uint8_t* const ring = ps + 2 * S::kP;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&p_empty[i], 1);
    }
    for (int i = 0; i < S::kVs; ++i) mbar_init(&v_full[i], 4);
    mbar_init(&o_empty, 8);
    mbar_init(&fin, 1);
    for (int i = 0; i < 4; ++i) mbar_init(&teams[i], 4);
    fence_mbarrier_init();
    prefetch_map(&map);
  }
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's units [u0, u1) of all U
  const int per = (p.n_seqs + kThreads - 1) / kThreads;
  const int my0 = min(p.n_seqs, (int)threadIdx.x * per), my1 = min(p.n_seqs, my0 + per);
  long long mine = 0;
  for (int s = my0; s < my1; ++s) mine += units_of(p, shape_of<NT>(p, s));
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_units[warp] = upto;
  __syncthreads();
  long long before = upto - mine, U = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warp_units[w];
    U += warp_units[w];
  }
  const long long grid = U < (long long)gridDim.x ? U : (long long)gridDim.x;
  if ((long long)blockIdx.x >= grid) return;
  const long long u0 = blockIdx.x * U / grid, u1 = (blockIdx.x + 1) * U / grid;
  if (u0 >= before && u0 < before + mine) {
    int s = my0;
    long long base = before;
    for (;; ++s) {
      const long long n = units_of(p, shape_of<NT>(p, s));
      if (u0 < base + n || s + 1 >= my1) break;
      base += n;
    }
    first_seq = s;
    first_base = base;
  }
  if (warp == 16) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // Every wait is bounded; a role that gave up leaves, and so do those that wait for it.
  auto wait = [&](uint64_t* bar, uint32_t parity) { return quick_wait(bar, parity, p.err); };

  // registers: 640 x 96 at launch = 256 x 128 + 256 x 96 + 128 x 32
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == 17) {
      // ---------------- the blocks in order, and the copies of their pages
      int s = first_seq, seg = -1, count = -1, it = 0, st = 0;
      long long base = first_base;
      Shape sh = shape_of<NT>(p, s);
      long long each = sh.blocks + kStart;
      int g = (int)((u0 - base) / each), blk = max(0, (int)((u0 - base) % each) - kStart);
      bool begin = true, stop = false;
      uint32_t phase = 1;  // of the wait for a free stage: the first round finds them free
      for (;; ++it) {
        if (blk >= sh.blocks) {
          blk = 0;
          begin = true;
          if (++g >= sh.tiles * p.nkv) {
            g = 0;
            base += units_of(p, sh);
            do {
              ++s;
              if (s >= p.n_seqs) break;
              sh = shape_of<NT>(p, s);
            } while (sh.nodes == 0);
            each = sh.blocks + kStart;
          }
        }
        const long long seg0 = base + (long long)g * each + kStart;  // unit of the segment's block 0
        stop = s >= p.n_seqs || seg0 + blk >= u1;
        int page = 0, valid = 0;
        const bool draft = blk + 1 == sh.blocks;
        if (!stop && !draft && lane < 2) {
          const int at = 2 * blk + lane;
          valid = min(kPageRows, sh.len - at * kPageRows);
          if (valid > 0) page = p.table[(int64_t)s * p.table_stride + at];
          if (valid < 0) valid = 0;
          if (page < 0 || page >= p.n_pages) {
            flag_position(p.err);
            valid = 0;
          }
        }
        if (begin) {
          ++count;
          seg = ((s * p.nkv) + g / max(sh.tiles, 1)) * p.most_tiles + g % max(sh.tiles, 1);
        }
        if (!wait(&empty[st], phase)) break;
        const int v0 = __shfl_sync(0xffffffffu, valid, 0), v1 = __shfl_sync(0xffffffffu, valid, 1);
        const int p0 = __shfl_sync(0xffffffffu, page, 0), p1 = __shfl_sync(0xffffffffu, page, 1);
        if (lane == 0) {
          Info f;
          if (stop) {
            f.flags = kStop;
          } else {
            const int kv = g / sh.tiles, tile = g % sh.tiles;
            const long long end = seg0 + sh.blocks - 1;
            const int c0 = (int)(((seg0 + 1) * grid - 1) / U), c1 = (int)(((end + 1) * grid - 1) / U);
            f.flags = (draft ? kDraft : 0) | (begin ? kFirst : 0) | (draft || seg0 + blk + 1 >= u1 ? kLast : 0) |
                      (c0 == c1 ? kAlone : 0) | (c0 == (int)blockIdx.x ? kOpens : 0);
            f.seq = s;
            f.kv = kv;
            f.seg = seg;
            f.r0 = sh.r0;
            f.nodes = sh.nodes;
            f.c0 = tile * sh.per;
            f.cols = min(sh.per, sh.nodes * p.hpk - f.c0);
            f.n = sh.per;
            f.valid[0] = draft ? min(sh.nodes, 64) : v0;
            f.valid[1] = draft ? max(sh.nodes - 64, 0) : v1;
            f.slot = 2 * blockIdx.x + (f.flags & kOpens ? 1 : 0);
            f.count = count;
            f.run = c1 - c0 + 1;
            f.first_cta = c0;
          }
          infos[it % kInfos] = f;
          uint8_t* dst = ring + (size_t)st * S::kStage;
          if (stop || draft) {
            mbar_arrive(&full[st]);
          } else {
            mbar_arrive_expect_tx(&full[st], (uint32_t)((v0 > 0) + (v1 > 0)) * S::kPage);
            if (v0 > 0) tma_load_2d(dst, &map, 0, (int)(((int64_t)p0 * p.nkv + f.kv) * (S::kPage / 128)), &full[st]);
            if (v1 > 0)
              tma_load_2d(dst + S::kPage, &map, 0, (int)(((int64_t)p1 * p.nkv + f.kv) * (S::kPage / 128)), &full[st]);
          }
        }
        __syncwarp();
        begin = false;
        if (++st == S::kStages) {
          st = 0;
          phase ^= 1;
        }
        if (stop) {
          ++it;
          break;
        }
        ++blk;
      }
      // copies in flight land before the CTA leaves
      for (int i = 0; i < S::kStages; ++i) {
        const int uses = it > i ? (it - i + S::kStages - 1) / S::kStages : 0;
        if (uses) warp_wait(&full[i], (uint32_t)(uses - 1) & 1u, p.err);
      }
    } else if (warp == 16) {
      // ---------------- products: S(0), S(1), PV(0), S(2), PV(1), ...
      const uint32_t fmt = 1u << 4;  // f16 operands, f32 sums; M = 128
      auto weighed = [&](int i) {    // O^T += V^T P^T of block i
        const Info& f = infos[i % kInfos];
        if (!wait(&v_full[i % S::kVs], (uint32_t)(i / S::kVs) & 1u) || !wait(&p_full[i & 1], (uint32_t)(i >> 1) & 1u))
          return false;
        if ((f.flags & kFirst) && f.count > 0 && !wait(&o_empty, (uint32_t)(f.count - 1) & 1u)) return false;
        tc_fence_after();
        const uint32_t idesc = fmt | (1u << 16) | ((uint32_t)(f.n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
        const uint32_t va = smem_addr(vs + (i % S::kVs) * S::kV), pa = smem_addr(ps + (i & 1) * S::kP);
        const bool first = f.flags & kFirst;
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
            for (int kk = 0; kk < kRows / 16; ++kk)
              umma_f16(tmem + S::kOCol + h * NT,
                       sw128_desc(va + (uint32_t)(h * 2 + kk / 4) * S::kERows * 128 + 32u * (kk % 4)),
                       sw128_desc_mn(pa + 2048u * kk, kRows * 128), idesc, first && kk == 0 ? 0u : 1u);
          umma_commit(&p_empty[i & 1]);
        }
        __syncwarp();
        return true;
      };
      int i = 0;
      for (;; ++i) {
        if (!wait(&k_full[i & 1], (uint32_t)(i >> 1) & 1u)) break;
        tc_fence_after();
        const Info& f = infos[i % kInfos];
        const bool stop = f.flags & kStop;
        if (!stop) {
          const uint32_t idesc = fmt | ((uint32_t)(f.n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
          const uint32_t qa = smem_addr(qs);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              umma_f16_ta(tmem + S::kSCol + (i & 1) * NT, tmem + (i & 1) * S::kKCols + 8u * kk,
                          sw128_desc(qa + (uint32_t)(kk / 4) * NT * 128 + 32u * (kk % 4)), idesc, kk > 0 ? 1u : 0u);
            umma_commit(&s_full[i & 1]);
          }
          __syncwarp();
        }
        if (i > 0 && !weighed(i - 1)) break;
        if (stop) {
          if (lane == 0) mbar_arrive(&s_full[i & 1]);
          break;
        }
      }
      if (elect_one()) umma_commit(&fin);
      __syncwarp();
    }
  } else if (warp >= 12) {
    // ---------------- V: two rows' pairs of values, transposed to rows of values
    const int tid = threadIdx.x - 12 * 32;
    Quartet team{&teams[3], nullptr, 0, p.err};
    int st = 0;
    uint32_t phase = 0;
    for (int i = 0;; ++i) {
      if (!wait(&full[st], phase)) break;
      const Info& f = infos[i % kInfos];
      if (f.flags & kStop) break;
      const int par = f.count & 3;
      if (f.flags & kFirst) {
        if (tid == 0) v_again[par] = 0;
        if (!team()) break;
      }
      // the place is free once PV(i - kVs) is done
      if (i >= S::kVs && !wait(&p_empty[(i - S::kVs) & 1], (uint32_t)((i - S::kVs) >> 1) & 1u)) break;
      uint8_t* const dst = vs + (i % S::kVs) * S::kV;
      if (!(f.flags & kDraft)) {
        const int o = tid >> 3, g = tid & 7;  // rows 8 o .. + 7 of the block, values 32 i + 8 n + g
        const uint8_t* const page = ring + (size_t)st * S::kStage + (o >> 3) * S::kPage;
        const int r = (o & 7) * 8, valid = f.valid[o >> 3];
        __half2 most = as_half2(0u);
#pragma unroll
        for (int P = 0; P < PL; ++P) {
          uint32_t w[4 * J];  // [t][i]
#pragma unroll
          for (int u = 0; u < J; ++u) {
            const uint4 x = *reinterpret_cast<const uint4*>(page + swizzled(40 * HD + P * 1024 * J + (r + g) * 16 * J + 16 * u));
            w[4 * u] = x.x;
            w[4 * u + 1] = x.y;
            w[4 * u + 2] = x.z;
            w[4 * u + 3] = x.w;
          }
          __half2 d[4][J], m[4][J];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int row = r + 2 * t;
            const bool even = row < valid, odd = row + 1 < valid;
#pragma unroll
            for (int k = 0; k < J; k += 2) {
              const int j = P * J + k;
              const uint32_t a = *reinterpret_cast<const uint32_t*>(page + swizzled(72 * HD + 2 * (row * G + j)));
              const uint32_t b = *reinterpret_cast<const uint32_t*>(page + swizzled(72 * HD + 2 * ((row + 1) * G + j)));
              const uint2 c = *reinterpret_cast<const uint2*>(page + swizzled(76 * HD + 4 * ((row >> 1) * G + j)));
              const uint32_t mask = (even ? 0x0000ffffu : 0u) | (odd ? 0xffff0000u : 0u);
              d[t][k] = as_half2(__byte_perm(a, b, 0x5410) & mask);
              d[t][k + 1] = as_half2(__byte_perm(a, b, 0x7632) & mask);
              m[t][k] = as_half2(c.x & mask);
              m[t][k + 1] = as_half2(c.y & mask);
              most = __hmax2(most, __hfma2(d[t][k], as_half2(0x4b804b80u), __habs2(m[t][k])));
              most = __hmax2(most, __hfma2(d[t][k + 1], as_half2(0x4b804b80u), __habs2(m[t][k + 1])));
            }
          }
#pragma unroll
          for (int k = 0; k < J; ++k) {
            uint32_t x[4][4];  // [t][n]
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              // (nibble n of the halves: the even row's and the odd row's)
              const uint32_t big = 0x64006400u, word = w[t * J + k], v = word >> 8;
              const __half2 less = as_half2(0xe400e400u), sixteenth = as_half2(0x2c002c00u), less64 = as_half2(0xd400d400u);
              x[t][0] = as_u32(__hfma2(__hadd2(as_half2(and_or(word, 0x000f000fu, big)), less), d[t][k], m[t][k]));
              x[t][1] = as_u32(__hfma2(__hfma2(as_half2(and_or(word, 0x00f000f0u, big)), sixteenth, less64), d[t][k], m[t][k]));
              x[t][2] = as_u32(__hfma2(__hadd2(as_half2(and_or(v, 0x000f000fu, big)), less), d[t][k], m[t][k]));
              x[t][3] = as_u32(__hfma2(__hfma2(as_half2(and_or(v, 0x00f000f0u, big)), sixteenth, less64), d[t][k], m[t][k]));
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int e = 32 * k + 8 * n + g;
              *reinterpret_cast<uint4*>(dst + (P * 2 + (o >> 3)) * S::kERows * 128 + e * 128 + (((o & 7) ^ g) << 4)) =
                  make_uint4(x[0][n], x[1][n], x[2][n], x[3][n]);
            }
          }
        }
        if (__hisinf(__low2half(most)) || __hisinf(__high2half(most))) v_again[par] = 1;
      } else {
        const int o = tid & 15, x = tid >> 4;  // rows 8 o .. + 7, values 8 (x + 8 c) .. + 7
        const T* src = static_cast<const T*>(p.v) + f.kv * p.v_head;
        auto load = [&](int c, uint4 (&w)[8]) {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            w[r] = 8 * o + r < f.nodes
                       ? *reinterpret_cast<const uint4*>(src + (int64_t)(f.r0 + 8 * o + r) * p.v_row + 8 * (x + 8 * c))
                       : make_uint4(0, 0, 0, 0);
        };
        uint32_t top = 0;
#pragma unroll 1
        for (int c = 0; c < HD / 64; ++c) {
          uint4 w[8];
          load(c, w);
#pragma unroll
          for (int r = 0; r < 8; ++r) top = max(top, top_bits<T>(w[r]));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) v_tops[warp & 3] = top;
        if (!team()) break;
        top = max(max(v_tops[0], v_tops[1]), max(v_tops[2], v_tops[3]));
        const float lift = lift_of(top);
#pragma unroll 1
        for (int c = 0; c < HD / 64; ++c) {
          uint4 w[8];
          load(c, w);
          const int e0 = 8 * (x + 8 * c);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            uint32_t y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float2 a = pair_of<T>((&w[2 * r].x)[k / 2]), b = pair_of<T>((&w[2 * r + 1].x)[k / 2]);
              y[r] = as_u32(__floats2half2_rn((k & 1 ? a.y : a.x) * lift, (k & 1 ? b.y : b.x) * lift));
            }
            const int e = e0 + k;
            *reinterpret_cast<uint4*>(dst + ((e >> 7) * 2 + (o >> 3)) * S::kERows * 128 + (e & 127) * 128 +
                                      (((o & 7) ^ (e & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
        if (!team()) break;  // v_tops is read
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&v_full[i % S::kVs]);
        mbar_arrive(&empty[st]);
      }
      if (++st == S::kStages) {
        st = 0;
        phase ^= 1;
      }
    }
  } else if (warp >= 8) {
    // ---------------- K: a row of keys per thread, into TMEM; and the tile's queries
    const int r = threadIdx.x - 8 * 32;
    Quartet team{&teams[2], nullptr, 0, p.err};
    int st = 0;
    uint32_t phase = 0;
    for (int i = 0;; ++i) {
      if (!wait(&full[st], phase)) break;
      const Info& f = infos[i % kInfos];
      const int flags = f.flags, par = f.count & 3;
      if (flags & kStop) {
        // (not before the products have seen the block two before, or they would miss its turn)
        if (i >= 2 && !wait(&s_full[i & 1], (uint32_t)((i - 2) >> 1) & 1u)) break;
        if (lane == 0) mbar_arrive(&k_full[i & 1]);
        break;
      }
      if (flags & kFirst) {
        // S of the segment before has read its queries
        if (i > 0 && !wait(&s_full[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1u)) break;
        if (r == 0) k_again[par] = 0;
        if (!team()) break;
        if (r < f.n) {
          const int c = f.c0 + r, head = f.kv * p.hpk + c % p.hpk;
          const T* src = static_cast<const T*>(p.q) + (int64_t)(f.r0 + c / p.hpk) * p.q_row + head * p.q_head;
          const bool some = r < f.cols;
          uint32_t top = 0;
          if (some)
#pragma unroll 8
            for (int x = 0; x < HD / 8; ++x) top = max(top, top_bits<T>(reinterpret_cast<const uint4*>(src)[x]));
          bool fine;
          const float s = to_one(top, fine);
          if (!fine) k_again[par] = 1;
#pragma unroll 4
          for (int x = 0; x < HD / 8; ++x) {
            uint32_t y[4] = {0, 0, 0, 0};
            if (some) scaled_pairs<T>(reinterpret_cast<const uint4*>(src)[x], s, y);
            const int j = x / 4, w = (j / J) * 4 * J + (x % 4) * J + j % J;  // its place among the words of a row of codes
            *reinterpret_cast<uint4*>(qs + (w / 8) * NT * 128 + sw128_off(r, w % 8)) = make_uint4(y[0], y[1], y[2], y[3]);
          }
          q_scale[par][r] = some ? p.scale / s : 0.f;
        }
        fence_proxy_async_smem();
      }
      // the place is free once S(i - 2) is done
      if (i >= 2 && !wait(&s_full[i & 1], (uint32_t)((i - 2) >> 1) & 1u)) break;
      tc_fence_after();
      const uint32_t dst = tmem + (i & 1) * S::kKCols + ((uint32_t)(32 * (warp & 3)) << 16);
      if (!(flags & kDraft)) {
        const int half = r >> 6, row = r & 63;
        const uint8_t* const page = ring + (size_t)st * S::kStage + half * S::kPage;
        uint32_t d[G / 2], m[G / 2];
#pragma unroll
        for (int k = 0; k < G / 2; ++k) {
          d[k] = *reinterpret_cast<const uint32_t*>(page + swizzled(32 * HD + 2 * (row * G + 2 * k)));
          m[k] = *reinterpret_cast<const uint32_t*>(page + swizzled(36 * HD + 2 * (row * G + 2 * k)));
        }
        __half2 most = as_half2(0u);
#pragma unroll
        for (int k = 0; k < G / 2; ++k) most = __hmax2(most, __hfma2(as_half2(d[k]), as_half2(0x4b804b80u), __habs2(as_half2(m[k]))));
        if (row < f.valid[half] && (__hisinf(__low2half(most)) || __hisinf(__high2half(most)))) k_again[par] = 1;
#pragma unroll
        for (int P = 0; P < PL; ++P)
#pragma unroll
          for (int q = 0; q < J; q += 2) {  // eight words, 32 columns
            uint32_t y[32];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint4 x = *reinterpret_cast<const uint4*>(page + swizzled(P * 1024 * J + row * 16 * J + 16 * (q + u)));
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int j = P * J + (4 * (q + u) + k) % J;
                const __half2 dd = j & 1 ? __high2half2(as_half2(d[j / 2])) : __low2half2(as_half2(d[j / 2]));
                const __half2 mm = j & 1 ? __high2half2(as_half2(m[j / 2])) : __low2half2(as_half2(m[j / 2]));
                uint32_t z[4];
                values_of((&x.x)[k], dd, mm, z);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[16 * u + 4 * k + e] = z[e];
              }
            }
            __syncwarp();
            tmem_st32(dst + P * 16 * J + q * 16, y);
          }
      } else {
        // drafted rows: to [1, 2) by a power of two each; what their V is lifted by; who sees whom
        const bool some = r < f.nodes;
        const T* src = static_cast<const T*>(p.k) + (int64_t)(f.r0 + r) * p.k_row + f.kv * p.k_head;
        const T* vsrc = static_cast<const T*>(p.v) + (int64_t)(f.r0 + r) * p.v_row + f.kv * p.v_head;
        uint32_t top = 0, vtop = 0;
        if (some)
#pragma unroll 4
          for (int x = 0; x < HD / 8; ++x) {
            top = max(top, top_bits<T>(reinterpret_cast<const uint4*>(src)[x]));
            vtop = max(vtop, top_bits<T>(reinterpret_cast<const uint4*>(vsrc)[x]));
          }
        bool fine;
        const float s = to_one(top, fine);
        if (!fine || vtop > kHalfMax) k_again[par] = 1;
        k_scale[par][r] = 1.f / s;
        vtop = __reduce_max_sync(0xffffffffu, vtop);
        if (lane == 0) k_tops[warp & 3] = vtop;
        uint4 bits = make_uint4(0, 0, 0, 0);
        int parent = -1;
        if (some) {
          (&bits.x)[r >> 5] = 1u << (r & 31);
          parent = p.parents ? p.parents[f.r0 + r] : r - 1;
          if (parent < -1 || parent >= r) {
            flag_position(p.err);
            parent = -1;
          }
        }
        seen[par][r] = bits;
        up[r] = parent;
        bool ok = team();
        if (r == 0) v_lift[par] = 1.f / lift_of(max(max(k_tops[0], k_tops[1]), max(k_tops[2], k_tops[3])));
        for (int n = 1; ok && n < f.nodes; n <<= 1) {  // ancestors up to 2 n rows above
          uint4 more = make_uint4(0, 0, 0, 0);
          int next = -1;
          if (parent >= 0) {
            more = seen[par][parent];
            next = up[parent];
          }
          ok = team();
          bits.x |= more.x;
          bits.y |= more.y;
          bits.z |= more.z;
          bits.w |= more.w;
          parent = next;
          seen[par][r] = bits;
          up[r] = parent;
          ok = ok && team();
        }
        if (!ok) break;
#pragma unroll
        for (int w0 = 0; w0 < HD / 8; w0 += 8) {  // eight words, 32 columns
          uint32_t y[32];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int w = w0 + k, P = w / (4 * J), t = w % (4 * J) / J, j = P * J + w % J;
            uint32_t z[4] = {0, 0, 0, 0};
            if (some) scaled_pairs<T>(reinterpret_cast<const uint4*>(src)[4 * j + t], s, z);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[4 * k + e] = z[e];
          }
          __syncwarp();
          tmem_st32(dst + 4 * w0, y);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k_full[i & 1]);
        mbar_arrive(&empty[st]);
      }
      if (++st == S::kStages) {
        st = 0;
        phase ^= 1;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    // ---------------- softmax: a KV row per thread, half of the columns
    const int h = warp >> 2, qd = warp & 3, r = threadIdx.x & 127;
    Quartet team{&teams[h], &votes[h][0][0], 0, p.err};
    const uint32_t sub = (uint32_t)(32 * qd) << 16;
    float l[kHalfCols];
    for (int i = 0;; ++i) {
      if (!wait(&s_full[i & 1], (uint32_t)(i >> 1) & 1u)) break;
      const Info& f = infos[i % kInfos];
      const int flags = f.flags;
      if (flags & kStop) break;
      tc_fence_after();
      const int par = f.count & 3, cols = f.n >> 1, x0 = h * cols;  // this half: columns x0 .. x0 + cols - 1 of the tile
      const bool first = flags & kFirst;
      if (first) {
        if (!team()) break;  // the segment before no longer reads its lines
        if (r < cols) line[x0 + r] = make_float2(q_scale[par][x0 + r], kBias);
#pragma unroll
        for (int x = 0; x < kHalfCols; ++x) l[x] = 0.f;
        if (!team()) break;
      }
      // the arguments of the weights' exponentials
      float a[kHalfCols];
      const uint32_t sc = tmem + S::kSCol + (i & 1) * NT + x0 + sub;
      __syncwarp();
#pragma unroll
      for (int x = 0; x < kHalfCols; x += 8)
        if (x < cols) tmem_ld8_async(sc + x, reinterpret_cast<uint32_t*>(a) + x);
      tmem_wait_ld();
      const bool here = (r & 63) < f.valid[r >> 6];
      float top = -INFINITY;
      if (flags & kDraft) {
        const float ks = k_scale[par][r];
        int token = (f.c0 + x0) / p.hpk, sub_head = (f.c0 + x0) % p.hpk;
        const uint32_t* bits = reinterpret_cast<const uint32_t*>(seen[par]) + qd;
#pragma unroll
        for (int x = 0; x < kHalfCols; ++x)
          if (x < cols) {
            const bool sees = x0 + x < f.cols && ((bits[4 * min(token, kMaxNodes - 1)] >> lane) & 1u);
            const float2 ln = line[x0 + x];
            a[x] = sees ? fmaf(a[x] * ks, ln.x, ln.y) : -INFINITY;
            top = fmaxf(top, a[x]);
            if (++sub_head == p.hpk) {
              sub_head = 0;
              ++token;
            }
          }
      } else {
#pragma unroll
        for (int x = 0; x < kHalfCols; x += 2)
          if (x < cols) {
            const float4 ln = *reinterpret_cast<const float4*>(&line[x0 + x]);
            a[x] = fmaf(a[x], ln.x, ln.y);
            a[x + 1] = fmaf(a[x + 1], ln.z, ln.w);
            top = fmaxf(top, fmaxf(a[x], a[x + 1]));
          }
        if (!__all_sync(0xffffffffu, here)) {
          top = here ? top : -INFINITY;
#pragma unroll
          for (int x = 0; x < kHalfCols; ++x) a[x] = here ? a[x] : -INFINITY;
        }
      }
      // a new maximum, where a weight would be larger than the lazy ones may be
      bool ok;
      const bool grown = team.any(first || top > kBias + kLazy, ok);
      if (!ok) break;
      if (grown) {
#pragma unroll
        for (int x = 0; x < kHalfCols; ++x)
          if (x < cols) {
            const float m = redux_max(a[x]);
            if (lane == 0) quad[h][qd][x] = m;
          }
        if (!team()) break;
        if (r < cols) {
          float m = fmaxf(fmaxf(quad[h][0][r], quad[h][1][r]), fmaxf(quad[h][2][r], quad[h][3][r])) - kBias;
          if (!first) m = fmaxf(m, 0.f);
          if (!(fabsf(m) < 1e37f)) m = 0.f;  // (no row, or a score that is not finite)
          change[h][r] = m;
          line[x0 + r].y -= m;
        }
        if (!team()) break;
        // (O of the blocks before is complete)
        if (!first && !wait(&p_empty[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1u)) break;
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < kHalfCols; ++x)
          if (x < cols) {
            a[x] -= change[h][x];
            if (!first) l[x] *= ex2(-change[h][x]);
          }
        if (!first) {
#pragma unroll 1
          for (int k = 0; k < S::kHalves; ++k)
#pragma unroll 1
            for (int x = 0; x < cols; x += 8) {
              const uint32_t oc = tmem + S::kOCol + k * NT + x0 + x + sub;
              uint32_t o[8];
              __syncwarp();
              tmem_ld8(oc, o);
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * ex2(-change[h][x + e]));
              tmem_st8(oc, o);
            }
          tmem_wait_st();
          tc_fence_before();
        }
        if (!team()) break;  // `change` and `quad` are read
      }
      // the weights, in P's place once PV(i - 2) is done
      if (i >= 2 && !wait(&p_empty[i & 1], (uint32_t)((i - 2) >> 1) & 1u)) break;
      uint8_t* const dst = ps + (i & 1) * S::kP;
      const float low = flags & kDraft ? v_lift[par] : 1.f;
#pragma unroll
      for (int x = 0; x < kHalfCols; x += 8)
        if (x < cols) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = ex2(a[x + 2 * e]), v = ex2(a[x + 2 * e + 1]);
            l[x + 2 * e] += u;
            l[x + 2 * e + 1] += v;
            w[e] = flags & kDraft ? as_u32(__floats2half2_rn(u * low, v * low)) : as_u32(__floats2half2_rn(u, v));
          }
          const int c = x0 + x;
          *reinterpret_cast<uint4*>(dst + (c >> 6) * (kRows * 128) + sw128_off(r, (c & 63) >> 3)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i & 1]);
      if (!(flags & kLast)) continue;

      // ---------------- the end of the segment, in this CTA
#pragma unroll
      for (int x = 0; x < kHalfCols; x += 32) {
        if (x >= cols) break;
        if constexpr (kHalfCols >= 32) {
          if (x + 32 <= kHalfCols) {
            float v[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = x + k < kHalfCols ? l[(x + k) % kHalfCols] : 0.f;
            quad[h][qd][x + lane] = transposed_sum(v);
          } else {
            float v[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) v[k] = l[(x + k) % kHalfCols];
            const float s = transposed_sum(v);
            if (lane < 16) quad[h][qd][x + lane] = s;
          }
        }
      }
      if (!wait(&p_empty[i & 1], (uint32_t)(i >> 1) & 1u)) break;
      tc_fence_after();
      if (!team()) break;
      const bool alone = flags & kAlone;
      if (r < cols) {
        const float s = (quad[h][0][r] + quad[h][1][r]) + (quad[h][2][r] + quad[h][3][r]);
        change[h][r] = alone ? 1.f / s : s;
        if (!alone) p.stats[(size_t)f.slot * NT + x0 + r] = make_float2(kBias - line[x0 + r].y, s);
      }
      if (!team()) break;
      if (threadIdx.x == 0) {
        const int again = k_again[par] | v_again[par];
        if (alone || (flags & kOpens)) p.runs[f.seg] = make_int4(f.first_cta, f.run, alone ? again : 0, 0);
        if (!alone) p.again[f.slot] = again;
      }
      if (qd * 32 < S::kERows) {
        const int used = min(cols, f.cols - x0);  // (columns past them are padding)
#pragma unroll 1
        for (int k = 0; k < S::kHalves; ++k) {
          const int e = 128 * k + 32 * qd + lane;
          int token = (f.c0 + x0) / p.hpk, sub_head = (f.c0 + x0) % p.hpk;
#pragma unroll 1
          for (int x = 0; x < used; x += 8) {
            uint32_t o[8];
            __syncwarp();
            tmem_ld8(tmem + S::kOCol + k * NT + x0 + x + sub, o);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              if (x + c >= used) break;
              if (alone)
                static_cast<T*>(p.out)[(f.r0 + token) * p.out_row + (int64_t)(f.kv * p.hpk + sub_head) * p.out_head + e] =
                    from_f32<T>(__uint_as_float(o[c]) * change[h][x + c]);
              else
                p.parts[((size_t)f.slot * NT + x0 + x + c) * HD + e] = __uint_as_float(o[c]);
              if (++sub_head == p.hpk) {
                sub_head = 0;
                ++token;
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    warp_wait(&fin, 0u, p.err);  // no product still runs when its TMEM is freed
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One row and KV head by four warps in 32-bit arithmetic, over the rows that it sees and no others; the
// query heads first .. end - 1 of the KV head's are written. Each warp takes every fourth row, lane l the
// values D l .. D l + D - 1 of a head.
template <int HD, typename T>
__device__ __noinline__ void plain_row(const TreeParams& p, int seq, int r0, int len, int row, int kv, int first, int end) {
  using B = Kv4Block<HD>;
  constexpr int D = HD / 32;
  __shared__ float joined[4][kMaxHpk][HD];
  __shared__ float tops[4][kMaxHpk], sums[4][kMaxHpk];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = D * lane;
  float q[kMaxHpk][D], o[kMaxHpk][D], m[kMaxHpk], l[kMaxHpk];
#pragma unroll
  for (int h = 0; h < kMaxHpk; ++h) {
    m[h] = kNone;
    l[h] = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) q[h][d] = o[h][d] = 0.f;
    if (h < p.hpk)
      load_vec<T, D>(static_cast<const T*>(p.q) + row * p.q_row + (int64_t)(kv * p.hpk + h) * p.q_head + e0, q[h]);
  }
  auto take = [&](const float (&k)[D], const float (&v)[D]) {
#pragma unroll
    for (int h = 0; h < kMaxHpk; ++h) {
      if (h >= p.hpk) break;
      float s = 0.f;
#pragma unroll
      for (int d = 0; d < D; ++d) s = fmaf(q[h][d], k[d], s);
      s = warp_sum(s) * p.scale;
      const float top = fmaxf(m[h], s), keep = ex2(m[h] - top), w = ex2(s - top);
      m[h] = top;
      l[h] = fmaf(l[h], keep, w);
#pragma unroll
      for (int d = 0; d < D; ++d) o[h][d] = fmaf(o[h][d], keep, w * v[d]);
    }
  };
  for (int at = warp; at < len; at += 4) {
    const int page = p.table[(int64_t)seq * p.table_stride + at / kPageRows], r = at % kPageRows;
    if (page < 0 || page >= p.n_pages) continue;
    const uint8_t* blk = p.pages + ((int64_t)page * p.nkv + kv) * B::kBytes;
    const uint8_t* vb = blk + B::kHalf;
    const int j = e0 / 32;
    const __half* ks = reinterpret_cast<const __half*>(blk + B::kCodes);
    const __half* vs = reinterpret_cast<const __half*>(vb + B::kCodes);
    const uint32_t word = reinterpret_cast<const uint32_t*>(blk)[B::k_word(r, j, e0 % 32 / 8)];
    const float kd = __half2float(ks[B::scale(r, j)]), km = __half2float(ks[HD * 2 + B::scale(r, j)]);
    const float vd = __half2float(vs[B::scale(r, j)]), vm = __half2float(vs[HD * 2 + B::v_min(r, j)]);
    float k[D], v[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int e = e0 + d;
      k[d] = fmaf((float)((word >> (4 * (e % 8))) & 15u), kd, km);
      const uint32_t c = reinterpret_cast<const uint16_t*>(vb)[B::v_half(r, j, e % 8)];
      v[d] = fmaf((float)((c >> (4 * (e % 32 / 8))) & 15u), vd, vm);
    }
    take(k, v);
  }
  // the row and its ancestors; a parent that does not lie before its child is none
  int node = row - r0;
  for (int step = 0; node >= 0; ++step) {
    if (step % 4 == warp) {
      float k[D], v[D];
      load_vec<T, D>(static_cast<const T*>(p.k) + (r0 + node) * p.k_row + kv * p.k_head + e0, k);
      load_vec<T, D>(static_cast<const T*>(p.v) + (r0 + node) * p.v_row + kv * p.v_head + e0, v);
      take(k, v);
    }
    const int above = p.parents ? p.parents[r0 + node] : node - 1;
    node = above < node ? above : -1;
  }
#pragma unroll
  for (int h = 0; h < kMaxHpk; ++h) {
    if (h >= p.hpk) break;
#pragma unroll
    for (int d = 0; d < D; ++d) joined[warp][h][e0 + d] = o[h][d];
    if (lane == 0) {
      tops[warp][h] = m[h];
      sums[warp][h] = l[h];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x + first * HD; i < end * HD; i += 128) {
    const int h = i / HD, e = i % HD;
    float top = kNone;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, tops[w][h]);
    float s = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float a = ex2(tops[w][h] - top);
      s = fmaf(a, sums[w][h], s);
      x = fmaf(a, joined[w][h][e], x);
    }
    static_cast<T*>(p.out)[row * p.out_row + (int64_t)(kv * p.hpk + h) * p.out_head + e] = from_f32<T>(x / s);
  }
  __syncthreads();
}

// Joins the parts of the tiles of one (sequence, KV head) in the order of the CTAs; a tile whose values f16
// does not hold is computed again in 32 bits.
template <int HD, int NT, typename T>
__global__ void __launch_bounds__(128) tree_join_kernel(const __grid_constant__ TreeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.x / p.nkv, kv = blockIdx.x % p.nkv;
  const Shape sh = shape_of<NT>(p, seq);
  for (int tile = 0; tile < sh.tiles; ++tile) {
    const int4 run = p.runs[(int64_t)blockIdx.x * p.most_tiles + tile];
    const int first_cta = run.x, n = run.y, c0 = tile * sh.per, cols = min(sh.per, sh.nodes * p.hpk - c0);
    if (n < 1 || first_cta < 0 || n > p.ctas - first_cta) continue;  // (nothing written where a wait gave up)
    bool again = run.z != 0;
    if (n > 1) {
      // the part that starts the segment is its CTA's slot 1, the others slot 0
      auto slot = [&](int i) { return (size_t)2 * (first_cta + i) + (i == 0 ? 1 : 0); };
      for (int i = 0; i < n; ++i) again |= p.again[slot(i)] != 0;
      if (!again)
        for (int x = blockIdx.y * 128 + threadIdx.x; x < cols * HD / 4; x += 128 * gridDim.y) {
          const int c = x / (HD / 4), e = 4 * (x % (HD / 4));
          float top = kNone, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
          for (int i = 0; i < n; ++i) top = fmaxf(top, __ldcg(&p.stats[slot(i) * NT + c]).x);
          for (int i = 0; i < n; ++i) {
            const float2 st = __ldcg(&p.stats[slot(i) * NT + c]);
            const float4 o = __ldcg(reinterpret_cast<const float4*>(p.parts + (slot(i) * NT + c) * HD + e));
            const float w = ex2(st.x - top);
            sum = fmaf(w, st.y, sum);
            v[0] = fmaf(w, o.x, v[0]);
            v[1] = fmaf(w, o.y, v[1]);
            v[2] = fmaf(w, o.z, v[2]);
            v[3] = fmaf(w, o.w, v[3]);
          }
          const float inv = 1.f / sum;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= inv;
          store_vec<T, 4>(static_cast<T*>(p.out) + (sh.r0 + (c0 + c) / p.hpk) * p.out_row +
                              (int64_t)(kv * p.hpk + (c0 + c) % p.hpk) * p.out_head + e, v);
        }
    }
    if (again)
      for (int token = c0 / p.hpk + blockIdx.y; token * p.hpk < c0 + cols; token += gridDim.y)
        plain_row<HD, T>(p, seq, sh.r0, sh.len, sh.r0 + token, kv, max(0, c0 - token * p.hpk), min(p.hpk, c0 + cols - token * p.hpk));
  }
}

template <int HD, int NT, typename T>
cudaError_t launch(const LaunchEnv& env, TreeParams p) {
  using S = Sizes<HD, NT>;
  CUtensorMap map{};
  if (p.n_pages > 0 && !encode_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.pages, 128, (uint64_t)p.n_pages * p.nkv * (S::kPage / 128),
                                  128, 128, S::kPage / 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  auto kern = tree_kernel<HD, NT, T>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  p.ctas = env.sm_count;
  p.most_tiles = (kMaxNodes * p.hpk + NT - 1) / NT;
  e = rrr_launch_pdl(kern, dim3(env.sm_count), dim3(kThreads), (size_t)S::kSmem, env.stream, env.pdl, map, p);
  if (e != cudaSuccess) return e;
  // few heads: their columns are shared by several CTAs
  const int64_t heads = (int64_t)p.n_seqs * p.nkv;
  int64_t across = (4 * (int64_t)env.sm_count + heads - 1) / heads;
  if (across > 64) across = 64;
  return rrr_launch_pdl(tree_join_kernel<HD, NT, T>, dim3((unsigned)heads, (unsigned)across), dim3(128), 0, env.stream, env.pdl, p);
}
template <int HD>
cudaError_t launch_type(const LaunchEnv& env, int type, const TreeParams& p) {
  if constexpr (HD < 256)
    if ((int64_t)p.rows * p.hpk > 64 * (int64_t)p.n_seqs)
      return type == RRR_F16 ? launch<HD, 96, __half>(env, p) : launch<HD, 96, __nv_bfloat16>(env, p);
  return type == RRR_F16 ? launch<HD, 64, __half>(env, p) : launch<HD, 64, __nv_bfloat16>(env, p);
}

// The workspace: runs, statistics, flags, parts; for the widest tiles
struct Layout {
  int64_t stats, again, parts, bytes;
};
Layout layout_of(const rrr_kv4_cache* c, int n_heads, int sms) {
  const int64_t hpk = n_heads / c->n_kv_heads, tiles = (kMaxNodes * hpk + 63) / 64, slots = 2 * (int64_t)sms;
  Layout l;
  l.stats = ((int64_t)c->n_seqs * c->n_kv_heads * tiles * 16 + 255) / 256 * 256;
  l.again = l.stats + slots * 96 * 8;
  l.parts = l.again + (slots * 4 + 255) / 256 * 256;
  l.bytes = l.parts + slots * 96 * c->head_dim * 4;
  return l;
}

int check_tree(rrr_ctx* ctx, const rrr_kv4_cache* c, int n_heads, int rows, const char* fn) {
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  const int rc = check_kv4_cache(ctx, c, fn);
  if (rc) return rc;
  if (n_heads < 1 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > kMaxHpk)
    return set_error(ctx, RRR_ERR_BAD_SHAPE,
                     "%s: n_heads must be a multiple of n_kv_heads, at most 8 query heads per KV head", fn);
  if (rows < 0 || rows > 1 << 24) return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: need 0 <= rows <= 2^24", fn);
  // (a page is addressed by its line of 128 bytes, and one launch has 2^31 CTAs)
  if (c->n_pages * c->n_kv_heads > INT32_MAX / (80 * c->head_dim / 128) || (int64_t)c->n_seqs * c->n_kv_heads > INT32_MAX / 16)
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: at most 2^38 bytes of pages and 2^27 sequences times heads", fn);
  return RRR_OK;
}

}  // namespace
}  // namespace rrr

using namespace rrr;

extern "C" {

int rrr_tree_workspace(rrr_ctx* ctx, const rrr_kv4_cache* c, int n_heads, int rows, int64_t* bytes) {
  const char* fn = "rrr_tree_workspace";
  const int rc = check_tree(ctx, c, n_heads, rows, fn);
  if (rc) return rc;
  if (!bytes) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  (void)rows;
  *bytes = layout_of(c, n_heads, ctx->sm_count).bytes;
  return RRR_OK;
}

int rrr_attention_tree_kv4(rrr_ctx* ctx, const rrr_kv4_cache* c, const rrr_tree_desc* d, const void* q, const void* k,
                           const void* v, const int32_t* cu_rows, const int32_t* parents, const int32_t* kv_lens,
                           void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "rrr_attention_tree_kv4";
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  if (!d) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null descriptor", fn);
  int64_t need = 0;
  int rc = rrr_tree_workspace(ctx, c, d->n_heads, d->rows, &need);
  if (rc) return rc;
  if (d->type != RRR_F16 && d->type != RRR_BF16)
    return set_error(ctx, RRR_ERR_BAD_QTYPE, "%s: type must be 1 (F16) or 30 (BF16)", fn);
  if (!workspace || (d->rows > 0 && (!q || !k || !v || !out)) || (c->n_seqs > 0 && (!cu_rows || !kv_lens)))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int hd = c->head_dim, nkv = c->n_kv_heads, nh = d->n_heads;
  const int64_t strides[8] = {d->q_row, d->q_head, d->k_row, d->k_head, d->v_row, d->v_head, d->out_row, d->out_head};
  for (int64_t s : strides) {
    if (s < hd || s > ((int64_t)1 << 38)) return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: a stride is shorter than a head, or over 2^38", fn);
    if (s % 8) return set_error(ctx, RRR_ERR_MISALIGNED, "%s: strides must be multiples of 8 elements", fn);
  }
  if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(out, 16))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: q, k, v and out must be 16-byte aligned", fn);
  if (!(d->scale >= 0.f) || d->scale > 3.4e38f)
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: scale must be finite, not negative", fn);
  if (!aligned_to(cu_rows, 4) || !aligned_to(parents, 4) || !aligned_to(kv_lens, 4) || !aligned_to(workspace, 16))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: the workspace must be 16-byte aligned", fn);
  if (workspace_bytes < need)
    return set_error(ctx, RRR_ERR_BUFFER_TOO_SMALL, "%s: the workspace needs %lld bytes", fn, (long long)need);
  const int64_t page_bytes = c->n_pages * nkv * 80 * hd;
  // out: rows of heads or heads of rows, without two elements in one place, apart from all else
  if (!(d->out_row >= (int64_t)(nh - 1) * d->out_head + hd || d->out_head >= (int64_t)(d->rows - 1) * d->out_row + hd))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows and heads of out overlap", fn);
  const HeadRows mine{out, d->rows, d->out_row, nh, d->out_head, hd};
  const HeadRows ws{workspace, 1, hd, 1, hd, need / 2}, pages{c->pages, page_bytes ? 1 : 0, hd, 1, hd, page_bytes / 2};
  bool fine = apart(mine, ws) && apart(mine, pages) && apart(ws, pages);
  for (const HeadRows& in : {HeadRows{q, d->rows, d->q_row, nh, d->q_head, hd}, HeadRows{k, d->rows, d->k_row, nkv, d->k_head, hd},
                             HeadRows{v, d->rows, d->v_row, nkv, d->v_head, hd}})
    fine = fine && apart(mine, in) && apart(ws, in);
  if (!fine) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: out and the workspace must overlap nothing", fn);
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  if (d->rows == 0 || c->n_seqs == 0) return RRR_OK;
  const LaunchEnv env = make_env(ctx, stream);
  TreeParams p{};
  p.pages = static_cast<const uint8_t*>(c->pages);
  p.n_pages = c->n_pages;
  p.table_stride = c->table_stride;
  p.table = c->page_table;
  p.n_seqs = c->n_seqs;
  p.max_pages = c->max_pages;
  p.nh = nh;
  p.nkv = nkv;
  p.hpk = nh / nkv;
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.q_row = d->q_row;
  p.q_head = d->q_head;
  p.k_row = d->k_row;
  p.k_head = d->k_head;
  p.v_row = d->v_row;
  p.v_head = d->v_head;
  p.out_row = d->out_row;
  p.out_head = d->out_head;
  p.cu = cu_rows;
  p.parents = parents;
  p.lens = kv_lens;
  p.rows = d->rows;
  p.scale = (d->scale == 0.f ? 1.f / sqrtf((float)hd) : d->scale) * 1.4426950408889634f;
  p.err = env.d_err;
  const Layout l = layout_of(c, nh, ctx->sm_count);
  char* w = static_cast<char*>(workspace);
  p.runs = reinterpret_cast<int4*>(w);
  p.stats = reinterpret_cast<float2*>(w + l.stats);
  p.again = reinterpret_cast<int*>(w + l.again);
  p.parts = reinterpret_cast<float*>(w + l.parts);
  cudaError_t e;
  switch (hd) {
    case 64: e = launch_type<64>(env, d->type, p); break;
    case 128: e = launch_type<128>(env, d->type, p); break;
    default: e = launch_type<256>(env, d->type, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_attention_tree_kv4 launch");
}

}  // extern "C"
