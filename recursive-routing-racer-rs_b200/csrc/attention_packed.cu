// attention_packed.cu — attention of packed prompts with grouped heads (rrr_attention_packed):
// the prefill form of the `attention` dispatch (src/model/phi4.rs:1284-1309, 1680-1688) for
// several sequences at once.
//
// Mathematics. One pass over a sequence's KV rows per tile of query rows with the running
// maximum m and sum l of the softmax in base 2: s = q . k * scale * log2(e), p = 2^(s - m), O <-
// O 2^(m_old - m) + p V, out = O / l. Products on the tensor cores in the inputs' type with
// 32-bit accumulators; p is rounded to that type for the second product (its rounding, half a
// step per weight, averages over the row and is of the size of the output's own).
//
// Where a tile begins. Tile x of the grid belongs to the last sequence s with floor(cu[s] /
// rows) + s <= x and starts at its row cu[s] + rows * (x - floor(cu[s] / rows) - s): sequences
// get disjoint runs of x that are long enough; a warp searches 32 sequences at a time.
//
// Which kernel. packed_tc_kernel: head_dim 64 and 128, two tiles of 128 (row, head) pairs per CTA.
// packed_wide_kernel: head_dim 256, one tile. Both share the KV rows of an item among the CTAs of a
// cluster where there are few items. packed_kernel (mma.sync): what neither can describe.
#include <math.h>

#include "serve_common.cuh"
#include "tile_common.cuh"

namespace rrr {
namespace {

constexpr int kQRows = 64, kKRows = 64, kThreads = 128;

struct PackedParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;
  const int* cu_q;
  const int* cu_kv;
  int n_seqs, nh, hpk, causal;
  int64_t q_rows, kv_rows;
  float scale;  // with log2(e)
  int* err;
};

// The sequence and rows of query tile x; false when the tile is empty.
struct Tile {
  int seq, q0, q1, row0;  // the sequence's query rows [q0, q1), the tile's first
  int k0, k1;             // its KV rows
};
__device__ __forceinline__ bool find_tile(const PackedParams& p, int rows, int x, Tile& t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.n_seqs;  // the last s with cu[s] / rows + s <= x lies in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, s < hi && p.cu_q[s] / rows + s <= x);
    lo += below ? (31 - __clz(below)) * step : 0;
    hi = min(hi, lo + step);
  }
  t.seq = lo;
  t.q0 = p.cu_q[lo];
  t.q1 = p.cu_q[lo + 1];
  t.k0 = p.cu_kv[lo];
  t.k1 = p.cu_kv[lo + 1];
  if (t.q0 < 0 || t.q1 < t.q0 || t.q1 > p.q_rows || t.k0 < 0 || t.k1 < t.k0 || t.k1 > p.kv_rows) {
    if ((threadIdx.x & 31) == 0) flag_position(p.err);
    return false;
  }
  const int64_t row0 = t.q0 + (int64_t)rows * (x - (t.q0 / rows + lo));
  if (row0 < t.q0 || row0 >= t.q1) return false;
  t.row0 = (int)row0;
  return true;
}
// KV rows of the sequence that query row `row` sees.
__device__ __forceinline__ int seen_by(const PackedParams& p, const Tile& t, int row) {
  const int lk = t.k1 - t.k0;
  return p.causal ? max(0, min(lk, row - t.q0 + 1 + lk - (t.q1 - t.q0))) : lk;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
struct Mma;
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p)));
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_addr(p)));
}

// Whether a row that came out not finite may owe that to what it does not see: a masked weight of
// zero times an infinite or NaN value is a NaN in a tile's product. Where the weights' sum is not
// a positive number the row's own scores made it so.
__device__ __forceinline__ bool doubtful(bool bad, float sum) { return bad && sum > 0.f && sum <= 3.402823466e38f; }
// One such query row by one warp: where the values that its tile took in beyond what it sees, up
// to row `reach` of the sequence, are finite, it stands; else it is computed again in 32-bit
// arithmetic over the rows that it sees and no others, so that the others never reach it.
template <int HD, typename T>
__device__ __noinline__ void slow_row(const PackedParams& p, const Tile& t, int row, int head, int reach) {
  constexpr int D = HD / 32, U = 4;  // rows at once
  const int lane = threadIdx.x & 31, kv = head / p.hpk, n = seen_by(p, t, row);
  const T* kp = static_cast<const T*>(p.k) + t.k0 * p.k_row + kv * p.k_head + D * lane;
  const T* vp = static_cast<const T*>(p.v) + t.k0 * p.v_row + kv * p.v_head + D * lane;
  bool finite = true;
  for (int j = n; j < reach; ++j) {
    float x[D];
    load_vec<T, D>(vp + j * p.v_row, x);
#pragma unroll
    for (int i = 0; i < D; ++i) finite &= fabsf(x[i]) <= 3.402823466e38f;
  }
  if (__all_sync(0xffffffffu, finite)) return;
  float q[D], o[D], m = -INFINITY, l = 0.f;
  load_vec<T, D>(static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head + D * lane, q);
#pragma unroll
  for (int i = 0; i < D; ++i) o[i] = 0.f;
  for (int j = 0; j < n; j += U) {
    float x[U][D], s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      load_vec<T, D>(kp + min(j + u, n - 1) * p.k_row, x[u]);
      s[u] = 0.f;
#pragma unroll
      for (int i = 0; i < D; ++i) s[u] = fmaf(q[i], x[u][i], s[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<T, D>(vp + min(j + u, n - 1) * p.v_row, x[u]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], k);
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = j + u < n ? s[u] * p.scale : -INFINITY;
      mn = fmaxf(mn, s[u]);
    }
    const float mu = mn == -INFINITY ? 0.f : mn, alpha = ex2(m - mu);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < D; ++i) o[i] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (j + u >= n) break;
      const float w = ex2(s[u] - mu);
      l += w;
#pragma unroll
      for (int i = 0; i < D; ++i) o[i] = fmaf(w, x[u][i], o[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < D; ++i) o[i] = n > 0 ? o[i] / l : 0.f;
  store_vec<T, D>(static_cast<T*>(p.out) + row * p.out_row + head * p.out_head + D * lane, o);
}

// 64 query rows of one head per CTA, 16 per warp, against 64 KV rows at a time in shared memory:
// for more than 128 query heads per KV head, whose rows fit no tile of the kernels below, and for
// batches without any KV row, which no tensor map describes.
template <int HD, typename T>
__global__ void __launch_bounds__(kThreads) packed_kernel(const __grid_constant__ PackedParams p) {
  constexpr int PITCH = HD + 8;  // rows 16 bytes apart in the banks: conflict-free ldmatrix
  constexpr int CH = HD / 8;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  T* qs = reinterpret_cast<T*>(smem_raw);
  T* ks = qs + kQRows * PITCH;
  T* vs = ks + kKRows * PITCH;
  pdl_launch_dependents();
  pdl_wait();
  Tile t;
  if (!find_tile(p, kQRows, (int)(gridDim.x - 1 - blockIdx.x), t)) return;
  const int head = blockIdx.y, kv = head / p.hpk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int rows = min(kQRows, t.q1 - t.row0);
  for (int i = threadIdx.x; i < kQRows * CH; i += kThreads) {
    const int r = i / CH, cc = i % CH;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < rows)
      w = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (t.row0 + r) * p.q_row + head * p.q_head + 8 * cc);
    *reinterpret_cast<uint4*>(qs + r * PITCH + 8 * cc) = w;
  }
  const int end = seen_by(p, t, t.row0 + rows - 1);  // KV rows that the tile's last row sees
  const int lk = t.k1 - t.k0;
  int seen[2];  // of this lane's rows g, g + 8 of the warp
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = t.row0 + 16 * warp + 8 * i + g;
    seen[i] = r < t.row0 + rows ? seen_by(p, t, r) : 0;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[HD / 8][4];
#pragma unroll
  for (int n = 0; n < HD / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
  for (int j0 = 0; j0 < end; j0 += kKRows) {
    __syncthreads();
    for (int i = threadIdx.x; i < kKRows * CH; i += kThreads) {
      const int r = i / CH, cc = i % CH;
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (j0 + r < lk) {
        const int64_t at = t.k0 + j0 + r;
        a = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.k) + at * p.k_row + kv * p.k_head + 8 * cc);
        b = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.v) + at * p.v_row + kv * p.v_head + 8 * cc);
      }
      *reinterpret_cast<uint4*>(ks + r * PITCH + 8 * cc) = a;
      *reinterpret_cast<uint4*>(vs + r * PITCH + 8 * cc) = b;
    }
    __syncthreads();
    float s[kKRows / 8][4];
#pragma unroll
    for (int n = 0; n < kKRows / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll 4
    for (int kk = 0; kk < HD / 16; ++kk) {
      uint32_t a[4];
      ldmatrix4(a, qs + (16 * warp + (lane & 15)) * PITCH + 16 * kk + 8 * (lane >> 4));
#pragma unroll
      for (int n = 0; n < kKRows / 8; n += 2) {
        uint32_t b[4];
        ldmatrix4(b, ks + (8 * n + 8 * (lane >> 4) + (lane & 7)) * PITCH + 16 * kk + 8 * ((lane >> 3) & 1));
        Mma<T>::run(s[n], a, b[0], b[1]);
        Mma<T>::run(s[n + 1], a, b[2], b[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < kKRows / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[n][2 * i + e];
          x = j0 + 8 * n + 2 * c + e < seen[i] ? x * p.scale : -INFINITY;
          top = fmaxf(top, x);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float mn = fmaxf(m[i], top), mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = ex2(m[i] - mu);
      m[i] = mn;
      l[i] *= alpha;
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        o[n][2 * i] *= alpha;
        o[n][2 * i + 1] *= alpha;
      }
#pragma unroll
      for (int n = 0; n < kKRows / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[n][2 * i + e] = ex2(s[n][2 * i + e] - mu);
          l[i] += s[n][2 * i + e];
        }
    }
#pragma unroll
    for (int kk = 0; kk < kKRows / 16; ++kk) {
      const uint32_t a[4] = {Mma<T>::pack(s[2 * kk][0], s[2 * kk][1]), Mma<T>::pack(s[2 * kk][2], s[2 * kk][3]),
                             Mma<T>::pack(s[2 * kk + 1][0], s[2 * kk + 1][1]),
                             Mma<T>::pack(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
      for (int n = 0; n < HD / 8; n += 2) {
        uint32_t b[4];
        ldmatrix4_t(b, vs + (16 * kk + (lane & 15)) * PITCH + 8 * n + 8 * (lane >> 4));
        Mma<T>::run(o[n], a, b[0], b[1]);
        Mma<T>::run(o[n + 1], a, b[2], b[3]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int r = 16 * warp + 8 * i + g;
    const float inv = seen[i] > 0 ? 1.f / l[i] : 0.f;
    bool bad = false;
    T* dst = static_cast<T*>(p.out) + (t.row0 + r) * p.out_row + head * p.out_head;
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      const float a = o[n][2 * i] * inv, b = o[n][2 * i + 1] * inv;
      bad |= !(fabsf(a) <= 3.402823466e38f) || !(fabsf(b) <= 3.402823466e38f);
      if (r < rows) *reinterpret_cast<uint32_t*>(dst + 8 * n + 2 * c) = Mma<T>::pack(a, b);
    }
    unsigned rows_bad = __ballot_sync(0xffffffffu, doubtful(bad, l[i]) && r < rows);
    for (int rr = 0; rr < 8; ++rr)
      if (rows_bad & (0xfu << (4 * rr))) {
        __syncwarp();
        slow_row<HD, T>(p, t, t.row0 + 16 * warp + 8 * i + rr, head, min(lk, (end + kKRows - 1) / kKRows * kKRows));
      }
  }
}

// ---- head_dim 64 and 128: tcgen05 ---------------------------------------------------------
//
// A CTA takes two tiles of 128 (query row, head) pairs that share a KV head, heads innermost:
// floor(128 / hpk) rows of hpk heads each, one TMA box; so grouped heads fill the tensor
// core's 128 rows whatever their number, and the rows of a tile end near the same KV row.
// Warps 0-3 and 4-7 are the tiles' softmax (one thread per tile row), warp 8 issues the MMAs,
// warp 9 the copies. Per 128 KV rows and tile: S = Q K^T (128 x 128 f32 in TMEM); a thread
// reads its row of S, takes its maximum, writes p in 16 bits over S, packed two a column, as
// the A operand of O += P V, whose accumulator stays in TMEM. The MMA thread alternates the
// tiles (P0 V, next S0, P1 V, next S1), so that one tile's products run during the other's
// softmax. O is rescaled only when a row's maximum has grown by over 2^kLazy since its last
// rescale: until then the weights are at most 2^kLazy, which neither 16-bit type rounds worse
// than values up to one.
// V rows behind the sequence are zeroed in shared memory before their product: other
// sequences' values, or none, may be anything.
//
// Measured (head_dim 128): a prompt of 16,384 rows of 24 heads 1575 us in a row of calls, at the power
// limit (1.05 PFLOP/s), and 1340 once at full clocks, two tiles' block in some 3600 clocks, of which the products need
// 2100 and the exponentials (16 a clock) 2050; short items pay 4 to 5 us for a CTA's start and end.
// Tried without gain: exponentials by a polynomial, weights handed over by halves, two threads per
// row, persistent CTAs with the longest items first.
constexpr int kTcThreads = 384;  // warps 10 and 11 only complete the third warpgroup
constexpr int kTile = 128;   // MMA rows, and KV rows per block
constexpr float kLazy = 8.f;

// Stages of the ring of K and V tiles beside the two of Q: what fits. (Two stages of K and two of
// V, freed apart, took 1756 us instead of 1720 for a prompt of 16,384 rows.)
template <int HD>
constexpr int tc_stages() { return HD == 128 ? 5 : 10; }

struct TcParams {
  PackedParams a;
  int tokens;  // query rows per tile
  int splits;  // CTAs of a cluster, each with a part of the KV rows (1, 2, 4 or 8)
  uint32_t idesc_s, idesc_o;
};

// One lane of a converged warp. (Under this predicate the compiler keeps descriptors in uniform
// registers: 64 products of 128 x 128 x 16 took 8 x 577 clocks against 8 x 676 issued by a
// branch on the lane number, 8 x 512 being the tensor core's own time.)
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  umma_bf16(d_tmem, a_desc, b_desc, idesc, accumulate);  // kind::f16: the types are in idesc
}
// The same with A in TMEM: 128 lanes, two 16-bit elements of K per 32-bit column
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Descriptor of an operand whose rows (K) of 64 elements lie 128 bytes apart, 128-byte swizzled
// (N contiguous): 8 rows every 1024 bytes (stride offset), the next 64 elements of N after
// `lead` bytes (leading offset).
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr, uint32_t lead) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(bar))
      : "memory");
}
// 32 columns of this thread's TMEM lane, without the wait
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
// Brings a tensor map on its way before the first copy wants it (a prompt of 77 rows 8.03 -> 7.89 us)
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
// 32 bytes of a row of out: every lane writes another row, so a store costs what it has of rows
__device__ __forceinline__ void store_32(void* p, const uint32_t (&a)[4], const uint32_t (&b)[4], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a[0]), "r"(a[1]), "r"(a[2]),
                 "r"(a[3]), "r"(b[0]), "r"(b[1]), "r"(b[2]), "r"(b[3])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(a[0], a[1], a[2], a[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(b[0], b[1], b[2], b[3]);
  }
}

// The softmax of one tile row, by one thread.
template <typename T>
struct RowSoftmax {
  float scale;
  bool mine;  // whether it is a query row of the tile's sequence: the others, of the next sequence or
              // of none, hold anything and have no vote (nor are their weights anyone's concern)
  float m;   // the maximum of the scaled scores, as of the last rescale
  float2 l;  // the weights' sum, of even and odd columns
  // the weights of 32 scores under the maximum m, stored over S as columns 32 part .. + 31; their
  // sum to l
  __device__ __forceinline__ void weights(uint32_t sc, const float* v, int part) {
    const float neg = m == -INFINITY ? 0.f : -m;
    const float2 neg2 = make_float2(neg, neg), scale2 = make_float2(scale, scale);
    float2 sum = make_float2(0.f, 0.f);
    uint32_t w[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const float2 e = __ffma2_rn(make_float2(v[2 * c], v[2 * c + 1]), scale2, neg2);
      const float2 q = make_float2(ex2(e.x), ex2(e.y));
      sum = __fadd2_rn(sum, q);
      w[c] = Mma<T>::pack(q.x, q.y);
    }
    l = __fadd2_rn(l, sum);
    tmem_st16(sc + 16 * part, w);
  }
  static __device__ __forceinline__ float top_of(const float* v) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
      top[0] = fmaxf(top[0], fmaxf(v[c], v[c + 1]));
      top[1] = fmaxf(top[1], fmaxf(v[c + 2], v[c + 3]));
    }
    return fmaxf(top[0], top[1]);
  }
  // takes over a larger maximum where a row's has grown by more than kLazy; whether any has.
  // scale_o(alpha) does that to the products so far.
  template <class F>
  __device__ __forceinline__ bool rescale(float m_new, F&& scale_o) {
    if (!__any_sync(0xffffffffu, mine && m_new > m + kLazy)) return false;
    const bool grow = mine && m_new > m;
    const float next = grow ? m_new : m;
    const float alpha = grow ? ex2(m - next) : 1.f;
    m = next;
    l.x *= alpha;
    l.y *= alpha;
    scale_o(alpha);
    return true;
  }
  // Block j: the scores in sc become weights. open: columns that this row sees; every row of the
  // warp sees all_see of them, none of its rows none_sees or more.
  template <class F>
  __device__ __forceinline__ void block(uint32_t sc, int j, int open, int all_see, int none_sees, F&& scale_o) {
    if (j > 0 && (j + 1) * kTile <= all_see) {
      // the weights under the old maximum; the new one is found meanwhile, and where it is too
      // large for the old one they are computed again
      uint32_t x[kTile];
      const float* v = reinterpret_cast<const float*>(x);
      tmem_ld32(sc, x);
      tmem_wait_ld();
      const float2 before = l;
      float top = -INFINITY;
#pragma unroll
      for (int part = 0; part < 4; ++part) {
        if (part < 3) tmem_ld32(sc + 32 * (part + 1), x + 32 * (part + 1));
        weights(sc, v + 32 * part, part);
        top = fmaxf(top, top_of(v + 32 * part));
        if (part < 3) tmem_wait_ld();
      }
      const float2 after = l;
      l = before;
      if (rescale(top * scale, scale_o)) {
#pragma unroll
        for (int part = 0; part < 4; ++part) weights(sc, v + 32 * part, part);
      } else {
        l = after;
      }
    } else {
      // the first block, or one with masked columns: the maximum first. A part of 32 columns
      // that no row of the warp sees has no weights, one that every row sees no mask.
      auto load = [&](int part, uint32_t* x) {
        const int at = j * kTile + 32 * part;
        tmem_ld32(sc + 32 * part, x);
        tmem_wait_ld();
        if (at + 32 > all_see) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (c >= open - at) x[c] = 0xff800000u;
        }
      };
      const int parts = min(4, (none_sees - j * kTile + 31) / 32);
      float m_new = -INFINITY;
#pragma unroll 1
      for (int part = 0; part < parts; ++part) {
        uint32_t x[32];
        load(part, x);
        m_new = fmaxf(m_new, top_of(reinterpret_cast<const float*>(x)));
      }
      rescale(m_new * scale, scale_o);
#pragma unroll 1
      for (int part = 0; part < 4; ++part) {
        uint32_t x[32];
        if (part < parts) {
          load(part, x);
          weights(sc, reinterpret_cast<const float*>(x), part);
        } else {
          const uint32_t zero[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
          tmem_st16(sc + 16 * part, zero);
        }
      }
    }
  }
};
// HD columns of this thread's row of O times alpha
template <int HD>
__device__ __forceinline__ void scale_row(uint32_t oc, float alpha) {
#pragma unroll 1
  for (int c = 0; c < HD; c += 16) {
    uint32_t v[16];
    tmem_ld16(oc + c, v);
    tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * alpha);
    tmem_st16(oc + c, v);
  }
}
// This thread's row of out from O (`some`: whether there are products) over the weights' sum;
// rows of the warp that need it are computed again.
template <int HD, typename T>
__device__ __forceinline__ void write_row(const PackedParams& p, const Tile& t, uint32_t oc, bool some, bool mine,
                                          int row, int head, int seen, float sum, int reach) {
  const float inv = seen > 0 ? 1.f / sum : 0.f;
  T* dst = static_cast<T*>(p.out) + row * p.out_row + (int64_t)head * p.out_head;
  bool bad = false;
  const bool wide = (reinterpret_cast<uintptr_t>(p.out) & 31) == 0 && p.out_row % 16 == 0 && p.out_head % 16 == 0;
  for (int c = 0; c < HD; c += 32) {
    uint32_t v[32];
    if (some) {
      tmem_ld32(oc + c, v);
      tmem_wait_ld();
    }
    uint32_t pair[4];
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = seen > 0 ? __uint_as_float(v[k + 2 * e]) * inv : 0.f;
        const float b = seen > 0 ? __uint_as_float(v[k + 2 * e + 1]) * inv : 0.f;
        bad |= !(fabsf(a) <= 3.402823466e38f) || !(fabsf(b) <= 3.402823466e38f);
        o[e] = Mma<T>::pack(a, b);
      }
      if (k % 16 == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) pair[e] = o[e];
      } else if (mine) {
        store_32(dst + c + k - 8, pair, o, wide);
      }
    }
  }
  unsigned again = __ballot_sync(0xffffffffu, doubtful(bad, sum) && mine);
  while (again) {
    const int from = __ffs(again) - 1;
    again &= again - 1;
    __syncwarp();
    slow_row<HD, T>(p, t, __shfl_sync(0xffffffffu, row, from), __shfl_sync(0xffffffffu, head, from), reach);
  }
}

// Where the tiles are too few for the SMs, a cluster of CTAs takes one item, each CTA an equal part
// of its blocks of KV rows, as if the sequence's rows began and ended there. Then every CTA sends
// its rows' maxima and sums to all, and of O's columns each CTA's share to it, over the cluster's
// shared memory; a CTA adds up its columns in the order of the parts and writes them.
__device__ __forceinline__ uint32_t in_cta(const void* local, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(local)), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void send2(uint32_t at, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(a), "f"(b) : "memory");
}
__device__ __forceinline__ void send4(uint32_t at, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

// The end of an item that a cluster shares, for one tile row (of ROWS in the CTA): m_own, l_own and
// the row of O at oc are of this CTA's part (`some`: whether it has products). All threads of the
// cluster pass three barriers.
template <int HD, typename T, int ROWS>
__device__ __forceinline__ void join_rows(const PackedParams& p, const Tile& t, uint8_t* qs, uint8_t* ring, int splits,
                                          int rank, int at, bool some, bool mine, int row, int head, int all_seen,
                                          float m_own, float l_own, uint32_t oc, int reach) {
  // in every CTA, once the products of all are done: maxima and sums [part][row] and, of the first,
  // what came out not finite [part][row] in Q's place; [part][4 columns][row] in the ring's
  const int width = HD / splits;
  float2* stats = reinterpret_cast<float2*>(qs);
  int* bad_rows = reinterpret_cast<int*>(qs + 8 * ROWS * sizeof(float2));
  cluster_barrier();
  const bool sends = some && mine;
  for (int c = 0; c < splits; ++c)
    send2(in_cta(stats + rank * ROWS + at, c), sends ? m_own : -INFINITY, sends ? l_own : 0.f);
  if (some)
    for (int c = 0; c < HD; c += 16) {
      uint32_t v[16];
      tmem_ld16(oc + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const int to = (c + k) / width, four = (c + k) % width / 4;
        if (sends) send4(in_cta(ring + ((size_t)(rank * (width / 4) + four) * ROWS + at) * 16, to), v + k);
      }
    }
  cluster_barrier();
  float top = -INFINITY, sum = 0.f;
  for (int c = 0; c < splits; ++c) top = fmaxf(top, stats[c * ROWS + at].x);
  const float use = top == -INFINITY ? 0.f : top;
  for (int c = 0; c < splits; ++c) sum = fmaf(ex2(stats[c * ROWS + at].x - use), stats[c * ROWS + at].y, sum);
  const float inv = all_seen > 0 ? 1.f / sum : 0.f;
  T* dst = static_cast<T*>(p.out) + row * p.out_row + (int64_t)head * p.out_head + rank * width;
  bool bad = false;
  for (int e = 0; e < width; e += 8) {
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < splits; ++c) {
      const float m = stats[c * ROWS + at].x;
      if (m == -INFINITY) continue;  // (nothing was sent, or nothing but zeros)
      const float w = ex2(m - use);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(ring + ((size_t)(c * (width / 4) + e / 4 + k) * ROWS + at) * 16);
        o[4 * k] = fmaf(w, x.x, o[4 * k]);
        o[4 * k + 1] = fmaf(w, x.y, o[4 * k + 1]);
        o[4 * k + 2] = fmaf(w, x.z, o[4 * k + 2]);
        o[4 * k + 3] = fmaf(w, x.w, o[4 * k + 3]);
      }
    }
    uint32_t packed[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = all_seen > 0 ? o[2 * k] * inv : 0.f, b = all_seen > 0 ? o[2 * k + 1] * inv : 0.f;
      bad |= !(fabsf(a) <= 3.402823466e38f) || !(fabsf(b) <= 3.402823466e38f);
      packed[k] = Mma<T>::pack(a, b);
    }
    if (mine) *reinterpret_cast<uint4*>(dst + e) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
  }
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(in_cta(bad_rows + rank * ROWS + at, 0)), "r"((int)bad) : "memory");
  cluster_barrier();
  if (rank == 0) {
    for (int c = 0; c < splits; ++c) bad |= bad_rows[c * ROWS + at] != 0;
    unsigned again = __ballot_sync(0xffffffffu, doubtful(bad, sum) && mine);
    while (again) {
      const int who = __ffs(again) - 1;
      again &= again - 1;
      __syncwarp();
      slow_row<HD, T>(p, t, __shfl_sync(0xffffffffu, row, who), __shfl_sync(0xffffffffu, head, who),
                      reach);
    }
  }
}

template <int HD, typename T, bool SPLIT>
__global__ void __launch_bounds__(kTcThreads, 1)
    packed_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TcParams tp) {
  constexpr int kChunks = HD / 64;                  // 128-byte wide pieces of a head
  constexpr uint32_t kPiece = kTile * 128;          // bytes of one
  constexpr uint32_t kOperand = kChunks * kPiece;   // a tile of Q, K or V
  constexpr int kStages = tc_stages<HD>();          // one ring of K0, V0, K1, V1, ...
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint64_t q_full, full[kStages], empty[kStages];
  __shared__ uint64_t s_full[2], p_full[2], o_full[2], fin;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const PackedParams& p = tp.a;
  uint8_t* smem = smem_dyn + ((1024u - (smem_addr(smem_dyn) & 1023u)) & 1023u);
  uint8_t* qs = smem;
  uint8_t* ring = smem + 2 * kOperand;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(&fin, 1);
    abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 9 && lane < 3) prefetch_map(lane == 0 ? &qmap : lane == 1 ? &kmap : &vmap);
  pdl_wait();
  Tile t;
  const int both = 2 * tp.tokens, nkv = p.nh / p.hpk;
  const int splits = SPLIT ? tp.splits : 1, rank = SPLIT ? blockIdx.x % splits : 0;
  const int item = blockIdx.x / splits, items = gridDim.x / splits;
  if (!find_tile(p, both, (items - 1 - item) / nkv, t)) return;
  if (warp == 8) tmem_alloc(&tmem_slot, 512);
  const int kv = item % nkv;
  const int rows = min(both, t.q1 - t.row0);
  // KV rows that each tile's last row sees, of those that this CTA takes: from row `from` of the
  // sequence on, `most` at the most; and the blocks of 128 of them
  int all_sees[2], sees[2], blocks[2], from = 0, most = INT32_MAX;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int last = min(rows, (i + 1) * tp.tokens) - 1;
    all_sees[i] = last >= i * tp.tokens ? seen_by(p, t, t.row0 + last) : 0;
  }
  if constexpr (SPLIT) {
    const int all = (max(all_sees[0], all_sees[1]) + kTile - 1) / kTile;
    from = all * rank / splits * kTile;
    most = all * (rank + 1) / splits * kTile - from;
  }
  auto part = [&](int seen) { return SPLIT ? max(0, min(seen - from, most)) : seen; };
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    sees[i] = part(all_sees[i]);
    blocks[i] = (sees[i] + kTile - 1) / kTile;
  }
  const int n = max(blocks[0], blocks[1]);

  // tile rows past the last whole query row: zeros, so that their scores are
  for (int k = tp.tokens * p.hpk * 8 + threadIdx.x; k < kTile * 8; k += kTcThreads)
    for (int c = 0; c < 2 * kChunks; ++c) *reinterpret_cast<uint4*>(qs + c * kPiece + 16 * k) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if constexpr (SPLIT) cluster_barrier();  // every CTA has begun
  const uint32_t s_col[2] = {tmem, tmem + kTile}, o_col[2] = {tmem + 2 * kTile, tmem + 2 * kTile + HD};

  // registers: 384 x 168 at launch = 256 x 232 + 128 x 40
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
  if (warp == 9) {
    // ---------------- copies
    if (lane == 0 && n > 0) {
      const uint32_t box = (uint32_t)(tp.tokens * p.hpk) * 128u;
      mbar_arrive_expect_tx(&q_full, 2 * kChunks * box);
      for (int i = 0; i < 2; ++i)
        for (int c = 0; c < kChunks; ++c)
          tma_load_3d(qs + i * kOperand + c * kPiece, &qmap, 64 * c, kv * p.hpk, t.row0 + i * tp.tokens, &q_full);
    }
    int issued = 0, s = 0;
    uint32_t phase = 1;  // the first round finds the stages free
    for (; issued < 2 * n; ++issued) {
      if (warp_aborted(&abort_flag) || !warp_wait(&empty[s], phase, p.err)) {
        abort_flag = 1;
        break;
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[s], kOperand);
        for (int c = 0; c < kChunks; ++c)
          tma_load_3d(ring + (size_t)s * kOperand + c * kPiece, issued & 1 ? &vmap : &kmap, 64 * c, kv,
                      t.k0 + from + (issued >> 1) * kTile, &full[s]);
      }
      __syncwarp();
      if (++s == kStages) {
        s = 0;
        phase ^= 1;
      }
    }
    // copies in flight land before the CTA leaves
    if (n > 0) warp_wait(&q_full, 0, p.err);
    for (int i = 0; i < kStages; ++i) {
      const int uses = issued > i ? (issued - i + kStages - 1) / kStages : 0;
      if (uses) warp_wait(&full[i], (uint32_t)(uses - 1) & 1u, p.err);
    }
  } else if (warp == 8) {
    // ---------------- products. A commit holds up the products behind it by some 120 clocks, so
    // there are two per block: each tile's S, which stands for the PV before it too; the softmax
    // frees the ring's stages on it.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (warp_wait(bar, parity, p.err)) return true;
      abort_flag = 1;
      return false;
    };
    // columns of block j that tile i's last row sees, in steps of the products' 16
    auto columns = [&](int i, int j) { return min(kTile, (sees[i] - j * kTile + 15) & ~15); };
    auto scores = [&](int i, int j, int stage) {  // S_i = Q_i K^T
      const uint32_t idesc = tp.idesc_s | ((uint32_t)(columns(i, j) >> 3) << 17);
      const uint32_t qa = smem_addr(qs + i * kOperand), ka = smem_addr(ring + (size_t)stage * kOperand);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (uint32_t)(kk / 4) * kPiece + 32u * (kk % 4);
          umma_f16(s_col[i], sw128_desc(qa + off), sw128_desc(ka + off), idesc, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[i]);
      }
      __syncwarp();
    };
    int s = 0;
    uint32_t phase = 0;
    auto next = [&]() {
      if (++s == kStages) {
        s = 0;
        phase ^= 1;
      }
    };
    bool ok = n == 0 || (wait(&q_full, 0) && wait(&full[0], 0));
    if (ok && n > 0) {
      tc_fence_after();
      for (int i = 0; i < 2; ++i)
        if (blocks[i] > 0) scores(i, 0, 0);
      next();
    }
    for (int j = 0; j < n && ok; ++j) {
      ok = wait(&full[s], phase);
      const int vst = s;
      next();
      bool have_k = false;
      for (int i = 0; i < 2 && ok; ++i) {
        if (j >= blocks[i]) continue;
        ok = wait(&p_full[i], (uint32_t)j & 1u);
        if (!ok) break;
        tc_fence_after();
        const uint32_t va = smem_addr(ring + (size_t)vst * kOperand);
        const int steps = columns(i, j) / 16;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk) {
            if (kk >= steps) break;
            umma_f16_ta(o_col[i], s_col[i] + 8u * kk, sw128_desc_mn(va + 2048u * kk, kPiece), tp.idesc_o,
                        j > 0 || kk > 0 ? 1u : 0u);
          }
          if (j + 1 >= blocks[i]) umma_commit(&o_full[i]);
        }
        __syncwarp();
        if (j + 1 < blocks[i]) {
          if (!have_k) ok = wait(&full[s], phase);
          if (!ok) break;
          tc_fence_after();
          have_k = true;
          scores(i, j + 1, s);
        }
      }
      if (j + 1 < n) next();
    }
    if (elect_one()) umma_commit(&fin);
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ---------------- softmax of tile i: thread r = row r
    const int i = warp >> 2, r = threadIdx.x & 127;
    const int token = r / p.hpk, head = kv * p.hpk + r % p.hpk;
    const int row = t.row0 + i * tp.tokens + token;  // query row
    const bool mine = token < tp.tokens && i * tp.tokens + token < rows;
    const int all_seen = mine ? seen_by(p, t, row) : 0, seen = part(all_seen);
    const int open = mine ? seen : INT32_MAX;  // tile rows of no query mask nothing
    const int all_see = (int)__reduce_min_sync(0xffffffffu, (unsigned)open);    // every row of the warp,
    const int none_sees = (int)__reduce_max_sync(0xffffffffu, (unsigned)seen);  // and none from here on
    const int lk = t.k1 - t.k0 - from;  // rows of the sequence from this CTA's first on
    const uint32_t sub = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t sc = s_col[i] + sub, oc = o_col[i] + sub;
    const int end_block = (lk - 1) / kTile;
    const bool zeroes = lk % kTile != 0 && i == (blocks[0] > end_block ? 0 : 1);
    const bool frees = i == (blocks[1] > 0 ? 1 : 0);  // the tile whose products come last
    RowSoftmax<T> rs{p.scale, mine, -INFINITY, make_float2(0.f, 0.f)};
    bool ok = true;
    for (int j = 0; j < blocks[i]; ++j) {
      if (!warp_wait(&s_full[i], (uint32_t)j & 1u, p.err)) {
        abort_flag = 1;
        ok = false;
        break;
      }
      tc_fence_after();
      if (frees && r == 0) {  // S_j is done, and with it PV of block j - 1, of both tiles
        mbar_arrive(&empty[2 * j % kStages]);
        if (j > 0) mbar_arrive(&empty[(2 * j - 1) % kStages]);
      }
      if (zeroes && j == end_block) {
        // V rows behind the sequence
        const int item = 2 * j + 1;
        if (!warp_wait(&full[item % kStages], (uint32_t)(item / kStages) & 1u, p.err)) {
          abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t* v = ring + (size_t)(item % kStages) * kOperand;
        const int left = lk - j * kTile;
        for (int c = 0; c < kChunks; ++c)
          for (int k = (threadIdx.x & 127); k < (kTile - left) * 8; k += 128)
            *reinterpret_cast<uint4*>(v + c * kPiece + (size_t)left * 128 + 16 * k) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      rs.block(sc, j, open, all_see, none_sees, [&](float alpha) {
        if (j > 0) scale_row<HD>(oc, alpha);
      });
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i]);
    }
    // ---------------- out
    if (ok && blocks[i] > 0) {
      ok = warp_wait(&o_full[i], 0, p.err);
      if (!ok) abort_flag = 1;
    }
    tc_fence_after();
    if constexpr (!SPLIT) {
      if (ok && i * tp.tokens < rows)
        write_row<HD, T>(p, t, oc, blocks[i] > 0, mine, row, head, seen, rs.l.x + rs.l.y, min(lk, (sees[i] + 15) & ~15));
    } else {
      join_rows<HD, T, 256>(p, t, qs, ring, splits, rank, threadIdx.x, ok && blocks[i] > 0, mine, row, head, all_seen,
                            rs.m, rs.l.x + rs.l.y, oc, min(t.k1 - t.k0, (all_sees[i] + 15) & ~15));
    }
    tc_fence_before();
  }
  if constexpr (SPLIT)
    if (warp >= 8)
      for (int k = 0; k < 3; ++k) cluster_barrier();

  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    warp_wait(&fin, 0u, p.err);  // no product still runs when its TMEM is freed
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- head_dim 256: tcgen05, one tile per CTA -------------------------------------------------
//
// O of 128 rows takes half of TMEM here, so a CTA has one tile, and S two places: S of block j + 1
// runs during the softmax of block j, S(0), S(1), PV(0), S(2), PV(1), ... A stage of the ring holds
// half a tile, 128 KV rows x 128 values, which is half of S's depth or of O's columns. The copying
// warp sees a stage free by the commit behind its products: s_full of K's, pv of V's.
// Measured: 8,000 rows of 8 heads 223 us, 1175 TFLOP/s, the tensor cores 60 % busy, the L2 36 %.
// Without the softmax it took 203 us, without the copies 211 (each product takes some 70 clocks of
// 64, each commit holds up the next by 120, and a CTA's start and end are not overlapped). The
// mma.sync kernel above took 2622 us.
constexpr int kWideThreads = 192;  // warps 0-3 softmax, 4 products, 5 copies

template <typename T, bool SPLIT>
__global__ void __launch_bounds__(kWideThreads, 1)
    packed_wide_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const __grid_constant__ TcParams tp) {
  constexpr int HD = 256, kChunks = HD / 64, kStages = 5;
  constexpr uint32_t kPiece = kTile * 128, kStage = 2 * kPiece;
  extern __shared__ uint8_t smem_dyn[];
  // p_full: one per place, as a warp may be through a block whose S came early while others are at the
  // one before; pv: the products of all but the last block
  __shared__ uint64_t q_full, full[kStages], s_full[2], p_full[2], pv, o_full, fin;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const PackedParams& p = tp.a;
  uint8_t* smem = smem_dyn + ((1024u - (smem_addr(smem_dyn) & 1023u)) & 1023u);
  uint8_t* qs = smem;
  uint8_t* ring = smem + kChunks * kPiece;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(&pv, 1);
    mbar_init(&o_full, 1);
    mbar_init(&fin, 1);
    abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 5 && lane < 3) prefetch_map(lane == 0 ? &qmap : lane == 1 ? &kmap : &vmap);
  pdl_wait();
  Tile t;
  const int nkv = p.nh / p.hpk;
  const int splits = SPLIT ? tp.splits : 1, rank = SPLIT ? blockIdx.x % splits : 0;
  const int tile = blockIdx.x / splits, tiles = gridDim.x / splits;
  if (!find_tile(p, tp.tokens, (tiles - 1 - tile) / nkv, t)) return;
  if (warp == 4) tmem_alloc(&tmem_slot, 512);
  const int kv = tile % nkv;
  const int rows = min(tp.tokens, t.q1 - t.row0);
  const int all_sees = seen_by(p, t, t.row0 + rows - 1);  // KV rows that the last row sees
  int from = 0, most = INT32_MAX;                         // those that this CTA takes
  if constexpr (SPLIT) {
    const int all = (all_sees + kTile - 1) / kTile;
    from = all * rank / splits * kTile;
    most = all * (rank + 1) / splits * kTile - from;
  }
  auto part = [&](int seen) { return SPLIT ? max(0, min(seen - from, most)) : seen; };
  const int sees = part(all_sees), lk = t.k1 - t.k0 - from;  // lk: rows of the sequence from there on
  const int n = (sees + kTile - 1) / kTile;

  // tile rows past the last whole query row: zeros, so that their scores are
  for (int k = tp.tokens * p.hpk * 8 + threadIdx.x; k < kTile * 8; k += kWideThreads)
    for (int c = 0; c < kChunks; ++c) *reinterpret_cast<uint4*>(qs + c * kPiece + 16 * k) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if constexpr (SPLIT) cluster_barrier();  // every CTA has begun
  const uint32_t tmem = tmem_slot, o_col = tmem + 2 * kTile;
  auto wait = [&](uint64_t* bar, int use) {  // the use-th completion of a barrier
    if (warp_wait(bar, (uint32_t)use & 1u, p.err)) return true;
    abort_flag = 1;
    return false;
  };

  if (warp == 5) {
    // ---------------- copies. Halves come in pairs u: K(0), K(1), V(0), K(2), V(1), ..., V(n - 1)
    auto is_v = [&](int u) { return u == 2 * n - 1 || (u > 0 && u % 2 == 0); };
    auto block_of = [&](int u) { return is_v(u) ? (u == 2 * n - 1 ? n - 1 : u / 2 - 1) : (u + 1) / 2; };
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(&q_full, kChunks * (uint32_t)(tp.tokens * p.hpk) * 128u);
      for (int c = 0; c < kChunks; ++c) tma_load_3d(qs + c * kPiece, &qmap, 64 * c, kv * p.hpk, t.row0, &q_full);
    }
    int issued = 0, s_seen = 0, v_seen = 0;  // blocks whose products are known to be done
    for (; issued < 4 * n; ++issued) {
      bool ok = !warp_aborted(&abort_flag);
      if (ok && issued >= kStages) {  // what the stage held before
        const int u = (issued - kStages) >> 1, j = block_of(u);
        if (is_v(u)) {
          if (j >= v_seen) ok = wait(&pv, j);
          v_seen = j + 1;
        } else {
          if (j >= s_seen) ok = wait(&s_full[j & 1], j >> 1);
          s_seen = j + 1;
        }
      }
      if (!ok) break;
      if (lane == 0) {
        const int u = issued >> 1, half = issued & 1, st = issued % kStages;
        mbar_arrive_expect_tx(&full[st], kStage);
        for (int c = 0; c < 2; ++c)
          tma_load_3d(ring + (size_t)st * kStage + c * kPiece, is_v(u) ? &vmap : &kmap, 128 * half + 64 * c, kv,
                      t.k0 + from + block_of(u) * kTile, &full[st]);
      }
      __syncwarp();
    }
    // copies in flight land before the CTA leaves
    if (n > 0) warp_wait(&q_full, 0, p.err);
    for (int i = 0; i < kStages; ++i) {
      const int uses = issued > i ? (issued - i + kStages - 1) / kStages : 0;
      if (uses) warp_wait(&full[i], (uint32_t)(uses - 1) & 1u, p.err);
    }
  } else if (warp == 4) {
    // ---------------- products
    auto columns = [&](int j) { return min(kTile, (sees - j * kTile + 15) & ~15); };
    int item = 0;
    auto landed = [&]() {
      const bool ok = wait(&full[item % kStages], item / kStages);
      tc_fence_after();
      return ok;
    };
    auto scores = [&](int j) {  // S(j) = Q K(j)^T
      const uint32_t idesc = tp.idesc_s | ((uint32_t)(columns(j) >> 3) << 17);
      for (int half = 0; half < 2; ++half, ++item) {
        if (!landed()) return false;
        const uint32_t qa = smem_addr(qs + half * kStage), ka = smem_addr(ring + (size_t)(item % kStages) * kStage);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const uint32_t off = (uint32_t)(kk / 4) * kPiece + 32u * (kk % 4);
            umma_f16(tmem + kTile * (j & 1), sw128_desc(qa + off), sw128_desc(ka + off), idesc,
                     half > 0 || kk > 0 ? 1u : 0u);
          }
          if (half == 1) umma_commit(&s_full[j & 1]);
        }
        __syncwarp();
      }
      return true;
    };
    bool ok = n == 0 || (wait(&q_full, 0) && scores(0));
    for (int j = 0; j < n && ok; ++j) {
      ok = (j + 1 >= n || scores(j + 1)) && wait(&p_full[j & 1], j >> 1);
      if (!ok) break;
      const int steps = columns(j) / 16;
      for (int half = 0; half < 2 && ok; ++half, ++item) {  // O's columns 128 half .. + 127
        ok = landed();
        if (!ok) break;
        const uint32_t va = smem_addr(ring + (size_t)(item % kStages) * kStage);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk) {
            if (kk >= steps) break;
            umma_f16_ta(o_col + 128 * half, tmem + kTile * (j & 1) + 8u * kk, sw128_desc_mn(va + 2048u * kk, kPiece),
                        tp.idesc_o, j > 0 || kk > 0 ? 1u : 0u);
          }
          if (half == 1) umma_commit(j + 1 < n ? &pv : &o_full);
        }
        __syncwarp();
      }
    }
    if (elect_one()) umma_commit(&fin);
    __syncwarp();
  } else {
    // ---------------- softmax: thread r = row r
    const int r = threadIdx.x, token = r / p.hpk, head = kv * p.hpk + r % p.hpk, row = t.row0 + token;
    const bool mine = token < tp.tokens && token < rows;
    const int all_seen = mine ? seen_by(p, t, row) : 0, seen = part(all_seen);
    const int open = mine ? seen : INT32_MAX;  // tile rows of no query mask nothing
    const int all_see = (int)__reduce_min_sync(0xffffffffu, (unsigned)open);
    const int none_sees = (int)__reduce_max_sync(0xffffffffu, (unsigned)seen);
    const uint32_t sub = (uint32_t)(32 * warp) << 16;
    const int end_block = (lk - 1) / kTile;
    RowSoftmax<T> rs{p.scale, mine, -INFINITY, make_float2(0.f, 0.f)};
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      ok = wait(&s_full[j & 1], j >> 1);
      if (!ok) break;
      tc_fence_after();
      if (lk % kTile != 0 && j == end_block) {  // V rows behind the sequence; j is n - 1
        const int left = lk - j * kTile;
        for (int half = 0; half < 2 && ok; ++half) {
          const int item = 4 * n - 2 + half;
          ok = wait(&full[item % kStages], item / kStages);
          uint8_t* v = ring + (size_t)(item % kStages) * kStage;
          for (int c = 0; c < 2 && ok; ++c)
            for (int k = r; k < (kTile - left) * 8; k += 128)
              *reinterpret_cast<uint4*>(v + c * kPiece + (size_t)left * 128 + 16 * k) = make_uint4(0, 0, 0, 0);
        }
        if (!ok) break;
        fence_proxy_async_smem();
      }
      rs.block(tmem + kTile * (j & 1) + sub, j, open, all_see, none_sees, [&](float alpha) {
        if (j == 0) return;
        ok = wait(&pv, j - 1);  // the products so far (those before S(j) was issued are done)
        tc_fence_after();
        scale_row<HD>(o_col + sub, alpha);
      });
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[j & 1]);
    }
    if (ok && n > 0) ok = wait(&o_full, 0);
    tc_fence_after();
    if constexpr (SPLIT) {
      join_rows<HD, T, 128>(p, t, qs, ring, splits, rank, r, ok && n > 0, mine, row, head, all_seen, rs.m,
                            rs.l.x + rs.l.y, o_col + sub, min(t.k1 - t.k0, (all_sees + 15) & ~15));
    } else if (ok) {
      write_row<HD, T>(p, t, o_col + sub, n > 0, mine, row, head, seen, rs.l.x + rs.l.y, min(lk, (sees + 15) & ~15));
    }
    tc_fence_before();
  }
  if constexpr (SPLIT)
    if (warp >= 4)
      for (int k = 0; k < 3; ++k) cluster_barrier();

  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    warp_wait(&fin, 0u, p.err);  // no product still runs when its TMEM is freed
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Tensor map of rows of heads: {head_dim, heads, rows}, boxes of 64 x box_heads x box_rows.
bool encode_heads(CUtensorMap* map, int type, const void* base, int hd, int64_t heads, int64_t rows, int64_t head_stride,
                  int64_t row_stride, int box_heads, int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows}, estr[3] = {1, 1, 1};
  return fn(map, type == RRR_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of heads of hd 16-bit values; strides in elements.
struct HeadRows {
  const void* p;
  int64_t rows, row, heads, head, hd;
};
// Whether two such arrays share no byte, for certain: their extents do not meet, or all of their
// places lie apart modulo a stride (both in one buffer whose rows or heads hold a part of each).
bool apart(const HeadRows& a, const HeadRows& b) {
  using Wide = __int128;
  if (a.rows < 1 || b.rows < 1) return true;
  auto from = [](const HeadRows& x) { return (Wide) reinterpret_cast<uintptr_t>(x.p); };
  // bytes from the first place to the end of the last, where multiples of m elements do not count
  auto width = [](const HeadRows& x, int64_t m) {
    Wide w = x.hd;
    if (m == 0 || x.row % m) w += (Wide)(x.rows - 1) * x.row;
    if (m == 0 || x.head % m) w += (Wide)(x.heads - 1) * x.head;
    return 2 * w;
  };
  const Wide between = from(b) - from(a);
  if (between >= width(a, 0) || -between >= width(b, 0)) return true;
  for (const int64_t m : {a.row, a.head, b.row, b.head}) {
    const Wide period = 2 * (Wide)m, off = (between % period + period) % period;
    if (off >= width(a, m) && off + width(b, m) <= period) return true;
  }
  return false;
}

// Query rows of a CTA of the tcgen05 kernels
int rows_per_cta(int hd, int hpk) { return (hd == 256 ? 1 : 2) * (kTile / hpk); }

template <int HD, typename T, bool SPLIT>
auto tc_kernel() {
  if constexpr (HD == 256)
    return &packed_wide_kernel<T, SPLIT>;
  else
    return &packed_tc_kernel<HD, T, SPLIT>;
}

template <int HD, typename T>
cudaError_t launch_tc(const LaunchEnv& env, int type, const PackedParams& p) {
  TcParams tp{};
  tp.a = p;
  tp.tokens = kTile / p.hpk;
  const uint32_t fmt = type == RRR_F16 ? 0u : 1u;
  // f32 accumulator, A and B of the type, B of the second product N-contiguous, N / 8, M / 16
  tp.idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kTile >> 4) << 24);  // N / 8: as wide as the block
  tp.idesc_o = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((uint32_t)((HD < 128 ? HD : 128) >> 3) << 17) |
               ((uint32_t)(kTile >> 4) << 24);
  CUtensorMap qmap, kmap, vmap;
  const int64_t nkv = p.nh / p.hpk;
  if (!encode_heads(&qmap, type, p.q, HD, p.nh, p.q_rows, p.q_head, p.q_row, p.hpk, tp.tokens) ||
      !encode_heads(&kmap, type, p.k, HD, nkv, p.kv_rows, p.k_head, p.k_row, 1, kTile) ||
      !encode_heads(&vmap, type, p.v, HD, nkv, p.kv_rows, p.v_head, p.v_row, 1, kTile))
    return cudaErrorInvalidValue;
  // nkv times the slots fits the grid: the caller's check
  const dim3 grid((unsigned)(nkv * (p.q_rows / rows_per_cta(HD, p.hpk) + p.n_seqs)));
  // Few tiles with many blocks of KV rows (of the mean sequence) go to clusters. Joining costs 3 to 5
  // us, and no more than some 9 clusters of 8 such CTAs run at once: 1 row of 24 heads on 9,000 rows
  // 123 us alone, 75, 44 and 28 by 2, 4 and 8 CTAs; 100 rows on 2,000 36.5, 32, 24 and, in two rounds,
  // 36; 1,000 on 1,000 with 8 heads on 2 23, 24.5 and 20.6; 500 rows on 500 16 and 20 (128 values;
  // with 256 1 row on 9,000 126 and 34).
  const int64_t deep = (p.kv_rows / p.n_seqs + kTile - 1) / kTile;
  tp.splits = 1;
  for (const int by : {8, 4, 2}) {
    if ((int64_t)grid.x * by > (by == 8 ? env.sm_count / 2 : env.sm_count) || deep < (by == 2 ? 12 : 2 * by)) continue;
    tp.splits = by;
    break;
  }
  const int smem = (HD == 256 ? 7 * kTile * 128 : (2 + tc_stages<HD>()) * kTile * HD) * 2 + 1024;
  auto kern = tp.splits > 1 ? tc_kernel<HD, T, true>() : tc_kernel<HD, T, false>();
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = env.pdl ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)tp.splits, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid.x * tp.splits);
  cfg.blockDim = dim3(HD == 256 ? kWideThreads : kTcThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = env.stream;
  cfg.attrs = attr;
  cfg.numAttrs = tp.splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, qmap, kmap, vmap, tp);
}

template <int HD, typename T>
cudaError_t launch(const LaunchEnv& env, const PackedParams& p) {
  auto kern = packed_kernel<HD, T>;
  const int smem = (kQRows + 2 * kKRows) * (HD + 8) * (int)sizeof(T);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)(p.q_rows / kQRows + p.n_seqs), p.nh);
  return rrr_launch_pdl(kern, grid, dim3(kThreads), (size_t)smem, env.stream, env.pdl, p);
}
template <int HD>
cudaError_t launch_type(const LaunchEnv& env, int type, const PackedParams& p) {
  if (p.hpk <= kTile && p.kv_rows > 0)
    return type == RRR_F16 ? launch_tc<HD, __half>(env, type, p) : launch_tc<HD, __nv_bfloat16>(env, type, p);
  return type == RRR_F16 ? launch<HD, __half>(env, p) : launch<HD, __nv_bfloat16>(env, p);
}

}  // namespace
}  // namespace rrr

using namespace rrr;

extern "C" int rrr_attention_packed(rrr_ctx* ctx, const rrr_packed_desc* d, const void* q, const void* k,
                                    const void* v, const int32_t* cu_q, const int32_t* cu_kv, void* out,
                                    void* stream) {
  const char* fn = "rrr_attention_packed";
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  if (!d || (d->n_seqs > 0 && (!cu_q || !cu_kv))) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (d->type != RRR_F16 && d->type != RRR_BF16)
    return set_error(ctx, RRR_ERR_BAD_QTYPE, "%s: type must be 1 (F16) or 30 (BF16)", fn);
  const int hd = d->head_dim;
  if ((hd != 64 && hd != 128 && hd != 256) || d->n_heads < 1 || d->n_kv_heads < 1 || d->n_heads % d->n_kv_heads ||
      d->n_heads > 65535 || d->n_seqs < 0 || d->q_rows < 0 || d->kv_rows < 0 || d->q_rows > INT32_MAX / 2 ||
      d->kv_rows > INT32_MAX / 2 || d->n_seqs > INT32_MAX / 4)
    return set_error(ctx, RRR_ERR_BAD_SHAPE,
                     "%s: need head_dim 64/128/256, n_heads a multiple of n_kv_heads (at most 65535) and counts "
                     "of 0 to 2^30 - 1",
                     fn);
  if (d->causal != 0 && d->causal != 1) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: causal is 0 or 1", fn);
  if (!(d->scale >= 0.f) || d->scale > 3.4e38f)
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: scale must be finite, not negative", fn);
  if (d->q_rows && (!q || !out)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (d->kv_rows && (!k || !v)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int64_t strides[8] = {d->q_row, d->q_head, d->k_row, d->k_head, d->v_row, d->v_head, d->out_row, d->out_head};
  for (int64_t s : strides) {
    if (s < hd || s > ((int64_t)1 << 38)) return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: a stride is shorter than a head, or over 2^38", fn);
    if (s % 8) return set_error(ctx, RRR_ERR_MISALIGNED, "%s: strides must be multiples of 8 elements", fn);
  }
  if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(out, 16) ||
      !aligned_to(cu_q, 4) || !aligned_to(cu_kv, 4))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: q, k, v and out must be 16-byte aligned", fn);
  // out: rows of heads or heads of rows, without two elements in one place, apart from the inputs.
  // (2^30 rows of 2^38 elements: extents take more than 64 bits)
  using Wide = __int128;
  const int64_t nh = d->n_heads, kvh = d->n_kv_heads;
  if (!(d->out_row >= (nh - 1) * d->out_head + hd || d->out_head >= (Wide)(d->q_rows - 1) * d->out_row + hd))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows and heads of out overlap", fn);
  const HeadRows mine{out, d->q_rows, d->out_row, nh, d->out_head, hd};
  for (const HeadRows& in : {HeadRows{q, d->q_rows, d->q_row, nh, d->q_head, hd},
                             HeadRows{k, d->kv_rows, d->k_row, kvh, d->k_head, hd},
                             HeadRows{v, d->kv_rows, d->v_row, kvh, d->v_head, hd}})
    if (!apart(mine, in)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: out overlaps an input", fn);
  const int64_t hpk = nh / kvh, per = hpk <= kTile ? rows_per_cta(hd, (int)hpk) : 1;
  if (kvh * (d->q_rows / per + d->n_seqs) > INT32_MAX)
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: too many rows, sequences and heads for one call", fn);
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  if (d->q_rows == 0 || d->n_seqs == 0) return RRR_OK;
  const LaunchEnv env = make_env(ctx, stream);
  PackedParams p{q, k, v, out, d->q_row, d->q_head, d->k_row, d->k_head, d->v_row, d->v_head, d->out_row, d->out_head,
                 cu_q, cu_kv, d->n_seqs, d->n_heads, d->n_heads / d->n_kv_heads, d->causal, d->q_rows, d->kv_rows,
                 (d->scale == 0.f ? 1.f / sqrtf((float)hd) : d->scale) * 1.4426950408889634f, env.d_err};
  cudaError_t e;
  switch (hd) {
    case 64: e = launch_type<64>(env, d->type, p); break;
    case 128: e = launch_type<128>(env, d->type, p); break;
    default: e = launch_type<256>(env, d->type, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_attention_packed launch");
}
