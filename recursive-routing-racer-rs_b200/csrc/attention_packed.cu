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
// get disjoint runs of x that are long enough, found by a binary search on the device.
#include <math.h>

#include "serve_common.cuh"

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
template <int ROWS>
__device__ __forceinline__ bool find_tile(const PackedParams& p, int x, Tile& t) {
  int lo = 0, hi = p.n_seqs - 1;  // the last s with cu[s] / ROWS + s <= x
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu_q[mid] / ROWS + mid <= x)
      lo = mid;
    else
      hi = mid - 1;
  }
  t.seq = lo;
  t.q0 = p.cu_q[lo];
  t.q1 = p.cu_q[lo + 1];
  t.k0 = p.cu_kv[lo];
  t.k1 = p.cu_kv[lo + 1];
  if (t.q0 < 0 || t.q1 < t.q0 || t.q1 > p.q_rows || t.k0 < 0 || t.k1 < t.k0 || t.k1 > p.kv_rows) {
    if (threadIdx.x == 0) flag_position(p.err);
    return false;
  }
  const int64_t row0 = t.q0 + (int64_t)ROWS * (x - (t.q0 / ROWS + lo));
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

// One query row by one warp in 32-bit arithmetic over the rows that it sees and no others. A
// masked weight of zero times an infinite or NaN value is a NaN in a tile's product, so a row
// that comes out not finite is computed again here: what a row does not see never reaches it.
template <int HD, typename T>
__device__ __noinline__ void slow_row(const PackedParams& p, const Tile& t, int row, int head) {
  constexpr int D = HD / 32;
  const int lane = threadIdx.x & 31, kv = head / p.hpk, n = seen_by(p, t, row);
  float q[D], o[D], m = -INFINITY, l = 0.f;
  load_vec<T, D>(static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head + D * lane, q);
#pragma unroll
  for (int i = 0; i < D; ++i) o[i] = 0.f;
  for (int j = 0; j < n; ++j) {
    float x[D], dot = 0.f;
    load_vec<T, D>(static_cast<const T*>(p.k) + (int64_t)(t.k0 + j) * p.k_row + kv * p.k_head + D * lane, x);
#pragma unroll
    for (int i = 0; i < D; ++i) dot = fmaf(q[i], x[i], dot);
    const float s = warp_sum(dot) * p.scale;
    const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = ex2(m - mu), w = ex2(s - mu);
    m = mn;
    l = fmaf(l, alpha, w);
    load_vec<T, D>(static_cast<const T*>(p.v) + (int64_t)(t.k0 + j) * p.v_row + kv * p.v_head + D * lane, x);
#pragma unroll
    for (int i = 0; i < D; ++i) o[i] = fmaf(o[i], alpha, w * x[i]);
  }
#pragma unroll
  for (int i = 0; i < D; ++i) o[i] = n > 0 ? o[i] / l : 0.f;
  store_vec<T, D>(static_cast<T*>(p.out) + row * p.out_row + head * p.out_head + D * lane, o);
}

// 64 query rows of one head per CTA, 16 per warp, against 64 KV rows at a time in shared memory.
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
  if (!find_tile<kQRows>(p, (int)(gridDim.x - 1 - blockIdx.x), t)) return;
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
    unsigned rows_bad = __ballot_sync(0xffffffffu, bad && r < rows);
    for (int rr = 0; rr < 8; ++rr)
      if (rows_bad & (0xfu << (4 * rr))) {
        __syncwarp();
        slow_row<HD, T>(p, t, t.row0 + 16 * warp + 8 * i + rr, head);
      }
  }
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
  if (!d || !cu_q || !cu_kv) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
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
  // out: rows of heads or heads of rows, without two elements in one place, apart from the inputs
  const int64_t nh = d->n_heads;
  if (!(d->out_row >= (nh - 1) * d->out_head + hd || d->out_head >= (d->q_rows - 1) * d->out_row + hd))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows and heads of out overlap", fn);
  auto extent = [&](int64_t rows, int64_t row, int64_t heads, int64_t head) {
    return rows < 1 ? (int64_t)0 : 2 * ((rows - 1) * row + (heads - 1) * head + hd);
  };
  const int64_t kvh = d->n_kv_heads;
  const RowSet parts[4] = {{out, 0, extent(d->q_rows, d->out_row, nh, d->out_head), 1},
                           {q, 0, extent(d->q_rows, d->q_row, nh, d->q_head), 1},
                           {k, 0, extent(d->kv_rows, d->k_row, kvh, d->k_head), 1},
                           {v, 0, extent(d->kv_rows, d->v_row, kvh, d->v_head), 1}};
  for (int i = 1; i < 4; ++i)
    if (!rows_disjoint(parts[0], parts[i]))
      return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: out overlaps an input", fn);
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
