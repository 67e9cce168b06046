// kv4_tree.cu — attention of drafted rows over the 4-bit KV cache (rrr_attention_tree_kv4): the
// `attention` dispatch (src/model/phi4.rs:1284-1309, 1680-1688) for the rows of a tree of drafted
// tokens per sequence, which see the sequence's cached rows and their own ancestors.
#include <math.h>

#include "kv4.cuh"

namespace rrr {
namespace {

constexpr int kMaxHpk = 8, kMaxNodes = 128;
constexpr float kNone = -3e38f;  // the maximum of no rows: finite, so that it may be subtracted from -inf

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
  float scale;  // with log2(e)
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The sequence of a packed row, by a warp: the last s with cu[s] <= row; false where there is none
__device__ __forceinline__ bool find_seq(const TreeParams& p, int row, int& seq) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.n_seqs;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, s < hi && p.cu[s] <= row);
    lo += below ? (31 - __clz(below)) * step : 0;
    hi = min(hi, lo + step);
  }
  seq = lo;
  return p.cu[lo] <= row && row < p.cu[lo + 1];
}

// One row and KV head by four warps in 32-bit arithmetic, each warp every fourth row: lane l has the
// values D l .. D l + D - 1 of a head.
template <int HD, typename T>
__global__ void __launch_bounds__(128) tree_plain_kernel(const __grid_constant__ TreeParams p) {
  using B = Kv4Block<HD>;
  constexpr int D = HD / 32;
  __shared__ float joined[4][kMaxHpk][HD];
  __shared__ float tops[4][kMaxHpk], sums[4][kMaxHpk];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, kv = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = D * lane;
  int seq;
  if (!find_seq(p, row, seq)) return;
  const int r0 = p.cu[seq], r1 = p.cu[seq + 1];
  if (r0 < 0 || r1 > p.rows || r1 - r0 > kMaxNodes) {
    if (threadIdx.x == 0) flag_position(p.err);
    return;
  }
  int len = p.lens[seq];
  if (len < 0 || len > p.max_pages * kPageRows) {
    if (threadIdx.x == 0) flag_position(p.err);
    len = 0;
  }
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
    if (page < 0 || page >= p.n_pages) {
      if (lane == 0) flag_position(p.err);
      continue;
    }
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
    const int up = p.parents ? p.parents[r0 + node] : node - 1;
    if (up < -1 || up >= node) {
      if (threadIdx.x == 0) flag_position(p.err);
      break;
    }
    node = up;
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
  for (int i = threadIdx.x; i < p.hpk * HD; i += 128) {
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
}

template <int HD, typename T>
cudaError_t launch(const LaunchEnv& env, const TreeParams& p) {
  return rrr_launch_pdl(tree_plain_kernel<HD, T>, dim3((unsigned)p.rows, (unsigned)p.nkv), dim3(128), 0, env.stream, env.pdl, p);
}
template <int HD>
cudaError_t launch_type(const LaunchEnv& env, int type, const TreeParams& p) {
  return type == RRR_F16 ? launch<HD, __half>(env, p) : launch<HD, __nv_bfloat16>(env, p);
}

int check_tree(rrr_ctx* ctx, const rrr_kv4_cache* c, int n_heads, int rows, const char* fn) {
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  const int rc = check_kv4_cache(ctx, c, fn);
  if (rc) return rc;
  if (n_heads < 1 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > kMaxHpk)
    return set_error(ctx, RRR_ERR_BAD_SHAPE,
                     "%s: n_heads must be a multiple of n_kv_heads, at most 8 query heads per KV head", fn);
  if (rows < 0 || rows > 1 << 24) return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: need 0 <= rows <= 2^24", fn);
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
  *bytes = 256;
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
  cudaError_t e;
  switch (hd) {
    case 64: e = launch_type<64>(env, d->type, p); break;
    case 128: e = launch_type<128>(env, d->type, p); break;
    default: e = launch_type<256>(env, d->type, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_attention_tree_kv4 launch");
}

}  // extern "C"
