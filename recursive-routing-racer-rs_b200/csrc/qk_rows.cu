// qk_rows.cu — packed QKV rows to rows of q, k and v: per-head RMS norm of queries and keys,
// rotation for the row's position and the rounding to the output type, in one pass
// (rrr_qk_norm_rope; apply_rope_cfg and rms_norm, src/model/phi4.rs:238-256, 593-599, are the
// reference's arithmetic of its parts).
//
// Mathematics. x' = (gamma x) / sqrt(mean(x^2) + eps); with c, s = af cos(2 pi t), af sin(2 pi
// t) a pair (a, b) becomes (a c - b s, a s + b c). t = pos * f / factor / 2 pi turns is wanted
// modulo 1 to 2^-24 at any position: f / factor / 2 pi is held modulo 1 as a 64-bit fraction F
// (from 64-bit floats, so to 2^-53 of itself), and pos * F modulo 2^64 is exact in integers.
// sincospi of its top 32 bits, taken as a signed fraction, needs no range reduction.
//
// Bound by memory: each value is read once and written once. A warp owns a run of heads of one
// row, lane l the values D*l .. D*l + D - 1 (D = head_dim / 32) of each, so that a row's sines
// are computed once for all its heads and a partner of a pair (i, i + rope_dim/2) sits in
// another lane at the same place (rope_dim a multiple of 2D).
#include <math.h>

#include "serve_common.cuh"

namespace rrr {
namespace {

constexpr int kMaxPairs = 64;
constexpr int kQkWarps = 4;
constexpr int kBatch = 4;  // heads in flight per warp

struct QkParams {
  const void* qkv;
  int64_t row_stride, q_stride, k_stride, v_stride;
  void* q;
  void* k;
  void* v;
  const int* positions;
  const float* q_gamma;
  const float* k_gamma;
  const float* factors;
  int n_factors;
  int rows, nh, nkv, heads;  // heads: with or without V
  int chunk, chunks;         // heads per warp, warps per row
  int half_dim, halves, max_pos;
  float eps, attn_factor;
  int* err;
  double turns[kMaxPairs];  // theta^(-2i/rope_dim) / 2 pi
};

template <int HD, typename TIN, typename TOUT>
__global__ void __launch_bounds__(32 * kQkWarps) qk_rows_kernel(const __grid_constant__ QkParams p) {
  constexpr int D = HD / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kQkWarps + (threadIdx.x >> 5);
  const int64_t row = item / p.chunks;
  if (row >= p.rows) return;
  const int h0 = (int)(item - row * p.chunks) * p.chunk, h1 = min(h0 + p.chunk, p.heads);
  const int pos = p.positions[row];
  if (pos < 0 || pos >= p.max_pos) {
    if (h0 == 0 && lane == 0) flag_position(p.err);
    return;
  }
  // cos and sin of this lane's values; a value outside the rotation has (1, 0)
  float cs[D], sn[D];
  const int e0 = D * lane;
#pragma unroll
  for (int d = 0; d < D; ++d) {
    const int e = e0 + d;
    cs[d] = 1.f;
    sn[d] = 0.f;
    if (e < 2 * p.half_dim && (p.halves || (d & 1) == 0)) {
      const int i = p.halves ? (e < p.half_dim ? e : e - p.half_dim) : e >> 1;
      double t = p.turns[i];
      if (i < p.n_factors) t /= (double)p.factors[i];
      t -= floor(t);
      const unsigned long long F = __double2ull_rd(t * 18446744073709551616.0);
      const unsigned long long a = F * (unsigned long long)(unsigned)pos;
      const float frac = (float)(int)(unsigned)(a >> 32) * 4.656612873077393e-10f;  // 2 x turns, in [-1, 1)
      float s, c;
      sincospif(frac, &s, &c);
      cs[d] = c * p.attn_factor;
      sn[d] = s * p.attn_factor;
      // the first of a pair subtracts its partner's product, the second adds it
      if (p.halves && e < p.half_dim) sn[d] = -sn[d];
    }
  }
  const int hop = p.half_dim / D;  // lanes between the partners of (i, i + half)
  const int partner = lane < hop ? lane + hop : lane - hop;
  const TIN* src = static_cast<const TIN*>(p.qkv) + row * p.row_stride;
  for (int h = h0; h < h1; h += kBatch) {
    float x[kBatch][D];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (h + b < h1) load_vec<TIN, D>(src + (int64_t)(h + b) * HD + e0, x[b]);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int hb = h + b;
      if (hb >= h1) break;
      TOUT* dst;
      if (hb < p.nh)
        dst = static_cast<TOUT*>(p.q) + row * p.q_stride + (int64_t)hb * HD;
      else if (hb < p.nh + p.nkv)
        dst = static_cast<TOUT*>(p.k) + row * p.k_stride + (int64_t)(hb - p.nh) * HD;
      else
        dst = static_cast<TOUT*>(p.v) + row * p.v_stride + (int64_t)(hb - p.nh - p.nkv) * HD;
      if (hb < p.nh + p.nkv) {
        const float* gamma = hb < p.nh ? p.q_gamma : p.k_gamma;
        if (gamma) {
          float sq = 0.f;
#pragma unroll
          for (int d = 0; d < D; ++d) sq = fmaf(x[b][d], x[b][d], sq);
          const float inv = 1.f / sqrtf(warp_sum(sq) * (1.f / HD) + p.eps);
#pragma unroll
          for (int d = 0; d < D; ++d) x[b][d] = (gamma[e0 + d] * x[b][d]) * inv;
        }
        if (p.halves) {
#pragma unroll
          for (int d = 0; d < D; ++d) {
            const float o = __shfl_sync(0xffffffffu, x[b][d], partner & 31);
            if (e0 + d < 2 * p.half_dim) x[b][d] = fmaf(o, sn[d], x[b][d] * cs[d]);
          }
        } else {
#pragma unroll
          for (int d = 0; d < D; d += 2)
            if (e0 + d < 2 * p.half_dim) {
              const float a = x[b][d], c = x[b][d + 1];
              x[b][d] = fmaf(-c, sn[d], a * cs[d]);
              x[b][d + 1] = fmaf(a, sn[d], c * cs[d]);
            }
        }
      }
      store_vec<TOUT, D>(dst + e0, x[b]);
    }
  }
}

template <int HD, typename TIN>
cudaError_t launch_out(const LaunchEnv& env, int out_type, dim3 grid, const QkParams& p) {
  const dim3 block(32 * kQkWarps);
  switch (out_type) {
    case RRR_F32: return rrr_launch_pdl(qk_rows_kernel<HD, TIN, float>, grid, block, 0, env.stream, env.pdl, p);
    case RRR_F16: return rrr_launch_pdl(qk_rows_kernel<HD, TIN, __half>, grid, block, 0, env.stream, env.pdl, p);
    default:
      return rrr_launch_pdl(qk_rows_kernel<HD, TIN, __nv_bfloat16>, grid, block, 0, env.stream, env.pdl, p);
  }
}
template <int HD>
cudaError_t launch_in(const LaunchEnv& env, int in_type, int out_type, dim3 grid, const QkParams& p) {
  switch (in_type) {
    case RRR_F32: return launch_out<HD, float>(env, out_type, grid, p);
    case RRR_F16: return launch_out<HD, __half>(env, out_type, grid, p);
    default: return launch_out<HD, __nv_bfloat16>(env, out_type, grid, p);
  }
}

}  // namespace
}  // namespace rrr

using namespace rrr;

extern "C" int rrr_qk_norm_rope(rrr_ctx* ctx, const rrr_attn_desc* a, int in_type, const void* qkv,
                                int64_t row_stride, int rows, const int32_t* positions,
                                const float* q_gamma, const float* k_gamma, float eps, int halves,
                                int out_type, void* q, int64_t q_stride, void* k, int64_t k_stride,
                                void* v, int64_t v_stride, void* stream) {
  const char* fn = "rrr_qk_norm_rope";
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  int rc = check_attn_desc(ctx, a, fn);
  if (rc) return rc;
  if (!row_type(in_type) || !row_type(out_type))
    return set_error(ctx, RRR_ERR_BAD_QTYPE, "%s: types must be 0 (F32), 1 (F16) or 30 (BF16)", fn);
  if (!qkv || !positions || !q || !k) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int hd = a->head_dim, nh = a->n_heads, nkv = a->n_kv_heads;
  if (rows < 0) return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows >= 0", fn);
  if (halves != 0 && halves != 1) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: halves is 0 or 1", fn);
  if (halves && a->rope_dim % (hd / 16))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rope_dim must be a multiple of head_dim / 16 with halves", fn);
  if (!(a->rope_theta > 0.f)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: rope_theta must be positive", fn);
  if (!(eps >= 0.f)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: eps must not be negative", fn);
  if (row_stride < (int64_t)(nh + 2 * nkv) * hd || q_stride < (int64_t)nh * hd ||
      k_stride < (int64_t)nkv * hd || (v && v_stride < (int64_t)nkv * hd))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: a row stride is shorter than its row", fn);
  if (!aligned_to(qkv, 16) || !aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(v, 16) ||
      row_stride % 8 || q_stride % 8 || k_stride % 8 || (v && v_stride % 8) || !aligned_to(positions, 4) ||
      !aligned_to(q_gamma, 4) || !aligned_to(k_gamma, 4))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: rows must be 16-byte aligned, strides multiples of 8 elements", fn);
  // each output is its own part of qkv, in place, or shares nothing with qkv and the others
  const int ei = elem_bytes(in_type), eo = elem_bytes(out_type);
  const RowSet in{qkv, row_stride * ei, (int64_t)(nh + 2 * nkv) * hd * ei, rows};
  const RowSet out[3] = {{q, q_stride * eo, (int64_t)nh * hd * eo, rows},
                         {k, k_stride * eo, (int64_t)nkv * hd * eo, rows},
                         {v, v_stride * eo, (int64_t)nkv * hd * eo, rows}};
  const int first[3] = {0, nh, nh + nkv};
  bool own_place[3];
  for (int i = 0; i < 3; ++i) {
    own_place[i] = out[i].p && in_type == out_type && (rows <= 1 || out[i].stride == in.stride) &&
                   out[i].p == static_cast<const char*>(qkv) + (int64_t)first[i] * hd * ei;
    bool fine = own_place[i] || rows_disjoint(in, out[i]);
    for (int j = 0; j < i; ++j) fine = fine && rows_disjoint(out[i], out[j]);
    if (!fine)
      return set_error(ctx, RRR_ERR_INVALID_ARG,
                       "%s: q, k and v must lie in their own place in qkv or overlap nothing", fn);
  }
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  if (rows == 0) return RRR_OK;
  QkParams p{};
  p.qkv = qkv;
  p.row_stride = row_stride;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.q = q;
  p.k = k;
  p.v = v;
  p.positions = positions;
  p.q_gamma = q_gamma;
  p.k_gamma = k_gamma;
  p.factors = a->rope_factors;
  p.n_factors = a->rope_factors ? a->n_rope_factors : 0;
  p.rows = rows;
  p.nh = nh;
  p.nkv = nkv;
  p.heads = nh + nkv + (v && !own_place[2] ? nkv : 0);
  p.half_dim = a->rope_dim / 2;
  p.halves = halves;
  p.max_pos = a->max_seq;
  p.eps = eps;
  p.attn_factor = a->rope_attn_factor;
  for (int i = 0; i < p.half_dim; ++i)
    p.turns[i] = pow((double)a->rope_theta, -2.0 * i / a->rope_dim) / 6.283185307179586476925;
  // all heads of a row in one warp once the rows alone fill the GPU's warps
  const int want = ctx->sm_count * 16;
  int chunks = (want + rows - 1) / rows;
  const int most = (p.heads + kBatch - 1) / kBatch;
  chunks = chunks < 1 ? 1 : chunks > most ? most : chunks;
  p.chunk = (p.heads + chunks - 1) / chunks;
  p.chunk = (p.chunk + kBatch - 1) / kBatch * kBatch;
  p.chunks = (p.heads + p.chunk - 1) / p.chunk;
  const int64_t blocks = ((int64_t)rows * p.chunks + kQkWarps - 1) / kQkWarps;
  const LaunchEnv env = make_env(ctx, stream);
  p.err = env.d_err;
  cudaError_t e;
  const dim3 grid((unsigned)blocks);
  switch (hd) {
    case 64: e = launch_in<64>(env, in_type, out_type, grid, p); break;
    case 128: e = launch_in<128>(env, in_type, out_type, grid, p); break;
    default: e = launch_in<256>(env, in_type, out_type, grid, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_qk_norm_rope launch");
}
