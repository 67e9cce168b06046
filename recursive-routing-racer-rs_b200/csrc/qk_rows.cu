// qk_rows.cu — packed QKV rows to rows of q, k and v: per-head RMS norm of queries and keys,
// rotation for the row's position and the rounding to the output type, in one pass
// (rrr_qk_norm_rope; apply_rope_cfg and rms_norm, src/model/phi4.rs:238-256, 593-599, are the
// reference's arithmetic of its parts).
//
// Mathematics. x' = (gamma x) / sqrt(mean(x^2) + eps); with c, s = af cos(2 pi t), af sin(2 pi
// t) a pair (a, b) becomes (a c - b s, a s + b c). t = pos * f / factor / 2 pi turns is wanted
// modulo 1 to 2^-24: f / factor / 2 pi is held modulo 1 as a 64-bit fraction F, and pos * F modulo
// 2^64 is exact in integers. sincospi of its top 32 bits, taken as a signed fraction, needs no range
// reduction; as a float it is off by 2^-25 turns at most. F comes from 64-bit floats: where f and 1 /
// factor are at most one it is off by less than 2^-52.5 turns (nine roundings of at most 2^-53 / 2 pi,
// those of the exponents included), which reaches the rest of 2^-24 at position 2^27.
//
// Bound by memory: each value is read once and written once. A warp owns a run of heads of one
// row, lane l the values D*l .. D*l + D - 1 (D = head_dim / 32) of each, so that a row's sines
// are computed once for all its heads and a partner of a pair (i, i + rope_dim/2) sits in
// another lane at the same place (rope_dim a multiple of 2D). Four heads are in flight per warp,
// and their sums of squares are reduced together: 16,000 rows of 48 heads of 128 values, f32 to
// bf16, take 100 us, 5.9 TB/s (124 us head by head, with the norm and the rotation decided per
// head). One row is 3 us of launch; it is spread over as many warps as it has fours of heads.
#include <math.h>

#include <type_traits>

#include "serve_common.cuh"

namespace rrr {
namespace {

constexpr int kMaxPairs = 64;
constexpr int kQkWarps = 4;
constexpr int kFew = 4;  // heads in flight per warp
// ... and of 128 values in 16 bits, where there are as many: 6,000 rows of 24 + 8 + 8 heads in bf16
// took 29.7 us with four at once and 23.9 with eight (with norms 33.0 and 28.6); heads of 64 and of
// 256 values, and of 32 bits, gain nothing
constexpr int kMany = 8;
template <int HD, typename TIN>
constexpr bool takes_many() { return HD == 128 && sizeof(TIN) == 2; }

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

template <int HD, bool HALVES, typename TIN, typename TOUT>
__global__ void __launch_bounds__(32 * kQkWarps) qk_rows_kernel(const __grid_constant__ QkParams p) {
  constexpr int D = HD / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, e0 = D * lane;
  const int item = blockIdx.x * kQkWarps + (threadIdx.x >> 5);
  const int row = item / p.chunks;
  if (row >= p.rows) return;
  const int h0 = (item - row * p.chunks) * p.chunk, h1 = min(h0 + p.chunk, p.heads);
  const int pos = p.positions[row];
  if (pos < 0 || pos >= p.max_pos) {
    if (h0 == 0 && lane == 0) flag_position(p.err);
    return;
  }
  // cos and sin of this lane's values; values outside the rotation keep theirs
  float cs[D], sn[D];
  bool turns[D];
#pragma unroll
  for (int d = 0; d < D; ++d) {
    const int e = e0 + d;
    turns[d] = e < 2 * p.half_dim;
    cs[d] = 1.f;
    sn[d] = 0.f;
    if (turns[d] && (HALVES || (d & 1) == 0)) {
      const int i = HALVES ? (e < p.half_dim ? e : e - p.half_dim) : e >> 1;
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
      if (HALVES && e < p.half_dim) sn[d] = -sn[d];
    }
  }
  const int hop = p.half_dim / D;  // lanes between the partners of (i, i + half)
  const int partner = (lane < hop ? lane + hop : lane - hop) & 31;
  const TIN* src = static_cast<const TIN*>(p.qkv) + row * p.row_stride + e0;

  // heads [a, b) of one kind; dst: where head a goes
  auto heads = [&](auto rotate, auto norm, int a, int b, TOUT* dst, const float* gamma) {
    float gm[D];
    if constexpr (decltype(norm)::value) {
#pragma unroll
      for (int d = 0; d < D; ++d) gm[d] = gamma[e0 + d];
    }
    auto some = [&](auto count, int h) {
      constexpr int kBatch = decltype(count)::value;
      float x[kBatch][D];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)  // (heads past the last are read as it)
        load_vec<TIN, D>(src + (int64_t)min(h + k, b - 1) * HD, x[k]);
      if constexpr (decltype(norm)::value) {
        float sq[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          sq[k] = 0.f;
#pragma unroll
          for (int d = 0; d < D; ++d) sq[k] = fmaf(x[k][d], x[k][d], sq[k]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int k = 0; k < kBatch; ++k) sq[k] += __shfl_xor_sync(0xffffffffu, sq[k], o);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const float inv = rsqrtf(fmaf(sq[k], 1.f / HD, p.eps));
#pragma unroll
          for (int d = 0; d < D; ++d) x[k][d] = (gm[d] * x[k][d]) * inv;
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if constexpr (decltype(rotate)::value && HALVES) {
#pragma unroll
          for (int d = 0; d < D; ++d) {
            const float o = __shfl_sync(0xffffffffu, x[k][d], partner);
            if (turns[d]) x[k][d] = fmaf(o, sn[d], x[k][d] * cs[d]);
          }
        } else if constexpr (decltype(rotate)::value) {
#pragma unroll
          for (int d = 0; d < D; d += 2) {
            const float u = x[k][d], v = x[k][d + 1];
            if (turns[d]) {
              x[k][d] = fmaf(-v, sn[d], u * cs[d]);
              x[k][d + 1] = fmaf(u, sn[d], v * cs[d]);
            }
          }
        }
        if (h + k < b) store_vec<TOUT, D>(dst + (int64_t)(h + k - a) * HD + e0, x[k]);
      }
    };
    int h = a;
    if constexpr (takes_many<HD, TIN>()) {
#pragma unroll 1
      for (; h + kMany <= b; h += kMany) some(std::integral_constant<int, kMany>{}, h);
    }
#pragma unroll 1
    for (; h < b; h += kFew) some(std::integral_constant<int, kFew>{}, h);
  };
  auto rotated = [&](int first, int count, void* out, int64_t stride, const float* gamma) {
    const int a = max(h0, first), b = min(h1, first + count);
    if (a >= b) return;
    TOUT* dst = static_cast<TOUT*>(out) + row * stride + (int64_t)(a - first) * HD;
    if (gamma)
      heads(std::true_type{}, std::true_type{}, a, b, dst, gamma);
    else
      heads(std::true_type{}, std::false_type{}, a, b, dst, gamma);
  };
  rotated(0, p.nh, p.q, p.q_stride, p.q_gamma);
  rotated(p.nh, p.nkv, p.k, p.k_stride, p.k_gamma);
  const int a = max(h0, p.nh + p.nkv);
  if (a < h1)
    heads(std::false_type{}, std::false_type{}, a, h1,
          static_cast<TOUT*>(p.v) + row * p.v_stride + (int64_t)(a - p.nh - p.nkv) * HD, nullptr);
}

template <int HD, typename TIN, typename TOUT>
cudaError_t launch(const LaunchEnv& env, dim3 grid, const QkParams& p) {
  const dim3 block(32 * kQkWarps);
  return p.halves ? rrr_launch_pdl(qk_rows_kernel<HD, true, TIN, TOUT>, grid, block, 0, env.stream, env.pdl, p)
                  : rrr_launch_pdl(qk_rows_kernel<HD, false, TIN, TOUT>, grid, block, 0, env.stream, env.pdl, p);
}
template <int HD, typename TIN>
cudaError_t launch_out(const LaunchEnv& env, int out_type, dim3 grid, const QkParams& p) {
  switch (out_type) {
    case RRR_F32: return launch<HD, TIN, float>(env, grid, p);
    case RRR_F16: return launch<HD, TIN, __half>(env, grid, p);
    default: return launch<HD, TIN, __nv_bfloat16>(env, grid, p);
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
  if (rows > 0 && (!qkv || !positions || !q || !k)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int hd = a->head_dim, nh = a->n_heads, nkv = a->n_kv_heads;
  if (rows < 0) return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows >= 0", fn);
  if (halves != 0 && halves != 1) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: halves is 0 or 1", fn);
  if (halves && a->rope_dim % (hd / 16))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rope_dim must be a multiple of head_dim / 16 with halves", fn);
  if (!(a->rope_theta > 0.f)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: rope_theta must be positive", fn);
  if (!(eps >= 0.f)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: eps must not be negative", fn);
  if (!stride_fits(row_stride, (int64_t)(nh + 2 * nkv) * hd) || !stride_fits(q_stride, (int64_t)nh * hd) ||
      !stride_fits(k_stride, (int64_t)nkv * hd) || (v && !stride_fits(v_stride, (int64_t)nkv * hd)))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: a row stride is shorter than its row, or over 2^38", fn);
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
  // theta^(-2i/rope_dim) / 2 pi as a product of two powers: 16 calls of pow and not 64
  double fine[8], coarse[kMaxPairs / 8];
  for (int i = 0; i < 8; ++i) fine[i] = pow((double)a->rope_theta, -2.0 * i / a->rope_dim);
  for (int i = 0; 8 * i < p.half_dim; ++i)
    coarse[i] = pow((double)a->rope_theta, -16.0 * i / a->rope_dim) / 6.283185307179586476925;
  for (int i = 0; i < p.half_dim; ++i) p.turns[i] = coarse[i / 8] * fine[i % 8];
  // all heads of a row in one warp once the rows alone fill the GPU's warps
  const int want = ctx->sm_count * 16;
  int chunks = (int)(((int64_t)want + rows - 1) / rows);
  const int most = (p.heads + kFew - 1) / kFew;
  chunks = chunks < 1 ? 1 : chunks > most ? most : chunks;
  p.chunk = (p.heads + chunks - 1) / chunks;
  p.chunk = (p.chunk + kFew - 1) / kFew * kFew;
  p.chunks = (p.heads + p.chunk - 1) / p.chunk;
  const int64_t blocks = ((int64_t)rows * p.chunks + kQkWarps - 1) / kQkWarps;
  if ((blocks + 1) * kQkWarps > INT32_MAX) return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: too many rows for one call", fn);
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
