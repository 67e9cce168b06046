// kv4_rows.cu — rows of the 4-bit KV cache (rrr_kv4_cache): packed K and V rows into its pages
// (rrr_kv4_store) and the values they stand for back into packed rows (rrr_kv4_load).
//
// Mathematics. A group of 32 values of a head becomes m = f16(min), d = f16((max - min) / 15)
// and codes round((x - m) / d), all with the f32 operations of that formula (no contraction,
// division rounded to nearest), so that a group's bits do not depend on where it is computed.
// The value read back is d*code + m: d*code is exact in f32 (11 + 4 bits), so it carries one
// rounding.
//
// Bound by memory: 2 bytes (16-bit rows) in and 5/8 out per value, or the reverse. One warp
// takes one (row, KV head): lane l holds the values D*l .. D*l + D - 1 of the head (D =
// head_dim / 32), a group is 32 / D lanes.
#include <math.h>

#include "kv4.cuh"

namespace rrr {

int check_kv4_cache(rrr_ctx* ctx, const rrr_kv4_cache* c, const char* fn) {
  if (!c || !c->pages || !c->page_table) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  if ((c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) || c->n_kv_heads < 1 ||
      c->n_kv_heads > 65535 || c->n_pages < 0 || c->n_seqs < 0 || c->max_pages < 0 ||
      c->max_pages > INT32_MAX / kPageRows || c->table_stride < c->max_pages ||
      (int64_t)c->n_seqs * c->n_kv_heads > INT32_MAX)
    return set_error(ctx, RRR_ERR_BAD_SHAPE,
                     "%s: need head_dim 64/128/256, 1 <= n_kv_heads <= 65535, counts >= 0, table_stride >= "
                     "max_pages, at most 2^31 - 64 rows per sequence and 2^31 - 1 sequences times heads",
                     fn);
  if (!aligned_to(c->pages, 16) || !aligned_to(c->page_table, 4))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: pages must be 16-byte aligned", fn);
  return RRR_OK;
}

namespace {

constexpr int kRowWarps = 8;

struct Kv4RowParams {
  uint8_t* pages;
  int64_t n_pages, table_stride;
  const int* table;
  int n_seqs, max_pages, nkv, rows;
  void* k;
  void* v;
  int64_t k_stride, v_stride;
  const int* cu;
  const int* lens;
  int* err;
};

// The block and the row in it of packed row `row`, KV head h; null when it has none.
template <int HD>
__device__ __forceinline__ uint8_t* find_row(const Kv4RowParams& p, int row, int h, int lane, int& in_page) {
  const int s = seq_of_row(p.cu, p.n_seqs, row);
  if (s < 0) return nullptr;  // behind the last sequence
  const int64_t pos = (int64_t)p.lens[s] - (p.cu[s + 1] - row);
  if (pos >= 0 && pos < (int64_t)p.max_pages * kPageRows) {
    const int page = p.table[(int64_t)s * p.table_stride + pos / kPageRows];
    if (page >= 0 && page < p.n_pages) {
      in_page = (int)(pos % kPageRows);
      return p.pages + ((int64_t)page * p.nkv + h) * Kv4Block<HD>::kBytes;
    }
  }
  if (lane == 0) flag_position(p.err);
  return nullptr;
}

// This lane's values of a head row as codes (4 bits each, value i at bit 4i) and the group's
// d and m, which every lane of the group gets.
template <int D>
__device__ __forceinline__ uint32_t quantise(const float (&x)[D], __half& d16, __half& m16) {
  constexpr int L = 32 / D;  // lanes per group
  float lo = x[0], hi = x[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < D; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad |= !(fabsf(x[i]) <= 3.402823466e38f);
  }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const unsigned lanes = __ballot_sync(0xffffffffu, bad) >> ((threadIdx.x & 31) & ~(L - 1));
  const bool any_bad = (lanes & (L == 32 ? 0xffffffffu : (1u << L) - 1u)) != 0;
  m16 = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
  d16 = __float2half_rn(fminf(__fdiv_rn(__fsub_rn(hi, lo), 15.f), 65504.f));
  if (any_bad) d16 = __ushort_as_half(0x7fff);
  const float d = __half2float(d16), m = __half2float(m16);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < D; ++i) {
    const float c = d > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[i], m), d)) : 0.f;
    codes |= (uint32_t)(int)fminf(fmaxf(c, 0.f), 15.f) << (4 * i);
  }
  return codes;
}

template <int HD, typename T>
__global__ void __launch_bounds__(32 * kRowWarps) kv4_store_kernel(const __grid_constant__ Kv4RowParams p) {
  using B = Kv4Block<HD>;
  constexpr int D = HD / 32, L = 32 / D;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int64_t row = item / p.nkv;
  if (row >= p.rows) return;
  const int h = (int)(item - row * p.nkv);
  int r;
  uint8_t* blk = find_row<HD>(p, (int)row, h, lane, r);
  if (!blk) return;
  const int j = lane / L, lg = lane % L;  // this lane's group and its place in it
  float x[D];
  __half d, m;
  load_vec<T, D>(static_cast<const T*>(p.k) + row * p.k_stride + (int64_t)h * HD + D * lane, x);
  uint32_t c = quantise<D>(x, d, m);
  {
    // the 8 elements of a word are 8 / D lanes
    uint8_t* codes = blk;
    const int t = lg * D / 8;
    if constexpr (D == 8)
      reinterpret_cast<uint32_t*>(codes)[B::k_word(r, j, t)] = c;
    else if constexpr (D == 4)
      reinterpret_cast<uint16_t*>(codes)[2 * B::k_word(r, j, t) + (lg & 1)] = (uint16_t)c;
    else
      codes[4 * B::k_word(r, j, t) + (lg & 3)] = (uint8_t)c;
    if (lg == 0) {
      reinterpret_cast<__half*>(blk + B::kCodes)[B::scale(r, j)] = d;
      reinterpret_cast<__half*>(blk + B::kCodes + B::kScales)[B::scale(r, j)] = m;
    }
  }
  load_vec<T, D>(static_cast<const T*>(p.v) + row * p.v_stride + (int64_t)h * HD + D * lane, x);
  c = quantise<D>(x, d, m);
  blk += B::kHalf;
  {
    // element e = 8n + g of the group is nibble n of half word g: every lane places its codes in
    // the eight half words (two per u32), the lanes of the group join them, and L lanes write
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const int e = lg * D + i, g = e & 7, n = e >> 3;
      const uint32_t v = ((c >> (4 * i)) & 15u) << (4 * n + 16 * (g & 1));
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q == g >> 1) w[q] |= v;
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] |= __shfl_xor_sync(0xffffffffu, w[q], o);
    uint16_t* codes = reinterpret_cast<uint16_t*>(blk);
#pragma unroll
    for (int g = 0; g < 8; ++g)
      if (g % L == lg) codes[B::v_half(r, j, g)] = (uint16_t)(w[g >> 1] >> (16 * (g & 1)));
    if (lg == 0) {
      reinterpret_cast<__half*>(blk + B::kCodes)[B::scale(r, j)] = d;
      reinterpret_cast<__half*>(blk + B::kCodes + B::kScales)[B::v_min(r, j)] = m;
    }
  }
}

template <int HD, typename T>
__global__ void __launch_bounds__(32 * kRowWarps) kv4_load_kernel(const __grid_constant__ Kv4RowParams p) {
  using B = Kv4Block<HD>;
  constexpr int D = HD / 32, L = 32 / D;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int64_t row = item / p.nkv;
  if (row >= p.rows) return;
  const int h = (int)(item - row * p.nkv);
  int r;
  const uint8_t* blk = find_row<HD>(p, (int)row, h, lane, r);
  if (!blk) return;
  const int j = lane / L, lg = lane % L;
  float x[D];
  if (p.k) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(blk)[B::k_word(r, j, lg * D / 8)];
    const float d = __half2float(reinterpret_cast<const __half*>(blk + B::kCodes)[B::scale(r, j)]);
    const float m = __half2float(reinterpret_cast<const __half*>(blk + B::kCodes + B::kScales)[B::scale(r, j)]);
#pragma unroll
    for (int i = 0; i < D; ++i) x[i] = fmaf((float)((w >> (4 * ((lg * D + i) & 7))) & 15u), d, m);
    store_vec<T, D>(static_cast<T*>(p.k) + row * p.k_stride + (int64_t)h * HD + D * lane, x);
  }
  if (p.v) {
    blk += B::kHalf;
    const float d = __half2float(reinterpret_cast<const __half*>(blk + B::kCodes)[B::scale(r, j)]);
    const float m = __half2float(reinterpret_cast<const __half*>(blk + B::kCodes + B::kScales)[B::v_min(r, j)]);
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const int e = lg * D + i;
      const uint32_t w = reinterpret_cast<const uint16_t*>(blk)[B::v_half(r, j, e & 7)];
      x[i] = fmaf((float)((w >> (4 * (e >> 3))) & 15u), d, m);
    }
    store_vec<T, D>(static_cast<T*>(p.v) + row * p.v_stride + (int64_t)h * HD + D * lane, x);
  }
}

template <int HD, typename T>
cudaError_t launch(const LaunchEnv& env, bool store, const Kv4RowParams& p) {
  const dim3 grid((unsigned)(((int64_t)p.rows * p.nkv + kRowWarps - 1) / kRowWarps)), block(32 * kRowWarps);
  return store ? rrr_launch_pdl(kv4_store_kernel<HD, T>, grid, block, 0, env.stream, env.pdl, p)
               : rrr_launch_pdl(kv4_load_kernel<HD, T>, grid, block, 0, env.stream, env.pdl, p);
}
template <int HD>
cudaError_t launch_type(const LaunchEnv& env, int type, bool store, const Kv4RowParams& p) {
  switch (type) {
    case RRR_F32: return launch<HD, float>(env, store, p);
    case RRR_F16: return launch<HD, __half>(env, store, p);
    default: return launch<HD, __nv_bfloat16>(env, store, p);
  }
}

int kv4_rows(rrr_ctx* ctx, const char* fn, bool store, const rrr_kv4_cache* c, int type, void* k,
             int64_t k_stride, void* v, int64_t v_stride, int rows, const int32_t* cu_rows,
             const int32_t* kv_lens, void* stream) {
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  int rc = check_kv4_cache(ctx, c, fn);
  if (rc) return rc;
  if (!row_type(type)) return set_error(ctx, RRR_ERR_BAD_QTYPE, "%s: type must be 0 (F32), 1 (F16) or 30 (BF16)", fn);
  if ((store ? !k || !v : !k && !v) || !cu_rows || !kv_lens)
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int64_t width = (int64_t)c->n_kv_heads * c->head_dim;
  if (rows < 0 || (int64_t)rows * c->n_kv_heads > (int64_t)INT32_MAX * kRowWarps || (k && k_stride < width) || (v && v_stride < width))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows >= 0 and strides of at least n_kv_heads * head_dim", fn);
  if (!aligned_to(k, 16) || !aligned_to(v, 16) || (k && k_stride % 8) || (v && v_stride % 8) ||
      !aligned_to(cu_rows, 4) || !aligned_to(kv_lens, 4))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: rows must be 16-byte aligned, strides multiples of 8 elements", fn);
  const int es = elem_bytes(type);
  const RowSet ks{k, k_stride * es, width * es, rows}, vs{v, v_stride * es, width * es, rows};
  const int64_t page_bytes = c->n_pages * c->n_kv_heads * 80 * c->head_dim;
  const RowSet pages{c->pages, page_bytes, page_bytes, page_bytes ? 1 : 0};
  if ((!store && !rows_disjoint(ks, vs)) || !rows_disjoint(ks, pages) || !rows_disjoint(vs, pages))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: the rows overlap each other or the pages", fn);
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  if (rows == 0 || c->n_seqs == 0) return RRR_OK;
  const LaunchEnv env = make_env(ctx, stream);
  const Kv4RowParams p{static_cast<uint8_t*>(c->pages), c->n_pages, c->table_stride, c->page_table, c->n_seqs,
                       c->max_pages, c->n_kv_heads, rows, k, v, k_stride, v_stride, cu_rows, kv_lens, env.d_err};
  cudaError_t e;
  switch (c->head_dim) {
    case 64: e = launch_type<64>(env, type, store, p); break;
    case 128: e = launch_type<128>(env, type, store, p); break;
    default: e = launch_type<256>(env, type, store, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, fn);
}

}  // namespace
}  // namespace rrr

using namespace rrr;

extern "C" {

int rrr_kv4_store(rrr_ctx* ctx, const rrr_kv4_cache* c, int type, const void* k, int64_t k_stride,
                  const void* v, int64_t v_stride, int rows, const int32_t* cu_rows,
                  const int32_t* kv_lens, void* stream) {
  return kv4_rows(ctx, "rrr_kv4_store", true, c, type, const_cast<void*>(k), k_stride, const_cast<void*>(v),
                  v_stride, rows, cu_rows, kv_lens, stream);
}

int rrr_kv4_load(rrr_ctx* ctx, const rrr_kv4_cache* c, int type, void* k, int64_t k_stride, void* v,
                 int64_t v_stride, int rows, const int32_t* cu_rows, const int32_t* kv_lens,
                 void* stream) {
  return kv4_rows(ctx, "rrr_kv4_load", false, c, type, k, k_stride, v, v_stride, rows, cu_rows, kv_lens, stream);
}

}  // extern "C"
