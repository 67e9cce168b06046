// kv4_append.cu — QKV rows into the 4-bit KV cache, with the rotation on the way
// (rrr_kv4_append): the rope_kv_store dispatch of the decode step (src/model/phi4.rs:1117-1119,
// 1284-1300) for packed rows and pages.
//
// Mathematics. qk_rows.cu's norm and rotation in 32 bits and kv4_rows.cu's groups of 32 values; the
// rotated K is quantised from its 32-bit value, without the rounding to a 16-bit row between. A
// code changes by a whole step where a value crosses a border, so that groups which 32 bits do not
// decide (the step, the minimum or a code within the arithmetic's error of a rounding border: about
// one group in a hundred; and all groups of a head whose squares leave the range of 32 bits) are normed
// and rotated again in 64 bits, as all others then would be too.
//
// A CTA takes up to eight rows of one sequence that lie in eight aligned rows of a page (two rows
// whose V codes share words are then one warp's), and a share of the heads. The rows' sines and
// cosines are computed once, into shared memory; a warp keeps those of its rows in registers and
// goes through heads of q and K, whose values it loads some heads ahead: lane (j, t) the values
// 32j + 8t .. + 7 of a row, which are one word of K's codes. Partners that lie half a rotation away
// come by shuffles.
//
// What bounds it. Instructions: 5,949 rows of 48 heads of 128, bf16 with norms, 60 us (151 MB, 23 us at the copy's rate),
// 260 instructions for eight values of 32 lanes on average, of which K and V take four fifths; 64 single rows 7.2 us,
// five dependent trips to memory. The 64-bit rotation takes 9 us of the 60; with sines computed again for each group it took
// 45.
#include "kv4.cuh"

namespace rrr {
namespace {

constexpr int kAppendWarps = 8, kBlockRows = 8;

struct AppendParams {
  const void* qkv;
  int64_t row_stride, q_stride;
  void* q;
  uint8_t* pages;
  int64_t n_pages, table_stride;
  const int* table;
  int n_seqs, max_pages, nh, nkv, rows, slots;
  const int* cu;
  const int* lens;
  const int* path;
  const int* counts;
  const int* positions;
  const float* q_gamma;
  const float* k_gamma;
  const float* factors;
  int n_factors;
  int half_dim, halves, max_pos;
  float eps, attn_factor;
  int* err;
  double turns[kMaxPairs];  // theta^(-2i/rope_dim) / 2 pi
};

// The rows of a CTA: rows in_page .. in_page + n - 1 of a page, of a sequence whose packed rows
// start at row0; the first of them is the sequence's appended row nth.
struct Rows {
  int64_t page;
  int row0, held, nth, at, n;  // held: packed rows of the sequence; at: the first's place in the cache
};
// Slot x belongs to the last sequence s with cu[s] / R + 2 s <= x (sequences get disjoint runs of
// slots that are long enough), searched by the warp 32 sequences at a time.
__device__ __forceinline__ bool find_rows(const AppendParams& p, int x, Rows& b) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.n_seqs;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + lane * step;
    const bool at = s < hi && p.cu[s] / kBlockRows + 2 * s <= x;
    const unsigned below = __ballot_sync(0xffffffffu, at);
    lo += below ? (31 - __clz(below)) * step : 0;
    hi = min(hi, lo + step);
  }
  const int r0 = p.cu[lo], r1 = p.cu[lo + 1], len = p.lens[lo], most = p.max_pages * kPageRows;
  const int rows = p.counts ? p.counts[lo] : r1 - r0;
  if (r0 < 0 || r1 < r0 || r1 > p.rows || rows < 0 || rows > r1 - r0) {
    if (lane == 0) flag_position(p.err);
    return false;
  }
  if (rows > 0 && (len < rows || len > most) && lane == 0) flag_position(p.err);
  // (rows at places that do not exist are left out)
  const int k = x - (r0 / kBlockRows + 2 * lo);  // the block among the sequence's
  if (k < 0 || len <= 0 || rows <= 0) return false;
  const int pos0 = len - rows, first = max(pos0, 0), end = min(len, most);
  const int64_t start = (int64_t)(first / kBlockRows + (int64_t)k) * kBlockRows;
  if (start >= end) return false;
  const int from = max(first, (int)start), to = min(end, (int)start + kBlockRows);
  if (from >= to) return false;
  b.page = p.table[(int64_t)lo * p.table_stride + from / kPageRows];
  if (b.page < 0 || b.page >= p.n_pages) {
    if (lane == 0) flag_position(p.err);
    return false;
  }
  b.row0 = r0;
  b.held = r1 - r0;
  b.nth = from - pos0;
  b.at = from;
  b.n = to - from;
  return true;
}

// Eight values (from e0) of a key head whose row starts at src, normed and rotated in 64 bits; turn:
// the row's cosines and sines. All lanes of a warp call it together.
template <int HD, typename TIN>
__device__ __forceinline__ void rotated_in_64_bits(const AppendParams& p, const TIN* src, const double2* turn, int e0,
                                                   float (&x)[8]) {
  const int half = p.half_dim;
  float v[8];
  load_vec<TIN, 8>(src + e0, v);
  double inv = 1.0;
  if (p.k_gamma) {
    double sq = 0.0;
#pragma unroll
    for (int d = 0; d < 8; ++d) sq = fma((double)v[d], (double)v[d], sq);
#pragma unroll
    for (int k = 1; k < HD / 8; k <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, k);
    inv = rsqrt(sq / HD + (double)p.eps);
  }
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    const int e = e0 + d;
    double z = (double)v[d] * inv;
    if (p.k_gamma) z *= (double)p.k_gamma[e];
    if (e < 2 * half) {
      const bool first = p.halves ? e < half : d % 2 == 0;
      const int f = p.halves ? (first ? e + half : e - half) : e ^ 1, i = p.halves ? min(e, f) : e / 2;
      const double2 w = turn[i];
      double y = (double)to_f32(src[f]) * inv;
      if (p.k_gamma) y *= (double)p.k_gamma[f];
      z = z * w.x + (first ? -w.y : w.y) * y;
    }
    x[d] = (float)z;
  }
}

template <int HD, typename TIN, typename TOUT>
__global__ void __launch_bounds__(32 * kAppendWarps, 3) kv4_append_kernel(const __grid_constant__ AppendParams p) {
  using B = Kv4Block<HD>;
  constexpr int G = B::kGroups, kLanes = 4 * G;   // lanes of a row
  constexpr int kRows = 32 / kLanes;              // rows of a warp
  constexpr int kAhead = 4, kParts = sizeof(TIN) / 2;  // heads whose values are on their way, 16 bytes each
  __shared__ uint4 ahead[kAppendWarps][kAhead][kParts][32];
  __shared__ Rows found;
  __shared__ int source[kBlockRows], place[kBlockRows];
  __shared__ double turns[kMaxPairs];
  __shared__ __align__(16) float2 turn[kBlockRows][kMaxPairs];
  __shared__ __align__(16) double2 turn64[kBlockRows][kMaxPairs];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = p.half_dim;
  if (warp == 0) {
    Rows b;
    b.n = 0;
    if (!find_rows(p, (int)blockIdx.x, b)) b.n = 0;
    if (lane < b.n) {
      int i = b.nth + lane;
      if (p.path) i = p.path[b.row0 + i];
      int row = i >= 0 && i < b.held ? b.row0 + i : -1;
      const int pos = row < 0 ? -1 : p.positions ? p.positions[row] : b.at + lane;
      if (pos < 0 || pos >= p.max_pos) row = -1;
      if (row < 0) flag_position(p.err);
      source[lane] = row;
      place[lane] = max(pos, 0);
    }
    if (lane == 0) found = b;
  } else {
    for (int i = threadIdx.x - 32; i < half; i += 32 * (kAppendWarps - 1))
      turns[i] = i < p.n_factors ? p.turns[i] / (double)p.factors[i] : p.turns[i];
  }
  __syncthreads();
  const Rows b = found;
  if (b.n == 0) return;
  for (int x = threadIdx.x; x < b.n * half; x += 32 * kAppendWarps) {
    const int r = x / half, i = x - r * half;
    float c, s;
    rope_turn(turns[i], place[r], p.attn_factor, c, s);
    turn[r][i] = make_float2(c, s);
    double c64, s64;
    rope_turn(turns[i], place[r], (double)p.attn_factor, c64, s64);
    turn64[r][i] = make_double2(c64, s64);
  }
  __syncthreads();
  const int in_page = b.at % kPageRows;
  const int j = lane / 4 % G, t = lane % 4, set = lane / kLanes, e0 = 32 * j + 8 * t;
  const TIN* qkv = static_cast<const TIN*>(p.qkv);

  // q and K: a warp takes kRows rows and every `stride`th head of them
  const int sets = (b.n + kRows - 1) / kRows, share = kAppendWarps / sets;  // warps of the same rows
  if (warp < sets * share) {
    const int nq = p.q ? p.nh : 0, heads = nq + p.nkv, stride = share * gridDim.y;
    const int r = warp % sets * kRows + set, rr = min(r, b.n - 1);  // (rows past the last are read as it)
    const int row = source[rr];
    const TIN* src = qkv + (int64_t)max(row, 0) * p.row_stride + e0;
    const bool paired = p.halves && half % 8 == 0;
    const int hop = e0 < half ? half : e0 < 2 * half ? -half : 0;  // where the partners lie (paired)
    float c[8], s[8];  // of the lane's values
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const int i = !p.halves ? (e0 + d) / 2 : e0 + d < half ? e0 + d : e0 + d - half;
      const bool turns_too = e0 + d < 2 * half;
      const float2 w = turns_too ? turn[rr][i] : make_float2(1.f, 0.f);
      c[d] = w.x;
      s[d] = (p.halves ? e0 + d < half : d % 2 == 0) ? -w.y : w.y;
    }
    // what the 32-bit norm and rotation can be off by, in units of the largest value: of a value
    // and its partner each 2^-21.7 (angle 2^-23.3, sine 2^-23, factor and products 2^-24 each);
    // with norms 2^-19.9 more (13 additions of squares, half of which counts, and the root)
    const float off = fmaxf(fabsf(p.attn_factor), 1.f) * (p.k_gamma ? 1.f / 524288 : 1.f / 1048576);
    float gamma[8];
    const TIN* heads_at = src + (p.q ? 0 : (int64_t)p.nh * HD);
    int k = warp / sets * gridDim.y + blockIdx.y;
    auto fetch = [&](int at, int slot) {
      if (at < heads)
#pragma unroll
        for (int n = 0; n < kParts; ++n) cp_async16(&ahead[warp][slot][n][lane], heads_at + (int64_t)at * HD + 8 / kParts * n);
      cp_async_commit();
    };
#pragma unroll
    for (int a = 0; a < kAhead - 1; ++a) fetch(k + a * stride, a);
#pragma unroll 1
    for (int nth = 0, key = -1; k < heads; k += stride, ++nth) {
      const bool normed = k >= nq ? p.k_gamma : p.q_gamma;
      if (key != (k >= nq)) {
        key = k >= nq;
        const float* of = key ? p.k_gamma : p.q_gamma;
#pragma unroll
        for (int d = 0; d < 8; ++d) gamma[d] = of ? of[e0 + d] : 1.f;
      }
      fetch(k + (kAhead - 1) * stride, (nth + kAhead - 1) % kAhead);  // where the last head's values were
      cp_async_wait<kAhead - 1>();
      Vec<TIN, 8> now;
#pragma unroll
      for (int n = 0; n < kParts; ++n)
        reinterpret_cast<uint4*>(&now)[n] = ahead[warp][nth % kAhead][n][lane];
      float x[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) x[d] = to_f32(now.v[d]);
      float inv = 1.f, ground = 1.f;
      if (normed) {
        float sq = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) sq = fmaf(x[d], x[d], sq);
#pragma unroll
        for (int m = 1; m < kLanes; m <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
        ground = fmaf(sq, 1.f / HD, p.eps);
        inv = rsqrtf(ground);
#pragma unroll
        for (int d = 0; d < 8; ++d) x[d] = (gamma[d] * x[d]) * inv;
      }
      float largest = 0.f;  // of the lane's values and their partners
      if (key)
#pragma unroll
      for (int d = 0; d < 8; ++d) largest = fmaxf(largest, fabsf(x[d]));
      if (!p.halves) {
#pragma unroll
        for (int d = 0; d < 8; d += 2) {
          const float u = x[d], v = x[d + 1];
          if (e0 + d < 2 * half) {
            x[d] = fmaf(v, s[d], u * c[d]);
            x[d + 1] = fmaf(u, s[d + 1], v * c[d + 1]);
          }
        }
      } else if (paired) {
        float y[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) y[d] = __shfl_sync(0xffffffffu, x[d], lane + hop / 8);
        if (key) largest = fmaxf(largest, __shfl_sync(0xffffffffu, largest, lane + hop / 8));
        if (hop)
#pragma unroll
          for (int d = 0; d < 8; ++d) x[d] = fmaf(y[d], s[d], x[d] * c[d]);
      } else {  // pairs that lie across lanes' borders
        const TIN* head = src - e0 + (int64_t)(key ? p.nh + k - nq : k) * HD;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const int e = e0 + d;
          if (e < 2 * half) {
            const int f = e < half ? e + half : e - half;
            float y = to_f32(head[f]);
            if (normed) y = ((key ? p.k_gamma : p.q_gamma)[f] * y) * inv;
            largest = fmaxf(largest, fabsf(y));
            x[d] = fmaf(y, s[d], x[d] * c[d]);
          }
        }
      }
      const bool stored = r < b.n && row >= 0;
      if (!key) {
        if (stored) store_vec<TOUT, 8>(static_cast<TOUT*>(p.q) + row * p.q_stride + (int64_t)k * HD + e0, x);
        continue;
      }
#pragma unroll
      for (int m = 1; m < 4; m <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, m));
      const int h = k - nq;
      __half d16, m16;
      bool unsure;
      uint32_t w = quantise<true>(x, d16, m16, off * largest, &unsure);
      // (and where 32 bits do not hold the squares or the largest values at all)
      unsure = unsure || !(ground > 7.9e-31f && ground < 1e38f) || !(off * largest < 1e30f);
      if (__any_sync(0xffffffffu, unsure)) {
        rotated_in_64_bits<HD>(p, src - e0 + (int64_t)(p.nh + h) * HD, turn64[rr], e0, x);
        w = quantise(x, d16, m16);
      }
      if (stored) {
        uint8_t* blk = p.pages + (b.page * p.nkv + h) * B::kBytes;
        reinterpret_cast<uint32_t*>(blk)[B::k_word(in_page + r, j, t)] = w;
        if (t == 0) {
          reinterpret_cast<__half*>(blk + B::kCodes)[B::scale(in_page + r, j)] = d16;
          reinterpret_cast<__half*>(blk + B::kCodes + B::kScales)[B::scale(in_page + r, j)] = m16;
        }
      }
    }
  }

  // V: a warp takes a head of kRows pairs of rows whose codes share words
  const int g = 2 * t, odd_first = in_page & 1, pairs = (b.n + odd_first + 1) / 2, turns_of = (pairs + kRows - 1) / kRows;
  const int tasks = p.nkv * turns_of, first = (kAppendWarps - 1 - warp) * gridDim.y + blockIdx.y;
#pragma unroll 1
  for (int task = first; task < tasks; task += kAppendWarps * gridDim.y) {
    const int h = task / turns_of, u = task % turns_of * kRows + set;
    uint8_t* vb = p.pages + (b.page * p.nkv + h) * B::kBytes + B::kHalf;
    const TIN* src = qkv + (int64_t)(p.nh + p.nkv + h) * HD + 32 * j + g;
    const int r = 2 * min(u, pairs - 1) - odd_first, row = in_page + r;  // the pair's even row
    uint32_t c[2];
    bool has[2];
    float v[2][8];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int from = source[min(max(r + o, 0), b.n - 1)];
      has[o] = u < pairs && r + o >= 0 && r + o < b.n && from >= 0;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float two[2];
        load_vec<TIN, 2>(src + (int64_t)max(from, 0) * p.row_stride + 8 * n, two);
        v[o][2 * n] = two[0];
        v[o][2 * n + 1] = two[1];
      }
    }
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      __half d, m;
      c[o] = quantise(v[o], d, m);
      if (t == 0 && has[o]) {
        reinterpret_cast<__half*>(vb + B::kCodes)[B::scale(row + o, j)] = d;
        reinterpret_cast<__half*>(vb + B::kCodes + B::kScales)[B::v_min(row + o, j)] = m;
      }
    }
    // nibbles 0, 2, 4, 6 are g's, the others g + 1's: four each to a half word
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t w[2];
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        uint32_t y = (c[o] >> (4 * e)) & 0x0f0f0f0fu;
        y = (y | y >> 4) & 0x00ff00ffu;
        w[o] = (y | y >> 8) & 0xffffu;
      }
      uint16_t* codes = reinterpret_cast<uint16_t*>(vb);
      if (has[0] && has[1])
        reinterpret_cast<uint32_t*>(vb)[B::v_half(row, j, g + e) / 2] = w[0] | w[1] << 16;
      else if (has[0])
        codes[B::v_half(row, j, g + e)] = (uint16_t)w[0];
      else if (has[1])
        codes[B::v_half(row + 1, j, g + e)] = (uint16_t)w[1];
    }
  }
}

template <int HD, typename TIN>
cudaError_t launch_out(const LaunchEnv& env, int out_type, dim3 grid, const AppendParams& p) {
  const dim3 block(32 * kAppendWarps);
  switch (out_type) {
    case RRR_F32: return rrr_launch_pdl(kv4_append_kernel<HD, TIN, float>, grid, block, 0, env.stream, env.pdl, p);
    case RRR_F16: return rrr_launch_pdl(kv4_append_kernel<HD, TIN, __half>, grid, block, 0, env.stream, env.pdl, p);
    default: return rrr_launch_pdl(kv4_append_kernel<HD, TIN, __nv_bfloat16>, grid, block, 0, env.stream, env.pdl, p);
  }
}
template <int HD>
cudaError_t launch_in(const LaunchEnv& env, int in_type, int out_type, dim3 grid, const AppendParams& p) {
  switch (in_type) {
    case RRR_F32: return launch_out<HD, float>(env, out_type, grid, p);
    case RRR_F16: return launch_out<HD, __half>(env, out_type, grid, p);
    default: return launch_out<HD, __nv_bfloat16>(env, out_type, grid, p);
  }
}

}  // namespace
}  // namespace rrr

using namespace rrr;

extern "C" int rrr_kv4_append(rrr_ctx* ctx, const rrr_attn_desc* a, const rrr_kv4_cache* c, int in_type,
                              const void* qkv, int64_t row_stride, int rows, const int32_t* cu_rows,
                              const int32_t* kv_lens, const int32_t* path, const int32_t* counts,
                              const int32_t* positions, const float* q_gamma, const float* k_gamma, float eps,
                              int halves, int out_type, void* q, int64_t q_stride, void* stream) {
  const char* fn = "rrr_kv4_append";
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  int rc = check_attn_desc(ctx, a, fn);
  if (rc || (rc = check_kv4_cache(ctx, c, fn))) return rc;
  if (!row_type(in_type) || (q && !row_type(out_type)))
    return set_error(ctx, RRR_ERR_BAD_QTYPE, "%s: types must be 0 (F32), 1 (F16) or 30 (BF16)", fn);
  if ((rows > 0 && !qkv) || (c->n_seqs > 0 && (!cu_rows || !kv_lens)))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (!path != !counts || (path && q))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: path and counts come together, and without q", fn);
  const int hd = a->head_dim, nh = a->n_heads, nkv = a->n_kv_heads;
  if (hd != c->head_dim || nkv != c->n_kv_heads)
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: the cache has other KV heads than the rows", fn);
  if (rows < 0 || rows > INT32_MAX / 4 || c->n_seqs > INT32_MAX / 8)
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows >= 0, and not too many rows and sequences for one call", fn);
  if (halves != 0 && halves != 1) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: halves is 0 or 1", fn);
  if (halves && a->rope_dim % (hd / 16))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rope_dim must be a multiple of head_dim / 16 with halves", fn);
  if (!(a->rope_theta > 0.f)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: rope_theta must be positive", fn);
  if (!(eps >= 0.f)) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: eps must not be negative", fn);
  if (!stride_fits(row_stride, (int64_t)(nh + 2 * nkv) * hd) || (q && !stride_fits(q_stride, (int64_t)nh * hd)))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: a row stride is shorter than its row, or over 2^38", fn);
  if (!aligned_to(qkv, 16) || !aligned_to(q, 16) || row_stride % 8 || (q && q_stride % 8) || !aligned_to(cu_rows, 4) ||
      !aligned_to(kv_lens, 4) || !aligned_to(path, 4) || !aligned_to(counts, 4) || !aligned_to(positions, 4) ||
      !aligned_to(q_gamma, 4) || !aligned_to(k_gamma, 4))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: rows must be 16-byte aligned, strides multiples of 8 elements", fn);
  const int ei = elem_bytes(in_type), eo = elem_bytes(out_type);
  const int64_t page_bytes = c->n_pages * c->n_kv_heads * 80 * hd;
  const RowSet in{qkv, row_stride * ei, (int64_t)(nh + 2 * nkv) * hd * ei, rows};
  const RowSet out{q, q_stride * eo, (int64_t)nh * hd * eo, rows}, pages{c->pages, page_bytes, page_bytes, page_bytes ? 1 : 0};
  if (!rows_disjoint(in, out) || !rows_disjoint(in, pages) || !rows_disjoint(out, pages))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: the rows, q and the pages must not overlap", fn);
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  if (rows == 0 || c->n_seqs == 0) return RRR_OK;
  AppendParams p{};
  p.qkv = qkv;
  p.row_stride = row_stride;
  p.q_stride = q_stride;
  p.q = q;
  p.pages = static_cast<uint8_t*>(c->pages);
  p.n_pages = c->n_pages;
  p.table_stride = c->table_stride;
  p.table = c->page_table;
  p.n_seqs = c->n_seqs;
  p.max_pages = c->max_pages;
  p.nh = nh;
  p.nkv = nkv;
  p.rows = rows;
  p.cu = cu_rows;
  p.lens = kv_lens;
  p.path = path;
  p.counts = counts;
  p.positions = positions;
  p.q_gamma = q_gamma;
  p.k_gamma = k_gamma;
  p.factors = a->rope_factors;
  p.n_factors = a->rope_factors ? a->n_rope_factors : 0;
  p.half_dim = a->rope_dim / 2;
  p.halves = halves;
  p.max_pos = a->max_seq;
  p.eps = eps;
  p.attn_factor = a->rope_attn_factor;
  rope_turns(p.turns, a->rope_theta, a->rope_dim);
  p.slots = rows / kBlockRows + 2 * c->n_seqs;
  // a CTA takes all heads of its rows once the blocks of rows alone fill the SMs
  const int tasks = 2 * nkv + (q ? nh : 0), most = (tasks + kAppendWarps - 1) / kAppendWarps;
  const int64_t blocks = (int64_t)rows / kBlockRows + c->n_seqs;
  int64_t shares = (4 * (int64_t)ctx->sm_count + blocks - 1) / blocks;
  if (shares > most) shares = most;
  const LaunchEnv env = make_env(ctx, stream);
  p.err = env.d_err;
  cudaError_t e;
  const dim3 grid((unsigned)p.slots, (unsigned)shares);
  switch (hd) {
    case 64: e = launch_in<64>(env, in_type, out_type, grid, p); break;
    case 128: e = launch_in<128>(env, in_type, out_type, grid, p); break;
    default: e = launch_in<256>(env, in_type, out_type, grid, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_kv4_append launch");
}
