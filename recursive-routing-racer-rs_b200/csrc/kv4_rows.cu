// kv4_rows.cu — rows of the 4-bit KV cache (rrr_kv4_cache): packed K and V rows into its pages
// (rrr_kv4_store) and the values they stand for back into packed rows (rrr_kv4_load).
//
// Mathematics. A group of 32 values of a head becomes m = f16(min), d = f16((max - min) / 15)
// and codes round((x - m) / d), all with the f32 operations of that formula (no contraction,
// division rounded to nearest), so that a group's bits do not depend on where it is computed.
// The value read back is d*code + m: d*code is exact in f32 (11 + 4 bits), so it carries one
// rounding.
//
// Bound by memory (2 bytes of a 16-bit row in and 5/8 out per value, or the reverse), and not far
// from it by instructions. One warp takes the rows of one block of 8 or 16 (aligned in the page, so
// that the two rows of a pair, whose V codes share words, are one warp's) of K or V of one head. K:
// a lane takes 8 consecutive values, which are one word of codes. V: a lane takes the values 32i +
// 8n + g, + 1 (n = 0..3, g even) of both rows of a pair, which are two words. A quotient is first
// taken by the reciprocal, and the lane's quotients are divided out where one comes close to a
// rounding border, which the first misses by less than 8e-6 of a code (the reciprocal by two units,
// its product with 1/15 and with the value by half a one each, and the division itself: 2^-21 of
// 15). (max - min) / 15 is rounded right by one correction of the product with 1/15 (Markstein's
// method), which the tests compare with the division.
//
// 5,960 rows of 8 x 128 are stored and read back in 27.6 us, 10 us being their bytes: the stores are
// bound by some 25 instructions a value, the loads by the way to memory. (29.0 with 64-bit divisions
// to find a warp's rows; first version, a warp per row with codes shuffled together and a division
// per value: 58.)
#include <math.h>

#include "kv4.cuh"

namespace rrr {

int check_kv4_cache(rrr_ctx* ctx, const rrr_kv4_cache* c, const char* fn) {
  if (!c) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  if ((c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) || c->n_kv_heads < 1 ||
      c->n_kv_heads > 65535 || c->n_pages < 0 || c->n_pages > INT32_MAX || c->n_seqs < 0 || c->max_pages < 0 ||
      c->max_pages > INT32_MAX / kPageRows || c->table_stride < c->max_pages ||
      (int64_t)c->n_seqs * c->n_kv_heads > INT32_MAX)
    return set_error(ctx, RRR_ERR_BAD_SHAPE,
                     "%s: need head_dim 64/128/256, 1 <= n_kv_heads <= 65535, counts >= 0, table_stride >= "
                     "max_pages, at most 2^31 - 1 pages, 2^31 - 64 rows per sequence and 2^31 - 1 sequences times heads",
                     fn);
  if ((c->n_pages > 0 && !c->pages) || (c->n_seqs > 0 && c->max_pages > 0 && !c->page_table))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
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
  int slots;  // blocks of rows, with room for the sequences' ends
  void* k;
  void* v;
  int64_t k_stride, v_stride;
  const int* cu;
  const int* lens;
  int* err;
};

// The rows of a warp: packed rows [row0, row0 + n) are the rows first .. first + n - 1 (first < R)
// of a block of R rows of a page, from row in_page of it on.
struct RowBlock {
  uint8_t* blk;
  int64_t row0;
  int in_page, first, n;
};

// Slot x belongs to the last sequence s with cu[s] / R + 2 s <= x (sequences get disjoint runs
// of slots that are long enough), searched by the warp 32 sequences at a time.
template <int HD, int R>
__device__ __forceinline__ bool find_rows(const Kv4RowParams& p, int x, int h, RowBlock& b) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.n_seqs;  // the sequence lies in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + lane * step;
    const bool at = s < hi && p.cu[s] / R + 2 * s <= x;
    const unsigned below = __ballot_sync(0xffffffffu, at);
    lo += below ? (31 - __clz(below)) * step : 0;
    hi = min(hi, lo + step);
  }
  const int r0 = p.cu[lo], r1 = p.cu[lo + 1], len = p.lens[lo], most = p.max_pages * kPageRows;
  if (r0 < 0 || r1 < r0 || r1 > p.rows) {
    if (lane == 0) flag_position(p.err);
    return false;
  }
  const int rows = r1 - r0, k = x - (r0 / R + 2 * lo);  // k: the block among the sequence's
  if (rows > 0 && (len < rows || len > most) && lane == 0) flag_position(p.err);
  // (rows at positions that do not exist are left out)
  if (k < 0 || len <= 0) return false;
  const int pos0 = len - rows;  // position of the sequence's first packed row
  const int at = max(pos0, 0), end = min(len, most);
  const int64_t start = (int64_t)(at / R + (int64_t)k) * R;
  if (start >= end) return false;
  const int from = max(at, (int)start), to = min(end, (int)start + R);  // (end <= 2^31 - 64)
  if (from >= to) return false;
  const int page = p.table[(int64_t)lo * p.table_stride + (unsigned)from / kPageRows];
  if (page < 0 || page >= p.n_pages) {
    if (lane == 0) flag_position(p.err);
    return false;
  }
  b.blk = p.pages + ((int64_t)page * p.nkv + h) * Kv4Block<HD>::kBytes;
  b.row0 = r0 + (from - pos0);
  b.in_page = from % kPageRows;
  b.first = from % R;
  b.n = to - from;
  return true;
}
// CTAs: a head of K (z even) or V each, kRowWarps slots in y and z
__device__ __forceinline__ int slot_of() {
  return (int)(((blockIdx.z >> 1) * gridDim.y + blockIdx.y) * kRowWarps + (threadIdx.x >> 5));
}

// The same eight values back
__device__ __forceinline__ void dequantise(uint32_t w, float d, float m, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = fmaf(__uint_as_float(((w >> (4 * i)) & 15u) | 0x4b000000u) - 8388608.f, d, m);
}

template <int HD, int R>
struct Lanes {  // of a warp of R rows: groups at once, and rows (K) or pairs of rows (V) at once
  static constexpr int kGroups = Kv4Block<HD>::kGroups;
  static constexpr int kRows = 32 / (4 * kGroups);
  static constexpr int kAhead = R / kRows < 4 ? (R / kRows < 1 ? 1 : R / kRows) : 4;  // rows in flight
  static constexpr int kPairsAhead = kRows >= 4 ? 1 : 2;
};

template <int HD, int R, typename T>
__global__ void __launch_bounds__(32 * kRowWarps) kv4_store_kernel(const __grid_constant__ Kv4RowParams p) {
  using B = Kv4Block<HD>;
  using L = Lanes<HD, R>;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int x = slot_of(), h = blockIdx.x;
  const bool is_v = blockIdx.z & 1;
  if (x >= p.slots) return;
  RowBlock b;
  if (!find_rows<HD, R>(p, x, h, b)) return;
  const int in_page = b.in_page;
  const int j = lane / 4 % L::kGroups, t = lane % 4, set = lane / (4 * L::kGroups);
  if (!is_v) {
    const T* src = static_cast<const T*>(p.k) + (int64_t)h * HD + 32 * j + 8 * t;
#pragma unroll 1
    for (int r0 = set; r0 < b.n + set; r0 += L::kAhead * L::kRows) {
      float v[L::kAhead][8];
#pragma unroll
      for (int a = 0; a < L::kAhead; ++a) {
        if (r0 - set + a * L::kRows >= b.n) break;
        const int r = min(r0 + a * L::kRows, b.n - 1);  // (rows past the last are read as it)
        load_vec<T, 8>(src + (b.row0 + r) * p.k_stride, v[a]);
      }
#pragma unroll
      for (int a = 0; a < L::kAhead; ++a) {
        if (r0 - set + a * L::kRows >= b.n) break;
        const int r = r0 + a * L::kRows;
        __half d, m;
        const uint32_t w = quantise(v[a], d, m);
        if (r < b.n) {
          const int row = in_page + r;
          reinterpret_cast<uint32_t*>(b.blk)[B::k_word(row, j, t)] = w;
          if (t == 0) {
            reinterpret_cast<__half*>(b.blk + B::kCodes)[B::scale(row, j)] = d;
            reinterpret_cast<__half*>(b.blk + B::kCodes + B::kScales)[B::scale(row, j)] = m;
          }
        }
      }
    }
  } else {
    uint8_t* vb = b.blk + B::kHalf;
    const int g = 2 * t;
    const T* src = static_cast<const T*>(p.v) + (int64_t)h * HD + 32 * j + g;
    const int odd_first = b.first & 1, pairs = (b.n + odd_first + 1) / 2;
#pragma unroll 1
    for (int u0 = set; u0 < pairs + set; u0 += L::kPairsAhead * L::kRows) {
      float v[L::kPairsAhead][2][8];  // [pair][row][2 n + (g, g + 1)]
#pragma unroll
      for (int a = 0; a < L::kPairsAhead; ++a) {
        if (u0 - set + a * L::kRows >= pairs) break;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int r = min(max(2 * (u0 + a * L::kRows) + o - odd_first, 0), b.n - 1);
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            float two[2];
            load_vec<T, 2>(src + (b.row0 + r) * p.v_stride + 8 * n, two);
            v[a][o][2 * n] = two[0];
            v[a][o][2 * n + 1] = two[1];
          }
        }
      }
#pragma unroll
      for (int a = 0; a < L::kPairsAhead; ++a) {
        if (u0 - set + a * L::kRows >= pairs) break;
        const int r = 2 * (u0 + a * L::kRows) - odd_first, row = in_page + r;  // the pair's even row
        const bool has[2] = {r >= 0 && r < b.n, r + 1 >= 0 && r + 1 < b.n};
        uint32_t c[2];
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          __half d, m;
          c[o] = quantise(v[a][o], d, m);
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
  }
}

template <int HD, int R, typename T>
__global__ void __launch_bounds__(32 * kRowWarps) kv4_load_kernel(const __grid_constant__ Kv4RowParams p) {
  using B = Kv4Block<HD>;
  using L = Lanes<HD, R>;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int x = slot_of(), h = blockIdx.x;
  const bool is_v = blockIdx.z & 1;
  if (x >= p.slots) return;
  if (!(is_v ? p.v : p.k)) return;
  RowBlock b;
  if (!find_rows<HD, R>(p, x, h, b)) return;
  const int in_page = b.in_page;
  const int j = lane / 4 % L::kGroups, t = lane % 4, set = lane / (4 * L::kGroups);
  if (!is_v) {
    T* dst = static_cast<T*>(p.k) + (int64_t)h * HD + 32 * j + 8 * t;
#pragma unroll 1
    for (int r0 = set; r0 < b.n; r0 += L::kAhead * L::kRows) {
      uint32_t w[L::kAhead];
      __half d[L::kAhead], m[L::kAhead];
#pragma unroll
      for (int a = 0; a < L::kAhead; ++a) {
        const int row = in_page + min(r0 + a * L::kRows, b.n - 1);
        w[a] = reinterpret_cast<const uint32_t*>(b.blk)[B::k_word(row, j, t)];
        d[a] = reinterpret_cast<const __half*>(b.blk + B::kCodes)[B::scale(row, j)];
        m[a] = reinterpret_cast<const __half*>(b.blk + B::kCodes + B::kScales)[B::scale(row, j)];
      }
#pragma unroll
      for (int a = 0; a < L::kAhead; ++a) {
        const int r = r0 + a * L::kRows;
        float v[8];
        dequantise(w[a], __half2float(d[a]), __half2float(m[a]), v);
        if (r < b.n) store_vec<T, 8>(dst + (b.row0 + r) * p.k_stride, v);
      }
    }
  } else {
    const uint8_t* vb = b.blk + B::kHalf;
    const int g = 2 * t;
    T* dst = static_cast<T*>(p.v) + (int64_t)h * HD + 32 * j + g;
    const int odd_first = b.first & 1, pairs = (b.n + odd_first + 1) / 2;
#pragma unroll 1
    for (int u0 = set; u0 < pairs; u0 += L::kPairsAhead * L::kRows) {
      uint32_t w[L::kPairsAhead][2], m[L::kPairsAhead];
      __half d[L::kPairsAhead][2];
#pragma unroll
      for (int a = 0; a < L::kPairsAhead; ++a) {
        const int row = in_page - odd_first + 2 * min(u0 + a * L::kRows, pairs - 1);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          w[a][e] = reinterpret_cast<const uint32_t*>(vb)[B::v_half(row, j, g + e) / 2];
          d[a][e] = reinterpret_cast<const __half*>(vb + B::kCodes)[B::scale(row + e, j)];
        }
        m[a] = reinterpret_cast<const uint32_t*>(vb + B::kCodes + B::kScales)[B::v_min(row, j) / 2];
      }
#pragma unroll
      for (int a = 0; a < L::kPairsAhead; ++a)
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int r = 2 * (u0 + a * L::kRows) + o - odd_first;
          // nibbles n of g and of g + 1
          const uint32_t both = __byte_perm(w[a][0], w[a][1], o ? 0x7632 : 0x5410);
          float v[8];
          dequantise(both, __half2float(d[a][o]), __half2float(__ushort_as_half((unsigned short)(m[a] >> (16 * o)))), v);
          if (r >= 0 && r < b.n)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const float two[2] = {v[n], v[4 + n]};
              store_vec<T, 2>(dst + (b.row0 + r) * p.v_stride + 8 * n, two);
            }
        }
    }
  }
}

template <int HD, int R, typename T>
cudaError_t launch_rows(const LaunchEnv& env, bool store, Kv4RowParams p) {
  p.slots = p.rows / R + 2 * p.n_seqs;
  const int64_t across = ((int64_t)p.slots + kRowWarps - 1) / kRowWarps, y = across < 65535 ? across : 65535;
  const dim3 grid(p.nkv, (unsigned)y, (unsigned)(2 * ((across + y - 1) / y))), block(32 * kRowWarps);
  return store ? rrr_launch_pdl(kv4_store_kernel<HD, R, T>, grid, block, 0, env.stream, env.pdl, p)
               : rrr_launch_pdl(kv4_load_kernel<HD, R, T>, grid, block, 0, env.stream, env.pdl, p);
}
template <int HD, typename T>
cudaError_t launch(const LaunchEnv& env, bool store, const Kv4RowParams& p) {
  // Blocks of 8 rows where those of 16 would not fill the SMs once or twice, and for long rows:
  // 12,000 rows of 2 x 128 stored and read back 15.7 us (16 rows: 18.5), of 8 x 128 47.5 (46.0), of
  // 1 x 256 18.1 (25.3), of 8 x 256 77.5 (78.2).
  if constexpr (HD < 256)
    if (2 * ((int64_t)p.rows / 16 + p.n_seqs) * p.nkv >= 32 * (int64_t)env.sm_count)
      return launch_rows<HD, 16, T>(env, store, p);
  return launch_rows<HD, 8, T>(env, store, p);
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
  if ((rows > 0 && (store ? !k || !v : !k && !v)) || (c->n_seqs > 0 && (!cu_rows || !kv_lens)))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  const int64_t width = (int64_t)c->n_kv_heads * c->head_dim;
  if (rows < 0 || (k && !stride_fits(k_stride, width)) || (v && !stride_fits(v_stride, width)))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: rows >= 0 and strides of n_kv_heads * head_dim to 2^38", fn);
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
  if (c->n_seqs > INT32_MAX / 4 || rows > INT32_MAX / 4)
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: too many rows and sequences for one call", fn);
  const LaunchEnv env = make_env(ctx, stream);
  const Kv4RowParams p{static_cast<uint8_t*>(c->pages), c->n_pages, c->table_stride, c->page_table, c->n_seqs,
                       c->max_pages, c->n_kv_heads, rows, 0, k, v, k_stride, v_stride, cu_rows, kv_lens, env.d_err};
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
