// kv4_tree.cu — attention of drafted rows over the 4-bit KV cache (rrr_attention_tree_kv4): the
// `attention` dispatch (src/model/phi4.rs:1284-1309, 1680-1688) for the rows of a tree of drafted
// tokens per sequence, which see the sequence's cached rows and their own ancestors.
//
// Mathematics. The columns of a tile are up to 64 or 96 (row, query head) pairs of a sequence and KV
// head, its blocks 128 cached rows each and at last the drafted ones: S = K Q^T, the weights P =
// 2^(S scale log2(e) - m + 10) with a column's reference m, O^T += V^T P, and the sums of the weights
// by a product with ones, so that they are the sums of what V is multiplied by. m is taken
// over anew where a weight would pass 2^15. Who sees whom in the drafted block is a bit mask per row. A
// query, and a drafted key, is scaled by a power of two, drafted values together by one, so
// that f16 operands hold both 16-bit types. A result that is not finite, and one that may owe something to a cached group or
// a drafted row that f16 does not hold, is computed again row by row in 32 bits.
//
// Layout. One CTA per SM and an equal run of blocks for each; a sequence's share that crosses the border of two CTAs is
// joined by a second kernel, in order. Keys are dequantised, a row per thread, straight into TMEM (operand A), values
// transposed into shared memory, queries lie on the products' N side: so few columns cost few product cycles.
// 27 warps: one copies pages (TMA), four each dequantise K and V, sixteen take the softmax, one each issues the two
// products.
//
// What bounds it. Not memory (1.3 TB/s) nor the tensor cores, but the roles' instructions and hand-overs: a warp gets one in
// about ten cycles, a block of 48 columns takes 3,400 cycles and of 96 3,600. Measured on 24 heads over 8 of 128: 64
// sequences of 16 rows on up to 8,190: 245 us (floor 54 by bytes); 60 rows on 131,000: 217-228 us (57 by operations). With
// dequantisation, weights and products left out (at 322 us for the 64 sequences) 207 and 125 us remained. Steps, for
// the 64 sequences: scalar products 14.8 ms, tensor cores 690 us, rolled loops 464 (the instruction cache), scores ahead of the
// weighted sums 333, two issuing warps and sixteen softmax warps 322, small code for what a segment does once 245.
//
// What f16 operands round. By their scales queries, drafted keys and drafted values no more than 2^-11 of a row's largest (the
// rows of values that are too small for that beside others are computed again). Cached keys and values d c + m, up to 15 bits
// and more, and weights to 11 bits each: beside a bf16 result's own rounding that is little: 1.69e-3 to 1.71e-3 against 64
// bits, 1.65e-3 to 1.66e-3 of it the rounding. Not so for f16 rows, where keys and weights are two f16 each: 2.4e-4 against
// 2.1e-4; with one each it was 4.3e-4 on 3,000 rows (and 24 trees of up to 33 rows took 108 us against 121).
#include <math.h>

#include <type_traits>

#include "kv4.cuh"
#include "tile_common.cuh"

namespace rrr {
namespace {

constexpr int kMaxHpk = 8, kMaxNodes = 128;
constexpr float kNone = -3e38f;  // the reference of no rows: finite, so that it may be subtracted from -inf
constexpr int kRows = 128;       // KV rows of a block: two pages, or the drafted rows
constexpr int kStart = 6;        // units in front of a segment's blocks
constexpr int kGroups = 4;       // of four softmax warps each: group h takes the columns 8 h .. + 7 of every 8 kGroups
constexpr int kKWarp = 4 * kGroups, kVWarp = kKWarp + 4, kSWarp = kVWarp + 4, kLoadWarp = kSWarp + 1, kPVWarp = kSWarp + 2;
constexpr int kThreads = 32 * (kSWarp + 4);
constexpr int kInfos = 16;
constexpr int kSumBlocks = 128;  // a power of two: blocks after which the sums in TMEM are moved out
constexpr int kNap = 100;        // ns
constexpr float kBias = 10.f;    // weights are 2^(s - m + kBias), at most 2^(kBias + kLazy)
constexpr float kLazy = 5.f;
constexpr uint32_t kF16 = 1u << 4 | (uint32_t)(kRows >> 4) << 24;  // products' descriptor: f16 operands, f32 sums, M = 128

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
  struct Opened* opened;  // [CTA]: the segment that it opened and shares
  float2* stats;          // [slot][column]: maximum, sum
  int* again;             // [slot][group of columns]
  float* parts;           // [slot][column][value]
  float2* held_stats;     // [CTA][quarter][column]: reference and sum of the weights moved out
  float* held;            // [CTA][column][value]
};
struct Opened {
  int run, seq, kv, r0, len, c0, cols, pad;  // run: CTAs that share it, 0 for none
};

// ---- what the sequences are
struct Shape {
  int r0, nodes, len, blocks, tiles, per;  // per: columns of a tile
};
template <int NT>
__device__ __noinline__ Shape shape_of(const TreeParams& p, int seq) {
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
__device__ __forceinline__ int units_of(const TreeParams& p, const Shape& s) {
  return s.nodes ? s.tiles * p.nkv * (s.blocks + kStart) : 0;
}
// The units of a CTA: U / G each, one more for the first U % G
struct Share {
  int each, more;
  __device__ __forceinline__ int first(int cta) const { return cta * each + min(cta, more); }
  __device__ __forceinline__ int cta_of(int unit) const {
    const int wide = more * (each + 1);
    return unit < wide ? unit / (each + 1) : more + (unit - wide) / each;
  }
};

// kOut: the sums are moved out after it; kAnew: they begin with it; kHeld: some of the segment's have been moved out before
enum { kDraft = 1, kFirst = 2, kLast = 4, kAlone = 8, kStop = 16, kOpens = 32, kOut = 64, kAnew = 128, kHeld = 1024 };
struct __align__(16) Info {  // of a block
  int flags;                // and the segment's number modulo 4 from bit 8 on
  int n, valid[2];          // columns with the padding; rows of each page that count
  int c0, cols, kv, count;  // the tile's columns c0 .. c0 + cols - 1 of the sequence's (row, head) pairs; the segment's number in this CTA
  int r0, nodes, seq, len;
  int run;                  // CTAs that share the segment
  int outs;                 // how often the sums in TMEM have been read so far
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
// in vain. (Out of line, with what else is not in the blocks' loops: with all of it in place the kernel was 165 KB of
// instructions, and half of the warps' time went into fetching them.)
__device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t parity, int* err) {
  bool ok = false;
#pragma unroll 1
  for (int k = 0; k < 32 && !ok; ++k) ok = mbar_try_wait(bar, parity);
  return __all_sync(0xffffffffu, ok) || warp_wait(bar, parity, err);
}
__device__ __forceinline__ bool quick_wait(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || wait_longer(bar, parity, err);
}
// The same for a role that works ahead of the others: asleep between the tries, which would take issue slots from them
__device__ __noinline__ bool sleep_longer(uint64_t* bar, uint32_t parity, int* err) {
  bool ok = false;
#pragma unroll 1
  for (int k = 0; k < 256 && !ok; ++k) {
    __nanosleep(kNap);
    ok = mbar_try_wait(bar, parity);
  }
  return __all_sync(0xffffffffu, ok) || warp_wait(bar, parity, err);
}
__device__ __forceinline__ bool sleepy_wait(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || sleep_longer(bar, parity, err);
}

// Bounded barrier of four warps.
struct Quartet {
  uint64_t* bar;
  uint32_t phase;
  int* err;
  __device__ __forceinline__ bool operator()() {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
    const bool ok = quick_wait(bar, phase, err);
    phase ^= 1;
    return ok;
  }
};
// A barrier of 128 threads that tells whether one of them says yes. (All of them pass as many of these, also where a
// wait gave up.)
__device__ __forceinline__ bool any_of_128(int id, bool yes) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((int)yes), "r"(id)
      : "memory");
  return r != 0;
}
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
// d c + m of two groups as the sum of two such values, the first of which f16 holds exactly where the
// group's values have both signs: d without its last four bits (a multiple of u, as 64 to 127 u), m
// rounded to a multiple of u, at most 2,048 u in all; and what is left, under 16 u, whose own
// rounding is 2^-17 of the value.
__device__ __forceinline__ void split(uint32_t& d, uint32_t& m, uint32_t& d_rest, uint32_t& m_rest) {
  const uint32_t most = d & 0xfff0fff0u;
  const float2 all = __half22float2(as_half2(m));
  auto multiple = [](float x, uint32_t bits) {
    const uint32_t e = max((bits >> 10) & 31u, 1u);  // u = 2^(e - 21)
    return rintf(x * __uint_as_float((148u - e) << 23)) * __uint_as_float((e + 106u) << 23);
  };
  const __half2 near = __floats2half2_rn(multiple(all.x, d), multiple(all.y, d >> 16));
  d_rest = as_u32(__hsub2(as_half2(d), as_half2(most)));
  m_rest = as_u32(__hsub2(as_half2(m), near));
  d = most;
  m = as_u32(near);
}
// Two weights as f16 and what that leaves of them
__device__ __forceinline__ void split(float a, float b, uint32_t& w, uint32_t& rest) {
  const __half2 x = __floats2half2_rn(a, b);
  const float2 y = __half22float2(x);
  w = as_u32(x);
  rest = as_u32(__floats2half2_rn(a - y.x, b - y.y));
}
// 128-byte swizzle of an offset from a 1024-byte border
__device__ __forceinline__ uint32_t swizzled(uint32_t off) { return off ^ (((off >> 7) & 7u) << 4); }
// N words (a power of two) at p
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x;
    w[1] = x.y;
    w[2] = x.z;
    w[3] = x.w;
  }
}
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
// The power of two that brings values of at most `top` into [1, 2) (1 where they are not finite)
__device__ __forceinline__ float to_one(uint32_t top) {
  const int e = (int)(top >> 23);  // (a subnormal top counts as 2^-126)
  return e == 255 || top == 0 ? 1.f : __uint_as_float((uint32_t)min(max(254 - e, 1), 254) << 23);
}
// Drafted values of at most `top` are multiplied by 2^0, 2^8 or 2^15, as far as f16 allows: those of rows that are far
// smaller (down to 2^-14, 2^-22 or 2^-29) are off by at most 2^-11 of their row's largest then. (And the rows' weights are
// divided by it, which have bits to spare.)
__device__ __forceinline__ int lift_of(uint32_t top) { return top >= 0x43000000u /* 2^7 */ ? 0 : top >= 0x3f800000u /* 1 */ ? 1 : 2; }
__device__ __forceinline__ float lifted_by(int lift) { return lift == 0 ? 1.f : lift == 1 ? 256.f : 32768.f; }
// Whether a row of values up to `top` loses more all the same: its largest is no normal f16. (Who sees that row alone, or with
// others like it, is computed again.) An f16 row has no bits to lose.
template <typename T>
__device__ __forceinline__ bool too_small(uint32_t top, int lift) {
  return !std::is_same<T, __half>::value && top != 0 && top < (lift == 0 ? 0x38800000u : lift == 1 ? 0x34800000u : 0x31000000u);
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
  static constexpr int kStatic = 18 * 1024;         // more than the static shared memory
  static constexpr int kFit = (227 * 1024 - kStatic - 1024 - kFixed) / kStage;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kFixed + kStages * kStage + 1024;
  // TMEM: keys, scores, sums of the weights, O, and ones times 2^0, 2^8 and 2^15
  static constexpr int kKs = 2 * kKCols + (3 + kHalves) * NT + 24 <= 512 ? 2 : 1;  // places for K
  static constexpr int kSCol = kKs * kKCols, kLCol = kSCol + 2 * NT, kOCol = kLCol + NT, kOnes = kOCol + kHalves * NT;
  static_assert(kStages >= 2 && kOnes + 24 <= 512, "");
};

// One row of one query head by one warp in 32-bit arithmetic, over the rows that it sees and no others:
// for what f16 does not hold (values that are not finite, or of 65,520 and more). Lane l has the values D l .. D l + D - 1.
template <int HD, typename T>
__device__ __noinline__ void plain_row(const TreeParams& p, int seq, int r0, int len, int row, int kv, int head) {
  using B = Kv4Block<HD>;
  constexpr int D = HD / 32;
  const int e0 = D * (threadIdx.x & 31);
  float q[D], o[D], m = kNone, l = 0.f;
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] = 0.f;
  load_vec<T, D>(static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head + e0, q);
  auto take = [&](const float (&k)[D], const float (&v)[D]) {
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) s = fmaf(q[d], k[d], s);
    s = warp_sum(s) * p.scale;
    const float top = fmaxf(m, s), keep = ex2(m - top), w = ex2(s - top);
    m = top;
    l = fmaf(l, keep, w);
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = fmaf(o[d], keep, w * v[d]);
  };
#pragma unroll 1
  for (int at = 0; at < len; ++at) {
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
#pragma unroll 1
  for (int node = row - r0; node >= 0;) {
    float k[D], v[D];
    load_vec<T, D>(static_cast<const T*>(p.k) + (r0 + node) * p.k_row + kv * p.k_head + e0, k);
    load_vec<T, D>(static_cast<const T*>(p.v) + (r0 + node) * p.v_row + kv * p.v_head + e0, v);
    take(k, v);
    const int above = p.parents ? p.parents[r0 + node] : node - 1;
    node = above < node ? above : -1;
  }
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] = o[d] / l;
  store_vec<T, D>(static_cast<T*>(p.out) + row * p.out_row + head * p.out_head + e0, o);
}

// What is done once in a segment is kept small: its instructions come from far away each time, which took longer than
// what they do. So rows are copied as they are to the places of what is made of them, all at once, and each thread then
// goes through its own 16 bytes in a loop. In place and not as calls, which read the parameters from memory: 64 sequences
// of 16 rows took 275 us with calls, 245 so.

// Eight 16-bit values at p, of a row that HD / 8 neighbouring lanes hold, to f16 in the order of K's words, the row brought
// to [1, 2) by a power of two, which is returned
template <int HD, typename T>
__device__ __forceinline__ float row_to_one(uint8_t* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  uint32_t top = top_bits<T>(v);
#pragma unroll
  for (int o = 1; o < HD / 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = to_one(top);
  uint32_t y[4];
  scaled_pairs<T>(v, s, y);
  *reinterpret_cast<uint4*>(p) = make_uint4(y[0], y[1], y[2], y[3]);
  return s;
}
// The tile's queries into shared memory, in the order of K's words: HD / 8 lanes per row, 8 values each; a row is
// brought to [1, 2) by a power of two, which its line takes back.
template <int HD, int NT, typename T>
__device__ __forceinline__ void queries(const TreeParams& p, const Info& f, int r, uint8_t* qs, float* line) {
  constexpr int J = HD < 128 ? HD / 32 : 4, kLanes = HD / 8, kAcross = 128 / kLanes;
  const int x = r % kLanes, j = x / 4, w = (j / J) * 4 * J + (x % 4) * J + j % J;  // the place among the words of a row of codes
  uint8_t* const to = qs + (w / 8) * NT * 128;
#pragma unroll 1
  for (int c = r / kLanes; c < f.n; c += kAcross) {
    const int column = f.c0 + min(c, f.cols - 1), token = column / p.hpk, head = f.kv * p.hpk + column - token * p.hpk;
    cp_async16_or_zero(to + sw128_off(c, w % 8),
                       static_cast<const T*>(p.q) + (int64_t)(f.r0 + token) * p.q_row + head * p.q_head + 8 * x, c < f.cols);
  }
  cp_async_commit();
  cp_async_wait<0>();
#pragma unroll 1
  for (int c = r / kLanes; c < f.n; c += kAcross) {
    const float s = row_to_one<HD, T>(to + sw128_off(c, w % 8));
    if (x == 0) {
      line[c] = c < f.cols ? p.scale / s : 0.f;
      line[NT + c] = kBias;
    }
  }
}
// Up to 64 drafted keys from row `first` on: HD / 8 lanes per row, 8 values each; a row is brought to [1, 2) by a power of two.
// They go to shared memory, from where their threads take them to TMEM.
template <int HD, typename T>
__device__ __forceinline__ void drafted_keys(const TreeParams& p, const Info& f, int r, int first, uint8_t* to, float* scales) {
  constexpr int J = HD < 128 ? HD / 32 : 4, kLanes = HD / 8, kAcross = 128 / kLanes;
  const int x = r % kLanes, j = x / 4, w = (j / J) * 4 * J + (x % 4) * J + j % J, rows = min(f.nodes - first, 64);
  const T* src = static_cast<const T*>(p.k) + (int64_t)(f.r0 + first) * p.k_row + f.kv * p.k_head + 8 * x;
  const int own = r / kLanes, end = own + rows;  // (whole warps go through the loops)
#pragma unroll 1
  for (int c = own; c < end; c += kAcross)
    cp_async16_or_zero(to + c * (2 * HD) + ((w ^ (c & 7)) << 4), src + min(c, rows - 1) * p.k_row, c < rows);
  cp_async_commit();
  cp_async_wait<0>();
#pragma unroll 1
  for (int c = own; c < end; c += kAcross) {
    const float s = row_to_one<HD, T>(to + c * (2 * HD) + ((w ^ (c & 7)) << 4));
    if (x == 0) scales[first + c] = 1.f / s;
  }
}
// Drafted values: a thread has rows 8 o .. + 7 (o = tid % 16) of values 8 (tid / 16 + 8 c) .. + 7, eight rows of 16 bytes
// which become eight values of 16 bytes. The rows into shared memory, to the values' places; the largest bits of row tid.
template <int HD>
__device__ __forceinline__ uint8_t* value_place(uint8_t* dst, int o, int e) {
  constexpr int kERows = HD < 128 ? HD : 128;
  return dst + ((e >> 7) * 2 + (o >> 3)) * kERows * 128 + (e & 127) * 128 + (((o & 7) ^ (e & 7)) << 4);
}
template <int HD, typename T>
__device__ __forceinline__ void drafted_rows(const TreeParams& p, const Info& f, int tid, uint8_t* dst) {
  const int o = tid & 15, e0 = 8 * (tid >> 4);
  const T* src = static_cast<const T*>(p.v) + f.kv * p.v_head + (int64_t)f.r0 * p.v_row + e0;
#pragma unroll 1
  for (int x = 0; x < HD / 8; ++x) {
    const int row = 8 * o + x % 8, c = x / 8;
    cp_async16_or_zero(value_place<HD>(dst, o, e0 + 64 * c + x % 8), src + min(row, f.nodes - 1) * p.v_row + 64 * c, row < f.nodes);
  }
  cp_async_commit();
  cp_async_wait<0>();
}
template <int HD, typename T>
__device__ __forceinline__ uint32_t row_top(int tid, uint8_t* dst) {
  uint32_t top = 0;
#pragma unroll 1
  for (int e = tid & 7; e < HD; e += 8) top = max(top, top_bits<T>(*reinterpret_cast<const uint4*>(value_place<HD>(dst, tid >> 3, e))));
  return top;
}
// The values of the rows there, lifted
template <int HD, typename T>
__device__ __forceinline__ void drafted_values(int tid, float lift, uint8_t* dst) {
  const int o = tid & 15;
#pragma unroll 1
  for (int c = 0; c < HD / 64; ++c) {
    const int e0 = 8 * ((tid >> 4) + 8 * c);
    uint4 w[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) w[r] = *reinterpret_cast<const uint4*>(value_place<HD>(dst, o, e0 + r));
    // two values of the eight rows at a time, the rows' next words in front then
#pragma unroll 1
    for (int k = 0; k < 8; k += 2) {
      uint32_t y[4], z[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float2 a = pair_of<T>(w[2 * r].x), b = pair_of<T>(w[2 * r + 1].x);
        y[r] = as_u32(__floats2half2_rn(a.x * lift, b.x * lift));
        z[r] = as_u32(__floats2half2_rn(a.y * lift, b.y * lift));
      }
      *reinterpret_cast<uint4*>(value_place<HD>(dst, o, e0 + k)) = make_uint4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<uint4*>(value_place<HD>(dst, o, e0 + k + 1)) = make_uint4(z[0], z[1], z[2], z[3]);
#pragma unroll
      for (int r = 0; r < 8; ++r) w[r] = make_uint4(w[r].y, w[r].z, w[r].w, 0u);
    }
  }
}

// The first block from blk on with a row on a page that exists, or else `last`. (A part begins with it, whose rows give the
// maxima their first values: from 0 on they would only rise, and the weights of scores far below 0 are lost in f16.)
__device__ __noinline__ int first_with_rows(const TreeParams& p, int seq, int len, int blk, int last) {
  const int lane = threadIdx.x & 31, pages = (len + kPageRows - 1) / kPageRows;
#pragma unroll 1
  for (; blk < last; blk += 16) {
    const int at = 2 * blk + lane;
    const int id = at < min(pages, 2 * last) ? p.table[(int64_t)seq * p.table_stride + at] : 0;
    if (id < 0 || id >= p.n_pages) flag_position(p.err);
    const unsigned there = __ballot_sync(0xffffffffu, at < min(pages, 2 * last) && id >= 0 && id < p.n_pages);
    if (there) return blk + (__ffs(there) - 1) / 2;
  }
  return last;
}

// The tensor core cuts off what does not fit a sum's 24 bits, eight or sixteen times a block and always towards zero: over
// 131,000 rows of one CTA's the results of f16 rows lost 4e-4, over 400,000 2.2e-3. So sums of kSumBlocks blocks are added up in
// memory, and come back to TMEM at the segment's end: sums in TMEM and those held become one, there or here. By the softmax
// warps, each its own columns and values, a column at a time (eight at once were 12 us slower for 60 rows on 131,000, whose
// instructions come from far away).
template <int HD, int NT>
__device__ __noinline__ void move_sums(const TreeParams& p, const Info& f, const float* line, uint32_t tmem) {
  using S = Sizes<HD, NT>;
  const int lane = threadIdx.x & 31, h = threadIdx.x >> 7, qd = (threadIdx.x >> 5) & 3;
  const bool out = f.flags & kOut, held = f.flags & kHeld;
  const uint32_t sub = (uint32_t)(32 * qd) << 16;
  float2* const stats = p.held_stats + (blockIdx.x * 4 + qd) * NT;
#pragma unroll 1
  for (int x = 8 * h; x < f.cols; x += x % 8 == 7 ? 8 * kGroups - 7 : 1) {
    uint32_t l, o;
    const float2 was = held ? stats[x] : make_float2(kNone, 0.f);
    __syncwarp();
    tmem_ld1(tmem + S::kLCol + x + sub, l);
    const float m = kBias - line[NT + x], keep = ex2(was.x - m), sum = fmaf(was.y, keep, __uint_as_float(l));  // (a reference only rises)
    if (!out) tmem_st1(tmem + S::kLCol + x + sub, __float_as_uint(sum));
    else if (lane == 0) stats[x] = make_float2(sum > 0.f ? m : kNone, sum);
    if (qd * 32 < S::kERows) {
#pragma unroll 1
      for (int k = 0; k < S::kHalves; ++k) {
        float* const to = p.held + ((size_t)blockIdx.x * NT + x) * HD + 128 * k + 32 * qd + lane;
        const float old = held ? *to : 0.f;
        __syncwarp();
        tmem_ld1(tmem + S::kOCol + k * NT + x + sub, o);
        const float v = fmaf(old, keep, __uint_as_float(o));
        if (out) *to = v;
        __syncwarp();
        if (!out) tmem_st1(tmem + S::kOCol + k * NT + x + sub, __float_as_uint(v));
      }
    }
  }
  tmem_wait_st();
  __syncwarp();
}

// The segments of a CTA's own whose bits are set, in 32 bits, a warp per column. All warps come here when the roles are done:
// the rows may take longer than a role waits.
constexpr int kBits = 1024;  // segments of a CTA with a bit each; those from the last on share it
template <int HD, int NT, typename T>
__device__ __noinline__ void compute_again(const TreeParams& p, int s, int base, int units, const uint32_t* bits) {
  const int warp = threadIdx.x >> 5;
  const Share share{units / (int)gridDim.x, units % (int)gridDim.x};
  const int u0 = share.first(blockIdx.x), u1 = share.first(blockIdx.x + 1);
  Shape sh = shape_of<NT>(p, s);
  int each = sh.blocks + kStart, g = (u0 - base) / each, blk = max(0, (u0 - base) % each - kStart);
#pragma unroll 1
  for (int count = 0; base + g * each + kStart + blk < u1; ++count, blk = 0) {
    const int seg0 = base + g * each + kStart, bit = min(count, kBits - 1), cta = (int)blockIdx.x;
    if (((bits[bit >> 5] >> (bit & 31)) & 1u) && share.cta_of(seg0) == cta && share.cta_of(seg0 + sh.blocks - 1) == cta) {
      const int kv = g / sh.tiles, c0 = (g - kv * sh.tiles) * sh.per, end = min(c0 + sh.per, sh.nodes * p.hpk);
#pragma unroll 1
      for (int c = c0 + warp; c < end; c += kThreads / 32)
        plain_row<HD, T>(p, s, sh.r0, sh.len, sh.r0 + c / p.hpk, kv, kv * p.hpk + c % p.hpk);
    }
    if (++g >= sh.tiles * p.nkv) {
      g = 0;
      base += units_of(p, sh);
      do {
        if (++s >= p.n_seqs) return;
        sh = shape_of<NT>(p, s);
      } while (sh.nodes == 0);
      each = sh.blocks + kStart;
    }
  }
}

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    tree_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ TreeParams p) {
  using S = Sizes<HD, NT>;
  constexpr int G = HD / 32, J = G < 4 ? G : 4, PL = G / J;  // groups, groups per plane, planes
  // f16 rows show what f16 operands lose, bf16 rows do not: with f16 rows cached keys and weights are sums of two f16
  // each. The two of a block of keys come one after the other; the weights have one place, in two halves.
  constexpr bool kTwice = std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], k_full[2], k_done[2], s_full[2], v_full[S::kVs], p_full[2], p_empty[2], o_empty, fin;
  __shared__ uint64_t told[kInfos];                // that the info of a segment's first block is there, or that there is none
  __shared__ uint64_t lifted[4];                  // v_lift is there, by the segment's number (every segment but the last has drafted rows here)
  __shared__ uint64_t teams[2];                   // of K's and V's warps
  __shared__ Info infos[kInfos];
  __shared__ uint4 seen[4][kMaxNodes];            // of a tree's row: the rows that it sees, as bits
  __shared__ int up[kMaxNodes];
  __shared__ float k_scale[4][kRows];
  __shared__ int v_lift[4];
  __shared__ int k_again[4], v_again[4];
  __shared__ uint32_t v_tops[4];
  __shared__ __align__(16) float lines[4][2 * NT];  // of a column c: the argument of a weight's exponential is score * [c] + [NT + c]
  __shared__ float quad[4][NT], change[NT];
  __shared__ int warp_units[kThreads / 32], first_base, first_seq, all_units, dead[kGroups];
  __shared__ uint32_t again[kBits / 32];  // a bit per segment of the CTA's own that f16 did not hold
  __shared__ uint32_t tmem_slot;
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
      mbar_init(&k_done[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4 * kGroups);
      mbar_init(&p_empty[i], 1);
      mbar_init(&teams[i], 4);
    }
    for (int i = 0; i < S::kVs; ++i) mbar_init(&v_full[i], 4);
    mbar_init(&o_empty, 4 * kGroups);
    for (int i = 0; i < kGroups; ++i) dead[i] = 0;
    for (int i = 0; i < kInfos; ++i) mbar_init(&told[i], 1);
    for (int i = 0; i < 4; ++i) mbar_init(&lifted[i], 1);
    mbar_init(&fin, 2);
    fence_mbarrier_init();
    if (p.n_pages > 0) prefetch_map(&map);  // (there is none without pages)
  }
  if (threadIdx.x < kBits / 32) again[threadIdx.x] = 0;
  if (warp == kSWarp) tmem_alloc(&tmem_slot, 512);
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's units [u0, u1) of all U
  const int per = (p.n_seqs + kThreads - 1) / kThreads;
  const int my0 = min(p.n_seqs, (int)threadIdx.x * per), my1 = min(p.n_seqs, my0 + per);
  int mine = 0;
  for (int s = my0; s < my1; ++s) mine += units_of(p, shape_of<NT>(p, s));
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) warp_units[warp] = upto;
  if (threadIdx.x == 0) p.opened[blockIdx.x].run = 0;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  int before = upto - mine, U = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warp_units[w];
    U += warp_units[w];
  }
  const Share share{U / (int)gridDim.x, U % (int)gridDim.x};
  const int u0 = share.first(blockIdx.x), u1 = share.first(blockIdx.x + 1);
  if (u0 >= before && u0 < before + mine) {
    int s = my0, base = before;
    for (;; ++s) {
      const int n = units_of(p, shape_of<NT>(p, s));
      if (u0 < base + n || s + 1 >= my1) break;
      base += n;
    }
    first_seq = s;
    first_base = base;
    all_units = U;
  }
  __syncthreads();
  // Every wait is bounded; a role that gave up leaves, and so do those that wait for it.
  auto wait = [&](uint64_t* bar, uint32_t parity) { return quick_wait(bar, parity, p.err); };
  auto doze = [&](uint64_t* bar, uint32_t parity) { return sleepy_wait(bar, parity, p.err); };

  if (u0 >= u1) {
    // nothing to do
    if (warp == kSWarp || warp == kPVWarp) {
      if (elect_one()) umma_commit(&fin);
      __syncwarp();
    }
  } else if (warp == kLoadWarp) {
    // ---------------- the blocks in order, and the copies of their pages
    int s = first_seq, count = -1, it = 0, st = 0, base = first_base;
    Shape sh = shape_of<NT>(p, s);
    int each = sh.blocks + kStart;
    int g = (u0 - base) / each, blk = max(0, (u0 - base) % each - kStart);
    int ids_at = 0, id = 0;  // page numbers of the segment
    int kv = 0, c0 = 0, cols = 0;
    int the = 0, run = 0, from = 0, outs = 0;  // (of lane 0) the segment's flags, its CTAs, its first block here
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
      const int seg0 = base + g * each + kStart;  // unit of the segment's block 0
      stop = s >= p.n_seqs || seg0 + blk >= u1;
      Info& f = infos[it % kInfos];
      if (begin || stop) {
        if (!stop) blk = first_with_rows(p, s, sh.len, blk, min(sh.blocks, u1 - seg0) - 1);
        kv = stop ? 0 : g / sh.tiles;
        c0 = (g - kv * sh.tiles) * sh.per;
        cols = min(sh.per, sh.nodes * p.hpk - c0);
        // what the segment is, before its first block is there; its rows on their way to L2
        if (lane == 0) {
          const int cta0 = share.cta_of(seg0), cta1 = share.cta_of(seg0 + sh.blocks - 1);
          ++count;
          the = (cta0 == cta1 ? kAlone : 0) | (cta0 == (int)blockIdx.x ? kOpens : 0) | (count & 3) << 8;
          run = cta1 - cta0 + 1;
          f.flags = stop ? kStop : the | kFirst;
          f.n = sh.per;
          f.c0 = c0;
          f.cols = cols;
          f.kv = kv;
          f.r0 = sh.r0;
          mbar_arrive(&told[it % kInfos]);
        }
        if (!stop) {
          constexpr int kLines = HD / 64;
          for (int x = lane; x < (cols + 2 * sh.nodes) * kLines; x += 32) {
            const int c = x / kLines, part = x % kLines * 64;
            const T* a;
            if (c < cols) {
              const int token = (c0 + c) / p.hpk;
              a = static_cast<const T*>(p.q) + (int64_t)(sh.r0 + token) * p.q_row + (kv * p.hpk + (c0 + c) - token * p.hpk) * p.q_head;
            } else if (c < cols + sh.nodes) {
              a = static_cast<const T*>(p.k) + (int64_t)(sh.r0 + c - cols) * p.k_row + kv * p.k_head;
            } else {
              a = static_cast<const T*>(p.v) + (int64_t)(sh.r0 + c - cols - sh.nodes) * p.v_row + kv * p.v_head;
            }
            asm volatile("prefetch.global.L2 [%0];" ::"l"(a + part));
          }
        }
      }
      const bool draft = blk + 1 == sh.blocks;
      // the numbers of the next 32 pages, one per lane
      if (!stop && !draft && (begin || 2 * blk + 2 > ids_at + 32)) {
        ids_at = 2 * blk;
        const int left = sh.len - (ids_at + lane) * kPageRows;
        id = left > 0 ? p.table[(int64_t)s * p.table_stride + ids_at + lane] : 0;
        if (left > 0 && (id < 0 || id >= p.n_pages)) {
          flag_position(p.err);
          id = -1;
        }
      }
      int p0 = 0, p1 = 0, v0 = 0, v1 = 0;
      if (!stop && !draft) {
        p0 = __shfl_sync(0xffffffffu, id, 2 * blk - ids_at);
        p1 = __shfl_sync(0xffffffffu, id, 2 * blk + 1 - ids_at);
        v0 = p0 < 0 ? 0 : min(kPageRows, sh.len - 2 * blk * kPageRows);
        v1 = p1 < 0 ? 0 : max(0, min(kPageRows, sh.len - (2 * blk + 1) * kPageRows));
      }
      if (!doze(&empty[st], phase)) break;
      if (lane == 0) {
        uint8_t* dst = ring + (size_t)st * S::kStage;
        if (v0 > 0) tma_load_2d(dst, &map, 0, (int)(((int64_t)p0 * p.nkv + kv) * (S::kPage / 128)), &full[st]);
        if (v1 > 0) tma_load_2d(dst + S::kPage, &map, 0, (int)(((int64_t)p1 * p.nkv + kv) * (S::kPage / 128)), &full[st]);
        if (stop) {
          f.flags = kStop;
        } else {
          from = begin ? blk : from;
          const int nth = (blk - from) % kSumBlocks;
          const bool last = draft || seg0 + blk + 1 >= u1, out = !last && nth == kSumBlocks - 1;
          f.flags = the | (draft ? kDraft : 0) | (begin ? kFirst : 0) | (last ? kLast : out ? kOut : 0) |
                    (nth == 0 ? kAnew : 0);
          the |= out ? kHeld : 0;
          f.outs = outs;
          outs += last || out;
          f.n = sh.per;
          f.valid[0] = v0;
          f.valid[1] = v1;
          f.c0 = c0;
          f.cols = cols;
          f.kv = kv;
          f.count = count;
          f.r0 = sh.r0;
          f.nodes = sh.nodes;
          f.seq = s;
          f.len = sh.len;
          f.run = run;
        }
        mbar_arrive_expect_tx(&full[st], (uint32_t)((v0 > 0) + (v1 > 0)) * S::kPage);
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
  } else if (warp == kSWarp) {
    // ---------------- scores: S = K Q^T of block i, in the place of S(i - 2) once its weights are there
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);  // (known to be the warp's, as what is derived from it)
    const uint64_t q_desc = sw128_desc(smem_addr(qs));
    int kc = 0;  // K's operands so far
#pragma unroll 1
    for (int i = 0;; ++i) {
      if (!wait(&k_full[kc & 1], (uint32_t)(kc >> 1) & 1u)) break;
      if (i >= 2 && !wait(&p_full[i & 1], (uint32_t)((i - 2) >> 1) & 1u)) break;
      const int2 f = *reinterpret_cast<const int2*>(&infos[i % kInfos]);  // flags, columns
      if (f.x & kStop) {
        if (lane == 0) mbar_arrive(&s_full[i & 1]);
        break;
      }
      const uint32_t odd = __shfl_sync(0xffffffffu, i & 1, 0), n = __shfl_sync(0xffffffffu, f.y, 0);
      const uint32_t idesc = kF16 | n >> 3 << 17, to = base + S::kSCol + odd * NT;
      const int times = kTwice && !(f.x & kDraft) ? 2 : 1;
      bool ok = true;
#pragma unroll 1
      for (int t = 0; t < times && ok; ++t, ++kc) {
        if (t) ok = wait(&k_full[kc & 1], (uint32_t)(kc >> 1) & 1u);
        if (!ok) break;
        const uint32_t k = base + (S::kKs == 2 ? __shfl_sync(0xffffffffu, kc & 1, 0) * S::kKCols : 0u);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            umma_f16_ta(to, k + 8u * kk, q_desc + (((kk / 4) * NT * 128 + 32 * (kk % 4)) >> 4), idesc, t + kk > 0 ? 1u : 0u);
          if (kTwice) umma_commit(&k_done[kc & 1]);
          if (t + 1 == times) umma_commit(&s_full[i & 1]);
        }
        __syncwarp();
      }
      if (!ok) break;
    }
    if (elect_one()) umma_commit(&fin);
    __syncwarp();
  } else if (warp == kPVWarp) {
    // ---------------- weighted sums: O^T += V^T P^T of block i, and the sums of the weights
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t v_desc = sw128_desc(smem_addr(vs)), p_desc = sw128_desc_mn(smem_addr(ps), kRows * 128);
#pragma unroll 1
    for (int i = 0;; ++i) {
      if (!wait(&v_full[i % S::kVs], (uint32_t)(i / S::kVs) & 1u)) break;
      const Info& f = infos[i % kInfos];
      const int2 head = *reinterpret_cast<const int2*>(&f);
      if (head.x & kStop) break;
      if (!wait(&p_full[i & 1], (uint32_t)(i >> 1) & 1u)) break;
      if ((head.x & kAnew) && f.outs > 0 && !wait(&o_empty, (uint32_t)(f.outs - 1) & 1u)) break;
      const uint32_t odd = __shfl_sync(0xffffffffu, i & 1, 0), flags = __shfl_sync(0xffffffffu, head.x, 0), n = __shfl_sync(0xffffffffu, head.y, 0);
      const uint32_t lift = __shfl_sync(0xffffffffu, flags & kDraft ? v_lift[(flags >> 8) & 3] : 0, 0);
      const uint32_t idesc = kF16 | 1u << 16 | n >> 3 << 17, more = flags & kAnew ? 0u : 1u, ones = base + S::kOnes + 8u * lift;
      const uint64_t v = v_desc + (S::kVs == 2 ? odd * (S::kV >> 4) : 0u), w = p_desc + (kTwice ? 0u : odd * (S::kP >> 4));
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int x = 0; x < (kTwice ? 2 : 1) * (kRows / 16); ++x) {
          const int kk = x % (kRows / 16);
          const uint64_t part = w + ((x / (kRows / 16) * S::kP + 2048 * kk) >> 4);
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h)
            umma_f16(base + S::kOCol + h * NT, v + (((h * 2 + kk / 4) * S::kERows * 128 + 32 * (kk % 4)) >> 4), part, idesc,
                     x > 0 ? 1u : more);
          umma_f16_ta(base + S::kLCol, ones, part, idesc, x > 0 ? 1u : more);
        }
        umma_commit(&p_empty[i & 1]);
      }
      __syncwarp();
    }
    if (elect_one()) umma_commit(&fin);
    __syncwarp();
  } else if (warp > kPVWarp) {
    // (no role)
  } else if (warp >= kVWarp) {
    // ---------------- V: pairs of rows, transposed to rows of values
    const int tid = threadIdx.x - 32 * kVWarp;
    // of a cached block a thread takes values 32 k + 8 n + g (of each plane) of every kPass-th eight rows. What lies within a
    // line of the pages is reached by an exclusive or.
    constexpr int kPass = 128 / (8 * J);
    const int g = tid & 7, k = (tid >> 3) % J, o0 = tid / (8 * J);
    const uint32_t pick = k & 1 ? 0x7632 : 0x5410;
    Quartet team{&teams[1], 0, p.err};
    int st = 0;
    uint32_t phase = 0;
#pragma unroll 1
    for (int i = 0;; ++i) {
      if (!doze(&full[st], phase)) break;
      const Info& f = infos[i % kInfos];
      const int flags = f.flags;
      if (flags & kStop) {
        // (not before the products have seen the block two before, as above)
        if (i >= S::kVs && !doze(&p_empty[(i - S::kVs) & 1], (uint32_t)((i - S::kVs) >> 1) & 1u)) break;
        if (lane == 0) mbar_arrive(&v_full[i % S::kVs]);
        break;
      }
      uint8_t* const stage = ring + (size_t)st * S::kStage;
      uint8_t* const dst = vs + (i % S::kVs) * S::kV;
      // the place is free once PV(i - kVs) is done
      auto free_place = [&]() {
        return i < S::kVs || doze(&p_empty[(i - S::kVs) & 1], (uint32_t)((i - S::kVs) >> 1) & 1u);
      };
      if (!(flags & kDraft)) {
        if (f.valid[0] < kPageRows || f.valid[1] < kPageRows) {
          // rows that do not count: d = m = 0
          const int half = tid >> 6, row = tid & 63;
          if (row >= f.valid[half])
            for (int j = 0; j < G; ++j) {
              *reinterpret_cast<uint16_t*>(stage + half * S::kPage + swizzled(72 * HD + 2 * (row * G + j))) = 0;
              *reinterpret_cast<uint16_t*>(stage + half * S::kPage + swizzled(76 * HD + 4 * ((row >> 1) * G + j) + 2 * (row & 1))) = 0;
            }
          if (!team()) break;
        }
        if (!free_place()) break;
        // (the loop stays small: five warps of four roles share a scheduler's instruction cache)
#pragma unroll 1
        for (int n = 0; n < 16 * PL / kPass; ++n) {
          const int P = n / (16 / kPass), o = n % (16 / kPass) * kPass + o0, r = (o & 7) * 8;  // rows 8 o .. + 7
          const uint8_t* const page = stage + (o >> 3) * S::kPage;
          const uint32_t codes = swizzled(40 * HD + P * 1024 * J + (r + g) * 16 * J) + 4 * (k % 4);
          const uint32_t steps = swizzled(72 * HD + 2 * r * G) ^ (HD == 256 ? 8 * P + 4 * (k >> 1) : 4 * (k >> 1));
          const uint32_t mins = swizzled(76 * HD + 2 * r * G) ^ (HD == 256 ? 16 * P + 4 * k : 4 * k);
          uint32_t x[4][4];  // [t][n]: nibble n of the halves, the even row's and the odd row's
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(page + (codes ^ (4 * J * t)));
            const uint32_t a = *reinterpret_cast<const uint32_t*>(page + (steps ^ (4 * G * t)));
            const uint32_t b = *reinterpret_cast<const uint32_t*>(page + (steps ^ (4 * G * t + 2 * G)));
            const uint32_t m = *reinterpret_cast<const uint32_t*>(page + (mins ^ (4 * G * t)));
            values_of(w, as_half2(__byte_perm(a, b, pick)), as_half2(m), x[t]);
          }
          uint8_t* const to = dst + (P * 2 + (o >> 3)) * S::kERows * 128 + (32 * k + g) * 128 + (((o & 7) ^ g) << 4);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<uint4*>(to + 8 * e * 128) = make_uint4(x[0][e], x[1][e], x[2][e], x[3][e]);
        }
      } else {
        if (!free_place()) break;
        drafted_rows<HD, T>(p, f, tid, dst);
        if (tid == 0) v_again[(flags >> 8) & 3] = 0;
        if (!team()) break;
        const uint32_t mine = row_top<HD, T>(tid, dst), most = __reduce_max_sync(0xffffffffu, mine);
        if (lane == 0) v_tops[warp & 3] = most;
        if (!team()) break;
        const int lift = lift_of(max(max(v_tops[0], v_tops[1]), max(v_tops[2], v_tops[3])));
        if (tid == 0) {
          v_lift[(flags >> 8) & 3] = lift;
          mbar_arrive(&lifted[(flags >> 8) & 3]);
        }
        if (too_small<T>(mine, lift)) v_again[(flags >> 8) & 3] = 1;
        drafted_values<HD, T>(tid, lifted_by(lift), dst);
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
  } else if (warp >= kKWarp) {
    // ---------------- K: a row of keys per thread, into TMEM; and the tile's queries
    const int r = threadIdx.x - 32 * kKWarp, half = r >> 6, row = r & 63;
    const uint32_t sub = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t k_codes = swizzled(row * 16 * J), k_steps = swizzled(32 * HD + 2 * row * G), k_mins = swizzled(36 * HD + 2 * row * G);
    Quartet team{&teams[0], 0, p.err};
    int st = 0;
    uint32_t phase = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint32_t ones[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) ones[e] = k == 0 ? 0x3c003c00u : k == 1 ? 0x5c005c00u : 0x78007800u;
      tmem_st8(tmem + S::kOnes + 8 * k + sub, ones);
    }
    bool begins = true;
    uint32_t turns = 0;  // of the waits for `told`
    int kc = 0;          // operands so far
#pragma unroll 1
    for (int i = 0;; ++i) {
      const Info& f = infos[i % kInfos];
      if (begins) {
        if (!doze(&told[i % kInfos], turns >> (i % kInfos) & 1u)) break;
        turns ^= 1u << (i % kInfos);
        if (!(f.flags & kStop)) {
          const int par = (f.flags >> 8) & 3;
          // S of the segment before has read its queries, so that weights three blocks before are there, and the end of a
          // segment four before, which has read what lies in the same place
          if (i > 0 && !doze(&s_full[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1u)) break;
          if (r == 0) k_again[par] = 0;
          queries<HD, NT, T>(p, f, r, qs, lines[par]);
          fence_proxy_async_smem();
          if (!team()) break;
        }
      }
      if (!doze(&full[st], phase)) break;
      const int flags = f.flags, par = (flags >> 8) & 3;
      begins = flags & kLast;
      if (flags & kStop) {
        // (not before the products have seen the block two before, or they would miss its turn)
        if (kc >= 2 && !doze(kTwice ? &k_done[kc & 1] : &s_full[kc & 1], (uint32_t)((kc - 2) >> 1) & 1u)) break;
        if (lane == 0) mbar_arrive(&k_full[kc & 1]);
        break;
      }
      uint32_t dst = 0;
      // the place is free once the products with the operand kKs before are done (kc = i where there is one per block)
      auto free_place = [&]() {
        const int last = kc - S::kKs;
        dst = tmem + (kc % S::kKs) * S::kKCols + sub;
        const bool ok = last < 0 || doze(kTwice ? &k_done[last & 1] : &s_full[last & 1], (uint32_t)(last >> 1) & 1u);
        tc_fence_after();
        return ok;
      };
      if (!(flags & kDraft)) {
        const uint8_t* const page = ring + (size_t)st * S::kStage + half * S::kPage;
        uint32_t d[G / 2], m[G / 2];
        load_words<G / 2>(page + k_steps, d);
        load_words<G / 2>(page + k_mins, m);
        __half2 most = as_half2(0u);
#pragma unroll
        for (int k = 0; k < G / 2; ++k) most = __hmax2(most, __hfma2(as_half2(d[k]), as_half2(0x4b804b80u), __habs2(as_half2(m[k]))));
        if (row < f.valid[half] && (__hisinf(__low2half(most)) || __hisinf(__high2half(most)))) k_again[par] = 1;
        uint32_t d_rest[G / 2], m_rest[G / 2];
        if (kTwice)
#pragma unroll
          for (int k = 0; k < G / 2; ++k) split(d[k], m[k], d_rest[k], m_rest[k]);
        if (!free_place()) break;
        bool ok = true;
#pragma unroll 1
        for (int t = 0; t < (kTwice ? 2 : 1); ++t) {
          if (kTwice && t) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[kc & 1]);
            ++kc;
            ok = free_place();
            if (!ok) break;
#pragma unroll
            for (int k = 0; k < G / 2; ++k) {
              d[k] = d_rest[k];
              m[k] = m_rest[k];
            }
          }
#pragma unroll
          for (int P = 0; P < PL; ++P) {
            __half2 dd[J], mm[J];
#pragma unroll
            for (int k = 0; k < J; ++k) {
              const int j = P * J + k;
              dd[k] = j & 1 ? __high2half2(as_half2(d[j / 2])) : __low2half2(as_half2(d[j / 2]));
              mm[k] = j & 1 ? __high2half2(as_half2(m[j / 2])) : __low2half2(as_half2(m[j / 2]));
            }
#pragma unroll 1
            for (int u = 0; u < J; ++u) {  // four words, 16 columns
              const uint4 x = *reinterpret_cast<const uint4*>(page + ((k_codes + P * 1024 * J) ^ (16 * u)));
              uint32_t y[16];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t z[4];
                values_of((&x.x)[k], dd[k % J], mm[k % J], z);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[4 * k + e] = z[e];
              }
              __syncwarp();
              tmem_st16(dst + P * 16 * J + 16 * u, y);
            }
          }
        }
        if (!ok) break;
      } else {
        // drafted rows: to [1, 2) by a power of two each; who sees whom
        uint8_t* const to = ring + (size_t)st * S::kStage;
        int parent = -1;
        if (r < f.nodes) {
          parent = p.parents ? p.parents[f.r0 + r] : r - 1;
          if (parent < -1 || parent >= r) {
            flag_position(p.err);
            parent = -1;
          }
        }
        up[r] = parent;
        bool ok = free_place();
#pragma unroll 1
        for (int first = 0; ok && first < f.nodes; first += 64) {
          drafted_keys<HD, T>(p, f, r, first, to, k_scale[par]);
          ok = team();
          if ((r & 64) == first) {
#pragma unroll 1
            for (int w = 0; w < HD / 8; w += 4) {  // four words, 16 columns
              uint32_t y[16];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint4 v = *reinterpret_cast<const uint4*>(to + (r & 63) * (2 * HD) + (((w + k) ^ (r & 7)) << 4));
                y[4 * k] = v.x;
                y[4 * k + 1] = v.y;
                y[4 * k + 2] = v.z;
                y[4 * k + 3] = v.w;
              }
              __syncwarp();
              tmem_st16(dst + 4 * w, y);
            }
          }
          if (first + 64 < f.nodes) ok = ok && team();
        }
        if (!ok) break;
        uint4 bits = make_uint4(0, 0, 0, 0);
#pragma unroll 1
        for (int node = r < f.nodes ? r : -1; node >= 0; node = up[node]) {
          const uint32_t bit = 1u << (node & 31);
          if (node < 64) {
            if (node < 32) bits.x |= bit; else bits.y |= bit;
          } else {
            if (node < 96) bits.z |= bit; else bits.w |= bit;
          }
        }
        seen[par][r] = bits;
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k_full[kc & 1]);
        mbar_arrive(&empty[st]);
      }
      ++kc;
      if (++st == S::kStages) {
        st = 0;
        phase ^= 1;
      }
    }
  } else {
    // ---------------- softmax: a KV row per thread, a share of the columns
    const int h = warp >> 2, qd = warp & 3, r = threadIdx.x & 127, bar = 1 + h;
    const uint32_t sub = (uint32_t)(32 * qd) << 16;
#pragma unroll 1
    for (int i = 0;; ++i) {
      bool ok = wait(&s_full[i & 1], (uint32_t)(i >> 1) & 1u);
      const Info& f = infos[i % kInfos];
      const int4 head = *reinterpret_cast<const int4*>(&f);
      const int flags = ok ? head.x : kStop, valid = r < 64 ? head.z : head.w;
      const int par = (flags >> 8) & 3, n = head.y;
      const bool first = flags & kFirst;
      const uint32_t sc = tmem + S::kSCol + (i & 1) * NT + sub;
      uint8_t* const dst = ps + (kTwice ? 0 : (i & 1) * S::kP) + (r >> 3) * 1024 + (r & 7) * 128;
      float* const line = lines[par];
      tc_fence_after();
      // P's place is free once PV(i - kPs) is done
      constexpr int kPs = kTwice ? 1 : 2;
      if (!(flags & kStop) && i >= kPs) ok = wait(&p_empty[(i - kPs) & 1], (uint32_t)((i - kPs) >> 1) & 1u);
      const bool plain = !(flags & kDraft) && (r & 32) + 32 <= valid;  // every row of the warp counts, for all columns
      float ks = 1.f, low = 1.f;
      if (flags & kDraft) {
        ok = ok && wait(&lifted[par], (uint32_t)(f.count >> 2) & 1u);
        ks = k_scale[par][r];
        low = 1.f / lifted_by(v_lift[par]);
      }
      // eight arguments from column x on; those that this row does not have are -inf
      auto arguments = [&](int x, float (&a)[8]) {
        __syncwarp();
        tmem_ld8(sc + x, reinterpret_cast<uint32_t(&)[8]>(a));
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = fmaf(a[e] * ks, line[x + e], line[NT + x + e]);
        if (flags & kDraft) {
          int token = (f.c0 + x) / p.hpk, sub_head = (f.c0 + x) - token * p.hpk;
          const uint32_t* bits = reinterpret_cast<const uint32_t*>(seen[par]) + qd;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (x + e >= f.cols || !((bits[4 * min(token, kMaxNodes - 1)] >> lane) & 1u)) a[e] = -INFINITY;
            if (++sub_head == p.hpk) {
              sub_head = 0;
              ++token;
            }
          }
        } else if ((r & 63) >= valid) {
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] = -INFINITY;
        }
      };
      auto put = [&](int c, const uint32_t (&w)[4], const uint32_t (&rest)[4]) {
        uint8_t* const to = dst + (c >> 6) * (kRows * 128) + ((((c & 63) >> 3) ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        if (kTwice) *reinterpret_cast<uint4*>(to + S::kP) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
      };
      // find: the largest arguments of all columns; otherwise their weights into P, and the largest argument. (One copy
      // of the general arguments for both.)
      auto columns = [&](bool find) {
        float top = -INFINITY;
        if (plain && !find) {
#pragma unroll 1
          for (int x = 8 * h; x < n; x += 8 * kGroups) {
            uint32_t sv[8], w[4], rest[4];
            tmem_ld8(sc + x, sv);
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
              const float4 a = *reinterpret_cast<const float4*>(line + x + e), b = *reinterpret_cast<const float4*>(line + NT + x + e);
              const float2 u = __ffma2_rn(make_float2(__uint_as_float(sv[e]), __uint_as_float(sv[e + 1])), make_float2(a.x, a.y), make_float2(b.x, b.y));
              const float2 v = __ffma2_rn(make_float2(__uint_as_float(sv[e + 2]), __uint_as_float(sv[e + 3])), make_float2(a.z, a.w), make_float2(b.z, b.w));
              top = fmaxf(top, fmaxf(u.x, u.y));
              top = fmaxf(top, fmaxf(v.x, v.y));
              if (kTwice) {
                split(ex2(u.x), ex2(u.y), w[e / 2], rest[e / 2]);
                split(ex2(v.x), ex2(v.y), w[e / 2 + 1], rest[e / 2 + 1]);
              } else {
                w[e / 2] = as_u32(__floats2half2_rn(ex2(u.x), ex2(u.y)));
                w[e / 2 + 1] = as_u32(__floats2half2_rn(ex2(v.x), ex2(v.y)));
              }
            }
            put(x, w, rest);
          }
          return top;
        }
#pragma unroll 1
        for (int x = 8 * h; x < n; x += 8 * kGroups) {
          float a[8];
          arguments(x, a);
          if (find) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float m = redux_max(a[e]);
              if (lane == 0) quad[qd][x + e] = m;
            }
          } else {
            uint32_t w[4], rest[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              top = fmaxf(top, fmaxf(a[2 * e], a[2 * e + 1]));
              split(ex2(a[2 * e]) * low, ex2(a[2 * e + 1]) * low, w[e], rest[e]);
            }
            put(x, w, rest);
          }
        }
        return top;
      };
      float top = -INFINITY;
      if (!ok) dead[h] = 1;
      bool leave = false;
      // weights, a vote; where one says so the largest arguments, and weights again
      bool vote = !ok || (flags & (kStop | kFirst));
#pragma unroll 1
      for (;;) {
        bool find = false;
        if (vote) {
          // a new maximum, where a weight would be larger than the lazy ones may be
          find = any_of_128(bar, first || top > kBias + kLazy);
          leave = (flags & kStop) || *reinterpret_cast<volatile int*>(&dead[h]);
          if (leave || !find) break;
        }
#pragma unroll 1
        for (;; find = false) {
          top = columns(find);
          if (!find) break;
          any_of_128(bar, false);
          const int mine = 8 * h + r % 8 + r / 8 * 8 * kGroups;  // a column of the group
          if (mine < n) {
            float m = fmaxf(fmaxf(quad[0][mine], quad[1][mine]), fmaxf(quad[2][mine], quad[3][mine])) - kBias;
            if (!first) m = fmaxf(m, 0.f);
            if (!(fabsf(m) < 1e37f)) m = 0.f;  // (no row, of which the second kernel knows by the sum, or a score that is not finite)
            change[mine] = ex2(-m);
            line[NT + mine] -= m;
          }
          // (O of the blocks before is complete)
          if (!first && !wait(&p_empty[(i - 1) & 1], (uint32_t)((i - 1) >> 1) & 1u)) dead[h] = 1;
          any_of_128(bar, false);
          leave = *reinterpret_cast<volatile int*>(&dead[h]);
          if (leave) break;
          tc_fence_after();
          if (!first) {
#pragma unroll 1
            for (int k = -1; k < S::kHalves; ++k)  // the sums of the weights, and O
#pragma unroll 1
              for (int x = 8 * h; x < n; x += 8 * kGroups) {
                const uint32_t oc = tmem + S::kOCol + k * NT + x + sub;
                uint32_t o[8];
                __syncwarp();
                tmem_ld8(oc, o);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * change[x + e]);
                tmem_st8(oc, o);
              }
            tmem_wait_st();
          }
        }
        if (leave || vote) break;
        vote = true;
      }
      if (leave) break;
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[i & 1]);
      if (!(flags & (kLast | kOut))) continue;

      // ---------------- the end of the segment, in this CTA, or of what the tensor core sums at a time
      // (where the wait gave up, the numbers are not the segment's, and the next vote ends the role)
      if (!wait(&p_empty[i & 1], (uint32_t)(i >> 1) & 1u)) dead[h] = 1;
      tc_fence_after();
      if (flags & (kOut | kHeld)) move_sums<HD, NT>(p, f, line, tmem);
      if (flags & kOut) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty);
        continue;
      }
      const bool alone = flags & kAlone;
      const int slot = 2 * blockIdx.x + (flags & kOpens ? 1 : 0);
      bool bad = k_again[par] != 0 || ((flags & kDraft) && v_again[par] != 0);
      if (qd * 32 < S::kERows) {
#pragma unroll 1
        for (int k = 0; k < S::kHalves; ++k) {
          const int e = 128 * k + 32 * qd + lane;
#pragma unroll 1
          for (int x = 8 * h; x < f.cols; x += 8 * kGroups) {  // (columns past f.cols are padding)
            uint32_t o[8], l[8];
            __syncwarp();
            tmem_ld8_async(tmem + S::kLCol + x + sub, l);
            tmem_ld8(tmem + S::kOCol + k * NT + x + sub, o);
            const int left = f.cols - x;
            if (alone) {
              const int token = (f.c0 + x) / p.hpk;
              int sub_head = (f.c0 + x) - token * p.hpk;
              T* out = static_cast<T*>(p.out) + (f.r0 + token) * p.out_row + (int64_t)(f.kv * p.hpk + sub_head) * p.out_head + e;
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const float v = __fdividef(__uint_as_float(o[c]), __uint_as_float(l[c]));
                if (c < left) {
                  bad |= !(fabsf(v) <= 3.402823466e38f);
                  *out = from_f32<T>(v);
                }
                out += p.out_head;
                if (++sub_head == p.hpk) {
                  sub_head = 0;
                  out += p.out_row - p.hpk * p.out_head;
                }
              }
            } else {
              float* part = p.parts + ((size_t)slot * NT + x) * HD + e;
#pragma unroll
              for (int c = 0; c < 8; ++c)
                if (c < left) {
                  bad |= !(fabsf(__uint_as_float(o[c])) <= 3.402823466e38f);
                  part[c * HD] = __uint_as_float(o[c]);
                }
              if (k == 0 && qd == 0) {
#pragma unroll
                for (int c = 0; c < 8; ++c)
                  if (lane == c && c < left)
                    p.stats[(size_t)slot * NT + x + c] = make_float2(kBias - line[NT + x + c], __uint_as_float(l[c]));
              }
            }
          }
        }
      }
      // what came out not finite, or may owe its value to an infinity of f16, is computed again: by the CTA at its end, or by
      // the second kernel
      bad = any_of_128(bar, bad);
      if (!alone) {
        if (r == 0) {
          p.again[kGroups * slot + h] = bad;
          if (h == 0 && (flags & kOpens)) p.opened[blockIdx.x] = Opened{f.run, f.seq, f.kv, f.r0, f.len, f.c0, f.cols, 0};
        }
      } else if (bad && r == 0) {
        const int bit = min(f.count, kBits - 1);
        atomicOr(&again[bit >> 5], 1u << (bit & 31));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSWarp) {
    warp_wait(&fin, 0u, p.err);  // no product still runs when its TMEM is freed
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (__any_sync(0xffffffffu, again[lane] != 0)) compute_again<HD, NT, T>(p, first_seq, first_base, all_units, again);
}

// Joins the parts of the segment that a CTA opened and others share, in the order of the CTAs; where f16 did not hold
// its values it is computed again in 32 bits.
constexpr int kJoinThreads = 256;
template <int HD, int NT, typename T>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ TreeParams p, int ctas) {
  constexpr int kAtOnce = 4;
  pdl_launch_dependents();
  pdl_wait();
  const Opened f = p.opened[blockIdx.x];
  if (f.run < 2 || f.run > ctas - (int)blockIdx.x) return;
  // the part that starts the segment is its CTA's slot 1, the others slot 0
  auto slot = [&](int i) { return (size_t)2 * (blockIdx.x + i) + (i == 0 ? 1 : 0); };
  int again = 0;
  for (int i = threadIdx.x & 31; i < f.run; i += 32)
    for (int h = 0; h < kGroups; ++h) again |= p.again[kGroups * slot(i) + h];
  if (__any_sync(0xffffffffu, again != 0)) {
    for (int c = blockIdx.y * (kJoinThreads / 32) + (threadIdx.x >> 5); c < f.cols; c += gridDim.y * (kJoinThreads / 32)) {
      const int token = (f.c0 + c) / p.hpk;
      plain_row<HD, T>(p, f.seq, f.r0, f.len, f.r0 + token, f.kv, f.kv * p.hpk + (f.c0 + c) - token * p.hpk);
    }
    return;
  }
  for (int x = blockIdx.y * kJoinThreads + threadIdx.x; x < f.cols * HD / 4; x += kJoinThreads * gridDim.y) {
    const int c = x / (HD / 4), e = 4 * (x % (HD / 4));
    float top = kNone, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < f.run; i0 += kAtOnce) {
      float2 st[kAtOnce];
      float4 o[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        st[k] = make_float2(kNone, 0.f);
        o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + k < f.run) {
          st[k] = __ldcg(&p.stats[slot(i0 + k) * NT + c]);
          o[k] = __ldcg(reinterpret_cast<const float4*>(p.parts + (slot(i0 + k) * NT + c) * HD + e));
        }
      }
      float next = top;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        if (!(st[k].y > 0.f)) st[k].x = kNone;  // (no row of this part counts for the column)
        next = fmaxf(next, st[k].x);
      }
      const float keep = ex2(top - next);
      top = next;
      sum *= keep;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= keep;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const float w = ex2(st[k].x - top);
        sum = fmaf(w, st[k].y, sum);
        v[0] = fmaf(w, o[k].x, v[0]);
        v[1] = fmaf(w, o[k].y, v[1]);
        v[2] = fmaf(w, o[k].z, v[2]);
        v[3] = fmaf(w, o[k].w, v[3]);
      }
    }
    const float inv = 1.f / sum;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= inv;
    const int token = (f.c0 + c) / p.hpk, head = f.kv * p.hpk + (f.c0 + c) - token * p.hpk;
    store_vec<T, 4>(static_cast<T*>(p.out) + (f.r0 + token) * p.out_row + head * p.out_head + e, v);
  }
}

template <int HD, int NT, typename T>
cudaError_t launch(const LaunchEnv& env, const TreeParams& p) {
  using S = Sizes<HD, NT>;
  CUtensorMap map{};
  if (p.n_pages > 0 && !encode_2d(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.pages, 128, (uint64_t)p.n_pages * p.nkv * (S::kPage / 128),
                                  128, 128, S::kPage / 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return cudaErrorInvalidValue;
  auto kern = tree_kernel<HD, NT, T>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
  if (e != cudaSuccess) return e;
  e = rrr_launch_pdl(kern, dim3(env.sm_count), dim3(kThreads), (size_t)S::kSmem, env.stream, env.pdl, map, p);
  if (e != cudaSuccess) return e;
  return rrr_launch_pdl(tree_join_kernel<HD, NT, T>, dim3(env.sm_count, 6), dim3(kJoinThreads), 0, env.stream, env.pdl, p,
                        env.sm_count);
}
template <int HD>
cudaError_t launch_type(const LaunchEnv& env, int type, const TreeParams& p) {
  // Tiles of 96 columns where a sequence's (row, query head) pairs do not fit one of 64 on average, since every tile reads
  // the pages: 32 sequences of 24 rows on up to 4,000, 24 heads on 8 of 128, 109 us (of 64: 164), one of 60 rows on 60,000
  // 116 (145), 24 of 12 rows, 64 heads on 8 of 64, 87 (119); and where they do fit the smaller tile, whose scores
  // and sums are fewer: 32 of 16 rows 92 (of 96: 98), 32 of 8 rows of 32 heads, f16, 107 (118). Heads of 256 leave no room in TMEM.
  if constexpr (HD < 256)
    if ((int64_t)p.rows * p.hpk > 64 * (int64_t)p.n_seqs)
      return type == RRR_F16 ? launch<HD, 96, __half>(env, p) : launch<HD, 96, __nv_bfloat16>(env, p);
  return type == RRR_F16 ? launch<HD, 64, __half>(env, p) : launch<HD, 64, __nv_bfloat16>(env, p);
}

// The workspace: segments opened, statistics, flags, sums moved out, parts; for the widest tiles
struct Layout {
  int64_t stats, again, held_stats, held, parts, bytes;
};
Layout layout_of(const rrr_kv4_cache* c, int sms) {
  const int64_t slots = 2 * (int64_t)sms;
  Layout l;
  l.stats = ((int64_t)sms * (int64_t)sizeof(Opened) + 255) / 256 * 256;
  l.again = l.stats + slots * 96 * 8;
  l.held_stats = l.again + (slots * 4 * kGroups + 255) / 256 * 256;
  l.held = l.held_stats + (int64_t)sms * 4 * 96 * 8;
  l.parts = l.held + (int64_t)sms * 96 * c->head_dim * 4;
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
  // (a page is addressed by its line of 128 bytes, the work counted in 32 bits)
  const int64_t tiles = (kMaxNodes * (int64_t)(n_heads / c->n_kv_heads) + 63) / 64;
  if (c->n_pages * c->n_kv_heads > INT32_MAX / (80 * c->head_dim / 128) ||
      (__int128)c->n_seqs * c->n_kv_heads * tiles * (c->max_pages / 2 + 2 + kStart) > INT32_MAX)
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: too many pages, or sequences times heads times pages of a sequence", fn);
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
  *bytes = layout_of(c, ctx->sm_count).bytes;
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
  const Layout l = layout_of(c, ctx->sm_count);
  char* w = static_cast<char*>(workspace);
  p.opened = reinterpret_cast<Opened*>(w);
  p.stats = reinterpret_cast<float2*>(w + l.stats);
  p.again = reinterpret_cast<int*>(w + l.again);
  p.parts = reinterpret_cast<float*>(w + l.parts);
  p.held_stats = reinterpret_cast<float2*>(w + l.held_stats);
  p.held = reinterpret_cast<float*>(w + l.held);
  cudaError_t e;
  switch (hd) {
    case 64: e = launch_type<64>(env, d->type, p); break;
    case 128: e = launch_type<128>(env, d->type, p); break;
    default: e = launch_type<256>(env, d->type, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_attention_tree_kv4 launch");
}

}  // extern "C"
