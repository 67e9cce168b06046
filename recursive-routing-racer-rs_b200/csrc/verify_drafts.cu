// verify_drafts.cu — which drafted tokens stand, given the target's logits and random numbers, and
// the token that follows them (rrr_verify_drafts). The greedy scan over one row of logits
// (src/model/phi4.rs:1172-1183) is the case of one row and temperature 0.
//
// Mathematics. With p = softmax(x / T) of a row of logits and a number u in [0, 1), the drawn token
// is the first i with p_0 + .. + p_i > u. Trees without the draft's logits: the token drawn at a
// row is the target's own sample; if a child of the row carries it, that child stands and the
// walk goes on there. Chains with the draft's logits, q = softmax(y / T): a drafted token x stands
// if u q(x) < p(x), and where the first does not, the token is drawn from max(p - q, 0), which
// leaves the target's distribution unchanged.
//
// Exactness. The border between two of 200,000 tokens moves with every rounding before it: at a
// relative error of 2^-24 one draw in some fifty would come out as a neighbour. So exponentials and
// sums are held in 64 bits; an error of 2^-44 leaves one in 10^7.
//
// Exponentials. (x - top) c = n + r, n the nearest multiple of 1/16 (the product added to 1.5 2^48 leaves
// 16 n in the low bits), |r| <= 1/32 from one more fma, exact; 2^n from a table of 16 in shared
// memory, which fills its 32 banks, and the exponent's bits; 2^r - 1 by a polynomial of degree 5
// (interpolated at Chebyshev nodes), off by 2^-46.6: eleven operations of 64 bits.
//
// A row is cut into chunks of 4 KB at 16-byte borders of memory. First kernel: per chunk the
// maximum, its first place and the sum of the exponentials under it, one warp each. Trees: a second
// kernel, one CTA per row, draws the row's token: its chunk from the chunks' sums, then the token
// inside it; a third, one CTA per sequence, walks. Chains with the draft's logits: one CTA per sequence
// compares, then the chunks of the row where the chain ends are summed as max(p - q, 0), and one CTA
// per sequence draws.
//
// What bounds it. Issue slots (70 % used) and latencies of the first kernel: 30 warp instructions for 32 values, of which
// eleven operations and a conversion go to the 64-bit pipe, half busy. 48 chains of 5 rows and their drafts on 200,064
// tokens, f32: 147 us (346 MB, 53 us), of which the first kernel takes 110, of greedy ones 70; 285 rows of trees, bf16:
// 62-72 us (114 MB, 17 us), some 60 of them, greedy 31. CUDA's exp2 took 302 and 327 us.
#include <float.h>

#include "serve_common.cuh"

namespace rrr {
namespace {

constexpr int kStatWarps = 8, kWalkThreads = 256, kKept = 2048;
constexpr int kChunkBytes = 4096, kRestChunk = 1024;

struct Stat {  // of one chunk
  double sum;  // of 2^((x - top) c)
  float top;
  int best;    // the first place of top
};
struct Ending {  // of a chain
  double pz, qz;  // the sums under the maxima
  float pm, qm;
  int last;       // the last row that stands
  int refused;    // whether the draft after it was refused, and the draw is from the rest
};

struct VerifyParams {
  const void* logits;
  const void* draft;
  int64_t logits_stride, draft_stride;
  const int* tokens;
  const int* cu;
  const int* parents;
  const float* uniforms;  // [rows][2]
  const float* temperature;
  int* path;
  int* counts;
  int* next;
  int rows, vocab, n_seqs, chunks, rest_chunks;
  Stat* p_stats;  // [rows][chunks]
  Stat* q_stats;
  Ending* endings;
  double* rest;   // [n_seqs][rest_chunks]
  int* drawn;     // [rows]
  int* err;
};

// x as the softmax takes it: NaN is no value, +inf the largest one
__device__ __forceinline__ float tidy(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }
// 2^y, y <= 0
__device__ __forceinline__ double exp2_of(double y) { return exp2(y); }
// The exponentials 2^((x - top) c) of values up to `top`; fine: whether they can be taken this way.
// Values that are 1000 binary orders and more under the top count as such, NaN too.
struct Powers {
  double c, top;
  float lowest;
  bool fine;
};
__device__ __forceinline__ Powers powers_of(float top, double c) {
  Powers w;
  w.c = c;
  w.top = (double)top;
  w.lowest = __double2float_rd(w.top - 1000. / c);
  const double span = (w.top - (double)w.lowest) * c;  // (roundings may leave it another one)
  w.fine = top < INFINITY && w.lowest >= -FLT_MAX && span > 980. && span < 1020.;
  return w;
}
__device__ __forceinline__ double power(const Powers& w, const double* table, float x) {
  constexpr double kMagic = 422212465065984.;  // 1.5 2^48
  const double v = (double)fmaxf(x, w.lowest) - w.top;
  const double t = fma(v, w.c, kMagic);
  const double r = fma(v, w.c, kMagic - t);
  double p = fma(r, 0.0013333744338239965, 0.009618317140580765);
  p = fma(r, p, 0.05550410866027587);
  p = fma(r, p, 0.24022650691319414);
  p = fma(r, p, 0.6931471805599453);
  const int n = __double2loint(t);
  const double step = table[n & 15];
  p = fma(step, r * p, step);
  return __hiloint2double(__double2hiint(p) + ((n & ~15) << 16), __double2loint(p));
}
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 16) table[threadIdx.x] = exp2(threadIdx.x * 0.0625);
  __syncthreads();
}
// The number that a row's draft stands by (0) or its token is drawn by (1); none that is negative, and 0 for NaN (draw() takes
// a negative one for none, and a draft without a chance would stand by it)
__device__ __forceinline__ double number_of(const VerifyParams& p, int64_t row, int which) {
  return fmax((double)p.uniforms[2 * row + which], 0.);
}
// log2(e) / T; 0 for temperature 0 (and, recorded, for one that is none)
__device__ __forceinline__ double sharpness(const VerifyParams& p, int seq) {
  const float t = p.temperature ? p.temperature[seq] : 1.f;
  if (t == 0.f) return 0.;
  if (!(t > 0.f) || t > FLT_MAX) {
    flag_position(p.err);
    return 0.;
  }
  return 1.4426950408889634 / (double)t;
}
// The elements before a row's first that its first 16 bytes of memory hold
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
// The sequence of a packed row, by a warp; false where there is none
__device__ __forceinline__ bool find_seq(const VerifyParams& p, int row, int& seq) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.n_seqs;  // the last s with cu[s] <= row
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, s = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, s < hi && p.cu[s] <= row);
    lo += below ? (31 - __clz(below)) * step : 0;
    hi = min(hi, lo + step);
  }
  seq = lo;
  return p.cu[lo] <= row && row < p.cu[lo + 1];
}
// The rows of a sequence; false (and recorded) where cu is wrong
__device__ __forceinline__ bool rows_of(const VerifyParams& p, int seq, int& r0, int& n) {
  r0 = p.cu[seq];
  const int r1 = p.cu[seq + 1];
  n = r1 - r0;
  if (r0 >= 0 && r1 >= r0 && r1 <= p.rows) return true;
  if (threadIdx.x == 0) flag_position(p.err);
  return false;
}

template <typename T>
__global__ void __launch_bounds__(32 * kStatWarps, 4) verify_stats_kernel(const __grid_constant__ VerifyParams p) {
  constexpr int kVec = 16 / (int)sizeof(T), kSteps = kChunkBytes / 512, kChunk = kChunkBytes / (int)sizeof(T);
  __shared__ double table[16];
  fill_table(table);
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kStatWarps + (threadIdx.x >> 5);
  const int64_t rows = item / p.chunks;
  const int chunk = (int)(item - rows * p.chunks);
  const bool is_q = rows >= p.rows;
  const int row = (int)(is_q ? rows - p.rows : rows);
  if (row >= p.rows || (is_q && !p.draft)) return;
  const T* x = is_q ? static_cast<const T*>(p.draft) + row * p.draft_stride
                    : static_cast<const T*>(p.logits) + row * p.logits_stride;
  const int shift = shift_of(x);
  const T* base = x - shift;
  union {
    uint4 raw[kSteps];
    T v[kSteps * kVec];
  } u;
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int at = chunk * kChunk + (k * 32 + lane) * kVec;
    if (at >= shift && at + kVec <= shift + p.vocab) {
      u.raw[k] = __ldcs(reinterpret_cast<const uint4*>(base + at));
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        u.v[k * kVec + i] = at + i >= shift && at + i < shift + p.vocab ? base[at + i] : from_f32<T>(-INFINITY);
    }
  }
  int seq;  // (sought while the values are on their way)
  Stat* const to = (is_q ? p.q_stats : p.p_stats) + (int64_t)row * p.chunks + chunk;
  if (!find_seq(p, row, seq) || (is_q && row == p.cu[seq])) {
    if (lane == 0) *to = Stat{0., -INFINITY, INT32_MAX};  // (sequences that overlap may come to it)
    return;
  }
  const double c = sharpness(p, seq);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSteps * kVec; ++i) top = fmaxf(top, to_f32(u.v[i]));
  const float mine = top = fminf(top, FLT_MAX);
  // (so that the words and not the values read from them stay in registers)
#pragma unroll
  for (int k = 0; k < kSteps; ++k) asm volatile("" : "+r"(u.raw[k].x), "+r"(u.raw[k].y), "+r"(u.raw[k].z), "+r"(u.raw[k].w));
  const bool infinite = __any_sync(0xffffffffu, mine == FLT_MAX);
  top = warp_max(top);
  int best = INT32_MAX;
  double sum = 0.;
  if (c == 0.) {
#pragma unroll
    for (int i = kSteps * kVec - 1; i >= 0; --i)
      if (to_f32(u.v[i]) >= top) best = i;
    if (mine < top || top == -INFINITY) best = INT32_MAX;
    if (best < INT32_MAX) best = chunk * kChunk + (best / kVec * 32 + lane) * kVec + best % kVec - shift;
    best = __reduce_min_sync(0xffffffffu, best);
  } else if (top > -INFINITY) {
    const Powers w = powers_of(top, c);
    if (w.fine && !infinite) {
#pragma unroll
      for (int i = 0; i < kSteps * kVec; ++i) sum += power(w, table, to_f32(u.v[i]));
    } else {
#pragma unroll 1
      for (int i = 0; i < kSteps * kVec; ++i) {
        const int at = chunk * kChunk + (i / kVec * 32 + lane) * kVec + i % kVec;
        const float v = at >= shift && at < shift + p.vocab ? tidy(to_f32(base[at])) : -INFINITY;
        if (v > -INFINITY) sum += exp2_of(((double)v - (double)top) * c);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (lane == 0) *to = Stat{sum, top, best};
}

// ---- one CTA of kWalkThreads threads per sequence
struct Shared {
  double sums[kWalkThreads / 32];
  float tops[kWalkThreads / 32];
  int low, high;
  double before;
  double kept[kKept];  // the weights of a draw, each read by the thread that wrote it
};
__device__ __forceinline__ double block_sum_before(Shared& sh, double v, double& total) {  // of the threads before
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double w = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += w;
  }
  if (lane == 31) sh.sums[warp] = upto;
  __syncthreads();
  double before = 0.;
  total = 0.;
#pragma unroll
  for (int w = 0; w < kWalkThreads / 32; ++w) {
    if (w < warp) before += sh.sums[w];
    total += sh.sums[w];
  }
  const double last = __shfl_up_sync(0xffffffffu, upto, 1);
  __syncthreads();
  return before + (lane ? last : 0.);
}
__device__ __forceinline__ float block_max(Shared& sh, float v) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) sh.tops[threadIdx.x >> 5] = v;
  __syncthreads();
  float m = sh.tops[0];
#pragma unroll
  for (int w = 1; w < kWalkThreads / 32; ++w) m = fmaxf(m, sh.tops[w]);
  __syncthreads();
  return m;
}
// The first i < n whose weights up to it, before + weight(0) + .. + weight(i), exceed the goal; with
// u >= 0 the goal becomes u times the weights' total. The last i with a weight where roundings leave
// none, -1 where there is no weight. *prior: the sum before i.
template <class F>
__device__ __forceinline__ int draw(Shared& sh, int n, double u, double& goal, double before, F&& weight, double* prior) {
  const int per = (n + kWalkThreads - 1) / kWalkThreads;
  const int a = min(n, (int)threadIdx.x * per), b = min(n, a + per);
  double mine = 0., total;
  int last = -1;
#pragma unroll 4
  for (int i = a; i < b; ++i) {
    const double w = weight(i);
    if (n <= kKept) sh.kept[i] = w;
    mine += w;
    if (w > 0.) last = i;
  }
  auto again = [&](int i) { return n <= kKept ? sh.kept[i] : weight(i); };
  if (threadIdx.x == 0) {
    sh.low = INT32_MAX;
    sh.high = -1;
  }
  double upto = before + block_sum_before(sh, mine, total);
  if (u >= 0.) goal = u * total;
  const double from = upto;
  if (last >= 0) {
    atomicMax(&sh.high, last);
    if (upto + mine > goal) {
      for (int i = a; i < b; ++i) {
        const double w = again(i);
        upto += w;
        if (w > 0. && upto > goal) {
          atomicMin(&sh.low, i);
          break;
        }
      }
    }
  }
  __syncthreads();
  const int got = sh.low != INT32_MAX ? sh.low : sh.high;
  if (prior && got >= a && got < b) {
    double s = from;
    for (int i = a; i < got; ++i) s += again(i);
    sh.before = s;
  }
  __syncthreads();
  if (prior) *prior = sh.before;
  __syncthreads();
  return got;
}

// The token drawn at a row (temperature 0, c = 0: the greedy one); -1 where no token has a weight.
template <typename T>
__device__ __forceinline__ int draw_token(Shared& sh, const VerifyParams& p, int row, double c, double u) {
  constexpr int kChunk = kChunkBytes / (int)sizeof(T);
  const Stat* st = p.p_stats + (int64_t)row * p.chunks;
  float top = -INFINITY;
  for (int i = threadIdx.x; i < p.chunks; i += kWalkThreads) top = fmaxf(top, st[i].top);
  top = block_max(sh, top);
  if (!(top > -INFINITY)) return -1;
  if (c == 0.) {
    if (threadIdx.x == 0) sh.low = INT32_MAX;
    __syncthreads();
    for (int i = threadIdx.x; i < p.chunks; i += kWalkThreads)
      if (st[i].top == top) atomicMin(&sh.low, st[i].best);
    __syncthreads();
    const int got = sh.low;
    __syncthreads();
    return got;
  }
  const double m = (double)top;
  auto chunk_weight = [&](int i) {
    const Stat s = st[i];
    return s.sum > 0. ? s.sum * exp2_of(((double)s.top - m) * c) : 0.;
  };
  double goal, before;
  const int chunk = draw(sh, p.chunks, u, goal, 0., chunk_weight, &before);
  if (chunk < 0) return -1;
  const T* x = static_cast<const T*>(p.logits) + row * p.logits_stride;
  const int first = max(0, chunk * kChunk - shift_of(x)), end = min(p.vocab, (chunk + 1) * kChunk - shift_of(x));
  const int got = draw(sh, end - first, -1., goal, before, [&](int i) {
    const float v = tidy(to_f32(x[first + i]));
    return v > -INFINITY ? exp2_of(((double)v - m) * c) : 0.;
  }, nullptr);
  return got < 0 ? -1 : first + got;
}

template <typename T>
__global__ void __launch_bounds__(kWalkThreads) verify_tokens_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ Shared sh;
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x;
  int seq;
  if (!find_seq(p, row, seq)) {
    if (threadIdx.x == 0) p.drawn[row] = -1;
    return;
  }
  const int token = draw_token<T>(sh, p, row, sharpness(p, seq), number_of(p, row, 1));
  if (threadIdx.x == 0) p.drawn[row] = token;
}
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ int child[2];
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.x;
  int r0, n;
  if (!rows_of(p, seq, r0, n)) n = 0;
  int at = 0, count = 0, token = -1;
  if (threadIdx.x == 0) child[0] = INT32_MAX;
  while (count < n) {
    int& next = child[count & 1];
    if (threadIdx.x == 0) p.path[r0 + count] = at;
    token = p.drawn[r0 + at];
    ++count;
    __syncthreads();
    if (threadIdx.x == 0) child[count & 1] = INT32_MAX;  // (all have read it)
    if (token < 0) break;
    // (a parent lies before its child)
    for (int i = at + 1 + threadIdx.x; i < n; i += kWalkThreads) {
      const int up = p.parents ? p.parents[r0 + i] : i - 1;
      if (up < -1 || up >= i) flag_position(p.err);
      if (up == at && p.tokens[r0 + i] == token) atomicMin(&next, i);
    }
    __syncthreads();
    if (next == INT32_MAX) break;
    at = next;
  }
  if (threadIdx.x == 0) {
    p.counts[seq] = count;
    p.next[seq] = token;
  }
  for (int i = count + threadIdx.x; i < n; i += kWalkThreads) p.path[r0 + i] = -1;
}

// The maximum and the sum of a row from its chunks, by a warp
__device__ __forceinline__ void warp_stats(const Stat* st, int n, double c, float& top, double& sum) {
  const int lane = threadIdx.x & 31;
  top = -INFINITY;
#pragma unroll 8
  for (int i = lane; i < n; i += 32) top = fmaxf(top, st[i].top);
  top = warp_max(top);
  sum = 0.;
  if (!(top > -INFINITY)) return;
#pragma unroll 4
  for (int i = lane; i < n; i += 32) {
    const Stat s = st[i];
    if (s.sum > 0.) sum += s.sum * exp2_of(((double)s.top - (double)top) * c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
}
__device__ __forceinline__ double share(float x, float top, double sum, double c) {
  x = tidy(x);
  return x > -INFINITY ? exp2_of(((double)x - (double)top) * c) / sum : 0.;
}

// Which drafts of a chain stand: a warp per draft, until the first that does not.
template <typename T>
__global__ void __launch_bounds__(kWalkThreads) verify_chain_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ int refused;
  __shared__ Ending ends[kWalkThreads / 32];  // of the drafts that are looked at together
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int r0, n;
  if (!rows_of(p, seq, r0, n)) n = 0;
  const double c = sharpness(p, seq);
  if (threadIdx.x == 0) refused = n;
  __syncthreads();
  for (int i0 = 1; i0 < n; i0 += kWalkThreads / 32) {
    const int i = i0 + warp;
    if (i < n) {
      const int64_t row = r0 + i;
      const int x = p.tokens[row];
      const Stat* st = p.p_stats + (row - 1) * p.chunks;
      float pm = 0.f, qm = 0.f;
      double pz = 0., qz = 0.;
      bool stands = false;
      if (c != 0.) {
        warp_stats(st, p.chunks, c, pm, pz);
        warp_stats(p.q_stats + row * p.chunks, p.chunks, c, qm, qz);
        if (lane == 0) ends[warp] = Ending{pz, qz, pm, qm, i - 1, pz > 0. && qz > 0.};
      }
      if (x < 0 || x >= p.vocab) {
        // no token: it does not stand
      } else if (c == 0.) {
        warp_stats(st, p.chunks, 0., pm, pz);
        int best = INT32_MAX;
        for (int k = lane; k < p.chunks; k += 32)
          if (st[k].top == pm) best = min(best, st[k].best);
        stands = pm > -INFINITY && __reduce_min_sync(0xffffffffu, best) == x;
      } else {
        const double pp = share(to_f32(static_cast<const T*>(p.logits)[(row - 1) * p.logits_stride + x]), pm, pz, c);
        const double q = share(to_f32(static_cast<const T*>(p.draft)[row * p.draft_stride + x]), qm, qz, c);
        stands = number_of(p, row, 0) * q < pp;
      }
      if (!stands && lane == 0) atomicMin(&refused, i);
    }
    __syncthreads();
    const bool stop = refused < n;
    __syncthreads();
    if (stop) break;
  }
  const int count = n ? refused : 0;
  if (threadIdx.x == 0 && n)
    p.endings[seq] = c != 0. && count < n ? ends[(count - 1) % (kWalkThreads / 32)] : Ending{0., 0., 0.f, 0.f, count - 1, 0};
  if (threadIdx.x == 0) p.counts[seq] = count;
  for (int i = threadIdx.x; i < n; i += kWalkThreads) p.path[r0 + i] = i < count ? i : -1;
}

// max(p - q, 0) of tokens where a chain ends, from their logits. The sums of chunks and the draw inside one are of the same
// terms, so that a chunk with a sum has a term to be drawn. power() gives values 1000 binary orders under the top, masked ones
// too, 2^-1000: beside a p of 2^-940 and more that is no q, and a smaller p is taken as it is, 0 where it is masked.
// Where the weights under p's and q's maxima are all equal, p and q are, and no rest is left, though their sums may be a rounding
// apart (rows that begin at other places of 16 bytes are summed in another order). A chunk of such weights alone has its sum with
// a minus.
struct Rest {
  Powers wp, wq;
  double sp, sq;
  float faint, none;  // x whose p is under 2^-940 of the top's, and 0 in 64 bits
  bool fast;
};
__device__ __forceinline__ Rest rest_from(const Ending& e, double c) {
  Rest r;
  r.wp = powers_of(e.pm, c);
  r.wq = powers_of(e.qm, c);
  r.sp = 1. / e.pz;
  r.sq = 1. / e.qz;
  r.faint = __double2float_ru(r.wp.top - 940. / c);
  r.none = __double2float_rd(r.wp.top - 1080. / c);
  // (tops of FLT_MAX may stand for infinities)
  r.fast = r.wp.fine && r.wq.fine && e.pm < FLT_MAX && e.qm < FLT_MAX;
  return r;
}
__device__ __noinline__ double rest_apart(float x, float y, const Ending& e, double c) {
  return fmax(share(x, e.pm, e.pz, c) - share(y, e.qm, e.qz, c), 0.);
}
// (with r.fast; the products rounded each by itself, so that of equal ones nothing is left) differ: bits where weights differ
__device__ __forceinline__ double rest_of(const Rest& r, const double* table, float x, float y, const Ending& e, double c,
                                          int& differ) {
  const double p = power(r.wp, table, x), q = power(r.wq, table, y);
  differ |= __double2hiint(p) ^ __double2hiint(q);
  differ |= __double2loint(p) ^ __double2loint(q);
  const double d = fmax(__dmul_rn(p, r.sp) - __dmul_rn(q, r.sq), 0.);
  if (x <= r.faint && x > r.none) {
    differ = 1;
    return rest_apart(x, y, e, c);
  }
  return x > r.faint ? d : 0.;
}
template <typename T>
__global__ void __launch_bounds__(32 * kStatWarps) verify_rest_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ double table[16];
  fill_table(table);
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.y, lane = threadIdx.x & 31, chunk = blockIdx.x * kStatWarps + (threadIdx.x >> 5);
  int r0, n;
  if (chunk >= p.rest_chunks || !rows_of(p, seq, r0, n) || n == 0) return;
  const Ending e = p.endings[seq];
  if (!e.refused) return;
  const double c = sharpness(p, seq);
  const T* x = static_cast<const T*>(p.logits) + (int64_t)(r0 + e.last) * p.logits_stride;
  const T* y = static_cast<const T*>(p.draft) + (int64_t)(r0 + e.last + 1) * p.draft_stride;
  double sum = 0.;
  const int first = chunk * kRestChunk, end = min(p.vocab, first + kRestChunk);
  const Rest rest = rest_from(e, c);
  int differ = 0;
  if (rest.fast) {
    constexpr int kStep = 8;
#pragma unroll 1
    for (int i0 = first + lane; i0 < end; i0 += 32 * kStep) {
      float a[kStep], b[kStep];
#pragma unroll
      for (int k = 0; k < kStep; ++k) {
        const int i = i0 + 32 * k;
        a[k] = i < end ? to_f32(x[i]) : -INFINITY;
        b[k] = i < end ? to_f32(y[i]) : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < kStep; ++k) sum += rest_of(rest, table, a[k], b[k], e, c, differ);
    }
  } else {
#pragma unroll 1
    for (int i = first + lane; i < end; i += 32) {
      const float v = tidy(to_f32(x[i])), w = tidy(to_f32(y[i]));
      differ |= (double)v - (double)e.pm != (double)w - (double)e.qm;
      sum += rest_apart(v, w, e, c);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (!__any_sync(0xffffffffu, differ)) sum = -sum;
  if (lane == 0) p.rest[(int64_t)seq * p.rest_chunks + chunk] = sum;
}
template <typename T>
__global__ void __launch_bounds__(kWalkThreads) verify_draw_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ Shared sh;
  __shared__ double table[16];
  fill_table(table);
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.x;
  int r0, n, token = -1;
  if (!rows_of(p, seq, r0, n)) n = 0;
  if (n > 0) {
    const Ending e = p.endings[seq];
    const double c = sharpness(p, seq), u = number_of(p, r0 + e.last, 1);
    if (e.refused) {
      const double* rest = p.rest + (int64_t)seq * p.rest_chunks;
      double goal, before;
      bool differ = false;
      for (int i = threadIdx.x; i < p.rest_chunks; i += kWalkThreads) differ = differ || !signbit(rest[i]);
      int chunk = -1;
      if (__syncthreads_or(differ)) chunk = draw(sh, p.rest_chunks, u, goal, 0., [&](int i) { return fabs(rest[i]); }, &before);
      if (chunk >= 0) {
        const T* x = static_cast<const T*>(p.logits) + (int64_t)(r0 + e.last) * p.logits_stride;
        const T* y = static_cast<const T*>(p.draft) + (int64_t)(r0 + e.last + 1) * p.draft_stride;
        const int first = chunk * kRestChunk, end = min(p.vocab, first + kRestChunk);
        const Rest terms = rest_from(e, c);
        const int got = draw(sh, end - first, -1., goal, before, [&](int i) {
          const float v = to_f32(x[first + i]), w = to_f32(y[first + i]);
          int unused = 0;
          return terms.fast ? rest_of(terms, table, v, w, e, c, unused) : rest_apart(v, w, e, c);
        }, nullptr);
        if (got >= 0) token = first + got;
      }
    }
    // (where p nowhere exceeds q, by roundings, p itself)
    if (token < 0) token = draw_token<T>(sh, p, r0 + e.last, c, u);
  }
  if (threadIdx.x == 0) p.next[seq] = token;
}

template <typename T>
cudaError_t launch(const LaunchEnv& env, const VerifyParams& p) {
  const int64_t items = (int64_t)p.rows * (p.draft ? 2 : 1) * p.chunks;
  if (p.rows > 0) {
    const cudaError_t e = rrr_launch_pdl(verify_stats_kernel<T>, dim3((unsigned)((items + kStatWarps - 1) / kStatWarps)),
                                         dim3(32 * kStatWarps), 0, env.stream, env.pdl, p);
    if (e != cudaSuccess) return e;
  }
  const dim3 seqs((unsigned)p.n_seqs), block(kWalkThreads);
  cudaError_t e = cudaSuccess;
  if (!p.draft) {
    if (p.rows > 0) e = rrr_launch_pdl(verify_tokens_kernel<T>, dim3((unsigned)p.rows), block, 0, env.stream, env.pdl, p);
    return e != cudaSuccess ? e : rrr_launch_pdl(verify_walk_kernel, seqs, block, 0, env.stream, env.pdl, p);
  }
  e = rrr_launch_pdl(verify_chain_kernel<T>, seqs, block, 0, env.stream, env.pdl, p);
  if (e == cudaSuccess)
    e = rrr_launch_pdl(verify_rest_kernel<T>, dim3((p.rest_chunks + kStatWarps - 1) / kStatWarps, (unsigned)p.n_seqs),
                       dim3(32 * kStatWarps), 0, env.stream, env.pdl, p);
  if (e == cudaSuccess) e = rrr_launch_pdl(verify_draw_kernel<T>, seqs, block, 0, env.stream, env.pdl, p);
  return e;
}

int64_t padded(int64_t n) { return (n + 255) / 256 * 256; }
struct Layout {
  int chunks, rest_chunks;
  int64_t q, endings, rest, drawn, bytes;
};
Layout layout_of(int rows, int vocab, int n_seqs, bool draft) {
  Layout l;
  l.chunks = (int)(((int64_t)vocab + 7 + 1023) / 1024);  // of 4 KB at most, wherever the row begins
  l.rest_chunks = (int)(((int64_t)vocab + kRestChunk - 1) / kRestChunk);
  l.q = padded((int64_t)rows * l.chunks * (int64_t)sizeof(Stat));
  l.endings = l.q * (draft ? 2 : 1);
  l.rest = l.endings + (draft ? padded((int64_t)n_seqs * (int64_t)sizeof(Ending)) : 0);
  l.drawn = l.rest + (draft ? padded((int64_t)n_seqs * l.rest_chunks * 8) : 0);
  l.bytes = l.drawn + (draft ? 0 : padded(4 * (int64_t)rows));
  if (l.bytes < 256) l.bytes = 256;
  return l;
}
int check_verify(rrr_ctx* ctx, int rows, int vocab, int n_seqs, const char* fn) {
  if (!ctx) return set_error(nullptr, RRR_ERR_INVALID_ARG, "null context");
  if (rows < 0 || n_seqs < 0 || vocab < 1 || vocab > 1 << 28 || rows > 1 << 24 || n_seqs > 65535 ||
      (int64_t)rows * ((vocab + 1030) / 1024) > (int64_t)1 << 32)
    return set_error(ctx, RRR_ERR_BAD_SHAPE,
                     "%s: need 0 <= rows <= 2^24, 1 <= vocab <= 2^28, 0 <= n_seqs <= 65535 and rows * vocab up to 2^42", fn);
  return RRR_OK;
}

}  // namespace
}  // namespace rrr

using namespace rrr;

extern "C" {

int rrr_verify_workspace(rrr_ctx* ctx, int rows, int vocab, int n_seqs, int with_draft, int64_t* bytes) {
  const char* fn = "rrr_verify_workspace";
  const int rc = check_verify(ctx, rows, vocab, n_seqs, fn);
  if (rc) return rc;
  if (!bytes) return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  *bytes = layout_of(rows, vocab, n_seqs, with_draft != 0).bytes;
  return RRR_OK;
}

int rrr_verify_drafts(rrr_ctx* ctx, int type, const void* logits, int64_t logits_stride, const void* draft,
                      int64_t draft_stride, int rows, int vocab, int n_seqs, const int32_t* cu_rows,
                      const int32_t* tokens, const int32_t* parents, const float* uniforms,
                      const float* temperature, int32_t* path, int32_t* counts, int32_t* next_tokens,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  const char* fn = "rrr_verify_drafts";
  int rc = check_verify(ctx, rows, vocab, n_seqs, fn);
  if (rc) return rc;
  if (!row_type(type)) return set_error(ctx, RRR_ERR_BAD_QTYPE, "%s: type must be 0 (F32), 1 (F16) or 30 (BF16)", fn);
  if (!workspace || (n_seqs > 0 && (!cu_rows || !counts || !next_tokens)) ||
      (rows > 0 && (!logits || !tokens || !uniforms || !path)))
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (draft && parents)
    return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: drafts with their logits are chains (parents NULL)", fn);
  if (!stride_fits(logits_stride, vocab) || (draft && !stride_fits(draft_stride, vocab)))
    return set_error(ctx, RRR_ERR_BAD_SHAPE, "%s: row strides of vocab to 2^38", fn);
  const int es = elem_bytes(type);
  if (!aligned_to(logits, es) || !aligned_to(draft, es) || !aligned_to(cu_rows, 4) || !aligned_to(tokens, 4) ||
      !aligned_to(parents, 4) || !aligned_to(uniforms, 4) || !aligned_to(temperature, 4) || !aligned_to(path, 4) ||
      !aligned_to(counts, 4) || !aligned_to(next_tokens, 4) || !aligned_to(workspace, 16))
    return set_error(ctx, RRR_ERR_MISALIGNED, "%s: arrays must be aligned to their elements, the workspace to 16 bytes", fn);
  const Layout l = layout_of(rows, vocab, n_seqs, draft != nullptr);
  if (workspace_bytes < l.bytes)
    return set_error(ctx, RRR_ERR_BUFFER_TOO_SMALL, "%s: the workspace needs %lld bytes", fn, (long long)l.bytes);
  const RowSet out[4] = {{path, 4 * (int64_t)rows, 4 * (int64_t)rows, rows ? 1 : 0},
                         {counts, 4 * (int64_t)n_seqs, 4 * (int64_t)n_seqs, n_seqs ? 1 : 0},
                         {next_tokens, 4 * (int64_t)n_seqs, 4 * (int64_t)n_seqs, n_seqs ? 1 : 0},
                         {workspace, l.bytes, l.bytes, 1}};
  const RowSet in[7] = {{logits, logits_stride * es, (int64_t)vocab * es, rows},
                        {draft, draft_stride * es, (int64_t)vocab * es, rows},
                        {tokens, 4 * (int64_t)rows, 4 * (int64_t)rows, rows ? 1 : 0},
                        {parents, 4 * (int64_t)rows, 4 * (int64_t)rows, rows ? 1 : 0},
                        {uniforms, 8 * (int64_t)rows, 8 * (int64_t)rows, rows ? 1 : 0},
                        {cu_rows, 4 * ((int64_t)n_seqs + 1), 4 * ((int64_t)n_seqs + 1), n_seqs ? 1 : 0},
                        {temperature, 4 * (int64_t)n_seqs, 4 * (int64_t)n_seqs, n_seqs ? 1 : 0}};
  for (int i = 0; i < 4; ++i) {
    bool fine = true;
    for (const RowSet& x : in) fine = fine && rows_disjoint(out[i], x);
    for (int j = 0; j < i; ++j) fine = fine && rows_disjoint(out[i], out[j]);
    if (!fine)
      return set_error(ctx, RRR_ERR_INVALID_ARG, "%s: path, counts, next_tokens and the workspace must overlap nothing", fn);
  }
  DeviceGuard dev(ctx);
  if (dev.rc) return dev.rc;
  if (n_seqs == 0) return RRR_OK;
  const LaunchEnv env = make_env(ctx, stream);
  char* ws = static_cast<char*>(workspace);
  const int chunk = kChunkBytes / es;
  const VerifyParams p{logits, draft, logits_stride, draft_stride, tokens, cu_rows, parents, uniforms, temperature,
                       path, counts, next_tokens, rows, vocab, n_seqs,
                       (int)(((int64_t)vocab + 16 / es - 1 + chunk - 1) / chunk), l.rest_chunks,
                       reinterpret_cast<Stat*>(ws), reinterpret_cast<Stat*>(ws + l.q),
                       reinterpret_cast<Ending*>(ws + l.endings), reinterpret_cast<double*>(ws + l.rest),
                       reinterpret_cast<int*>(ws + l.drawn), env.d_err};
  cudaError_t e;
  switch (type) {
    case RRR_F32: e = launch<float>(env, p); break;
    case RRR_F16: e = launch<__half>(env, p); break;
    default: e = launch<__nv_bfloat16>(env, p); break;
  }
  return e == cudaSuccess ? RRR_OK : cuda_error(ctx, e, "rrr_verify_drafts launch");
}

}  // extern "C"
