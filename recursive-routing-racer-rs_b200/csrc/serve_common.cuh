// serve_common.cuh — pieces shared by the packed-batch operators (qk_rows.cu, kv4_rows.cu,
// kv4_attention.cu, attention_packed.cu): element types, vector loads and stores of a lane's
// values, the argument rules that they share, and the current device's guard of their entry
// points.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_internal.h"
#include "internal.h"
#include "rrr_common.cuh"

namespace rrr {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive values in words of up to 16 bytes (p aligned to min(16, N * sizeof(T))).
template <int BYTES>
struct Words {
  static constexpr int kN = BYTES / 16;
  uint4 w[kN];
};
template <>
struct Words<8> {
  uint2 w[1];
};
template <>
struct Words<4> {
  uint32_t w[1];
};
template <typename T, int N>
union Vec {
  Words<N * (int)sizeof(T)> raw;
  T v[N];
  __device__ Vec() {}
};
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  Vec<T, N> u;
  u.raw = *reinterpret_cast<const Words<N * (int)sizeof(T)>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f32(u.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  Vec<T, N> u;
#pragma unroll
  for (int i = 0; i < N; ++i) u.v[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Words<N * (int)sizeof(T)>*>(p) = u.raw;
}

// cos and sin (times af) of a rotation by pos * t turns, t = f / factor / 2 pi (qk_rows.cu has the
// mathematics and the error).
__device__ __forceinline__ void rope_turn(double t, int pos, float af, float& c, float& s) {
  t -= floor(t);
  const unsigned long long F = __double2ull_rd(t * 18446744073709551616.0);
  const unsigned long long a = F * (unsigned long long)(unsigned)pos;
  const float frac = (float)(int)(unsigned)(a >> 32) * 4.656612873077393e-10f;  // 2 x turns, in [-1, 1)
  sincospif(frac, &s, &c);
  c *= af;
  s *= af;
}
// The same in 64 bits
__device__ __forceinline__ void rope_turn(double t, int pos, double af, double& c, double& s) {
  t -= floor(t);
  const unsigned long long a = __double2ull_rd(t * 18446744073709551616.0) * (unsigned long long)(unsigned)pos;
  sincospi((double)(long long)a * 1.0842021724855044e-19, &s, &c);  // 2 x turns, in [-1, 1]
  c *= af;
  s *= af;
}
constexpr int kMaxPairs = 64;  // rope_dim / 2
// turns[i] = theta^(-2i/rope_dim) / 2 pi as a product of two powers: 16 calls of pow and not 64
inline void rope_turns(double (&turns)[kMaxPairs], float theta, int rope_dim) {
  double fine[8], coarse[kMaxPairs / 8];
  for (int i = 0; i < 8; ++i) fine[i] = pow((double)theta, -2.0 * i / rope_dim);
  for (int i = 0; 16 * i < rope_dim; ++i) coarse[i] = pow((double)theta, -16.0 * i / rope_dim) / 6.283185307179586476925;
  for (int i = 0; 2 * i < rope_dim; ++i) turns[i] = coarse[i / 8] * fine[i % 8];
}

__device__ __forceinline__ void flag_position(int* err) {
  if (err) atomicCAS(err, 0, (int)kDevErrPosition);
}

inline int elem_bytes(int type) { return type == RRR_F32 ? 4 : 2; }
inline bool row_type(int type) { return type == RRR_F32 || type == RRR_F16 || type == RRR_BF16; }
inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// A row stride in elements that rows of `width` fit and whose products stay in 64 bits
inline bool stride_fits(int64_t stride, int64_t width) { return stride >= width && stride <= (int64_t)1 << 38; }

// Rows of `width` bytes at a pitch of `stride` bytes.
struct RowSet {
  const void* p;
  int64_t stride, width, rows;
};
// Whether two row sets share no byte (rows of one pitch may interleave).
inline bool rows_disjoint(const RowSet& a, const RowSet& b) {
  if (!a.p || !b.p || a.rows < 1 || b.rows < 1) return true;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  const __int128 ea = (__int128)pa + (__int128)(a.rows - 1) * a.stride + a.width;
  const __int128 eb = (__int128)pb + (__int128)(b.rows - 1) * b.stride + b.width;
  if (ea <= (__int128)pb || eb <= (__int128)pa) return true;
  if (a.stride != b.stride || a.stride < 1) return false;
  const int64_t d = (int64_t)(pb - pa) % a.stride, off = d < 0 ? d + a.stride : d;
  return off >= a.width && off + b.width <= a.stride;
}

// Rows of heads of hd 16-bit values; strides in elements.
struct HeadRows {
  const void* p;
  int64_t rows, row, heads, head, hd;
};
// Whether two such arrays share no byte, for certain: their extents do not meet, or all of their
// places lie apart modulo a stride (both in one buffer whose rows or heads hold a part of each).
inline bool apart(const HeadRows& a, const HeadRows& b) {
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

// Makes the context's device current for one call and puts the caller's back.
struct DeviceGuard {
  int before = -1;
  int rc;
  explicit DeviceGuard(rrr_ctx* ctx) {
    if (cudaGetDevice(&before) != cudaSuccess) before = -1;
    rc = bind_device(ctx);
    if (before == ctx->device) before = -1;
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
};

}  // namespace rrr
