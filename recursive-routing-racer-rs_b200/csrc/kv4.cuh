// kv4.cuh — the page layout of the 4-bit KV cache (rrr_kv4_cache) shared by the kernels that
// write it, read it back and attend over it. Offsets in bytes inside the block of one (page,
// KV head); the order of the codes is the order in which lane (g, t) = (lane / 4, lane % 4)
// of a warp feeds them to mma.m16n8k16 as A operands (kv4_attention.cu). And the codes of eight
// values, as rrr_kv4_store and rrr_kv4_append take them (kv4_rows.cu has the mathematics).
#pragma once
#include "serve_common.cuh"

namespace rrr {

constexpr int kPageRows = 64;

template <int HD>
struct Kv4Block {
  static constexpr int kGroups = HD / 32;                 // groups of 32 values per head
  static constexpr int kJ = kGroups < 4 ? kGroups : 4;    // groups per plane
  static constexpr int kPlanes = kGroups / kJ;
  static constexpr int kPlaneWords = kPageRows * 4 * kJ;  // u32 of codes per plane
  static constexpr int kCodes = 32 * HD, kScales = 4 * HD;
  static constexpr int kHalf = kCodes + 2 * kScales;      // K, then V
  static constexpr int kBytes = 2 * kHalf;
  // u32 index of the K codes of (row, group j, elements 32j + 8t ..)
  __device__ static constexpr int k_word(int row, int j, int t) {
    return (j / kJ) * kPlaneWords + (row * 4 + t) * kJ + j % kJ;
  }
  // u16 index of the V codes of (row, group j, elements 32j + g, + 8, + 16, + 24)
  __device__ static constexpr int v_half(int row, int j, int g) {
    return 2 * ((j / kJ) * kPlaneWords + (((row >> 3) * 8 + g) * 4 + ((row & 7) >> 1)) * kJ + j % kJ) + (row & 1);
  }
  // f16 index of a row's d and of K's m, and of V's m
  __device__ static constexpr int scale(int row, int j) { return row * kGroups + j; }
  __device__ static constexpr int v_min(int row, int j) { return ((row >> 1) * kGroups + j) * 2 + (row & 1); }
};

// Codes of four values by the division itself (out of line: rarely called)
static __device__ __noinline__ uint32_t divided(float a, float b, float c, float e, float m, float d) {
  auto code = [&](float x) {
    return (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x, m), d)), 0.f), 15.f);
  };
  return code(a) | code(b) << 4 | code(c) << 8 | code(e) << 12;
}
// The least and the largest of three, NaN where one is
__device__ __forceinline__ float least(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float largest(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Eight values of a group of 32, which four neighbouring lanes hold: their codes, value i at bit
// 4i, and the group's d and m. With kOff, whether values that are off by up to `off` (the group's)
// could have this lane's codes, d or m other than these.
template <bool kOff = false>
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], __half& d16, __half& m16, float off = 0.f,
                                             bool* unsure = nullptr) {
  const float inf = __int_as_float(0x7f800000);
  float lo = least(least(x[0], x[1], x[2]), least(x[3], x[4], x[5]), least(x[6], x[7], x[7]));
  float hi = largest(largest(x[0], x[1], x[2]), largest(x[3], x[4], x[5]), largest(x[6], x[7], x[7]));
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float l = __shfl_xor_sync(0xffffffffu, lo, o), h = __shfl_xor_sync(0xffffffffu, hi, o);
    lo = least(lo, l, l);
    hi = largest(hi, h, h);
  }
  const bool finite = fabsf(lo) < inf && fabsf(hi) < inf;
  // (hi - lo) / 15 by the product with 1/15 and its remainder
  const float range = __fsub_rn(hi, lo), first = __fmul_rn(range, 1.f / 15.f);
  const float step = fmaf(fmaf(-15.f, first, range), 1.f / 15.f, first);
  m16 = __float2half_rn(fminf(fmaxf(lo, -65504.f), 65504.f));
  d16 = finite ? __float2half_rn(fminf(range > 1e6f ? 65504.f : step, 65504.f)) : __ushort_as_half(0x7fff);
  const float d = __half2float(d16), m = __half2float(m16);
  const float inv = d > 0.f ? __fdividef(1.f / 15.f, d) : 0.f;
  float furthest = 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = __saturatef(__fmul_rn(__fsub_rn(x[i], m), inv));  // in units of 15, within 0..15
    const float t = fmaf(q, 15.f, 12582912.f);                      // the nearest integer in the low bits
    furthest = fmaxf(furthest, fabsf(fmaf(q, 15.f, 12582912.f - t)));
    w += __float_as_uint(t) << (4 * i);
  }
  // what 12582912's own bits added
  w -= 0x4b400000u + 0xb4000000u + 0x40000000u;
  if (furthest > 0.49999f && d > 0.f)
    w = divided(x[0], x[1], x[2], x[3], m, d) | divided(x[4], x[5], x[6], x[7], m, d) << 16;
  if (kOff) {
    auto apart = [](float at, float by) {
      return __half_as_ushort(__float2half_rn(at - by)) != __half_as_ushort(__float2half_rn(at + by));
    };
    *unsure = finite && (apart(lo, off) || apart(step, off * 0.134f) || furthest > fmaf(off, -15.1f * inv, 0.49998f));
  }
  return w;
}
// Argument rules of an rrr_kv4_cache (kv4_rows.cu).
int check_kv4_cache(rrr_ctx* ctx, const rrr_kv4_cache* c, const char* fn);

}  // namespace rrr
