// kv4.cuh — the page layout of the 4-bit KV cache (rrr_kv4_cache) shared by the kernels that
// write it, read it back and attend over it. Offsets in bytes inside the block of one (page,
// KV head); the order of the codes is the order in which lane (g, t) = (lane / 4, lane % 4)
// of a warp feeds them to mma.m16n8k16 as A operands (kv4_attention.cu).
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

// Argument rules of an rrr_kv4_cache (kv4_rows.cu).
int check_kv4_cache(rrr_ctx* ctx, const rrr_kv4_cache* c, const char* fn);

}  // namespace rrr
