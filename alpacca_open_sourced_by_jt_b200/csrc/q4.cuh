// The 4-bit cache: how a pool holds its rows.
//
// 32 consecutive values of a row (a block) are d * (code - 8): codes of 4 bits
// and a f16 scale of 8 significant bits, so that every value is exact in f16
// (11 bits).  16 consecutive rows of one KV head are a granule of 18 D bytes:
//   8 D  K codes    [D / (32 NBP) planes][16 rows][4 words of a block][NBP blocks]
//   8 D  V codes    [D / 8 words of the row][16 rows]
//   D    K scales   [16 rows][D / 32 blocks] f16
//   D    V scales   the same
// with NBP = min(4, D / 32) and words of 8 consecutive dims: dim 2i in bits
// 4i .. 4i + 3, dim 2i + 1 in bits 4i + 16 .. 4i + 19.
//
// Why so: a page of a head is one run of granules, so one bulk copy brings K and
// V of any number of rows, and a granule is what a warp's MMAs take (16 keys).
// Masked with 0x000f000f (0x00f000f0) a word is a pair of f16 subnormals, code x
// 2^-24 (2^-20), of two neighbouring dims: MMA operands without a conversion.
// The words that a lane needs, its dims of every block of a plane for K, its
// dims of four rows for V, are 16 bytes side by side.
#pragma once

#include "b2a_common.cuh"

namespace b2a {

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}

namespace q4 {

__host__ __device__ constexpr int granule_bytes(int D) { return 18 * D; }

// Byte offsets inside a granule: the word of dims 8u .. 8u + 7 of row r, the
// scale of block b.
__device__ __forceinline__ int k_word(int D, int r, int u) {
  const int lg = D >= 128 ? 2 : 1, b = u >> 2;  // 4 or 2 blocks in a plane
  return ((b >> lg) << (8 + lg)) + (r << (4 + lg)) + ((u & 3) << (2 + lg)) + (b & ((1 << lg) - 1)) * 4;
}
__device__ __forceinline__ int v_word(int D, int r, int u) { return 8 * D + u * 64 + r * 4; }
__device__ __forceinline__ int k_scale(int D, int r, int b) { return 16 * D + (r * (D / 32) + b) * 2; }
__device__ __forceinline__ int v_scale(int D, int r, int b) { return 17 * D + (r * (D / 32) + b) * 2; }

// A pool as the kernels see it; page_bytes apart, heads inside a page dense.
struct Pool {
  unsigned char* base;
  long long page_bytes;
  int page_shift;  // log2 of a page's rows; table-less caches: -1
  int head_bytes;  // a page's granules of one head
  int n_pages;
};

// Granule that holds row `in_page` of a page, for KV head h.
__device__ __forceinline__ unsigned char* granule(const Pool& p, int D, long long page, int h,
                                                  int in_page) {
  return p.base + page * p.page_bytes + static_cast<long long>(h) * p.head_bytes +
         static_cast<long long>(in_page >> 4) * granule_bytes(D);
}

}  // namespace q4
}  // namespace b2a
