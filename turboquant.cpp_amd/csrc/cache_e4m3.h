// Pages of keys and values in 8 bits: e4m3 codes with a scale, a power of two, for each block of 16 positions of a layer's kv
// head, keys and values apart.
//
// A pool holds [pages][layers][kv heads][page_size * hd] codes; a page's positions come in tiles of 64.  Within a tile
//   keys    lie [hd / 16][64 positions][16 numbers]: lane (r, c) of an operand of 16 rows reads 16 bytes, the numbers 16 c .. 16 c + 15
//           of 64 of its row, and 16 rows are 256 bytes in a row: whole lines, whatever the head size;
//   values  lie [hd][4][4][4], position 16 j + 4 c + i at [c][j][i]: the 16 bytes of dimension d and quarter c are the 16 keys
//           whose scores lane (., c) holds when the first product is done, in the order in which it holds them.
// A number is code * scale.  Why powers of two: code * scale is then exact in bfloat16 (4 significant bits), so the matrix cores see
// the numbers themselves, one instruction makes two of them from codes and scale, and a block that takes a larger scale because a
// later token is larger moves its codes' exponents only (what falls below 2^-6 of the new scale is rounded once more).
// The scale is the smallest power of two, 2^-100 at least, whose 448 fold is no smaller than the block's largest magnitude.
// A row whose key or value holds a number that is not finite (or is 2^120 or more) keeps NaN for its key and 0 for its value:
// whoever sees the row gets NaN, and 0 times NaN never reaches those who do not.
#pragma once
#include "common.h"

#define E4M3_BLOCK 16
#define E4M3_TILE 64
#define E4M3_LEAST (-100)
#define E4M3_TOO_LARGE 1.329227995784916e36f      // 2^120

struct E4m3Pages {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;               // [pages][layers][kv heads][page_size / 16]
  float* v_scale;
  float* weight;                // null, or [pages][layers][kv heads][page_size]: the attention weight each position has received
  const int* table;             // [slots][bt_stride]
  int bt_stride, page_size, heads, head0, hd;      // heads: layers * kv heads; head0: the layer's first
};

// Where the tile with position 64 t of the sequence with that row of the table lies: the index of (page, layer, kv head), or -1, and
// the tile within the page.
__device__ __forceinline__ int64_t e4m3_head_of(const E4m3Pages& p, const int* row, int t, int kvh, int& in_page) {
  const int per = p.page_size / E4M3_TILE;
  in_page = t % per;
  const int page = row[t / per];
  return page < 0 ? -1 : (int64_t)page * p.heads + p.head0 + kvh;
}
__device__ __forceinline__ int64_t e4m3_tile_at(const E4m3Pages& p, int64_t head, int in_page) {
  return (head * p.page_size + in_page * E4M3_TILE) * p.hd;
}
__device__ __forceinline__ int64_t e4m3_scale_at(const E4m3Pages& p, int64_t head, int in_page) {
  return (head * p.page_size + in_page * E4M3_TILE) / E4M3_BLOCK;
}

// The scale of a block whose largest magnitude is `top` (finite, 0 or more).
__device__ __forceinline__ float e4m3_scale(float top) {
  const uint32_t b = __float_as_uint(top);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
  if (e < E4M3_LEAST) e = E4M3_LEAST;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// 1 / scale for a scale that e4m3_scale gave; 0 for 0.
__device__ __forceinline__ float e4m3_inverse(float scale) {
  return scale == 0.f ? 0.f : __uint_as_float(0x7f000000u - __float_as_uint(scale));
}

// Four numbers to codes, rounded to the nearest, ties to even.
__device__ __forceinline__ uint32_t e4m3_codes(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// Four codes to numbers, times `by`, to codes again.
__device__ __forceinline__ uint32_t e4m3_rescale(uint32_t w, float a, float b, float c, float d) {
  return e4m3_codes(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * a, __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * b,
                    __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * c, __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * d);
}

// Whether the sizes are such as every kernel of these pages takes.
static inline bool e4m3_pages_fit(int page_size, int heads, int head0, int nkv, int hd) {
  return page_size >= E4M3_TILE && page_size % E4M3_TILE == 0 && hd >= 16 && hd <= 256 && hd % 16 == 0 && nkv > 0 && nkv <= 65535 &&
         head0 >= 0 && heads >= head0 + nkv;
}
