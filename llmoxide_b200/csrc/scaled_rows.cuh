// Cached rows of 8 bits with one float32 scale a row, and what their writers and readers share.
//
// A row x of D numbers (a token's key or value of one kv head) is held as y = round(x * (m / a)) with the scale s = a / m,
// a = max |x|; it stands for y * s.  m = 127 and whole numbers (int8, ties to even), or m = 448 and e4m3.  Rows whose a is
// below 2^-100 are held as zeros with scale 0; a row with an infinity or a NaN as zeros with scale NaN, so that whatever
// sees it is NaN, as it would be over the row itself.  The cache is [pages][G][64][D] bytes and [pages][G][64] scales.
//
// The attention kernels multiply the held numbers as float16, which holds each of them exactly (8 and 4 significant bits), and
// apply the scales to the float32 scores and probabilities.  What meets them in a product is float16 too: queries times a
// power of two a row, chosen so that bfloat16 queries stay exact, and probabilities with the values' scales in them, relative
// to the row's largest such weight, rounded to 11 bits.  float16 rather than bfloat16: three bits more in
// the probabilities, and two instructions a pair of int8 numbers where bfloat16 takes three.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "tc_ptx.cuh"

enum { ROWS_INT8 = 0, ROWS_E4M3 = 1 };
template <int FMT> __device__ __forceinline__ constexpr float rows_max() { return FMT == ROWS_INT8 ? 127.f : 448.f; }
#define ROWS_TINY 7.888609052210118e-31f          // 2^-100

// What a row of largest magnitude `a` is multiplied by, and its scale.
template <int FMT>
__device__ __forceinline__ void rows_scale(float a, float& inv, float& scale) {
  const bool fine = a < INFINITY;                  // false for a NaN too
  const bool tiny = a < ROWS_TINY;
  inv = rows_max<FMT>() / a, scale = a / rows_max<FMT>();
  if (tiny) inv = scale = 0.f;
  if (!fine) inv = 0.f, scale = __int_as_float(0x7fc00000);
}
// Four numbers as four bytes.  (inv 0: zeros, also for what is not finite.)
template <int FMT>
__device__ __forceinline__ uint32_t rows_pack4(float x0, float x1, float x2, float x3, float inv) {
  if (inv == 0.f) return 0u;
  x0 *= inv, x1 *= inv, x2 *= inv, x3 *= inv;
  if (FMT == ROWS_INT8)
    return (uint32_t)(__float2int_rn(x0) & 255) | ((uint32_t)(__float2int_rn(x1) & 255) << 8) |
           ((uint32_t)(__float2int_rn(x2) & 255) << 16) | ((uint32_t)__float2int_rn(x3) << 24);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x0, x1), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x2, x3), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Four bytes as four float32 numbers.
template <int FMT>
__device__ __forceinline__ float4 rows_unpack4(uint32_t w) {
  if (FMT == ROWS_INT8)
    return make_float4((float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24));
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffff), __NV_E4M3);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
  const float2 x = __half22float2(__half2(a)), y = __half22float2(__half2(b));
  return make_float4(x.x, x.y, y.x, y.y);
}

// Two bytes as a pair of float16.  int8: the bytes lie in the low byte of each half of `t`; 1024 + 128 + y is a float16 number
// one masked exclusive-or away, and 1152 is subtracted: two instructions.  e4m3: they lie side by side in the low half, and
// one conversion makes both.
template <int FMT>
__device__ __forceinline__ uint32_t rows_pair(uint32_t t) {
  uint32_t r;
  if (FMT == ROWS_INT8) {
    const uint32_t a = (t & 0x00ff00ffu) ^ 0x64806480u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x64806480u));
  } else {
    const uint16_t h = (uint16_t)t;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  }
  return r;
}
// The four numbers of a word as two pairs, in the order that costs least: int8 0 2 and 1 3, e4m3 0 1 and 2 3.  (Whatever they
// are multiplied with is laid out in the same order: rows_second is the number that follows 0.)
template <int FMT> __device__ __forceinline__ constexpr int rows_second() { return FMT == ROWS_INT8 ? 2 : 1; }
template <int FMT> __device__ __forceinline__ uint32_t rows_low(uint32_t w) { return rows_pair<FMT>(w); }
template <int FMT> __device__ __forceinline__ uint32_t rows_high(uint32_t w) { return rows_pair<FMT>(FMT == ROWS_INT8 ? w >> 8 : w >> 16); }
// Bytes E and E + 1 (E 0 or 2) of two words, as a pair of the words' bytes E and one of their bytes E + 1.
template <int FMT, int E>
__device__ __forceinline__ void rows_across(uint32_t w0, uint32_t w1, uint32_t& first, uint32_t& second) {
  if (FMT == ROWS_INT8) {
    first = rows_pair<FMT>(__byte_perm(w0, w1, E * 0x0011 + (4 + E) * 0x1100));
    second = rows_pair<FMT>(__byte_perm(w0, w1, (E + 1) * 0x0011 + (5 + E) * 0x1100));
  } else {
    const uint32_t t = __byte_perm(w0, w1, E + (4 + E) * 0x10 + (E + 1) * 0x100 + (5 + E) * 0x1000);
    first = rows_pair<FMT>(t), second = rows_pair<FMT>(t >> 16);
  }
}

// Numbers in float16 terms: x = the sum of TERMS terms, to 11 TERMS bits.
template <int TERMS>
__device__ __forceinline__ void rows_split2(float x, float y, uint32_t (&out)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    const __half2 h = __floats2half2_rn(x, y);
    out[i] = *reinterpret_cast<const uint32_t*>(&h);
    if (i + 1 < TERMS) x -= __low2float(h), y -= __high2float(h);
  }
}
__device__ __forceinline__ uint32_t rows_bf16x2(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The power of two that brings a magnitude to [2^target, 2^(target+1)), and its inverse; at most 2^118, so that the inverse is
// a normal number with room for a further factor, and never 0.
__device__ __forceinline__ void rows_power(float largest, int target, float& mul, float& inverse) {
  const int e = min(245, target + 254 - (int)(__float_as_uint(largest) >> 23 & 255u));
  mul = __uint_as_float((uint32_t)e << 23), inverse = __uint_as_float((uint32_t)(254 - e) << 23);
}
#define ROWS_QUERY_POWER 13       // queries: largest of a row below 2^14
// Weights: exp(s_j - r) vs_j, the probability of a key with its value's scale in it.  The reference r of a row follows the
// largest s_j + log(vs_j) that the row sees, not the largest s_j, so that the largest weight comes to 2^13 whatever the
// scales: float16 ends at 2^16 and steps by 2^-24 at its lower end, so a weight 2^-27 of the row's largest loses digits and one
// below 2^-38 vanishes, and neither a key that a row does not see nor one that it gives no weight has a say in that.  The
// row's sum of exp(s_j - r) goes by the same reference, which leaves it far from float32's ends: r is off the largest s_j by the
// log of one scale.
#define ROWS_WEIGHT_POWER 13.f
// log2 of a value's scale, for that reference.  A scale of zeros, or of next to nothing, counts as 2^-96: the sum of such a
// row's exponentials stays finite.
__device__ __forceinline__ float rows_log2(float scale) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fabsf(scale)));
  return fmaxf(y, -96.f);                          // (also for a NaN, which the weight itself carries on)
}

// The bytes [rows, cols] of a cache, in boxes of [box_rows x box_cols], laid down with the swizzle of box_cols bytes
// (64 or 128; none with `plain`).
static int make_rows_map(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t cols, uint32_t box_rows,
                         uint32_t box_cols, bool plain) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return 1;
  cuuint64_t dims[2] = {cols, rows};
  cuuint64_t strides[1] = {cols};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t elem[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE,
                  plain ? CU_TENSOR_MAP_SWIZZLE_NONE
                        : box_cols == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 2;
}
