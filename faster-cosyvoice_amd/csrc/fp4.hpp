// Shared pieces of the 4-bit operators (linear_fp4.hip, kv_fp4.hip, attention_fp4.hip): conversions
// between 4-bit numbers and the types that the matrix instructions take, and a page's parts.
#pragma once

#include <type_traits>

#include "../../include/fcv_fp4.h"
#include "lm.hpp"

namespace fcv {
namespace lm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 2^(b - 127) of a scale byte as the conversions take it: they look at the exponent alone, where 0 stands
// for 2^-127 and 255 makes their result NaN.
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b << 23); }

// The two codes of byte `kByte` of w, times a power of two, as a pair of E's elements: v_cvt_scalef32_pk_*
// (the low half of the byte in the low half of the pair).
template <class E, int kByte>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  if constexpr (std::is_same<E, Half>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, kByte));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte));
}

// The 8 codes of a word.
template <class E>
__device__ __forceinline__ s16x8 fp4_octet(uint32_t w, float scale) {
  const u32x4 v = {fp4_pair<E, 0>(w, scale), fp4_pair<E, 1>(w, scale), fp4_pair<E, 2>(w, scale),
                   fp4_pair<E, 3>(w, scale)};
  return __builtin_bit_cast(s16x8, v);
}

// Limits of a group's exponent: every code times 2^e is a number of the type.
__host__ __device__ constexpr int fp4_min_exp(bool f16) { return f16 ? -23 : -125; }
__host__ __device__ constexpr int fp4_max_exp(bool f16) { return f16 ? 13 : 125; }

// The scale byte of a group from the bits of its largest magnitude (fp32): the smallest exponent e with
// magnitude < 7 2^e.  1.75 2^x = 7 2^(x - 2), so e is x - 2 or, from that on, x - 1.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t top, bool f16) {
  if (top >= 0x7f800000u) return 255;
  const int e = (int)(top >> 23) - 127 - 2 + ((top & 0x7fffffu) >= 0x600000u);
  return (uint32_t)(min(max(e, fp4_min_exp(f16)), fp4_max_exp(f16)) + 127);
}

// 8 values over a power of two to codes: to the nearest number, ties to the even code, 6 at most.
__device__ __forceinline__ uint32_t fp4_word(const float* v, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
}

// Byte offsets of a page's parts of one head.
template <int D>
struct Page {
  static constexpr int kTokens = FCV_FP4_PAGE;
  static constexpr int kKey = D / 2;                       // bytes of a token's key
  static constexpr int kKeyScales = D / 32;
  static constexpr int kValues = kTokens * D / 2;          // offsets
  static constexpr int kScales = kTokens * D;
  static constexpr int kValueScales = kScales + kTokens * kKeyScales;
  static constexpr int kBytes = kValueScales + kTokens;
};

// Whether pages lie as the kernels read and write them: on 16-byte boundaries, none over another.
inline bool pages_fit(const void* pages, int64_t page_stride, int64_t head_stride, int32_t n_pages,
                      int32_t n_kv_heads, int32_t head_dim) {
  const int64_t bytes = FCV_FP4_PAGE * (head_dim + head_dim / 32 + 1), far = 1LL << 40;
  if (!aligned(pages, 16)) return false;
  if (n_pages > 1 && (page_stride < bytes || page_stride > far || page_stride % 16)) return false;
  if (n_kv_heads > 1 && (head_stride < bytes || head_stride > far || head_stride % 16)) return false;
  return n_pages <= 1 || n_kv_heads <= 1 || page_stride >= (n_kv_heads - 1) * head_stride + bytes ||
         head_stride >= (n_pages - 1) * page_stride + bytes;
}

}  // namespace lm
}  // namespace fcv
