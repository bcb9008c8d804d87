// Shared pieces of the speech language model's operators (linear.hip, qk_norm_rope.hip,
// prefix_attention.hip): the two 16-bit element types and their matrix instructions.
#pragma once

#include <string>

#include "../../include/fcv_lm.h"
#include "common.hpp"
#include "status.hpp"

namespace fcv {
namespace lm {

typedef short s16x8 __attribute__((ext_vector_type(8)));  // 8 elements of either type, as bits
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Element types: bits <-> fp32 (to the nearest, ties to even) and D = A B + C on fragments.
struct Half {
  typedef f16x2 T2;
  static constexpr short kInf = 0x7C00;        // +inf, and the exponent's mask
  // Softmax: a row's running maximum follows the true one when that is kLag (in powers of two) above
  // it, so that sums are rescaled seldom, and weights are held at 2^kShift times their size.  fp16:
  // no weight passes 2^15, and one is in the normal range down to 2^-25 of the row's largest (many
  // small weights can carry most of a long row's sum).
  static constexpr float kShift = 11.0f, kLag = 4.0f;
  static __device__ __forceinline__ float to_f32(short b) { return (float)__builtin_bit_cast(f16, b); }
  static __device__ __forceinline__ short from_f32(float v) {
    return __builtin_bit_cast(short, f2h(v));
  }
  static __device__ __forceinline__ f32x16 mfma32(const s16x8& a, const s16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(const s16x8& a, const s16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

struct Bf16 {
  typedef __bf16 T2 __attribute__((ext_vector_type(2)));
  static constexpr short kInf = 0x7F80;
  // bf16 has fp32's range: sums of 2^16 of its largest values do not pass fp32's
  static constexpr float kShift = -24.0f, kLag = 8.0f;
  static __device__ __forceinline__ float to_f32(short b) {
    return __uint_as_float((uint32_t)(uint16_t)b << 16);
  }
  static __device__ __forceinline__ short from_f32(float v) {
    return __builtin_bit_cast(short, (__bf16)v);
  }
  static __device__ __forceinline__ f32x16 mfma32(const s16x8& a, const s16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(const s16x8& a, const s16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// Whether 16-byte accesses fit a dimension of `count` entries; the stride of a single one says nothing.
inline bool stride_fits(int64_t stride, int64_t count) {
  return count <= 1 || (stride >= 0 && stride % 8 == 0);
}

inline bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

constexpr int kCus = 256;  // compute units of the MI355X

}  // namespace lm
}  // namespace fcv
