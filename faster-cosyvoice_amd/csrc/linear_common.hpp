// What the linear layers share (linear.hip, linear_fp4.hip): the epilogue act(sum + bias) + residual, the
// join of cut K ranges, row loads from any boundary, and the pieces of a tile kernel.
#pragma once

#include <algorithm>
#include <type_traits>

#include "lm.hpp"

namespace fcv {
namespace lm {
namespace {

struct Args {
  FcvLmLinear p;
  bool vec;                 // four columns of y, the residual and the bias are on the boundary of four
  int splits, slices;       // ranges of K, and the slices of one: of 64, or of 128 over 4-bit weights
  float* part;              // [splits][m][part_ld] sums of the ranges
  int part_ld;
};

// ---- the epilogue -------------------------------------------------------------------------------

template <int ACT>
__device__ __forceinline__ float act(float z) {
  if constexpr (ACT == FCV_LM_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
  if constexpr (ACT == FCV_LM_ACT_SILU) return silu(z);
  if constexpr (ACT == FCV_LM_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  if constexpr (ACT == FCV_LM_ACT_GELU_TANH) return gelu_tanh(z);
  return z;
}

// f(integral_constant) of the call's activation: one branch around a whole epilogue.
template <class F>
__device__ __forceinline__ void with_act(int kind, const F& f) {
  switch (kind) {
    case FCV_LM_ACT_RELU: return f(std::integral_constant<int, FCV_LM_ACT_RELU>{});
    case FCV_LM_ACT_SILU: return f(std::integral_constant<int, FCV_LM_ACT_SILU>{});
    case FCV_LM_ACT_GELU: return f(std::integral_constant<int, FCV_LM_ACT_GELU>{});
    case FCV_LM_ACT_GELU_TANH: return f(std::integral_constant<int, FCV_LM_ACT_GELU_TANH>{});
    default: return f(std::integral_constant<int, FCV_LM_ACT_NONE>{});
  }
}

template <int ACT>
__device__ __forceinline__ f32x4 act4(f32x4 z) {
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = act<ACT>(z[e]);
  return z;
}
__device__ __forceinline__ f32x4 act4(f32x4 z, int kind) {
  with_act(kind, [&](auto k) { z = act4<decltype(k)::value>(z); });
  return z;
}

template <class E>
__device__ __forceinline__ float element(const void* p, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : E::to_f32(static_cast<const short*>(p)[i]);
}

// Four elements from any element's boundary: the same instruction as an aligned access.
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef s16x4 s16x4_any __attribute__((aligned(2)));

template <class E>
__device__ __forceinline__ f32x4 load4(const void* p, bool f32, int64_t i) {
  if (f32) return *reinterpret_cast<const f32x4_any*>(static_cast<const float*>(p) + i);
  const s16x4 b = *reinterpret_cast<const s16x4_any*>(static_cast<const short*>(p) + i);
  return f32x4{E::to_f32(b[0]), E::to_f32(b[1]), E::to_f32(b[2]), E::to_f32(b[3])};
}

template <class E>
__device__ __forceinline__ void store4(void* p, bool f32, int64_t i, const f32x4& v) {
  if (f32)
    *reinterpret_cast<f32x4_any*>(static_cast<float*>(p) + i) = v;
  else
    *reinterpret_cast<s16x4_any*>(static_cast<short*>(p) + i) =
        s16x4{E::from_f32(v[0]), E::from_f32(v[1]), E::from_f32(v[2]), E::from_f32(v[3])};
}

// Column n of row m from its sum.
template <class E>
__device__ __forceinline__ void finish1(const FcvLmLinear& p, int m, int n, float z) {
  if (p.bias) z += element<E>(p.bias, p.bias_dtype == FCV_LM_F32, n);
  with_act(p.activation, [&](auto k) { z = act<decltype(k)::value>(z); });
  if (p.residual) z += element<E>(p.residual, p.residual_dtype == FCV_LM_F32, (int64_t)m * p.ldr + n);
  const int64_t at = (int64_t)m * p.ldy + n;
  if (p.y_dtype == FCV_LM_F32)
    static_cast<float*>(p.y)[at] = z;
  else
    static_cast<short*>(p.y)[at] = E::from_f32(z);
}

// Four columns n .. n + 3 of row m from their sums: at once, or those below N one at a time.  What is not
// there is not added where an access is off its boundary (`vec` false), so that a sum of -0 stays one as in
// finish1.
template <class E>
__device__ __forceinline__ void finish4(const FcvLmLinear& p, bool vec, int m, int n, f32x4 v,
                                        const f32x4& bias, const f32x4& residual) {
  if (n + 3 < p.n) {
    if (vec || p.bias) v += bias;
    v = act4(v, p.activation);
    if (vec || p.residual) v += residual;
    store4<E>(p.y, p.y_dtype == FCV_LM_F32, (int64_t)m * p.ldy + n, v);
    return;
  }
  const int count = p.n - n;
#pragma unroll 1
  for (int e = 0; e < count; ++e) {
    finish1<E>(p, m, n + e, v[0]);
    v = f32x4{v[1], v[2], v[3], 0.0f};
  }
}

template <class E>
__device__ __forceinline__ f32x4 bias4(const FcvLmLinear& p, bool whole, int n) {
  return whole && p.bias ? load4<E>(p.bias, p.bias_dtype == FCV_LM_F32, n) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

template <class E>
__device__ __forceinline__ f32x4 residual4(const FcvLmLinear& p, bool whole, int m, int n) {
  return whole && p.residual ? load4<E>(p.residual, p.residual_dtype == FCV_LM_F32, (int64_t)m * p.ldr + n)
                    : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// ---- rows from any element's boundary -------------------------------------------------------------

// 8 elements from any element's boundary (the same load instruction as an aligned one).
__device__ __forceinline__ s16x8 load8_any(const short* p) {
  typedef s16x8 any __attribute__((aligned(2)));
  return *reinterpret_cast<const any*>(p);
}

// Elements k .. k + 7 of a row of `len`, zeros past its end.
__device__ __forceinline__ s16x8 row_chunk(const short* row, int k, int len) {
  if (k + 8 <= len) return load8_any(row + k);
  s16x8 v = {};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < len) v[e] = row[k + e];
  return v;
}

// ---- tiles --------------------------------------------------------------------------------------

constexpr int kXcds = 8;
constexpr int kSlice = 64;  // K is split over workgroups in slices of 64
__device__ __attribute__((aligned(16))) uint32_t zeros16[4];  // what a copy past K reads

// WM x WN waves of (BM / WM) x (BN / WN) outputs each; a ring of STAGES slices.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int BK_ = 64>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, BK = BK_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int kChunks = BK / 8, kCopyRows = 64 / kChunks;  // 16-byte chunks of a row; rows of a copy
  static constexpr int kXCopies = BM / kCopyRows / kWaves, kWCopies = BN / kCopyRows / kWaves;
  static constexpr int kCopies = kXCopies + kWCopies;
  static constexpr int kStage = (BM + BN) * BK;  // elements
  static constexpr int kLds = STAGES * kStage * 2;
  static constexpr int kGroupM = 1024 / BM > 0 ? 1024 / BM : 1;
  static constexpr int kPerCu = 160 * 1024 / kLds;
  // waves a SIMD that the registers have to leave room for
  static constexpr int kWavesPerSimd = kPerCu * kWaves >= 8 ? 2 : 1;
  // small tiles: a whole slice's fragments are read at once, under the products of the slice before
  static constexpr bool kWhole = TM * TN == 1;
  static_assert(BM % (kCopyRows * kWaves) == 0 && BN % (kCopyRows * kWaves) == 0, "copy split");
  static_assert((STAGES - 2) * kCopies < 64, "copies in flight");
};

// LDS position of 16-byte chunk c of row r: 16 rows read at one chunk index touch all banks.
template <int BK>
__device__ __forceinline__ int swz(int r, int c) {
  return BK == 128 ? c ^ (r & 15) : BK == 64 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3);
}

template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int L, int A>
__device__ __forceinline__ void wait_ahead(int ahead) {
  if constexpr (A > 0) {
    if (ahead >= A) {
      wait_copies<A * L>();
      return;
    }
    wait_ahead<L, A - 1>(ahead);
  } else {
    wait_copies<0>();
  }
}

// The epilogue of a tile kernel whose waves have TM x TN blocks of 32 x 32 outputs each in `acc`: waves at
// (wm0, wn0) of the tile at row m0 and column n0, `smem` the workgroup's LDS (its kLds bytes are free).
template <class E, class C, int kLds>
__device__ __forceinline__ void store_tile(const Args& a, const f32x16 (&acc)[C::TM][C::TN], short* smem,
                                           int split, int n0, int wn0, int wm0, int m0) {
  constexpr int TM = C::TM, TN = C::TN;
  const FcvLmLinear& p = a.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 31, fh = lane >> 5;
  // The accumulators go through LDS 32 rows at a time, so that a store covers whole runs of a row.
  constexpr int kCols = TN * 32, kPitch = kCols + 4, kLanes = kCols / 4;
  constexpr int kPassRows = 64 / kLanes, kPasses = 32 / kPassRows;
  static_assert(C::kWaves * 32 * kPitch * 4 <= kLds, "epilogue staging");
  __syncthreads();
  float* stg = reinterpret_cast<float*>(smem) + wave * 32 * kPitch;
  const int rr = lane / kLanes, rc = (lane % kLanes) * 4;
  const int col = n0 + wn0 + rc;
  auto park = [&](int i) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(stg + fr * kPitch + j * 32 + g * 8 + fh * 4) =
            f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
    wave_fence();
  };
  const float* mine = stg + rr * kPitch + rc;  // the lane's columns of the block's row rr
  if (a.splits > 1) {
    // part_ld is n, up to a multiple of 4
    float* part = a.part + (int64_t)split * p.m * a.part_ld + col;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      park(i);
#pragma unroll
      for (int q = 0; q < kPasses; ++q) {
        const int row = m0 + wm0 + i * 32 + rr + q * kPassRows;
        if (row < p.m && col < p.n)
          *reinterpret_cast<f32x4*>(part + (int64_t)row * a.part_ld) =
              *reinterpret_cast<const f32x4*>(mine + q * kPassRows * kPitch);
      }
      wave_fence();
    }
    return;
  }
  // where N ends inside a lane's four columns, the one to three below it have a pass of their own
  const bool whole = col + 3 < p.n;
  const int left = p.n - n0 - wn0, edge = left > 0 && left < kCols ? left & 3 : 0;
  with_act(p.activation, [&](auto kind) {
    const f32x4 bias = bias4<E>(p, whole, col);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row0 = m0 + wm0 + i * 32 + rr;
      f32x4 r[kPasses];
      // a block's residuals are asked for together, before its stores
#pragma unroll
      for (int q = 0; q < kPasses; ++q)
        r[q] = residual4<E>(p, whole, min(row0 + q * kPassRows, p.m - 1), col);
      park(i);
      f32x4 v[kPasses];
#pragma unroll
      for (int q = 0; q < kPasses; ++q)
        v[q] = *reinterpret_cast<const f32x4*>(mine + q * kPassRows * kPitch);
      if (edge) {
        const int row = m0 + wm0 + i * 32 + fr;
        for (int e = fh; e < edge && row < p.m; e += 2) {
          const int at = left - edge + e, n = n0 + wn0 + at;
          const float b = p.bias ? element<E>(p.bias, p.bias_dtype == FCV_LM_F32, n) : 0.0f;
          const float z = act<decltype(kind)::value>(stg[fr * kPitch + at] + b) +
                          (p.residual ? element<E>(p.residual, p.residual_dtype == FCV_LM_F32,
                                                   (int64_t)row * p.ldr + n)
                                      : 0.0f);
          if (p.y_dtype == FCV_LM_F32)
            static_cast<float*>(p.y)[(int64_t)row * p.ldy + n] = z;
          else
            static_cast<short*>(p.y)[(int64_t)row * p.ldy + n] = E::from_f32(z);
        }
      }
      wave_fence();
#pragma unroll
      for (int q = 0; q < kPasses; ++q) {
        const f32x4 z = act4<decltype(kind)::value>(v[q] + bias) + r[q];
        const int row = row0 + q * kPassRows;
        if (row < p.m && whole) store4<E>(p.y, p.y_dtype == FCV_LM_F32, (int64_t)row * p.ldy + col, z);
      }
    }
  });
}

// Sums of the ranges in their order, then the epilogue; a thread has four columns of a row.
template <class E>
__global__ __launch_bounds__(256) void linear_join_kernel(const Args a) {
  const FcvLmLinear& p = a.p;
  const int quads = a.part_ld / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)p.m * quads) return;
  const int row = (int)(i / quads), col = (int)(i % quads) * 4;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  const float* part = a.part + (int64_t)row * a.part_ld + col;
  const int64_t range = (int64_t)p.m * a.part_ld;
  for (int s0 = 0; s0 < a.splits; s0 += 4) {  // four asked for at once
    f32x4 u[4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
      u[s] = s0 + s < a.splits ? *reinterpret_cast<const f32x4*>(part + (s0 + s) * range)
                               : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; ++s) v += u[s];
  }
  const bool whole = col + 3 < p.n;
  finish4<E>(p, a.vec, row, col, v, bias4<E>(p, whole, col), residual4<E>(p, whole, row, col));
}

inline int element_size(int dtype) { return dtype == FCV_LM_F32 ? 4 : 2; }

}  // namespace
}  // namespace lm
}  // namespace fcv
