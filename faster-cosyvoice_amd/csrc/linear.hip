// y = act(x W^T + bias) + residual on the matrix cores, for any row count, width and stride.
//
// x and W are read as they lie (K contiguous in both).  W is the A operand and x the B operand, so that a
// lane's accumulator holds four consecutive columns of one row of y per register group; sums are fp32, the
// epilogue is fp32, and y is rounded once.
//
// Three kernels (plan_of chooses by an estimate):
//   linear_tile_kernel  tiles of y from operand slices that are copied straight into LDS (a ring of two to
//                       four slices of 64 of K), K cut over several workgroups where the tiles are few;
//   linear_few_kernel   up to 16 rows, W read once into registers;
//   linear_any_kernel   more rows off 16-byte boundaries, or K no multiple of 8: through registers.
//
// Bound and rate: large products by the matrix pipes, 8192 x 4096 x 8192 bf16 with bias and SiLU 446 to 490
// us (1.1 to 1.2 PFLOP/s; 61 to 66 % of the cycles at the clock the card holds under it, and the same within
// 10 % with three to five slices of 32, with the copies asked for at once, and with four waves of 128 x 128);
// 9184 x 1024 x 2048 with tanh-GELU 60 us, half of it rounds that are not full and stores that all CUs send at
// once (gemm.hip's 128 x 128 form takes 52 us for that one; of the shapes here 192 x 256 is the fastest, 128 x
// 128 takes 70).  Small products by the latency of the few slices that one workgroup a CU has in flight, and
// 32 rows are copied as 64: 32 x 4096 x 4096 12 us.
#include <algorithm>
#include <type_traits>

#include "lm.hpp"

namespace fcv {
namespace lm {
namespace {

struct Args {
  FcvLmLinear p;
  bool vec;                 // four columns of y, the residual and the bias are one aligned access
  int splits, slices;       // ranges of K, and the 64-wide slices of one
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

template <class E>
__device__ __forceinline__ f32x4 load4(const void* p, bool f32, int64_t i) {
  if (f32) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  const s16x4 b = *reinterpret_cast<const s16x4*>(static_cast<const short*>(p) + i);
  return f32x4{E::to_f32(b[0]), E::to_f32(b[1]), E::to_f32(b[2]), E::to_f32(b[3])};
}

template <class E>
__device__ __forceinline__ void store4(void* p, bool f32, int64_t i, const f32x4& v) {
  if (f32)
    *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
  else
    *reinterpret_cast<s16x4*>(static_cast<short*>(p) + i) =
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

// Four columns n .. n + 3 of row m from their sums: those below N one at a time, or all of them
// where they are one aligned access (`vec`).
template <class E>
__device__ __forceinline__ void finish4(const FcvLmLinear& p, bool vec, int m, int n, f32x4 v,
                                        const f32x4& bias, const f32x4& residual) {
  if (vec) {
    v = act4(v + bias, p.activation) + residual;
    store4<E>(p.y, p.y_dtype == FCV_LM_F32, (int64_t)m * p.ldy + n, v);
    return;
  }
  const int count = min(4, p.n - n);
#pragma unroll 1
  for (int e = 0; e < count; ++e) {
    finish1<E>(p, m, n + e, v[0]);
    v = f32x4{v[1], v[2], v[3], 0.0f};
  }
}

template <class E>
__device__ __forceinline__ f32x4 bias4(const FcvLmLinear& p, bool vec, int n) {
  return vec && p.bias ? load4<E>(p.bias, p.bias_dtype == FCV_LM_F32, n) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

template <class E>
__device__ __forceinline__ f32x4 residual4(const FcvLmLinear& p, bool vec, int m, int n) {
  return vec && p.residual ? load4<E>(p.residual, p.residual_dtype == FCV_LM_F32, (int64_t)m * p.ldr + n)
                    : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// ---- any alignment: operands through registers --------------------------------------------------

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

constexpr int kTile = 64, kDepth = 64, kPitch = kDepth + 8;

// Tiles of 64 x 64, the next slice's elements in registers while this one's products run.  Bound by the
// loads, whose chunks cross lines, and by the one step of lookahead: 4000 x 3001 x 4000 336 us (0.29
// PFLOP/s), 1 x 1001 x 2000 (linear_few_kernel) 6 us.
template <class E>
__global__ __launch_bounds__(256) void linear_any_kernel(const Args a) {
  __shared__ __attribute__((aligned(16))) short sx[kTile][kPitch];
  __shared__ __attribute__((aligned(16))) short sw[kTile][kPitch];
  const FcvLmLinear& p = a.p;
  const int tiles_n = (p.n + kTile - 1) / kTile;
  const int m0 = blockIdx.x / tiles_n * kTile, n0 = blockIdx.x % tiles_n * kTile;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 31, fh = lane >> 5;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  const int lr = threadIdx.x >> 3, lc = (threadIdx.x & 7) * 8;
  const int first = blockIdx.y * a.slices * kDepth, end = min(first + a.slices * kDepth, p.k);
  const short *x[2], *w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[i] = static_cast<const short*>(p.x) + (int64_t)min(m0 + lr + 32 * i, p.m - 1) * p.ldx;
    w[i] = static_cast<const short*>(p.w) + (int64_t)min(n0 + lr + 32 * i, p.n - 1) * p.ldw;
  }
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
  s16x8 rx[2], rw[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    rx[i] = row_chunk(x[i], first + lc, end);
    rw[i] = row_chunk(w[i], first + lc, end);
  }
  for (int k0 = first; k0 < end; k0 += kDepth) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<s16x8*>(&sx[lr + 32 * i][lc]) = rx[i];
      *reinterpret_cast<s16x8*>(&sw[lr + 32 * i][lc]) = rw[i];
    }
    __syncthreads();
    if (k0 + kDepth < end) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        rx[i] = row_chunk(x[i], k0 + kDepth + lc, end);
        rw[i] = row_chunk(w[i], k0 + kDepth + lc, end);
      }
    }
#pragma unroll
    for (int ks = 0; ks < kDepth / 16; ++ks) {
      const s16x8 fx = *reinterpret_cast<const s16x8*>(&sx[wm + fr][ks * 16 + fh * 8]);
      const s16x8 fw = *reinterpret_cast<const s16x8*>(&sw[wn + fr][ks * 16 + fh * 8]);
      acc = E::mfma32(fw, fx, acc);
    }
  }
  const int m = m0 + wm + fr;
  if (m >= p.m) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int n = n0 + wn + g * 8 + fh * 4;
    if (n >= p.n) break;
    const f32x4 v = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    if (a.splits > 1) {
      *reinterpret_cast<f32x4*>(a.part + ((int64_t)blockIdx.y * p.m + m) * a.part_ld + n) = v;
      continue;
    }
    const bool vec = a.vec && n + 3 < p.n;
    finish4<E>(p, vec, m, n, v, bias4<E>(p, vec, n), residual4<E>(p, vec, m, n));
  }
}

// ---- tiles: operands by copies into LDS ----------------------------------------------------------

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
  return BK == 64 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3);
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

// LDS written by a wave is read by the same wave: in order, once the compiler keeps it so.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <class E, class C>
__global__ __launch_bounds__(C::kThreads, C::kWavesPerSimd) void linear_tile_kernel(const Args a) {
  constexpr int BM = C::BM, BN = C::BN, TM = C::TM, TN = C::TN, S = C::STAGES, BK = C::BK;
  __shared__ __attribute__((aligned(1024))) short smem[S * C::kStage];
  const FcvLmLinear& p = a.p;
  const int tiles_m = (p.m + BM - 1) / BM, tiles_n = (p.n + BN - 1) / BN;
  // blocks are dealt round-robin over the XCDs: each takes a contiguous range of the tiles, visited
  // in groups of kGroupM row tiles x all column tiles
  int split, n0, m0;
  {
    const int total = tiles_m * tiles_n * a.splits;
    const int xcd = blockIdx.x % kXcds, idx = blockIdx.x / kXcds;
    const int base = total / kXcds, extra = total % kXcds;
    int t = xcd * base + min(xcd, extra) + idx;
    split = t / (tiles_m * tiles_n);
    t -= split * tiles_m * tiles_n;
    const int g = t / (C::kGroupM * tiles_n), first = g * C::kGroupM;
    const int gm = min(C::kGroupM, tiles_m - first), r = t - g * C::kGroupM * tiles_n;
    m0 = (first + r % gm) * BM;
    n0 = r / gm * BN;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm0 = wave / C::WN * (BM / C::WM), wn0 = wave % C::WN * (BN / C::WN);

  const int slice0 = split * a.slices * (kSlice / BK);  // in units of BK
  const int all = (p.k + BK - 1) / BK;
  const int KT = min(a.slices * (kSlice / BK), all - slice0);
  const bool ragged = p.k % BK != 0 && slice0 + KT == all;  // the last slice passes K

  // byte offset of each copy's source from the tile's first row; rows past the matrix read its last
  const char* xb = reinterpret_cast<const char*>(static_cast<const short*>(p.x) + (int64_t)m0 * p.ldx +
                                                 (int64_t)slice0 * BK);
  const char* wb = reinterpret_cast<const char*>(static_cast<const short*>(p.w) + (int64_t)n0 * p.ldw +
                                                 (int64_t)slice0 * BK);
  const int crow = lane / C::kChunks, cpos = lane % C::kChunks;
  uint32_t x_off[C::kXCopies], w_off[C::kWCopies];
#pragma unroll
  for (int i = 0; i < C::kXCopies; ++i) {
    const int row = (wave * C::kXCopies + i) * C::kCopyRows + crow;
    x_off[i] = (uint32_t)min(row, p.m - 1 - m0) * (uint32_t)(p.ldx * 2) + swz<BK>(row, cpos) * 16;
  }
#pragma unroll
  for (int i = 0; i < C::kWCopies; ++i) {
    const int row = (wave * C::kWCopies + i) * C::kCopyRows + crow;
    w_off[i] = (uint32_t)min(row, p.n - 1 - n0) * (uint32_t)(p.ldw * 2) + swz<BK>(row, cpos) * 16;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
  const uint32_t lds_x = lds0 + wave * C::kXCopies * 1024;
  const uint32_t lds_w = lds0 + BM * BK * 2 + wave * C::kWCopies * 1024;
  // copies [c0, c1) of slice kt (x's first, then W's) into a stage
  auto issue = [&](int kt, int stage, int c0, int c1) {
    const char* xk = xb + kt * (BK * 2);
    const char* wk = wb + kt * (BK * 2);
    const uint32_t at = stage * (C::kStage * 2);
    if (ragged && kt == KT - 1) {
      const int left = p.k - (slice0 + kt) * BK;  // columns of the slice below K, a multiple of 8
#pragma unroll
      for (int c = 0; c < C::kCopies; ++c) {
        if (c < c0 || c >= c1) continue;
        const bool is_x = c < C::kXCopies;
        const int i = is_x ? c : c - C::kXCopies;
        const int row = (wave * (is_x ? C::kXCopies : C::kWCopies) + i) * C::kCopyRows + crow;
        const void* src = is_x ? xk + x_off[is_x ? i : 0] : wk + w_off[is_x ? 0 : i];
        lds_dma16_at(swz<BK>(row, cpos) * 8 < left ? src : zeros16,
                     (is_x ? lds_x : lds_w) + at + i * 1024);
      }
      return;
    }
#pragma unroll
    for (int c = 0; c < C::kCopies; ++c) {
      if (c < c0 || c >= c1) continue;
      if (c < C::kXCopies)
        lds_dma16(xk, x_off[c], lds_x + at + c * 1024);
      else
        lds_dma16(wk, w_off[c - C::kXCopies], lds_w + at + (c - C::kXCopies) * 1024);
    }
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  const int fr = lane & 31, fh = lane >> 5;
  constexpr int KS = BK / 16, kSets = C::kWhole ? 2 * KS : 2;
  s16x8 fx[kSets][TM], fw[kSets][TN];
  auto load = [&](int buf, int ks, int st) {
    const short* sx = smem + st * C::kStage;
    const short* sw = sx + BM * BK;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = wm0 + i * 32 + fr;
      fx[buf][i] = *reinterpret_cast<const s16x8*>(sx + row * BK + swz<BK>(row, ks * 2 + fh) * 8);
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int row = wn0 + j * 32 + fr;
      fw[buf][j] = *reinterpret_cast<const s16x8*>(sw + row * BK + swz<BK>(row, ks * 2 + fh) * 8);
    }
  };
  auto mma = [&](int buf) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = E::mfma32(fw[buf][j], fx[buf][i], acc[i][j]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int st = 0; st < S - 1; ++st)
    if (st < KT) issue(st, st, 0, C::kCopies);
  wait_ahead<C::kCopies, S - 2>(KT - 1);
  __syncthreads();
  int kt = 0, stage = 0;
  if constexpr (C::kWhole) {
    // The fragments of slice kt are asked for after the barrier that publishes it and used after the
    // next one, so that an LDS read's latency passes once a slice and under products.  The barrier
    // also frees the stage before, which the copies of slice kt + S - 1 fill.
    auto load_all = [&](auto set) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) load(decltype(set)::value * KS + ks, ks, stage);
    };
    auto mma_all = [&](auto set) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = E::mfma32(fw[decltype(set)::value * KS + ks][j],
                                  fx[decltype(set)::value * KS + ks][i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    auto step = [&](auto set, auto before) {
      wait_ahead<C::kCopies, S - 2>(KT - 1 - kt);
      __syncthreads();
      const int freed = stage;
      stage = stage == S - 1 ? 0 : stage + 1;
      load_all(set);
      if (kt + S - 1 < KT) issue(kt + S - 1, freed, 0, C::kCopies);
      mma_all(before);
    };
    if (S - 1 < KT) issue(S - 1, S - 1, 0, C::kCopies);
    load_all(even);
    for (kt = 1; kt < KT;) {
      step(odd, even);
      if (++kt == KT) break;
      step(even, odd);
      ++kt;
    }
    if (KT & 1)
      mma_all(even);
    else
      mma_all(odd);
  } else {
    // The loop is rotated by one step of 16: a slice's last step runs from registers after the barrier
    // that publishes the next slice, while that slice's first fragments are read.  The barrier also
    // frees the stage before it (every wave holds the last fragments of that slice), which the copies
    // of slice kt + S - 1 then fill, a few of them before each step's products: asked for all at once
    // they would hold every wave at the copies' address unit (16 cycles each) while the matrix pipes idle.
    constexpr int kPhases = S == 2 ? KS - 1 : KS;  // two stages: the copies need the last step's time to land
    constexpr int kPer = (C::kCopies + kPhases - 1) / kPhases;
    auto copies = [&](int phase) {
      if (kt + S - 1 < KT)
        issue(kt + S - 1, stage == 0 ? S - 1 : stage - 1, phase * kPer, phase * kPer + kPer);
    };
    auto head = [&](int st) {
#pragma unroll
      for (int ks = 0; ks + 1 < KS; ++ks) {
        load((ks + 1) & 1, ks + 1, st);
        copies(ks + 1);
        mma(ks & 1);
      }
    };
    copies(0);
    load(0, 0, 0);
    head(0);
    for (kt = 1; kt < KT; ++kt) {
      const int next = stage == S - 1 ? 0 : stage + 1;
      wait_ahead<C::kCopies, S - 2>(KT - 1 - kt);
      __syncthreads();
      stage = next;
      load(0, 0, stage);
      copies(0);
      mma(1);
      head(stage);
    }
    mma(1);
  }

  // The accumulators go through LDS 32 rows at a time, so that a store covers whole runs of a row.
  constexpr int kCols = TN * 32, kPitch = kCols + 4, kLanes = kCols / 4;
  constexpr int kPassRows = 64 / kLanes, kPasses = 32 / kPassRows;
  static_assert(C::kWaves * 32 * kPitch * 4 <= (int)sizeof(smem), "epilogue staging");
  __syncthreads();
  float* stg = reinterpret_cast<float*>(smem) + wave * 32 * kPitch;
  const int rr = lane / kLanes, rc = (lane % kLanes) * 4;
  const int col = n0 + wn0 + rc;
  const bool inside = col < p.n;
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
  if (__all(a.vec && (!inside || col + 3 < p.n))) {
    with_act(p.activation, [&](auto kind) {
      const f32x4 bias = bias4<E>(p, inside, col);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row0 = m0 + wm0 + i * 32 + rr;
        f32x4 r[kPasses];
        // a block's residuals are asked for together, before its stores
#pragma unroll
        for (int q = 0; q < kPasses; ++q)
          r[q] = residual4<E>(p, inside, min(row0 + q * kPassRows, p.m - 1), col);
        park(i);
        f32x4 v[kPasses];
#pragma unroll
        for (int q = 0; q < kPasses; ++q)
          v[q] = *reinterpret_cast<const f32x4*>(mine + q * kPassRows * kPitch);
        wave_fence();
#pragma unroll
        for (int q = 0; q < kPasses; ++q) {
          const f32x4 z = act4<decltype(kind)::value>(v[q] + bias) + r[q];
          const int row = row0 + q * kPassRows;
          if (row < p.m && inside) store4<E>(p.y, p.y_dtype == FCV_LM_F32, (int64_t)row * p.ldy + col, z);
        }
      }
    });
    return;
  }
  // rows off their boundaries, or N no multiple of four: a column a lane, neighbouring lanes along a row
  static_assert(64 % kCols == 0, "a lane keeps its column");
  const int n = n0 + wn0 + lane % kCols;
  const float bias1 = p.bias && n < p.n ? element<E>(p.bias, p.bias_dtype == FCV_LM_F32, n) : 0.0f;
  with_act(p.activation, [&](auto kind) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      park(i);
      const int row0 = m0 + wm0 + i * 32 + lane / kCols;
#pragma unroll 1
      for (int q0 = 0; q0 < kCols / 2; q0 += 8) {  // 8 of the block's passes of 64 / kCols rows
        float r[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int row = row0 + (q0 + q) * (64 / kCols);
          r[q] = p.residual && row < p.m && n < p.n
                     ? element<E>(p.residual, p.residual_dtype == FCV_LM_F32, (int64_t)row * p.ldr + n)
                     : 0.0f;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int row = row0 + (q0 + q) * (64 / kCols);
          const float v = stg[(row - m0 - wm0 - i * 32) * kPitch + lane % kCols];
          const float z = act<decltype(kind)::value>(v + bias1) + r[q];
          if (row >= p.m || n >= p.n) continue;
          const int64_t at = (int64_t)row * p.ldy + n;
          if (p.y_dtype == FCV_LM_F32)
            static_cast<float*>(p.y)[at] = z;
          else
            static_cast<short*>(p.y)[at] = E::from_f32(z);
        }
      }
      wave_fence();
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
  const bool vec = a.vec && col + 3 < p.n;
  finish4<E>(p, vec, row, col, v, bias4<E>(p, vec, col), residual4<E>(p, vec, row, col));
}

// ---- up to 16 rows: the weights straight into registers -------------------------------------------
//
// v_mfma_f32_16x16x32 with 16 rows of W and the rows of x (lane l holds row l % 16, elements
// 8 (l / 16) .. + 7 of 32 of either).  One workgroup has 16 rows of W; its waves take turns in K, four
// steps of 32 at a time, and are summed through LDS.
//
// Bound: one CU takes in about 40 B/ns, so the weights are spread over as many workgroups as there are,
// and K over several (blockIdx.y, joined by linear_join_kernel) where W has few rows.  Measured, weights
// from HBM: 1 x 4096 x 4096 8.2 us (4.1 TB/s), 16 x 4096 x 4096 10.5 us, 1 x 1024 x 2048 3.8 us.  Eight
// or sixteen steps at a time, 16 waves, and 32 rows of W a workgroup were no faster.
constexpr int kFewRows = 16, kFewWaves = 8, kFewSteps = 4;

template <class E>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_kernel(const Args a) {
  __shared__ __attribute__((aligned(16))) f32x4 sums[kFewWaves][64];
  const FcvLmLinear& p = a.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fk = (lane >> 4) * 8;
  const int n0 = blockIdx.x * kFewRows;
  const int k0 = blockIdx.y * a.slices * kSlice, k1 = min(k0 + a.slices * kSlice, p.k);
  const short* w = static_cast<const short*>(p.w) + (int64_t)min(n0 + fr, p.n - 1) * p.ldw + fk;
  const short* x = static_cast<const short*>(p.x) + (int64_t)min(fr, p.m - 1) * p.ldx + fk;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = k0 + wave * kFewSteps * 32; k < k1; k += kFewWaves * kFewSteps * 32) {
    s16x8 fw[kFewSteps], fx[kFewSteps];
    if (k + kFewSteps * 32 <= k1) {
#pragma unroll
      for (int u = 0; u < kFewSteps; ++u) {
        fw[u] = load8_any(w + k + u * 32);
        fx[u] = load8_any(x + k + u * 32);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kFewSteps; ++u) {
        fw[u] = row_chunk(w, k + u * 32, k1 - fk);  // w and x begin at the lane's element fk
        fx[u] = row_chunk(x, k + u * 32, k1 - fk);
      }
    }
#pragma unroll
    for (int u = 0; u < kFewSteps; ++u) acc = E::mfma16(fw[u], fx[u], acc);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
  f32x4 v = sums[0][lane];
#pragma unroll
  for (int s = 1; s < kFewWaves; ++s) v += sums[s][lane];
  const int m = fr, n = n0 + (lane >> 4) * 4;
  if (m >= p.m || n >= p.n) return;
  if (a.splits > 1) {
    *reinterpret_cast<f32x4*>(a.part + ((int64_t)blockIdx.y * p.m + m) * a.part_ld + n) = v;
    return;
  }
  const bool vec = a.vec && n + 3 < p.n;
  finish4<E>(p, vec, m, n, v, bias4<E>(p, vec, n), residual4<E>(p, vec, m, n));
}

// ---- host ---------------------------------------------------------------------------------------

int element_size(int dtype) { return dtype == FCV_LM_F32 ? 4 : 2; }

int check(const FcvLmLinear* p) {
  FCV_CHECK(p, FCV_ERR_INVALID, "null arguments");
  FCV_CHECK(p->dtype == FCV_LM_F16 || p->dtype == FCV_LM_BF16, FCV_ERR_INVALID,
            "dtype must be FCV_LM_F16 or FCV_LM_BF16");
  FCV_CHECK((p->bias_dtype == p->dtype || p->bias_dtype == FCV_LM_F32) &&
                (p->residual_dtype == p->dtype || p->residual_dtype == FCV_LM_F32) &&
                (p->y_dtype == p->dtype || p->y_dtype == FCV_LM_F32),
            FCV_ERR_INVALID, "bias, residual and y must be of dtype or FCV_LM_F32");
  FCV_CHECK(p->activation >= FCV_LM_ACT_NONE && p->activation <= FCV_LM_ACT_GELU_TANH,
            FCV_ERR_INVALID, "unknown activation");
  FCV_CHECK(p->m >= 0 && p->n >= 1 && p->k >= 1, FCV_ERR_INVALID, "need m >= 0, n >= 1 and k >= 1");
  FCV_CHECK(p->k <= (1 << 28), FCV_ERR_INVALID, "k is limited to 2^28");
  FCV_CHECK(p->m <= (1 << 22) && p->n <= (1 << 22) && (int64_t)p->m * p->n <= (1LL << 34),
            FCV_ERR_INVALID, "m and n are limited to 2^22 each and their product to 2^34");
  FCV_CHECK(p->ldx >= 0 && p->ldw >= 0 && p->ldr >= 0, FCV_ERR_INVALID, "negative row stride");
  FCV_CHECK(p->ldy >= p->n || p->m <= 1, FCV_ERR_INVALID, "y's row stride is shorter than its row");
  if (p->m == 0) return FCV_OK;
  FCV_CHECK(p->x && p->w && p->y, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(aligned(p->x, 2) && aligned(p->w, 2) && aligned(p->y, element_size(p->y_dtype)) &&
                aligned(p->bias, element_size(p->bias_dtype)) &&
                aligned(p->residual, element_size(p->residual_dtype)),
            FCV_ERR_INVALID, "a tensor does not start on an element's boundary");
  return FCV_OK;
}

// Which kernel, and into how many ranges K is cut: the least of the estimates
//   rounds (slices slice_us + tile_us) + 3 us,   rounds = blocks over the CUs, `per_cu` each, rounded up,
// and for a cut K a second launch that reads the ranges' sums.  slice_us and tile_us are fits to full
// rounds of each shape at K 512, 2048 and 8192 (alone: one block a CU of those that share one).
// 128x128 tiles have three stages (kTile128Deep) while one a CU holds them all (88 against 115 us at 2048 x
// 8192 x 2048) and two, two a CU, above (146 us for 4096 x 8192 x 2048).
enum Form {
  kAny, kFew, kTile64, kTile64x128, kTile128, kTile128x256, kTile192x256, kTile256, kTile128Deep
};

struct Shape {
  Form form;
  int bm, bn, per_cu;
  float alone_us, slice_us, tile_us;
};
constexpr Shape kShapes[] = {
    {kAny, 64, 64, 4, 0.85f, 1.75f, 2.0f},
    {kTile64, 64, 64, 2, 0.29f, 0.45f, 1.3f},       {kTile64x128, 64, 128, 2, 0.44f, 0.67f, 2.5f},
    {kTile128, 128, 128, 2, 0.62f, 1.10f, 5.0f},    {kTile128x256, 128, 256, 1, 0.96f, 0.96f, 5.6f},
    {kTile192x256, 192, 256, 1, 1.40f, 1.40f, 7.5f}, {kTile256, 256, 256, 1, 1.65f, 1.65f, 9.4f}};
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr int kMinSlices = 4;  // of a range

struct Plan {
  Form form;
  int splits, slices;
};

int64_t tiles_of(const FcvLmLinear& p, int bm, int bn) {
  return (int64_t)((p.m + bm - 1) / bm) * ((p.n + bn - 1) / bn);
}

float join_us(const FcvLmLinear& p, int splits) {
  return splits > 1 ? 3.0f + (float)p.m * (float)p.n * 8.0f * splits / 4.0e6f : 0.0f;
}

Plan plan_of(const FcvLmLinear& p) {
  const bool chunks = aligned(p.x, 16) && aligned(p.w, 16) && (p.ldx % 8 == 0 || p.m == 1) &&
                      (p.ldw % 8 == 0 || p.n == 1) && p.k % 8 == 0 && p.ldx < (1 << 22) &&
                      p.ldw < (1 << 22);  // a tile's rows lie within 32-bit byte offsets
  const int slices = (p.k + kSlice - 1) / kSlice;
  Plan best{kAny, 1, slices};
  float best_us = 3.0e38f;
  auto consider = [&](Form form, int splits, float us) {
    us += join_us(p, splits);
    if (us >= best_us) return;
    best_us = us;
    const int per = (slices + splits - 1) / splits;
    best = Plan{form, (slices + per - 1) / per, per};
  };
  for (int splits : kSplits) {
    if (splits > 1 && slices < splits * kMinSlices) break;
    const float per = (float)((slices + splits - 1) / splits);
    if (p.m <= kFewRows) {
      const int64_t blocks = (int64_t)((p.n + kFewRows - 1) / kFewRows) * splits;
      const float bytes = per * kSlice * 2.0f * (float)(kFewRows + p.m);
      consider(kFew, splits, 3.4f + (float)((blocks + kCus - 1) / kCus) * bytes / 40.0e3f);
    }
    for (const Shape& s : kShapes) {
      if (chunks == (s.form == kAny)) continue;
      const int64_t blocks = tiles_of(p, s.bm, s.bn) * splits;
      const bool alone = blocks <= kCus;
      const int64_t round = alone ? kCus : (int64_t)kCus * s.per_cu;
      const float rounds = (float)((blocks + round - 1) / round);
      consider(s.form, splits, 3.0f + rounds * (per * (alone ? s.alone_us : s.slice_us) + s.tile_us));
    }
  }
  if (best.form == kTile128 && tiles_of(p, 128, 128) * best.splits <= kCus) best.form = kTile128Deep;
  return best;
}

int part_ld(const FcvLmLinear& p) { return (p.n + 3) / 4 * 4; }

size_t workspace_bytes(const FcvLmLinear& p, const Plan& plan) {
  return plan.splits > 1 ? (size_t)plan.splits * p.m * part_ld(p) * 4 : 0;
}

template <class E, class C>
void launch_tiles(const Args& a, hipStream_t stream) {
  const unsigned blocks = (unsigned)(tiles_of(a.p, C::BM, C::BN) * a.splits);
  hipLaunchKernelGGL((linear_tile_kernel<E, C>), dim3(blocks), dim3(C::kThreads), 0, stream, a);
}

template <class E>
void launch(const FcvLmLinear& p, const Plan& plan, void* workspace, hipStream_t stream) {
  auto quad = [](const void* t, int dtype, int64_t ld) {
    return t == nullptr || (aligned(t, dtype == FCV_LM_F32 ? 16 : 8) && ld % 4 == 0);
  };
  const Args a{p, quad(p.y, p.y_dtype, p.ldy) && quad(p.residual, p.residual_dtype, p.ldr) &&
                      quad(p.bias, p.bias_dtype, 0),
               plan.splits, plan.slices, static_cast<float*>(workspace), part_ld(p)};
  switch (plan.form) {
    case kAny:
      hipLaunchKernelGGL((linear_any_kernel<E>),
                         dim3((unsigned)tiles_of(p, kTile, kTile), (unsigned)a.splits), dim3(256), 0,
                         stream, a);
      break;
    case kFew:
      hipLaunchKernelGGL((linear_few_kernel<E>),
                         dim3((unsigned)((p.n + kFewRows - 1) / kFewRows), (unsigned)a.splits),
                         dim3(64 * kFewWaves), 0, stream, a);
      break;
    case kTile64: launch_tiles<E, Tile<64, 64, 2, 2, 4>>(a, stream); break;
    case kTile64x128: launch_tiles<E, Tile<64, 128, 2, 2, 3>>(a, stream); break;
    case kTile128: launch_tiles<E, Tile<128, 128, 2, 2, 2>>(a, stream); break;
    case kTile128Deep: launch_tiles<E, Tile<128, 128, 2, 2, 3>>(a, stream); break;
    case kTile128x256: launch_tiles<E, Tile<128, 256, 2, 4, 3>>(a, stream); break;
    case kTile192x256: launch_tiles<E, Tile<192, 256, 2, 4, 2>>(a, stream); break;
    case kTile256: launch_tiles<E, Tile<256, 256, 2, 4, 2>>(a, stream); break;
  }
  if (a.splits > 1) {
    const int64_t quads = (int64_t)p.m * (a.part_ld / 4);
    hipLaunchKernelGGL((linear_join_kernel<E>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0,
                       stream, a);
  }
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" size_t fcv_lm_linear_workspace_bytes(const FcvLmLinear* args) {
  if (fcv::lm::check(args) || args->m == 0) return 0;
  return fcv::lm::workspace_bytes(*args, fcv::lm::plan_of(*args));
}

extern "C" int fcv_lm_linear_plan(const FcvLmLinear* args, int32_t* form, int32_t* ranges) {
  if (int rc = fcv::lm::check(args)) return rc;
  FCV_CHECK(form && ranges, FCV_ERR_INVALID, "null argument");
  const fcv::lm::Plan plan = fcv::lm::plan_of(*args);
  *form = plan.form;
  *ranges = plan.splits;
  return FCV_OK;
}

extern "C" int fcv_lm_linear(const FcvLmLinear* args, void* workspace, size_t workspace_bytes,
                             hipStream_t stream) {
  if (int rc = fcv::lm::check(args)) return rc;
  if (args->m == 0) return FCV_OK;
  const fcv::lm::Plan plan = fcv::lm::plan_of(*args);
  const size_t need = fcv::lm::workspace_bytes(*args, plan);
  FCV_CHECK(need == 0 || workspace, FCV_ERR_INVALID, "null workspace");
  FCV_CHECK(workspace_bytes >= need, FCV_ERR_INVALID,
            "workspace too small: need " + std::to_string(need) + " bytes");
  FCV_CHECK(need == 0 || fcv::lm::aligned(workspace, 256), FCV_ERR_INVALID,
            "workspace must be 256-byte aligned");
  if (args->dtype == FCV_LM_F16)
    fcv::lm::launch<fcv::lm::Half>(*args, plan, workspace, stream);
  else
    fcv::lm::launch<fcv::lm::Bf16>(*args, plan, workspace, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}
