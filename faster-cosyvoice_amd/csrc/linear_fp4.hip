// y = act(x W^T + bias) + residual over 4-bit weights, and the quantization of such weights.
//
// W is read in 4 bits and becomes x's 16-bit type in registers (one instruction for two codes and their
// scale, exact), so that products and sums are those of the 16-bit layer: fp32 on the matrix cores, one
// rounding at the end.  W is the A operand and x the B operand, as in linear.hip.
//
// A lane's share of W is the 16 bytes of one group: 32 codes, one scale.  The matrix instruction wants 8
// elements of K a lane; which ones is free as long as x agrees, so step j of a group takes its elements
// 8 j .. 8 j + 7 from both, and nothing is moved between lanes.
#include <string>

#include "fp4.hpp"
#include "linear_common.hpp"

namespace fcv {
namespace lm {
namespace {

struct Fp4Args {
  Args a;  // the epilogue's fields, x, the ranges of K
  const uint8_t *codes, *scales;
  int64_t ld_codes, ld_scales;
  int32_t k;  // of the weights: a.p.k may be that of an x laid out
};

// The codes of a word that holds elements at .. at + 7 of a row of k: those past k as zeros.  x is 0 there, but a
// scale can make an infinity of a code, and NaN of its product.
__device__ __forceinline__ uint32_t codes_below(uint32_t w, int at, int k) {
  const int n = min(max(k - at, 0), 8);
  return n == 8 ? w : w & ((1u << (4 * n)) - 1);
}

// ---- few rows: the weights straight into registers -------------------------------------------------
//
// v_mfma_f32_16x16x32: lane l has row l % 16 of W and group l / 16 of a span of four groups, 128 of K.  A
// workgroup has NT blocks of 16 rows of W and all rows of x (MT blocks of 16); its waves take turns in K, the
// codes of kAhead spans asked for at once, and are summed through LDS.
//
// Bound: a CU takes in about 48 B/ns, and a workgroup reads all of x beside its rows of W: of 32 rows eight
// times what 16 rows of W are.  Hence NT, and K cut over workgroups (blockIdx.y, joined by
// linear_join_kernel), where that leaves each CU less to read.
constexpr int kFewN = 16, kFewWaves = 8, kSpan = 128;

template <class E, int MT, int NT>
__global__ __launch_bounds__(64 * kFewWaves, 2) void linear_fp4_few_kernel(const Fp4Args f) {
  constexpr int kAhead = NT == 4 ? 2 : 4;
  constexpr int kTiles = MT * NT;
  __shared__ __attribute__((aligned(16))) f32x4 sums[kFewWaves][kTiles][64];
  const FcvLmLinear& p = f.a.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fb = lane >> 4;
  const int n0 = blockIdx.x * (kFewN * NT);
  const int groups = (p.k + FCV_FP4_GROUP - 1) / FCV_FP4_GROUP;
  const uint8_t *codes[NT], *scales[NT];
  const short* x[MT];
  f32x4 acc[MT][NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const int64_t row = min(n0 + 16 * u + fr, p.n - 1);
    codes[u] = f.codes + row * f.ld_codes;
    scales[u] = f.scales + row * f.ld_scales;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    x[t] = static_cast<const short*>(p.x) + (int64_t)min(16 * t + fr, p.m - 1) * p.ldx;
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int first = blockIdx.y * f.a.slices, end = min(first + f.a.slices, (p.k + kSpan - 1) / kSpan);
  s16x8 fx[2][MT][4];
  auto load_x = [&](int buf, int span) {
    const int k = span * kSpan + fb * FCV_FP4_GROUP;
    if ((span + 1) * kSpan <= p.k) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) fx[buf][t][j] = load8_any(x[t] + k + 8 * j);
    } else {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) fx[buf][t][j] = row_chunk(x[t], k + 8 * j, p.k);
    }
  };
  for (int span0 = first + wave; span0 < end; span0 += kFewWaves * kAhead) {
    u32x4 w[kAhead][NT];
    uint32_t s[kAhead][NT];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int span = span0 + i * kFewWaves, g = span * 4 + fb;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        w[i][u] = u32x4{0, 0, 0, 0};
        s[i][u] = 127;
        if (span < end && g < groups) {
          w[i][u] = *reinterpret_cast<const u32x4*>(codes[u] + (int64_t)g * 16);
          s[i][u] = scales[u][g];
        }
      }
    }
    load_x(0, span0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int span = span0 + i * kFewWaves;
      if (span >= end) break;
      if (i + 1 < kAhead && span + kFewWaves < end) load_x((i + 1) & 1, span + kFewWaves);
      if ((span + 1) * kSpan > p.k && p.k % FCV_FP4_GROUP) {
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[i][u][j] = codes_below(w[i][u][j], span * kSpan + fb * FCV_FP4_GROUP + 8 * j, p.k);
      }
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float scale = scale_of(s[i][u]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const s16x8 fw = fp4_octet<E>(w[i][u][j], scale);
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[t][u] = E::mfma16(fw, fx[i & 1][t][j], acc[t][u]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) sums[wave][t * NT + u][lane] = acc[t][u];
  __syncthreads();
  for (int i = wave; i < kTiles; i += kFewWaves) {
    f32x4 v = sums[0][i][lane];
#pragma unroll
    for (int s = 1; s < kFewWaves; ++s) v += sums[s][i][lane];
    const int m = 16 * (i / NT) + fr, n = n0 + 16 * (i % NT) + fb * 4;
    if (m >= p.m || n >= p.n) continue;
    if (f.a.splits > 1) {
      *reinterpret_cast<f32x4*>(f.a.part + ((int64_t)blockIdx.y * p.m + m) * f.a.part_ld + n) = v;
      continue;
    }
    const bool whole = n + 3 < p.n;
    finish4<E>(p, f.a.vec, m, n, v, bias4<E>(p, whole, n), residual4<E>(p, whole, m, n));
  }
}

// ---- many rows: operands by copies into LDS ---------------------------------------------------------
//
// The ring of slices of linear.hip: x as it lies there, W's slice in 4 bits (a quarter of the LDS and of the
// copies) and a row's four scales of 128 elements.  Rows of scales start on any byte: both words that the four lie
// in are copied, and shifted together where they are used.  A lane of the 32 x 32 x 16 instruction has one group in 64 of K: its codes are
// one read, and become fragments a step ahead of the products that take them.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int BK_>
struct Fp4Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, BK = BK_;
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int kChunks = BK / 8, kXRows = 64 / kChunks;       // 16-byte chunks of a row of x; rows of a copy
  static constexpr int kGroups = BK / 32, kWRows = 64 / kGroups;      // and of a row of codes
  static constexpr int kXCopies = BM / kXRows / kWaves;
  static constexpr int kWParts = BN / kWRows, kSParts = 2 * (BN / 64);
  static constexpr int kWCopies = kWParts > kWaves ? kWParts / kWaves : 1;
  static constexpr int kCopies = kXCopies + kWCopies + 1;
  static constexpr int kW = BM * BK * 2, kS = kW + BN * BK / 2, kStage = kS + BN * 8;  // bytes
  static constexpr int kLds = STAGES * kStage;
  static constexpr int kGroupM = 1024 / BM > 0 ? 1024 / BM : 1;
  static constexpr int kPerCu = 160 * 1024 / kLds;
  static constexpr int kWavesPerSimd = kPerCu * kWaves >= 8 ? 2 : 1;
  // small tiles: a whole slice's operands are read at once, under the products of the slice before
  static constexpr bool kWhole = TM * TN <= 2;
  static_assert(BM % (kXRows * kWaves) == 0 && kSParts <= kWaves, "copy split");
  static_assert((STAGES - 2) * kCopies < 64, "copies in flight");
};

// Place of group g of row r in a slice of codes: 16 rows read at one group touch all banks.
template <int BK>
__device__ __forceinline__ int swz_w(int r, int g) {
  return BK == 128 ? g ^ ((r >> 2) & 3) : g ^ ((r >> 3) & 1);
}

// kCut: K ends inside a group, whose other codes are cleared.  As a branch of one kernel that took 3 to 8 % of calls
// without such a group (2000 x 4096 x 2000 48.2 -> 50.4 us).
template <class E, class C, bool kCut>
__global__ __launch_bounds__(C::kThreads, C::kWavesPerSimd) void linear_fp4_tile_kernel(const Fp4Args f) {
  constexpr int BM = C::BM, BN = C::BN, TM = C::TM, TN = C::TN, S = C::STAGES, BK = C::BK;
  __shared__ __attribute__((aligned(1024))) char smem[C::kLds];
  const FcvLmLinear& p = f.a.p;
  const int tiles_m = (p.m + BM - 1) / BM, tiles_n = (p.n + BN - 1) / BN;
  int split, n0, m0;  // blocks are dealt over the XCDs as in linear.hip
  {
    const int total = tiles_m * tiles_n * f.a.splits;
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

  const int slice0 = split * f.a.slices * (kSpan / BK);  // in units of BK
  const int all = (p.k + BK - 1) / BK;
  const int KT = min(f.a.slices * (kSpan / BK), all - slice0);
  const bool ragged = p.k % BK != 0 && slice0 + KT == all;  // the last slice passes K

  // byte offset of each copy's source from the tile's first row; rows past the matrix read its last
  const char* xb = reinterpret_cast<const char*>(static_cast<const short*>(p.x) + (int64_t)m0 * p.ldx +
                                                 (int64_t)slice0 * BK);
  const char* wb =
      reinterpret_cast<const char*>(f.codes + (int64_t)n0 * f.ld_codes + (int64_t)slice0 * (BK / 2));
  const uintptr_t s_first = (uintptr_t)f.scales + (int64_t)n0 * f.ld_scales;
  const char* sb = reinterpret_cast<const char*>(s_first & ~(uintptr_t)3);
  auto scale_at = [&](int row) {  // of the tile, in bytes from sb
    return (uint32_t)(s_first & 3) + (uint32_t)min(row, p.n - 1 - n0) * (uint32_t)f.ld_scales;
  };
  const int crow = lane / C::kChunks, cpos = lane % C::kChunks;
  uint32_t x_off[C::kXCopies], w_off[C::kWCopies];
#pragma unroll
  for (int i = 0; i < C::kXCopies; ++i) {
    const int row = (wave * C::kXCopies + i) * C::kXRows + crow;
    x_off[i] = (uint32_t)min(row, p.m - 1 - m0) * (uint32_t)(p.ldx * 2) + swz<BK>(row, cpos) * 16;
  }
  // where a slice has fewer copies of codes or scales than waves, several waves make the same one
  const int w_part = wave * C::kWCopies % C::kWParts, s_part = wave % C::kSParts;
  const int grow = lane / C::kGroups, gpos = lane % C::kGroups;
#pragma unroll
  for (int i = 0; i < C::kWCopies; ++i) {
    const int row = (w_part + i) * C::kWRows + grow;
    w_off[i] = (uint32_t)min(row, p.n - 1 - n0) * (uint32_t)f.ld_codes + swz_w<BK>(row, gpos) * 16;
  }
  const uint32_t s_at = scale_at(s_part / 2 * 64 + lane);
  const uint32_t s_off = (s_at & ~3u) + (s_part & 1) * 4;
  // the last span's groups; a second word without one of them is not read (it may lie behind the scales)
  const int last_span = (p.k - 1) / kSpan;
  const int last_groups = (p.k + FCV_FP4_GROUP - 1) / FCV_FP4_GROUP - 4 * last_span;
  const uint32_t s_last = (s_at & ~3u) + ((s_part & 1) && (int)(s_at & 3) + last_groups > 4 ? 4 : 0);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
  const uint32_t lds_x = lds0 + wave * C::kXCopies * 1024;
  const uint32_t lds_w = lds0 + C::kW + w_part * 1024;
  const uint32_t lds_s = lds0 + C::kS + s_part * 256;
  // copies [c0, c1) of slice kt (scales, codes, x) into a stage
  auto issue = [&](int kt, int stage, int c0, int c1) {
    const uint32_t at = stage * C::kStage;
    const int slice = slice0 + kt;
    const bool last = ragged && kt == KT - 1;
    const int left = p.k - slice * BK;  // columns of the slice below K, a multiple of 8
    const char* xk = xb + kt * (BK * 2);
    const char* wk = wb + kt * (BK / 2);
#pragma unroll
    for (int c = 0; c < C::kCopies; ++c) {
      if (c < c0 || c >= c1) continue;
      if (c == 0) {
        const int span = slice * BK / kSpan;
        lds_dma4(sb + span * 4, span == last_span ? s_last : s_off, lds_s + at);
      } else if (c < 1 + C::kWCopies) {
        const int i = c - 1;
        if (last) {
          const int row = (w_part + i) * C::kWRows + grow;
          lds_dma16_at(swz_w<BK>(row, gpos) * 32 < left ? static_cast<const void*>(wk + w_off[i]) : zeros16,
                       lds_w + at + i * 1024);
        } else {
          lds_dma16(wk, w_off[i], lds_w + at + i * 1024);
        }
      } else {
        const int i = c - 1 - C::kWCopies;
        if (last) {
          const int row = (wave * C::kXCopies + i) * C::kXRows + crow;
          lds_dma16_at(swz<BK>(row, cpos) * 8 < left ? static_cast<const void*>(xk + x_off[i]) : zeros16,
                       lds_x + at + i * 1024);
        } else {
          lds_dma16(xk, x_off[i], lds_x + at + i * 1024);
        }
      }
    }
  };

  // slice kt is in LDS: codes past K in the last one's last group become 0
  auto trim = [&](int kt, int st) {
    if constexpr (kCut) {
      if (kt != KT - 1 || slice0 + KT != all) return;
      const int left = f.k - (slice0 + kt) * BK, g = left / FCV_FP4_GROUP;
      for (int row = threadIdx.x; row < BN; row += C::kThreads) {
        u32x4* at = reinterpret_cast<u32x4*>(smem + st * C::kStage + C::kW + row * (BK / 2) + swz_w<BK>(row, g) * 16);
        u32x4 w = *at;
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = codes_below(w[q], 8 * q, left % FCV_FP4_GROUP);
        *at = w;
      }
      __syncthreads();
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
  constexpr int KS = BK / 16, kHalves = BK / 64;  // steps; groups of a lane
  constexpr int kSets = C::kWhole ? 2 : 1;
  s16x8 fx[C::kWhole ? 2 * KS : 2][TM], fw[2][TN];
  u32x4 wc[kSets][TN][kHalves];
  uint32_t ws[TN][2], ss[kSets][TN];  // scales as they lie, and in their places
  const uint32_t s_shift = (uint32_t)(s_first + (uint32_t)fr * (uint32_t)f.ld_scales) % 4 * 8;  // rows 32 apart alike
  auto load_w = [&](int set, int st) {
    const char* w = smem + st * C::kStage + C::kW;
    const char* s = smem + st * C::kStage + C::kS;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int row = wn0 + j * 32 + fr;
#pragma unroll
      for (int u = 0; u < kHalves; ++u)
        wc[set][j][u] =
            *reinterpret_cast<const u32x4*>(w + row * (BK / 2) + swz_w<BK>(row, 2 * u + fh) * 16);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        ws[j][u] = *reinterpret_cast<const uint32_t*>(s + row / 64 * 512 + u * 256 + row % 64 * 4);
    }
  };
  // step ks: elements 8 (ks % 4) .. + 7 of group 2 (ks / 4) + fh
  auto load_x = [&](int buf, int ks, int st) {
    const short* sx = reinterpret_cast<const short*>(smem + st * C::kStage);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = wm0 + i * 32 + fr;
      fx[buf][i] = *reinterpret_cast<const s16x8*>(
          sx + row * BK + swz<BK>(row, ks / 4 * 8 + 4 * fh + ks % 4) * 8);
    }
  };
  // the scales of slice kt; what lies past K is 1
  auto place = [&](int set, int kt) {
    const bool last = (slice0 + kt) * BK / kSpan == last_span && last_groups < 4;
    const uint32_t keep = last ? (1u << (8 * last_groups)) - 1 : ~0u;
#pragma unroll
    for (int j = 0; j < TN; ++j)
      ss[set][j] = (__builtin_amdgcn_alignbit(ws[j][1], ws[j][0], s_shift) & keep) | (0x7f7f7f7fu & ~keep);
  };
  // `odd`: the slice is the second one of its span (BK 64)
  auto convert = [&](int buf, int set, int ks, int odd) {
    const int shift = ((ks / 4 + odd) * 2 + fh) * 8;
#pragma unroll
    for (int j = 0; j < TN; ++j)
      fw[buf][j] = fp4_octet<E>(wc[set][j][ks / 4][ks % 4], scale_of((ss[set][j] >> shift) & 255));
  };
  auto parity = [&](int kt) { return BK == 64 ? (slice0 + kt) & 1 : 0; };
#pragma unroll
  for (int st = 0; st < S - 1; ++st)
    if (st < KT) issue(st, st, 0, C::kCopies);
  wait_ahead<C::kCopies, S - 2>(KT - 1);
  __syncthreads();
  int kt = 0, stage = 0;
  trim(kt, stage);
  if constexpr (C::kWhole) {
    // as in linear.hip: slice kt's operands are asked for after the barrier that publishes it and used after
    // the next one
    auto load_all = [&](auto set) {
      load_w(decltype(set)::value, stage);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) load_x(decltype(set)::value * KS + ks, ks, stage);
    };
    auto mma_all = [&](auto set, int kt) {
      __builtin_amdgcn_sched_barrier(0);
      const int odd = parity(kt);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        convert(ks & 1, decltype(set)::value, ks, odd);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = E::mfma32(fw[ks & 1][j], fx[decltype(set)::value * KS + ks][i], acc[i][j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    auto step = [&](auto set, auto before) {
      wait_ahead<C::kCopies, S - 2>(KT - 1 - kt);
      __syncthreads();
      const int freed = stage;
      stage = stage == S - 1 ? 0 : stage + 1;
      trim(kt, stage);
      load_all(set);
      if (kt + S - 1 < KT) issue(kt + S - 1, freed, 0, C::kCopies);
      mma_all(before, kt - 1);
      place(decltype(set)::value, kt);
    };
    if (S - 1 < KT) issue(S - 1, S - 1, 0, C::kCopies);
    load_all(even);
    place(0, 0);
    for (kt = 1; kt < KT;) {
      step(odd, even);
      if (++kt == KT) break;
      step(even, odd);
      ++kt;
    }
    if (KT & 1)
      mma_all(even, KT - 1);
    else
      mma_all(odd, KT - 1);
  } else {
    // rotated by one step as in linear.hip: a slice's last step runs from registers after the barrier that
    // publishes the next slice and frees the one before
    auto products = [&](int buf) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = E::mfma32(fw[buf][j], fx[buf][i], acc[i][j]);
    };
    auto mma = [&](int buf) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      products(buf);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    };
    // step ks - 1's products, and between them the conversions for step ks
    auto mma_convert = [&](int ks, int odd) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      convert(ks & 1, 0, ks, odd);
      products((ks - 1) & 1);
#pragma unroll
      for (int i = 0; i < TM * TN; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
        __builtin_amdgcn_sched_group_barrier(0x002, (6 * TN + TM * TN - 1) / (TM * TN), 0);  // vector instructions
      }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int kPhases = S == 2 ? KS - 1 : KS;
    constexpr int kPer = (C::kCopies + kPhases - 1) / kPhases;
    auto copies = [&](int phase) {
      if (kt + S - 1 < KT)
        issue(kt + S - 1, stage == 0 ? S - 1 : stage - 1, phase * kPer, phase * kPer + kPer);
    };
    auto head = [&](int st) {
#pragma unroll
      for (int ks = 0; ks + 1 < KS; ++ks) {
        load_x((ks + 1) & 1, ks + 1, st);
        copies(ks + 1);
        mma_convert(ks + 1, parity(kt));
      }
    };
    copies(0);
    load_w(0, 0);
    load_x(0, 0, 0);
    place(0, 0);
    convert(0, 0, 0, parity(0));
    head(0);
    for (kt = 1; kt < KT; ++kt) {
      const int next = stage == S - 1 ? 0 : stage + 1;
      wait_ahead<C::kCopies, S - 2>(KT - 1 - kt);
      __syncthreads();
      stage = next;
      trim(kt, stage);
      load_w(0, stage);
      load_x(0, 0, stage);
      copies(0);
      mma(1);
      place(0, kt);
      convert(0, 0, 0, parity(kt));
      head(stage);
    }
    mma(1);
  }
  store_tile<E, C, C::kLds>(f.a, acc, reinterpret_cast<short*>(smem), split, n0, wn0, wm0, m0);
}

// Copies rows of x from any boundary to 16-byte ones, with zeros up to a multiple of 8.  A thread has 8 elements.
__global__ __launch_bounds__(256) void lay_out_kernel(const FcvLmLinear p, short* x, int64_t ldx, int64_t units) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < units; i += (int64_t)gridDim.x * 256) {
    const int64_t per = ldx / 8, row = i / per;
    const int k = (int)(i % per) * 8;
    *reinterpret_cast<s16x8*>(x + row * ldx + k) =
        row_chunk(static_cast<const short*>(p.x) + row * p.ldx, k, p.k);
  }
}

// ---- quantization ---------------------------------------------------------------------------------

// A thread has a group of 32.
template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(const FcvFp4Quantize p) {
  const int groups = (p.k + FCV_FP4_GROUP - 1) / FCV_FP4_GROUP;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)p.n * groups) return;
  const int row = (int)(i / groups), g = (int)(i % groups);
  const T* w = static_cast<const T*>(p.w) + (int64_t)row * p.ldw + (int64_t)g * FCV_FP4_GROUP;
  const int count = min(FCV_FP4_GROUP, p.k - g * FCV_FP4_GROUP);
  float v[FCV_FP4_GROUP];
  uint32_t top = 0;  // the largest magnitude's bits: infinities and NaN come out on top
#pragma unroll
  for (int e = 0; e < FCV_FP4_GROUP; ++e) {
    v[e] = e < count ? (float)w[e] : 0.0f;
    top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  constexpr bool kHalf = std::is_same<T, f16>::value;
  const uint32_t b = fp4_scale_byte(top, kHalf);
  u32x4 c = {0, 0, 0, 0};
  if (b != 255) {
    const float scale = scale_of(b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = fp4_word(v + 8 * e, scale);
  }
  *reinterpret_cast<u32x4*>(p.codes + row * p.ld_codes + (int64_t)g * 16) = c;
  p.scales[row * p.ld_scales + g] = (uint8_t)b;
}

// ---- host ---------------------------------------------------------------------------------------

int check(const FcvFp4Linear* p) {
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
  FCV_CHECK(p->k <= (1 << 21), FCV_ERR_INVALID, "k is limited to 2^21");
  FCV_CHECK(p->m <= (1 << 22) && p->n <= (1 << 22) && (int64_t)p->m * p->n <= (1LL << 34),
            FCV_ERR_INVALID, "m and n are limited to 2^22 each and their product to 2^34");
  FCV_CHECK(p->ldx >= 0 && p->ld_codes >= 0 && p->ld_scales >= 0 && p->ldr >= 0, FCV_ERR_INVALID,
            "negative row stride");
  FCV_CHECK(p->n == 1 || (p->ld_codes < (1 << 24) && p->ld_scales < (1 << 24)), FCV_ERR_INVALID,
            "row strides of codes and scales are limited to 2^24");
  FCV_CHECK(p->ldy >= p->n || p->m <= 1, FCV_ERR_INVALID, "y's row stride is shorter than its row");
  if (p->m == 0) return FCV_OK;
  FCV_CHECK(p->x && p->codes && p->scales && p->y, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(aligned(p->codes, 16) && (p->n == 1 || p->ld_codes % 16 == 0), FCV_ERR_INVALID,
            "rows of codes must start on 16-byte boundaries");
  FCV_CHECK(aligned(p->x, 2) && aligned(p->y, element_size(p->y_dtype)) &&
                aligned(p->bias, element_size(p->bias_dtype)) &&
                aligned(p->residual, element_size(p->residual_dtype)),
            FCV_ERR_INVALID, "a tensor does not start on an element's boundary");
  return FCV_OK;
}

// Which kernel, and into how many ranges K is cut: the least of estimates in us, fits to measurements.
// Tiles:  rounds (spans span_us + tile_us) + 2.9,   rounds = blocks over the CUs, `per_cu` each, rounded up;
//   span_us of full rounds at K 4096 (alone: one block a CU of those that share one).  32 x 4096 x 16384 by
//   tiles of 64 x 64 23, by few rows 19.  By tiles of 128 x 256, 192 x 256 and 256 x 256 9184 x 1024 x 2048 take
//   61, 54 and 64 us, 2048 x 4096 x 4096 72, 84 and 88, 8192 x 4096 x 8192 545, 542 and 464.
// Few rows, up to 32:  2.9 + what W takes, 3.5 TB/s from all CUs or 18 B/ns to one, + 21 ns for each KB of x
//   that a CU reads.  In us by blocks of 16, 32 and 64 rows of W: 1 x 4096 x 4096 5.3, 7.2 and 11; 32 x 4096 x
//   16384 39, 26 and 19; 32 x 4096 x 4096 11.8, 13.5 and 17.5, with K in 1, 2 and 4 ranges 11.8, 10.7 and 9.8.
//   (x loaded in whole lines, W's words changing places between lanes instead: no faster.)
// A cut K adds the join's 1.8 (3.5 to few rows: what the second launch takes of the host, which calls that
// short wait for) and its sums' way, an x off its boundaries the pass that lays it out (the same
// for every tile).
enum Form { kFew, kTile64, kTile64x128, kTile128, kTile128x256, kTile192x256, kTile256 };

struct Shape {
  Form form;
  int bm, bn, per_cu;
  float alone_us, span_us, tile_us;
};
constexpr Shape kShapes[] = {
    {kTile64, 64, 64, 1, 0.60f, 0.62f, 1.2f},    {kTile64x128, 64, 128, 2, 0.76f, 1.25f, 1.5f},
    {kTile128, 128, 128, 2, 1.50f, 2.24f, 1.5f}, {kTile128x256, 128, 256, 1, 2.08f, 2.08f, 2.0f},
    {kTile192x256, 192, 256, 1, 2.75f, 2.75f, 3.0f},
    {kTile256, 256, 256, 1, 3.56f, 3.56f, 4.0f}};
constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr int kMinSpans = 2;  // of a range
constexpr int kFewMost = 32;  // rows of x

struct Plan {
  Form form;
  int nt;              // of kFew: blocks of 16 rows of W
  int splits, spans;   // ranges of K, and the spans of 128 of one
  bool lay_x;          // x is laid out first
};

int part_ld(int n) { return (n + 3) / 4 * 4; }

float join_us(const FcvFp4Linear& p, int splits) {
  return splits > 1 ? (p.m <= kFewMost ? 3.5f : 1.8f) + (float)p.m * (float)p.n * 8.0f * splits / 5.0e6f : 0.0f;
}

Plan plan_of(const FcvFp4Linear& p) {
  const bool lay_x = !(aligned(p.x, 16) && (p.ldx % 8 == 0 || p.m == 1) && p.k % 8 == 0 && p.ldx < (1 << 22));
  const int spans = (p.k + kSpan - 1) / kSpan;
  Plan best{};
  float best_us = 3.0e38f;
  auto consider = [&](Form form, int nt, int splits, float us) {
    us += join_us(p, splits);
    if (us >= best_us) return;
    best_us = us;
    const int per = (spans + splits - 1) / splits;
    best = Plan{form, nt, (spans + per - 1) / per, per, form != kFew && lay_x};
  };
  for (int splits : kSplits) {
    if (splits > 1 && spans < splits * kMinSpans) break;
    const float per = (float)((spans + splits - 1) / splits);
    if (p.m <= kFewMost) {
      for (int nt = 1; nt <= 4; nt *= 2) {
        const int64_t blocks = (int64_t)((p.n + kFewN * nt - 1) / (kFewN * nt)) * splits;
        const float rounds = (float)((blocks + kCus - 1) / kCus);
        const float w = per * nt * 1088.0f;  // bytes of a block
        consider(kFew, nt, splits,
                 2.9f + std::max((float)blocks * w / 3.5e6f, rounds * w / 18.0e3f) +
                     rounds * per * (float)p.m * 256.0f * 21.0e-6f);
      }
      continue;
    }
    for (const Shape& s : kShapes) {
      const int64_t blocks = (int64_t)((p.m + s.bm - 1) / s.bm) * ((p.n + s.bn - 1) / s.bn) * splits;
      const bool alone = blocks <= kCus;
      const int64_t round = alone ? kCus : (int64_t)kCus * s.per_cu;
      const float rounds = (float)((blocks + round - 1) / round);
      consider(s.form, 0, splits, 2.9f + rounds * (per * (alone ? s.alone_us : s.span_us) + s.tile_us));
    }
  }
  return best;
}

int64_t laid_ldx(const FcvFp4Linear& p) { return (p.k + 7) / 8 * 8; }
size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

// The workspace: sums of the ranges, then x laid out.
size_t part_bytes(const FcvFp4Linear& p, const Plan& plan) {
  return plan.splits > 1 ? round_up((size_t)plan.splits * p.m * part_ld(p.n) * 4) : 0;
}
size_t x_bytes(const FcvFp4Linear& p, const Plan& plan) {
  return plan.lay_x ? round_up((size_t)p.m * laid_ldx(p) * 2) : 0;
}
size_t workspace_bytes(const FcvFp4Linear& p, const Plan& plan) {
  return part_bytes(p, plan) + x_bytes(p, plan);
}

template <class E, class C>
void launch_tiles(const Fp4Args& f, hipStream_t stream) {
  const int64_t tiles = (int64_t)((f.a.p.m + C::BM - 1) / C::BM) * ((f.a.p.n + C::BN - 1) / C::BN);
  const dim3 grid((unsigned)(tiles * f.a.splits)), block(C::kThreads);
  if (f.k % FCV_FP4_GROUP)
    hipLaunchKernelGGL((linear_fp4_tile_kernel<E, C, true>), grid, block, 0, stream, f);
  else
    hipLaunchKernelGGL((linear_fp4_tile_kernel<E, C, false>), grid, block, 0, stream, f);
}

template <class E, int MT>
void launch_few(const Fp4Args& f, int nt, hipStream_t stream) {
  const dim3 grid((f.a.p.n + kFewN * nt - 1) / (kFewN * nt), f.a.splits), block(64 * kFewWaves);
  if (nt == 1)
    hipLaunchKernelGGL((linear_fp4_few_kernel<E, MT, 1>), grid, block, 0, stream, f);
  else if (nt == 2)
    hipLaunchKernelGGL((linear_fp4_few_kernel<E, MT, 2>), grid, block, 0, stream, f);
  else
    hipLaunchKernelGGL((linear_fp4_few_kernel<E, MT, 4>), grid, block, 0, stream, f);
}

template <class E>
void launch(const FcvFp4Linear& p, const Plan& plan, void* workspace, hipStream_t stream) {
  auto quad = [](const void* t, int dtype, int64_t ld) {
    return t == nullptr || (aligned(t, dtype == FCV_LM_F32 ? 16 : 8) && ld % 4 == 0);
  };
  FcvLmLinear e{};
  e.x = p.x, e.bias = p.bias, e.residual = p.residual, e.y = p.y;
  e.ldx = p.ldx, e.ldr = p.ldr, e.ldy = p.ldy, e.m = p.m, e.n = p.n, e.k = p.k;
  e.dtype = p.dtype, e.bias_dtype = p.bias_dtype, e.residual_dtype = p.residual_dtype;
  e.y_dtype = p.y_dtype, e.activation = p.activation;
  const Args a{e, quad(p.y, p.y_dtype, p.ldy) && quad(p.residual, p.residual_dtype, p.ldr) &&
                      quad(p.bias, p.bias_dtype, 0),
               plan.splits, plan.spans, static_cast<float*>(workspace), part_ld(p.n)};
  Fp4Args f{a, p.codes, p.scales, p.ld_codes, p.ld_scales, p.k};
  if (plan.lay_x) {
    short* x = reinterpret_cast<short*>(static_cast<char*>(workspace) + part_bytes(p, plan));
    const int64_t units = p.m * (laid_ldx(p) / 8);
    const int64_t blocks = std::min<int64_t>((units + 255) / 256, 1 << 20);
    hipLaunchKernelGGL(lay_out_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, f.a.p, x, laid_ldx(p), units);
    f.a.p.x = x, f.a.p.ldx = laid_ldx(p), f.a.p.k = (int32_t)laid_ldx(p);
  }
  switch (plan.form) {
    case kFew:
      if (p.m <= 16)
        launch_few<E, 1>(f, plan.nt, stream);
      else
        launch_few<E, 2>(f, plan.nt, stream);
      break;
    case kTile64: launch_tiles<E, Fp4Tile<64, 64, 2, 2, 4, 128>>(f, stream); break;
    case kTile64x128: launch_tiles<E, Fp4Tile<64, 128, 2, 2, 3, 128>>(f, stream); break;
    case kTile128: launch_tiles<E, Fp4Tile<128, 128, 2, 2, 3, 64>>(f, stream); break;
    case kTile128x256: launch_tiles<E, Fp4Tile<128, 256, 2, 4, 3, 64>>(f, stream); break;
    case kTile192x256: launch_tiles<E, Fp4Tile<192, 256, 2, 4, 3, 64>>(f, stream); break;
    case kTile256: launch_tiles<E, Fp4Tile<256, 256, 2, 4, 3, 64>>(f, stream); break;
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

extern "C" int fcv_fp4_quantize(const FcvFp4Quantize* args, hipStream_t stream) {
  using namespace fcv::lm;
  const FcvFp4Quantize* p = args;
  FCV_CHECK(p, FCV_ERR_INVALID, "null arguments");
  FCV_CHECK(p->dtype >= FCV_LM_F16 && p->dtype <= FCV_LM_F32, FCV_ERR_INVALID,
            "dtype must be FCV_LM_F16, FCV_LM_BF16 or FCV_LM_F32");
  FCV_CHECK(p->n >= 0 && p->k >= 1 && p->n <= (1 << 22) && p->k <= (1 << 26), FCV_ERR_INVALID,
            "need 0 <= n <= 2^22 and 1 <= k <= 2^26");
  if (p->n == 0) return FCV_OK;
  const int64_t groups = (p->k + FCV_FP4_GROUP - 1) / FCV_FP4_GROUP;
  FCV_CHECK(p->w && p->codes && p->scales, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(aligned(p->w, element_size(p->dtype)), FCV_ERR_INVALID,
            "w does not start on an element's boundary");
  FCV_CHECK(aligned(p->codes, 16) && (p->n == 1 || p->ld_codes % 16 == 0), FCV_ERR_INVALID,
            "rows of codes must start on 16-byte boundaries");
  FCV_CHECK(p->n == 1 || (p->ldw >= 0 && p->ld_codes >= 16 * groups && p->ld_scales >= groups),
            FCV_ERR_INVALID, "rows of codes or scales overlap");
  FCV_CHECK(p->n * groups <= (1LL << 31), FCV_ERR_INVALID, "at most 2^31 groups in a call");
  const int64_t blocks = (p->n * groups + 255) / 256;
  const dim3 grid((unsigned)blocks);
  if (p->dtype == FCV_LM_F16)
    hipLaunchKernelGGL(quantize_kernel<fcv::f16>, grid, dim3(256), 0, stream, *p);
  else if (p->dtype == FCV_LM_BF16)
    hipLaunchKernelGGL(quantize_kernel<__bf16>, grid, dim3(256), 0, stream, *p);
  else
    hipLaunchKernelGGL(quantize_kernel<float>, grid, dim3(256), 0, stream, *p);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}

extern "C" size_t fcv_fp4_linear_workspace_bytes(const FcvFp4Linear* args) {
  if (fcv::lm::check(args) || args->m == 0) return 0;
  return fcv::lm::workspace_bytes(*args, fcv::lm::plan_of(*args));
}

extern "C" int fcv_fp4_linear_plan(const FcvFp4Linear* args, int32_t* form, int32_t* ranges) {
  if (int rc = fcv::lm::check(args)) return rc;
  FCV_CHECK(form && ranges, FCV_ERR_INVALID, "null argument");
  const fcv::lm::Plan plan = fcv::lm::plan_of(*args);
  *form = plan.form;
  *ranges = plan.splits;
  return FCV_OK;
}

extern "C" int fcv_fp4_linear(const FcvFp4Linear* args, void* workspace, size_t workspace_bytes,
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
