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
};

// ---- few rows: the weights straight into registers -------------------------------------------------
//
// v_mfma_f32_16x16x32: lane l has row l % 16 of W and group l / 16 of a span of four groups, 128 of K.
constexpr int kFewN = 16, kFewWaves = 8, kSpan = 128;

// MT blocks of 16 rows of x.
template <class E, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void linear_fp4_few_kernel(const Fp4Args f) {
  __shared__ __attribute__((aligned(16))) f32x4 sums[kFewWaves][MT][64];
  const FcvLmLinear& p = f.a.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fb = lane >> 4;
  const int n0 = blockIdx.x * kFewN, m0 = blockIdx.z * (16 * MT);
  const int groups = (p.k + FCV_FP4_GROUP - 1) / FCV_FP4_GROUP;
  const int64_t row = min(n0 + fr, p.n - 1);
  const uint8_t* codes = f.codes + row * f.ld_codes;
  const uint8_t* scales = f.scales + row * f.ld_scales;
  const short* x[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    x[t] = static_cast<const short*>(p.x) + (int64_t)min(m0 + 16 * t + fr, p.m - 1) * p.ldx;
    acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int first = blockIdx.y * f.a.slices, end = min(first + f.a.slices, (p.k + kSpan - 1) / kSpan);
  for (int span = first + wave; span < end; span += kFewWaves) {
    const int g = span * 4 + fb;
    const bool there = g < groups;
    u32x4 w = {0, 0, 0, 0};
    uint32_t s = 127;
    if (there) {
      w = *reinterpret_cast<const u32x4*>(codes + (int64_t)g * 16);
      s = scales[g];
    }
    const float scale = scale_of(s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const s16x8 fw = fp4_octet<E>(w[j], scale);
#pragma unroll
      for (int t = 0; t < MT; ++t)
        acc[t] = E::mfma16(fw, row_chunk(x[t], g * FCV_FP4_GROUP + 8 * j, p.k), acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave >= MT) return;
  f32x4 v = sums[0][wave][lane];
#pragma unroll
  for (int s = 1; s < kFewWaves; ++s) v += sums[s][wave][lane];
  const int m = m0 + 16 * wave + fr, n = n0 + fb * 4;
  if (m >= p.m || n >= p.n) return;
  if (f.a.splits > 1) {
    *reinterpret_cast<f32x4*>(f.a.part + ((int64_t)blockIdx.y * p.m + m) * f.a.part_ld + n) = v;
    return;
  }
  const bool vec = f.a.vec && n + 3 < p.n;
  finish4<E>(p, vec, m, n, v, bias4<E>(p, vec, n), residual4<E>(p, vec, m, n));
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
  FCV_CHECK(p->k <= (1 << 26), FCV_ERR_INVALID, "k is limited to 2^26");
  FCV_CHECK(p->m <= (1 << 22) && p->n <= (1 << 22) && (int64_t)p->m * p->n <= (1LL << 34),
            FCV_ERR_INVALID, "m and n are limited to 2^22 each and their product to 2^34");
  FCV_CHECK(p->ldx >= 0 && p->ld_codes >= 0 && p->ld_scales >= 0 && p->ldr >= 0, FCV_ERR_INVALID,
            "negative row stride");
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

struct Plan {
  int mt;              // blocks of 16 rows of x
  int splits, slices;  // ranges of K, and the spans of one
};

Plan plan_of(const FcvFp4Linear& p) {
  const int spans = (p.k + kSpan - 1) / kSpan;
  return Plan{p.m <= 16 ? 1 : 2, 1, spans};
}

int part_ld(const FcvFp4Linear& p) { return (p.n + 3) / 4 * 4; }

size_t workspace_bytes(const FcvFp4Linear& p, const Plan& plan) {
  return plan.splits > 1 ? (size_t)plan.splits * p.m * part_ld(p) * 4 : 0;
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
               plan.splits, plan.slices, static_cast<float*>(workspace), part_ld(p)};
  const Fp4Args f{a, p.codes, p.scales, p.ld_codes, p.ld_scales};
  const dim3 grid((p.n + kFewN - 1) / kFewN, plan.splits, (p.m + 16 * plan.mt - 1) / (16 * plan.mt));
  if (plan.mt == 1)
    hipLaunchKernelGGL((linear_fp4_few_kernel<E, 1>), grid, dim3(64 * kFewWaves), 0, stream, f);
  else
    hipLaunchKernelGGL((linear_fp4_few_kernel<E, 2>), grid, dim3(64 * kFewWaves), 0, stream, f);
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
