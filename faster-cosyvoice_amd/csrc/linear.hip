// y = act(x W^T + bias) + residual on the matrix cores, for any row count, width and stride.
//
// The product runs on v_mfma_f32_32x32x16 with W as the A operand and x as the B operand, so that a
// lane's accumulator holds four consecutive columns of one row of y per register group.
#include <algorithm>

#include "lm.hpp"

namespace fcv {
namespace lm {
namespace {

struct Args {
  FcvLmLinear p;
  bool x_chunks, w_chunks;  // rows start on 16-byte boundaries
};

// ---- the epilogue -------------------------------------------------------------------------------

__device__ __forceinline__ float act(float z, int kind) {
  switch (kind) {
    case FCV_LM_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays
    case FCV_LM_ACT_SILU: return silu(z);
    case FCV_LM_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case FCV_LM_ACT_GELU_TANH: return gelu_tanh(z);
    default: return z;
  }
}

template <class E>
__device__ __forceinline__ float element(const void* p, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : E::to_f32(static_cast<const short*>(p)[i]);
}

// Four columns n .. n + 3 of row m (those below N), from their sums.
template <class E>
__device__ __forceinline__ void finish4(const FcvLmLinear& p, int m, int n, f32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= p.n) break;
    float z = v[e];
    if (p.bias) z += element<E>(p.bias, p.bias_dtype == FCV_LM_F32, n + e);
    z = act(z, p.activation);
    if (p.residual)
      z += element<E>(p.residual, p.residual_dtype == FCV_LM_F32, (int64_t)m * p.ldr + n + e);
    const int64_t at = (int64_t)m * p.ldy + n + e;
    if (p.y_dtype == FCV_LM_F32)
      static_cast<float*>(p.y)[at] = z;
    else
      static_cast<short*>(p.y)[at] = E::from_f32(z);
  }
}

// ---- any alignment: operands through registers --------------------------------------------------

// Elements k .. k + 7 of a row of `len`, zeros past its end.
__device__ __forceinline__ s16x8 row_chunk(const short* row, int k, int len, bool chunks) {
  s16x8 v = {};
  if (chunks && k + 8 <= len) return *reinterpret_cast<const s16x8*>(row + k);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < len) v[e] = row[k + e];
  return v;
}

constexpr int kTile = 64, kDepth = 64, kPitch = kDepth + 8;

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
  f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
  for (int k0 = 0; k0 < p.k; k0 += kDepth) {
    s16x8 rx[2], rw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int m = min(m0 + lr + 32 * i, p.m - 1), n = min(n0 + lr + 32 * i, p.n - 1);
      rx[i] = row_chunk(static_cast<const short*>(p.x) + (int64_t)m * p.ldx, k0 + lc, p.k, a.x_chunks);
      rw[i] = row_chunk(static_cast<const short*>(p.w) + (int64_t)n * p.ldw, k0 + lc, p.k, a.w_chunks);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<s16x8*>(&sx[lr + 32 * i][lc]) = rx[i];
      *reinterpret_cast<s16x8*>(&sw[lr + 32 * i][lc]) = rw[i];
    }
    __syncthreads();
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
  for (int g = 0; g < 4; ++g)
    finish4<E>(p, m, n0 + wn + g * 8 + fh * 4,
               f32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]});
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

template <class E>
void launch(const FcvLmLinear& p, hipStream_t stream) {
  Args a{p, aligned(p.x, 16) && (p.ldx % 8 == 0 || p.m == 1),
         aligned(p.w, 16) && (p.ldw % 8 == 0 || p.n == 1)};
  hipLaunchKernelGGL((linear_any_kernel<E>),
                     dim3((unsigned)((int64_t)((p.n + kTile - 1) / kTile) * ((p.m + kTile - 1) / kTile))),
                     dim3(256), 0, stream, a);
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" size_t fcv_lm_linear_workspace_bytes(const FcvLmLinear* args) {
  (void)args;
  return 0;
}

extern "C" int fcv_lm_linear(const FcvLmLinear* args, void* workspace, size_t workspace_bytes,
                             hipStream_t stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (int rc = fcv::lm::check(args)) return rc;
  if (args->m == 0) return FCV_OK;
  if (args->dtype == FCV_LM_F16)
    fcv::lm::launch<fcv::lm::Half>(*args, stream);
  else
    fcv::lm::launch<fcv::lm::Bf16>(*args, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}
