// Norms of queries and keys per head, the position rotation and the cache append in one pass.
//
// Per head x of D elements:  y = x / sqrt(mean(x^2) + eps) * w;  the first R elements are rotated
// in pairs, (a, b) -> (a cos - b sin, b cos + a sin).  Everything between the load and the store is
// fp32; a value is rounded once.
//
// Bound: bandwidth (each element is read once and written once; the tables' row, 2 R bytes a token,
// is shared by all of the token's heads), or the launch itself for a few tokens.
// Split: a head takes D / 16 lanes, each with two 16-byte chunks.  A lane's chunks are j and
// j + R / 16 inside the rotated part, so that both members of a pair (i, i + R / 2) are in one lane
// (pairs (2 i, 2 i + 1) are inside a chunk anyway), and 2 j, 2 j + 1 behind it: no exchange but the
// sum of squares over 4 or 8 neighbouring lanes.
#include "lm.hpp"

namespace fcv {
namespace lm {
namespace {

constexpr int kThreads = 256;

template <class E>
__device__ __forceinline__ void load8(const void* w, bool f32, int i, float (&out)[8]) {
  if (f32) {
    const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(w) + i);
    const f32x4 lo = p[0], hi = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      out[e] = lo[e];
      out[e + 4] = hi[e];
    }
  } else {
    const s16x8 v = *reinterpret_cast<const s16x8*>(static_cast<const short*>(w) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = E::to_f32(v[e]);
  }
}

// Sum of squares of a head, whose L lanes have 16 elements each.
template <int L>
__device__ __forceinline__ float squares(const float (&a)[8], const float (&b)[8]) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
  ss += dpp_f<0xB1>(ss);                  // lanes 1 apart, then 2
  ss += dpp_f<0x4E>(ss);
  if constexpr (L == 8) ss += dpp_f<0x141>(ss);  // the other four of eight
  return ss;
}

// heads_inv: 2^32 / heads, rounded up.
template <class E, int D>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(const FcvLmQkNormRope p, uint32_t total,
                                                                uint32_t heads_inv) {
  constexpr int L = D / 16;  // lanes of a head
  const uint32_t heads = p.n_heads + 2 * p.n_kv_heads;
  const uint32_t unit = (blockIdx.x * (uint32_t)kThreads + threadIdx.x) / L;
  const int j = threadIdx.x % L;
  if (unit >= total) return;  // whole heads: lanes that sum together leave together
  // unit / heads: the product is at most one too large
  uint32_t token = __umulhi(unit, heads_inv);
  if (token * heads > unit) --token;
  const int head = (int)(unit - token * heads);

  const bool is_q = head < p.n_heads, is_v = head >= p.n_heads + p.n_kv_heads;
  const int half_chunks = p.rope_dim / 16;  // chunks of half the rotated part
  const bool turned = j < half_chunks;
  const int c0 = turned ? j : 2 * j, c1 = turned ? j + half_chunks : 2 * j + 1;

  const short* src =
      static_cast<const short*>(p.qkv) + (int64_t)token * p.qkv_row + (int64_t)head * D;
  s16x8 x0 = *reinterpret_cast<const s16x8*>(src + c0 * 8);
  s16x8 x1 = *reinterpret_cast<const s16x8*>(src + c1 * 8);

  short* dst;
  bool store = true;
  if (is_q) {
    dst = static_cast<short*>(p.q_out) + (int64_t)token * p.q_row + (int64_t)head * D;
  } else {
    const int32_t row = p.cache_rows[token];
    store = row >= 0 && (int64_t)row < (int64_t)p.sessions * p.capacity;
    const uint32_t r = store ? (uint32_t)row : 0;
    const uint32_t session = p.sessions == 1 ? 0 : r / (uint32_t)p.capacity;
    const uint32_t at = r - session * (uint32_t)p.capacity;
    const int h = head - p.n_heads - (is_v ? p.n_kv_heads : 0);
    dst = is_v ? static_cast<short*>(p.v_cache) + session * p.v_session + at * p.v_row + h * p.v_head
               : static_cast<short*>(p.k_cache) + session * p.k_session + at * p.k_row + h * p.k_head;
  }

  if (!is_v) {
    // the table's entries of both chunks: four pairs each of 2 i, 2 i + 1, or the same eight of i, i + R / 2
    float cs[8], sn[8];
    if (turned) {
      const int pos = min(max(p.positions[token], 0), p.max_pos - 1);
      const int64_t row = (int64_t)pos * (p.rope_dim / 2);
      const int i0 = p.interleaved ? c0 * 4 : c0 * 8, i1 = p.interleaved ? c1 * 4 : c0 * 8 + 4;
      const f32x4 ca = *reinterpret_cast<const f32x4*>(p.rope_cos + row + i0);
      const f32x4 cb = *reinterpret_cast<const f32x4*>(p.rope_cos + row + i1);
      const f32x4 sa = *reinterpret_cast<const f32x4*>(p.rope_sin + row + i0);
      const f32x4 sb = *reinterpret_cast<const f32x4*>(p.rope_sin + row + i1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cs[e] = ca[e];
        cs[e + 4] = cb[e];
        sn[e] = sa[e];
        sn[e + 4] = sb[e];
      }
    }
    float a[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[e] = E::to_f32(x0[e]);
      b[e] = E::to_f32(x1[e]);
    }
    const void* w = is_q ? p.q_weight : p.k_weight;
    if (w) {
      float mean = fmaf(squares<L>(a, b), 1.0f / D, p.eps);
      if (mean > 0x1p100f || mean < 0x1p-60f) {
        // The squares of bf16's largest values pass fp32 and those of its smallest vanish: x s has the norm
        // of x where eps is eps s^2.  Seldom runs.
        const float s = mean > 1.0f ? 0x1p-70f : 0x1p70f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] *= s;
          b[e] *= s;
        }
        mean = fmaf(squares<L>(a, b), 1.0f / D, p.eps * s * s);
      }
      const float inv = 1.0f / sqrtf(mean);
      const bool wf = p.weight_dtype == FCV_LM_F32;
      float wa[8], wb[8];
      load8<E>(w, wf, c0 * 8, wa);
      load8<E>(w, wf, c1 * 8, wb);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a[e] *= inv * wa[e];
        b[e] *= inv * wb[e];
      }
    }
    if (turned) {
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float u0 = a[e], u1 = a[e + 1], v0 = b[e], v1 = b[e + 1];
          a[e] = fmaf(u0, cs[e / 2], -(u1 * sn[e / 2]));
          a[e + 1] = fmaf(u1, cs[e / 2], u0 * sn[e / 2]);
          b[e] = fmaf(v0, cs[4 + e / 2], -(v1 * sn[4 + e / 2]));
          b[e + 1] = fmaf(v1, cs[4 + e / 2], v0 * sn[4 + e / 2]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = a[e], v = b[e];
          a[e] = fmaf(u, cs[e], -(v * sn[e]));
          b[e] = fmaf(v, cs[e], u * sn[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x0[e] = E::from_f32(a[e]);
      x1[e] = E::from_f32(b[e]);
    }
  }
  if (store) {
    *reinterpret_cast<s16x8*>(dst + c0 * 8) = x0;
    *reinterpret_cast<s16x8*>(dst + c1 * 8) = x1;
  }
}

int check(const FcvLmQkNormRope* p) {
  FCV_CHECK(p, FCV_ERR_INVALID, "null arguments");
  FCV_CHECK(p->dtype == FCV_LM_F16 || p->dtype == FCV_LM_BF16, FCV_ERR_INVALID,
            "dtype must be FCV_LM_F16 or FCV_LM_BF16");
  FCV_CHECK(p->head_dim == 64 || p->head_dim == 128, FCV_ERR_INVALID, "head_dim must be 64 or 128");
  FCV_CHECK(p->tokens >= 0 && p->n_heads >= 1 && p->n_kv_heads >= 1 && p->n_heads <= 4096 &&
                p->n_kv_heads <= 4096,
            FCV_ERR_INVALID, "need tokens >= 0 and 1 to 4096 query and key heads");
  FCV_CHECK((int64_t)p->tokens * (p->n_heads + 2 * p->n_kv_heads) < (1LL << 28), FCV_ERR_INVALID,
            "too many tokens: tokens * heads must stay below 2^28");
  FCV_CHECK(p->rope_dim >= 16 && p->rope_dim <= p->head_dim && p->rope_dim % 16 == 0,
            FCV_ERR_INVALID, "rope_dim must be a multiple of 16 from 16 to head_dim");
  FCV_CHECK(p->max_pos >= 1, FCV_ERR_INVALID, "the rotation tables are empty");
  FCV_CHECK(p->sessions >= 1 && p->capacity >= 1 &&
                (int64_t)p->sessions * p->capacity <= 0x7fffffffLL,
            FCV_ERR_INVALID, "sessions * capacity must be in [1, 2^31)");
  FCV_CHECK((p->q_weight == nullptr) == (p->k_weight == nullptr), FCV_ERR_INVALID,
            "q_weight and k_weight come together");
  FCV_CHECK(p->weight_dtype == p->dtype || p->weight_dtype == FCV_LM_F32, FCV_ERR_INVALID,
            "weight_dtype must be dtype or FCV_LM_F32");
  FCV_CHECK(p->eps >= 0.0f && p->eps < __builtin_inff(), FCV_ERR_INVALID, "eps must be finite and >= 0");
  if (p->tokens == 0) return FCV_OK;
  FCV_CHECK(p->qkv && p->positions && p->cache_rows && p->rope_cos && p->rope_sin && p->q_out &&
                p->k_cache && p->v_cache,
            FCV_ERR_INVALID, "null argument");
  FCV_CHECK(aligned(p->qkv, 16) && aligned(p->q_out, 16) && aligned(p->k_cache, 16) &&
                aligned(p->v_cache, 16) && aligned(p->rope_cos, 16) && aligned(p->rope_sin, 16) &&
                aligned(p->q_weight, 16) && aligned(p->k_weight, 16),
            FCV_ERR_INVALID,
            "qkv, q_out, the caches, the tables and the weights must start on 16-byte boundaries");
  const int64_t strides[][2] = {{p->qkv_row, p->tokens},     {p->q_row, p->tokens},
                                {p->k_session, p->sessions}, {p->k_row, p->capacity},
                                {p->k_head, p->n_kv_heads},  {p->v_session, p->sessions},
                                {p->v_row, p->capacity},     {p->v_head, p->n_kv_heads}};
  for (const auto& v : strides) {
    FCV_CHECK(v[1] <= 1 || v[0] >= 0, FCV_ERR_INVALID, "negative stride");
    FCV_CHECK(stride_fits(v[0], v[1]), FCV_ERR_INVALID, "strides must be multiples of 8 elements");
  }
  FCV_CHECK(p->tokens == 1 || p->q_row >= (int64_t)p->n_heads * p->head_dim, FCV_ERR_INVALID,
            "rows of q_out overlap");
  return FCV_OK;
}

template <class E>
void launch(const FcvLmQkNormRope& p, hipStream_t stream) {
  const uint32_t total = (uint32_t)p.tokens * (uint32_t)(p.n_heads + 2 * p.n_kv_heads);
  const uint32_t heads = p.n_heads + 2 * p.n_kv_heads;
  const uint32_t heads_inv = (uint32_t)(((1ULL << 32) + heads - 1) / heads);
  const uint32_t per_block = kThreads * 16 / p.head_dim;
  const dim3 grid((total + per_block - 1) / per_block);
  if (p.head_dim == 64)
    hipLaunchKernelGGL((qk_norm_rope_kernel<E, 64>), grid, dim3(kThreads), 0, stream, p, total,
                       heads_inv);
  else
    hipLaunchKernelGGL((qk_norm_rope_kernel<E, 128>), grid, dim3(kThreads), 0, stream, p, total,
                       heads_inv);
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" int fcv_lm_qk_norm_rope(const FcvLmQkNormRope* args, hipStream_t stream) {
  if (int rc = fcv::lm::check(args)) return rc;
  if (args->tokens == 0) return FCV_OK;
  if (args->dtype == FCV_LM_F16)
    fcv::lm::launch<fcv::lm::Half>(*args, stream);
  else
    fcv::lm::launch<fcv::lm::Bf16>(*args, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}
