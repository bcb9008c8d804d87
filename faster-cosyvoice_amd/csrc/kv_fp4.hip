// Norms of queries and keys per head, the position rotation and the append of keys and values to a cache
// of 4-bit pages, in one pass; and the pages' tokens read back as 16-bit numbers.
//
// Per head x of D elements:  y = x / sqrt(mean(x^2) + eps) * w;  the first R elements are rotated in pairs,
// (a, b) -> (a cos - b sin, b cos + a sin).  Queries are rounded to 16 bits once; keys go to 4 bits in
// groups of 32, values of a head in one group.  All of it runs in 64 bits: a value next to the border of
// two codes, whose step is a third of it, goes where the formula puts it, and squares have the room.
//
// Bound: bandwidth (each element is read once and written once), or the launch itself for a few tokens.
// Split: a head takes D / 16 lanes, each with 16 consecutive elements; it reads the chunks that hold the
// other members of its pairs, too (from cache: they are a neighbour's), so that nothing is exchanged but the
// head's sum of squares and the groups' largest magnitudes.
#include "fp4.hpp"

namespace fcv {
namespace lm {
namespace {

constexpr int kThreads = 256;

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, false);
}
template <int kCtrl>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = dpp_u<kCtrl>((uint32_t)u), hi = dpp_u<kCtrl>((uint32_t)(u >> 32));
  return __builtin_bit_cast(double, hi << 32 | lo);
}

// To fp32, to the odd one of the two neighbours: on the same side of every border as the value in 64 bits.
__device__ __forceinline__ float to_odd(double v) {
  const float f = (float)v;
  const double rest = v - (double)f;
  uint32_t u = __float_as_uint(f);
  if ((u & 1) == 0 && (rest > 0.0 || rest < 0.0)) u += (rest > 0.0) == ((u >> 31) == 0) ? 1 : -1;
  return __uint_as_float(u);
}

template <class E>
__device__ __forceinline__ float weight(const void* w, bool f32, int i) {
  return f32 ? static_cast<const float*>(w)[i] : E::to_f32(static_cast<const short*>(w)[i]);
}

// 8 elements from `at` of a head, normed.
template <class E>
__device__ __forceinline__ void normed8(const short* head, int at, const void* w, bool wf, double inv,
                                        double (&out)[8]) {
  const s16x8 v = *reinterpret_cast<const s16x8*>(head + at);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    out[e] = E::to_f32(v[e]);
    if (w) out[e] *= inv * (double)weight<E>(w, wf, at + e);
  }
}

// Heads in order: every token's query heads, then its key heads, then its value heads.
template <class E, int D>
__global__ __launch_bounds__(kThreads) void append_fp4_kernel(const FcvFp4Append p) {
  constexpr int L = D / 16;  // lanes of a head
  constexpr bool kHalf = std::is_same<E, Half>::value;
  using P = Page<D>;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  const int j = threadIdx.x % L;
  const int64_t n_q = (int64_t)p.tokens * p.n_heads, n_kv = (int64_t)p.tokens * p.n_kv_heads;
  if (unit >= n_q + 2 * n_kv) return;  // whole heads: lanes that meet leave together
  const bool is_q = unit < n_q, is_v = unit >= n_q + n_kv;
  const uint32_t local = (uint32_t)(is_q ? unit : is_v ? unit - n_q - n_kv : unit - n_q);
  const uint32_t heads = is_q ? p.n_heads : p.n_kv_heads;
  const uint32_t token = local / heads;
  const int h = (int)(local - token * heads);
  const short* head = static_cast<const short*>(p.qkv) + (int64_t)token * p.qkv_row +
                      (int64_t)(is_q ? h : is_v ? p.n_heads + p.n_kv_heads + h : p.n_heads + h) * D;

  uint8_t* page = nullptr;
  int place = 0;
  if (!is_q) {
    const int32_t row = p.cache_rows[token];
    if (row >= 0 && row / P::kTokens < p.n_pages) {
      page = p.pages + (int64_t)(row / P::kTokens) * p.page_stride + (int64_t)h * p.head_stride;
      place = row % P::kTokens;
    }
  }

  if (is_v) {
    const s16x8 v0 = *reinterpret_cast<const s16x8*>(head + 16 * j);
    const s16x8 v1 = *reinterpret_cast<const s16x8*>(head + 16 * j + 8);
    float v[16];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      v[e] = E::to_f32(e < 8 ? v0[e] : v1[e - 8]);
      top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    top = max(top, dpp_u<0xB1>(top));                          // lanes 1 apart, then 2
    top = max(top, dpp_u<0x4E>(top));
    if constexpr (L == 8) top = max(top, dpp_u<0x141>(top));   // the other four of eight
    const uint32_t b = fp4_scale_byte(top, kHalf);
    uint32_t c[2] = {0, 0};
    if (b != 255) {
      c[0] = fp4_word(v, scale_of(b));
      c[1] = fp4_word(v + 8, scale_of(b));
    }
    if (!page) return;
    uint8_t* to = page + P::kValues + 8 * j * P::kTokens + place;
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e * P::kTokens] = (uint8_t)(c[e / 4] >> (8 * (e % 4)));
    if (j == 0) page[P::kValueScales + place] = (uint8_t)b;
    return;
  }

  const void* w = is_q ? p.q_weight : p.k_weight;
  const bool wf = p.weight_dtype == FCV_LM_F32;
  double inv = 1.0;
  if (w) {
    const s16x8 v0 = *reinterpret_cast<const s16x8*>(head + 16 * j);
    const s16x8 v1 = *reinterpret_cast<const s16x8*>(head + 16 * j + 8);
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double a = E::to_f32(v0[e]), b = E::to_f32(v1[e]);
      ss = fma(a, a, fma(b, b, ss));
    }
    ss += dpp_d<0xB1>(ss);
    ss += dpp_d<0x4E>(ss);
    if constexpr (L == 8) ss += dpp_d<0x141>(ss);
    inv = 1.0 / sqrt(ss / D + (double)p.eps);
  }
  const int pos = min(max(p.positions[token], 0), p.max_pos - 1);
  const float* cos_row = p.rope_cos + (int64_t)pos * (p.rope_dim / 2);
  const float* sin_row = p.rope_sin + (int64_t)pos * (p.rope_dim / 2);
  const int half = p.rope_dim / 2;
  float y[16];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = 16 * j + 8 * i;  // rope_dim / 2 is a multiple of 8: a chunk is on one side of it
    double a[8];
    normed8<E>(head, at, w, wf, inv, a);
    if (at < p.rope_dim) {
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const double c = cos_row[at / 2 + e / 2], s = sin_row[at / 2 + e / 2];
          const double u = a[e], v = a[e + 1];
          a[e] = fma(u, c, -(v * s));
          a[e + 1] = fma(v, c, u * s);
        }
      } else {
        const bool second = at >= half;
        const int t = second ? at - half : at;
        double o[8];
        normed8<E>(head, second ? t : at + half, w, wf, inv, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double c = cos_row[t + e], s = sin_row[t + e];
          a[e] = fma(a[e], c, second ? o[e] * s : -(o[e] * s));
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[8 * i + e] = is_q ? (float)a[e] : to_odd(a[e]);
  }
  if (is_q) {
    short* to = static_cast<short*>(p.q_out) + (int64_t)token * p.q_row + (int64_t)h * D + 16 * j;
    s16x8 r[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) r[e / 8][e % 8] = E::from_f32(y[e]);
    *reinterpret_cast<s16x8*>(to) = r[0];
    *reinterpret_cast<s16x8*>(to + 8) = r[1];
    return;
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(y[e]) & 0x7fffffffu);
  top = max(top, dpp_u<0xB1>(top));
  const uint32_t b = fp4_scale_byte(top, kHalf);
  u32x2 c = {0, 0};
  if (b != 255) {
    c[0] = fp4_word(y, scale_of(b));
    c[1] = fp4_word(y + 8, scale_of(b));
  }
  if (!page) return;
  *reinterpret_cast<u32x2*>(page + place * P::kKey + 8 * j) = c;
  if (j % 2 == 0) page[P::kScales + place * P::kKeyScales + j / 2] = (uint8_t)b;
}

// A thread has 16 elements of a token's key head or value head.
template <class E, int D>
__global__ __launch_bounds__(kThreads) void read_fp4_kernel(const FcvFp4Read p) {
  constexpr int L = D / 16;
  using P = Page<D>;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  const int j = threadIdx.x % L;
  const int64_t n = (int64_t)p.tokens * p.n_kv_heads;
  if (unit >= 2 * n) return;
  const bool is_v = unit >= n;
  const uint32_t local = (uint32_t)(is_v ? unit - n : unit);
  const uint32_t token = local / p.n_kv_heads;
  const int h = (int)(local - token * p.n_kv_heads);
  const int32_t row = p.rows[token];
  s16x8 r[2] = {};
  if (row >= 0 && row / P::kTokens < p.n_pages) {
    const uint8_t* page = p.pages + (int64_t)(row / P::kTokens) * p.page_stride + (int64_t)h * p.head_stride;
    const int place = row % P::kTokens;
    u32x2 c = {0, 0};
    uint32_t b;
    if (is_v) {
      b = page[P::kValueScales + place];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        c[e / 4] |= (uint32_t)page[P::kValues + (8 * j + e) * P::kTokens + place] << (8 * (e % 4));
    } else {
      b = page[P::kScales + place * P::kKeyScales + j / 2];
      c = *reinterpret_cast<const u32x2*>(page + place * P::kKey + 8 * j);
    }
    r[0] = fp4_octet<E>(c[0], scale_of(b));
    r[1] = fp4_octet<E>(c[1], scale_of(b));
  }
  short* to = static_cast<short*>(is_v ? p.v : p.k) + (int64_t)token * (is_v ? p.v_row : p.k_row) +
              (int64_t)h * D + 16 * j;
  *reinterpret_cast<s16x8*>(to) = r[0];
  *reinterpret_cast<s16x8*>(to + 8) = r[1];
}

int check(const FcvFp4Append* p) {
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
  FCV_CHECK(p->n_pages >= 1 && p->n_pages <= (1 << 24), FCV_ERR_INVALID,
            "n_pages must be in [1, 2^24]");
  FCV_CHECK((p->q_weight == nullptr) == (p->k_weight == nullptr), FCV_ERR_INVALID,
            "q_weight and k_weight come together");
  FCV_CHECK(p->weight_dtype == p->dtype || p->weight_dtype == FCV_LM_F32, FCV_ERR_INVALID,
            "weight_dtype must be dtype or FCV_LM_F32");
  FCV_CHECK(p->eps >= 0.0f && p->eps < __builtin_inff(), FCV_ERR_INVALID, "eps must be finite and >= 0");
  if (p->tokens == 0) return FCV_OK;
  FCV_CHECK(p->qkv && p->positions && p->cache_rows && p->rope_cos && p->rope_sin && p->q_out &&
                p->pages,
            FCV_ERR_INVALID, "null argument");
  FCV_CHECK(aligned(p->qkv, 16) && aligned(p->q_out, 16) && aligned(p->rope_cos, 16) &&
                aligned(p->rope_sin, 16) && aligned(p->q_weight, 16) && aligned(p->k_weight, 16),
            FCV_ERR_INVALID, "qkv, q_out, the tables and the weights must start on 16-byte boundaries");
  FCV_CHECK(pages_fit(p->pages, p->page_stride, p->head_stride, p->n_pages, p->n_kv_heads,
                      p->head_dim),
            FCV_ERR_INVALID, "pages must lie on 16-byte boundaries, none over another");
  FCV_CHECK(stride_fits(p->qkv_row, p->tokens) && stride_fits(p->q_row, p->tokens), FCV_ERR_INVALID,
            "row strides must be multiples of 8 elements, and not negative");
  FCV_CHECK(p->tokens == 1 || p->q_row >= (int64_t)p->n_heads * p->head_dim, FCV_ERR_INVALID,
            "rows of q_out overlap");
  return FCV_OK;
}

int check(const FcvFp4Read* p) {
  FCV_CHECK(p, FCV_ERR_INVALID, "null arguments");
  FCV_CHECK(p->dtype == FCV_LM_F16 || p->dtype == FCV_LM_BF16, FCV_ERR_INVALID,
            "dtype must be FCV_LM_F16 or FCV_LM_BF16");
  FCV_CHECK(p->head_dim == 64 || p->head_dim == 128, FCV_ERR_INVALID, "head_dim must be 64 or 128");
  FCV_CHECK(p->tokens >= 0 && p->n_kv_heads >= 1 && p->n_kv_heads <= 4096 &&
                (int64_t)p->tokens * p->n_kv_heads < (1LL << 27),
            FCV_ERR_INVALID, "need tokens >= 0 and 1 to 4096 key heads, tokens * heads below 2^27");
  FCV_CHECK(p->n_pages >= 1 && p->n_pages <= (1 << 24), FCV_ERR_INVALID,
            "n_pages must be in [1, 2^24]");
  if (p->tokens == 0) return FCV_OK;
  FCV_CHECK(p->pages && p->rows && p->k && p->v, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(aligned(p->k, 16) && aligned(p->v, 16) && stride_fits(p->k_row, p->tokens) &&
                stride_fits(p->v_row, p->tokens),
            FCV_ERR_INVALID, "rows of k and v must start on 16-byte boundaries");
  const int64_t width = (int64_t)p->n_kv_heads * p->head_dim;
  FCV_CHECK(p->tokens == 1 || (p->k_row >= width && p->v_row >= width), FCV_ERR_INVALID,
            "rows of k or v overlap");
  FCV_CHECK(pages_fit(p->pages, p->page_stride, p->head_stride, p->n_pages, p->n_kv_heads,
                      p->head_dim),
            FCV_ERR_INVALID, "pages must lie on 16-byte boundaries, none over another");
  return FCV_OK;
}

template <class E>
void launch(const FcvFp4Append& p, hipStream_t stream) {
  const int64_t units = (int64_t)p.tokens * (p.n_heads + 2 * p.n_kv_heads);
  const int per_block = kThreads * 16 / p.head_dim;
  const dim3 grid((unsigned)((units + per_block - 1) / per_block));
  if (p.head_dim == 64)
    hipLaunchKernelGGL((append_fp4_kernel<E, 64>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((append_fp4_kernel<E, 128>), grid, dim3(kThreads), 0, stream, p);
}

template <class E>
void launch(const FcvFp4Read& p, hipStream_t stream) {
  const int64_t units = 2 * (int64_t)p.tokens * p.n_kv_heads;
  const int per_block = kThreads * 16 / p.head_dim;
  const dim3 grid((unsigned)((units + per_block - 1) / per_block));
  if (p.head_dim == 64)
    hipLaunchKernelGGL((read_fp4_kernel<E, 64>), grid, dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((read_fp4_kernel<E, 128>), grid, dim3(kThreads), 0, stream, p);
}

template <class A>
int run(const A* args, hipStream_t stream) {
  if (int rc = check(args)) return rc;
  if (args->tokens == 0) return FCV_OK;
  if (args->dtype == FCV_LM_F16)
    launch<Half>(*args, stream);
  else
    launch<Bf16>(*args, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" size_t fcv_fp4_page_bytes(int32_t head_dim) {
  return head_dim == 64    ? (size_t)fcv::lm::Page<64>::kBytes
         : head_dim == 128 ? (size_t)fcv::lm::Page<128>::kBytes
                           : 0;
}

extern "C" int fcv_fp4_append(const FcvFp4Append* args, hipStream_t stream) {
  return fcv::lm::run(args, stream);
}

extern "C" int fcv_fp4_read(const FcvFp4Read* args, hipStream_t stream) {
  return fcv::lm::run(args, stream);
}
