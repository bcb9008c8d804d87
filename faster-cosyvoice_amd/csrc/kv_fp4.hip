// Norms of queries and keys per head, the position rotation and the append of keys and values to a cache
// of 4-bit pages, in one pass; and the pages' tokens read back as 16-bit numbers.
//
// Per head x of D elements:  y = x / sqrt(mean(x^2) + eps) * w;  the first R elements are rotated in pairs,
// (a, b) -> (a cos - b sin, b cos + a sin).  Queries are rounded to 16 bits once; keys go to 4 bits in
// groups of 32, values of a head in one group.  Keys are computed in 64 bits: one next to the border of two
// codes, whose step is a third of it, goes where the formula puts it.
//
// Bound: bandwidth (each element is read once and written once), or the launch itself for a few tokens.
// Split: a head takes D / 16 lanes with two chunks of 8 each (rope.hpp), so that nothing is exchanged but the
// head's sum of squares and its groups' largest magnitudes.  A workgroup has heads of one kind; of keys and
// values a wave has 8 neighbouring tokens of a head, whose bytes lie side by side in a page.
#include "fp4.hpp"
#include "rope.hpp"

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

// Keys and values are dealt out 8 tokens of a head at a time: unit -> (token, head).
constexpr int kTokens = 8;
struct Unit {
  uint32_t token;
  int head;
};
__device__ __forceinline__ Unit unit_of(uint32_t u, uint32_t heads) {
  const uint32_t v = u / kTokens, block = v / heads;
  return Unit{block * kTokens + u % kTokens, (int)(v - block * heads)};
}
int64_t units_of(int64_t tokens, int64_t heads) { return (tokens + kTokens - 1) / kTokens * kTokens * heads; }

// Workgroups of keys, of values, then of queries.
struct AppendArgs {
  FcvFp4Append p;
  uint32_t kv_blocks;  // of the keys, and of the values
};

template <class E, int D>
__global__ __launch_bounds__(kThreads) void append_fp4_kernel(const AppendArgs a) {
  constexpr int L = D / 16, kHeads = kThreads / L, kChunks = D / 8;
  constexpr bool kHalf = std::is_same<E, Half>::value;
  using P = Page<D>;
  __shared__ __attribute__((aligned(16))) uint32_t tops[kHeads][kChunks];
  const FcvFp4Append& p = a.p;
  const int j = threadIdx.x % L, local = threadIdx.x / L;
  const int half_chunks = p.rope_dim / 16;  // chunks of half the rotated part
  const bool turned = j < half_chunks;
  const int c0 = turned ? j : 2 * j, c1 = turned ? j + half_chunks : 2 * j + 1;

  if (blockIdx.x >= 2 * a.kv_blocks) {
    const uint32_t unit = (blockIdx.x - 2 * a.kv_blocks) * kHeads + local;
    if (unit >= (uint32_t)p.tokens * (uint32_t)p.n_heads) return;  // whole heads leave together
    const uint32_t token = unit / (uint32_t)p.n_heads, h = unit - token * (uint32_t)p.n_heads;
    const short* src = static_cast<const short*>(p.qkv) + (int64_t)token * p.qkv_row + (int64_t)h * D;
    s16x8 x0 = *reinterpret_cast<const s16x8*>(src + c0 * 8);
    s16x8 x1 = *reinterpret_cast<const s16x8*>(src + c1 * 8);
    norm_rotate<E, D>(p, token, p.q_weight, turned, c0, c1, x0, x1);
    short* to = static_cast<short*>(p.q_out) + (int64_t)token * p.q_row + (int64_t)h * D;
    *reinterpret_cast<s16x8*>(to + c0 * 8) = x0;
    *reinterpret_cast<s16x8*>(to + c1 * 8) = x1;
    return;
  }

  const bool is_v = blockIdx.x >= a.kv_blocks;
  const Unit u = unit_of((blockIdx.x - (is_v ? a.kv_blocks : 0)) * kHeads + local, p.n_kv_heads);
  if (u.token >= (uint32_t)p.tokens) return;
  const int32_t row = p.cache_rows[u.token];
  if (row < 0 || row / P::kTokens >= p.n_pages) return;
  uint8_t* page = p.pages + (int64_t)(row / P::kTokens) * p.page_stride + (int64_t)u.head * p.head_stride;
  const int place = row % P::kTokens;
  const short* head = static_cast<const short*>(p.qkv) + (int64_t)u.token * p.qkv_row +
                      (int64_t)(p.n_heads + (is_v ? p.n_kv_heads : 0) + u.head) * D;

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
    uint8_t* to = page + P::kValues + 8 * j * P::kTokens + place;
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e * P::kTokens] = (uint8_t)(c[e / 4] >> (8 * (e % 4)));
    if (j == 0) page[P::kValueScales + place] = (uint8_t)b;
    return;
  }

  const s16x8 x0 = *reinterpret_cast<const s16x8*>(head + c0 * 8);
  const s16x8 x1 = *reinterpret_cast<const s16x8*>(head + c1 * 8);
  double k0[8], k1[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    k0[e] = E::to_f32(x0[e]);
    k1[e] = E::to_f32(x1[e]);
  }
  if (p.k_weight) {
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fma(k0[e], k0[e], fma(k1[e], k1[e], ss));
    ss += dpp_d<0xB1>(ss);
    ss += dpp_d<0x4E>(ss);
    if constexpr (L == 8) ss += dpp_d<0x141>(ss);
    const double inv = 1.0 / sqrt(ss / D + (double)p.eps);
    const bool wf = p.weight_dtype == FCV_LM_F32;
    float w0[8], w1[8];
    load8<E>(p.k_weight, wf, c0 * 8, w0);
    load8<E>(p.k_weight, wf, c1 * 8, w1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      k0[e] *= inv * (double)w0[e];
      k1[e] *= inv * (double)w1[e];
    }
  }
  if (turned) {
    const int pos = min(max(p.positions[u.token], 0), p.max_pos - 1);
    const float* cos_row = p.rope_cos + (int64_t)pos * (p.rope_dim / 2);
    const float* sin_row = p.rope_sin + (int64_t)pos * (p.rope_dim / 2);
    if (p.interleaved) {
      auto turn = [&](double (&k)[8], int c) {
        const f32x4 cs = *reinterpret_cast<const f32x4*>(cos_row + c * 4);
        const f32x4 sn = *reinterpret_cast<const f32x4*>(sin_row + c * 4);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const double x = k[e], y = k[e + 1], cd = cs[e / 2], sd = sn[e / 2];
          k[e] = fma(x, cd, -(y * sd));
          k[e + 1] = fma(y, cd, x * sd);
        }
      };
      turn(k0, c0);
      turn(k1, c1);
    } else {
#pragma unroll
      for (int q = 0; q < 8; q += 4) {
        const f32x4 cs = *reinterpret_cast<const f32x4*>(cos_row + c0 * 8 + q);
        const f32x4 sn = *reinterpret_cast<const f32x4*>(sin_row + c0 * 8 + q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const double x = k0[q + e], y = k1[q + e], cd = cs[e], sd = sn[e];
          k0[q + e] = fma(x, cd, -(y * sd));
          k1[q + e] = fma(y, cd, x * sd);
        }
      }
    }
  }
  float y0[8], y1[8];
  uint32_t t0 = 0, t1 = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y0[e] = to_odd(k0[e]);
    y1[e] = to_odd(k1[e]);
    t0 = max(t0, __float_as_uint(y0[e]) & 0x7fffffffu);
    t1 = max(t1, __float_as_uint(y1[e]) & 0x7fffffffu);
  }
  // a group's four chunks may be in any lanes of the head
  tops[local][c0] = t0;
  tops[local][c1] = t1;
  wave_fence();
  auto store = [&](const float (&y)[8], int c) {
    const u32x4 t = *reinterpret_cast<const u32x4*>(&tops[local][c & ~3]);
    const uint32_t b = fp4_scale_byte(max(max(t[0], t[1]), max(t[2], t[3])), kHalf);
    *reinterpret_cast<uint32_t*>(page + place * P::kKey + 4 * c) = b == 255 ? 0 : fp4_word(y, scale_of(b));
    if (c % 4 == 0) page[P::kScales + place * P::kKeyScales + c / 4] = (uint8_t)b;
  };
  store(y0, c0);
  store(y1, c1);
}

// A thread has 16 elements of a token's key head or value head.
template <class E, int D>
__global__ __launch_bounds__(kThreads) void read_fp4_kernel(const FcvFp4Read p, uint32_t blocks) {
  constexpr int L = D / 16, kHeads = kThreads / L;
  using P = Page<D>;
  const int j = threadIdx.x % L;
  const bool is_v = blockIdx.x >= blocks;
  const Unit u = unit_of((blockIdx.x - (is_v ? blocks : 0)) * kHeads + threadIdx.x / L, p.n_kv_heads);
  if (u.token >= (uint32_t)p.tokens) return;
  const int32_t row = p.rows[u.token];
  s16x8 r[2] = {};
  if (row >= 0 && row / P::kTokens < p.n_pages) {
    const uint8_t* page =
        p.pages + (int64_t)(row / P::kTokens) * p.page_stride + (int64_t)u.head * p.head_stride;
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
  short* to = static_cast<short*>(is_v ? p.v : p.k) + (int64_t)u.token * (is_v ? p.v_row : p.k_row) +
              (int64_t)u.head * D + 16 * j;
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

uint32_t blocks_of(int64_t units, int head_dim) {
  const int heads = kThreads * 16 / head_dim;
  return (uint32_t)((units + heads - 1) / heads);
}

template <class E>
void launch(const FcvFp4Append& p, hipStream_t stream) {
  const AppendArgs a{p, blocks_of(units_of(p.tokens, p.n_kv_heads), p.head_dim)};
  const dim3 grid(2 * a.kv_blocks + blocks_of((int64_t)p.tokens * p.n_heads, p.head_dim));
  if (p.head_dim == 64)
    hipLaunchKernelGGL((append_fp4_kernel<E, 64>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((append_fp4_kernel<E, 128>), grid, dim3(kThreads), 0, stream, a);
}

template <class E>
void launch(const FcvFp4Read& p, hipStream_t stream) {
  const uint32_t blocks = blocks_of(units_of(p.tokens, p.n_kv_heads), p.head_dim);
  if (p.head_dim == 64)
    hipLaunchKernelGGL((read_fp4_kernel<E, 64>), dim3(2 * blocks), dim3(kThreads), 0, stream, p, blocks);
  else
    hipLaunchKernelGGL((read_fp4_kernel<E, 128>), dim3(2 * blocks), dim3(kThreads), 0, stream, p, blocks);
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
