// Causal attention of a batch over a cache of 4-bit pages.
//
//   s = scale q.k,  out = sum exp(s) v / sum exp(s)  over a query's visible keys, in one pass: a wave keeps
// the running maximum m of its rows and sums of 2^(s - m) and of 2^(s - m) v, in fp32.
//
// A page of 64 tokens is a tile.  v_mfma_f32_16x16x32 computes S^T = K Q^T (16 keys, 16 rows of queries: the
// heads that share a key head, token after token) and O^T += V^T P.  Codes become 16-bit numbers in
// registers, the keys' scales with them.  The order of a tile's keys is chosen so that nothing moves between
// lanes: key 16 c + 4 t + j is row 4 c + j of the t-th S^T tile, so lane block c holds the weights of keys
// 16 c .. 16 c + 15, and as the right operand of the second product lane block c wants 8 of those at a time.
// The values lie in the page as the left operand wants them, bytes of 16 neighbouring keys; a byte's two
// numbers are two elements of one token, so two conversions and two byte permutations give a pair of keys
// of either element.
//
// A value's scale goes into its weight, in fp32; the weight then goes in as two bf16 numbers, its rounding
// and the rest's (16 bits of the weight), so the result's error is its own rounding.
#include <algorithm>
#include <string>

#include "fp4.hpp"

namespace fcv {
namespace lm {
namespace {

constexpr int kPage = FCV_FP4_PAGE;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// bf16's weights times values are held at 2^-24 times their size: sums of 2^24 of its largest values do not
// pass fp32's.
template <class E>
constexpr float kHeld = std::is_same<E, Bf16>::value ? 0x1p-24f : 1.0f;

struct AttendArgs {
  FcvFp4Attention p;
  int group;                 // query heads of a key head
  int row_tiles;             // tiles of 16 rows of a sequence's longest query range
  int splits, pages_per;     // ranges of keys, and the pages of one
  float* part;               // [splits][tokens][n_heads][D]
  float* part_ml;            // [splits][tokens][n_heads][2]
};

__device__ __forceinline__ float across_max(float v) {  // over the lane blocks l / 16
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float across_sum(float v) { return swap32_sum(swap16_sum(v)); }

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
}

// What a lane reads of a page.
template <int D>
struct Raw {
  static constexpr int kU = D / 32;  // tiles of 16 byte rows of the values
  uint32_t k[4][D / 32];             // 4 tiles: the lane's D / 4 codes of its key
  uint32_t ks[4];
  u32x4 v[kU];
  u32x4 vs;
};

template <class E, int D>
__global__ __launch_bounds__(256, 2) void attend_fp4_kernel(const AttendArgs a) {
  using P = Page<D>;
  constexpr int kWaves = 4, kU = D / 32, kJ = D / 32;  // value tiles; steps of 32 of the first product
  __shared__ __attribute__((aligned(16))) float so[kWaves - 1][16][D + 4];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  const FcvFp4Attention& p = a.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, blk = lane >> 4;
  int b, first, n;  // the sequence, its first row of q, its queries
  const int kv = blockIdx.x % p.n_kv_heads, tile = blockIdx.x / p.n_kv_heads % a.row_tiles;
  b = blockIdx.x / p.n_kv_heads / a.row_tiles;
  if (p.cu_q) {
    first = min(max(p.cu_q[b], 0), p.tokens);
    n = min(max(p.cu_q[b + 1], first), p.tokens) - first;
  } else {
    n = p.tokens / p.batch;
    first = b * n;
  }
  const int64_t rows = (int64_t)n * a.group;
  const int length = min(max(p.lengths[b], 0), (int)min((int64_t)p.max_pages * kPage, (int64_t)0x7fffffff));
  const int32_t* table = p.table + (int64_t)b * p.table_row;
  const uint8_t* pool = p.pages + (int64_t)kv * p.head_stride;

  // a batch whose sequence has more rows than max_q said: the tiles take turns
  for (int64_t row0 = (int64_t)tile * 16; row0 < rows; row0 += (int64_t)a.row_tiles * 16) {
    const int64_t row = row0 + col;
    const bool there = row < rows;
    const int token = (int)(min(row, rows - 1) / a.group);
    const int head = kv * a.group + (int)(min(row, rows - 1) % a.group);
    const int limit = there ? length - n + token + 1 : 0;  // the row's visible keys
    const int last_token = (int)(min(row0 + 15, rows - 1) / a.group);
    const int reach = min(max(length - n + last_token + 1, 0), length);  // of the whole tile
    const int all_pages = (reach + kPage - 1) / kPage;
    int page0 = blockIdx.y * a.pages_per, page1 = min(page0 + a.pages_per, all_pages);
    if (blockIdx.y == (unsigned)a.splits - 1) page1 = all_pages;  // and what max_length left out

    s16x8 fq[kJ];
    {
      const short* q = static_cast<const short*>(p.q) + (int64_t)(first + token) * p.q_row +
                       (int64_t)head * p.q_head + blk * (D / 4);
#pragma unroll
      for (int j = 0; j < kJ; ++j) fq[j] = *reinterpret_cast<const s16x8*>(q + 8 * j);
    }
    const float scale = p.scale * kLog2e;
    f32x4 o[kU][2];
#pragma unroll
    for (int u = 0; u < kU; ++u)
      for (int h = 0; h < 2; ++h) o[u][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -__builtin_inff(), l = 0.0f;

    for (int page = page0 + wave; page < page1; page += kWaves) {
      int id = table[page];
      const bool good = id >= 0 && id < p.n_pages;
      if (!good) continue;
      const uint8_t* at = pool + (int64_t)id * p.page_stride;
      Raw<D> r;
      const int key0 = 16 * (col >> 2) + (col & 3);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int key = key0 + 4 * t;
        if constexpr (D == 128) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(at + key * P::kKey + blk * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) r.k[t][j] = w[j];
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2*>(at + key * P::kKey + blk * 8);
          r.k[t][0] = w[0];
          r.k[t][1] = w[1];
        }
        r.ks[t] = at[P::kScales + key * P::kKeyScales + (D == 128 ? blk : blk >> 1)];
      }
#pragma unroll
      for (int u = 0; u < kU; ++u)
        r.v[u] = *reinterpret_cast<const u32x4*>(at + P::kValues + (16 * u + col) * kPage + 16 * blk);
      r.vs = *reinterpret_cast<const u32x4*>(at + P::kValueScales + 16 * blk);

      f32x4 s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const float ks = scale_of(r.ks[t]);
#pragma unroll
        for (int j = 0; j < kJ; ++j) s[t] = E::mfma16(fp4_octet<E>(r.k[t][j], ks), fq[j], s[t]);
      }
      const int seen = limit - page * kPage - 16 * blk;  // the lane's visible keys of its 16
      float top = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[t][j] = 4 * t + j < seen ? s[t][j] * scale : -__builtin_inff();
          top = fmaxf(top, s[t][j]);
        }
      top = across_max(top);
      const float next = fmaxf(m, top);
      const float base = next == -__builtin_inff() ? 0.0f : next;
      const float alpha = hw_exp2(m - base);  // 0 before the first visible key
      m = next;
      l *= alpha;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        o[u][0] *= alpha;
        o[u][1] *= alpha;
      }
      uint32_t hi[2][4], lo[2][4];  // the weights of keys 8 s .. 8 s + 7 of the lane's 16
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float w[4], rest[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool vis = 4 * t + j < seen;
          const float e = vis ? hw_exp2(s[t][j] - base) : 0.0f;
          l += e;
          w[j] = vis ? e * kHeld<E> * scale_of((r.vs[t] >> (8 * j)) & 255) : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const uint32_t u = bf16_pair(w[j], w[j + 1]);
          rest[j] = w[j] - __uint_as_float(u << 16);
          rest[j + 1] = w[j + 1] - __uint_as_float(u & 0xffff0000u);
          hi[t >> 1][(t & 1) * 2 + j / 2] = u;
          lo[t >> 1][(t & 1) * 2 + j / 2] = bf16_pair(rest[j], rest[j + 1]);
        }
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const s16x8 ph = __builtin_bit_cast(s16x8, u32x4{hi[st][0], hi[st][1], hi[st][2], hi[st][3]});
        const s16x8 pl = __builtin_bit_cast(s16x8, u32x4{lo[st][0], lo[st][1], lo[st][2], lo[st][3]});
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          u32x4 even, odd;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w = r.v[u][2 * st + i];
            const uint32_t x0 = fp4_pair<Bf16, 0>(w, 1.0f), x1 = fp4_pair<Bf16, 1>(w, 1.0f);
            const uint32_t x2 = fp4_pair<Bf16, 2>(w, 1.0f), x3 = fp4_pair<Bf16, 3>(w, 1.0f);
            even[2 * i] = __builtin_amdgcn_perm(x1, x0, 0x05040100);
            even[2 * i + 1] = __builtin_amdgcn_perm(x3, x2, 0x05040100);
            odd[2 * i] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
            odd[2 * i + 1] = __builtin_amdgcn_perm(x3, x2, 0x07060302);
          }
          const s16x8 ve = __builtin_bit_cast(s16x8, even), vo = __builtin_bit_cast(s16x8, odd);
          o[u][0] = Bf16::mfma16(ve, ph, o[u][0]);
          o[u][1] = Bf16::mfma16(vo, ph, o[u][1]);
          o[u][0] = Bf16::mfma16(ve, pl, o[u][0]);
          o[u][1] = Bf16::mfma16(vo, pl, o[u][1]);
        }
      }
    }

    // the waves' sums, in their order
    l = across_sum(l);
    if (blk == 0) {
      sm[wave][col] = m;
      sl[wave][col] = l;
    }
    if (wave > 0) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float* to = &so[wave - 1][col][32 * u + 8 * blk];
        *reinterpret_cast<f32x4*>(to) = f32x4{o[u][0][0], o[u][1][0], o[u][0][1], o[u][1][1]};
        *reinterpret_cast<f32x4*>(to + 4) = f32x4{o[u][0][2], o[u][1][2], o[u][0][3], o[u][1][3]};
      }
    }
    __syncthreads();
    if (wave == 0) {
      float top = m;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w][col]);
      const float base = top == -__builtin_inff() ? 0.0f : top;
      const float f0 = hw_exp2(m - base);
      l *= f0;
      f32x4 r[kU][2];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        r[u][0] = f32x4{o[u][0][0], o[u][1][0], o[u][0][1], o[u][1][1]} * f0;
        r[u][1] = f32x4{o[u][0][2], o[u][1][2], o[u][0][3], o[u][1][3]} * f0;
      }
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        const float f = hw_exp2(sm[w][col] - base);
        l += sl[w][col] * f;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const float* from = &so[w - 1][col][32 * u + 8 * blk];
          r[u][0] += *reinterpret_cast<const f32x4*>(from) * f;
          r[u][1] += *reinterpret_cast<const f32x4*>(from + 4) * f;
        }
      }
      if (there) {
        const int64_t at = (int64_t)(first + token) * p.n_heads + head;
        if (a.splits > 1) {
          const int64_t i = (int64_t)blockIdx.y * p.tokens * p.n_heads + at;
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            float* to = a.part + i * D + 32 * u + 8 * blk;
            *reinterpret_cast<f32x4*>(to) = r[u][0];
            *reinterpret_cast<f32x4*>(to + 4) = r[u][1];
          }
          if (blk == 0) {
            a.part_ml[2 * i] = top;
            a.part_ml[2 * i + 1] = l;
          }
        } else {
          // a query that sees no key: 0.  A sum of 0 otherwise has NaN weights.
          const float inv = l == 0.0f ? 0.0f : 1.0f / (l * kHeld<E>);
          short* to = static_cast<short*>(p.out) + (int64_t)(first + token) * p.out_row +
                      (int64_t)head * p.out_head + 8 * blk;
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            s16x8 v;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = E::from_f32(r[u][e / 4][e % 4] * inv);
            *reinterpret_cast<s16x8*>(to + 32 * u) = v;
          }
          if (p.lse && blk == 0) p.lse[at] = (top + __builtin_amdgcn_logf(l)) * kLn2;
        }
      }
    }
    __syncthreads();
  }
}

// The ranges' sums, in their order.  A thread has 8 elements of a row's head.
template <class E, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(const AttendArgs a) {
  const FcvFp4Attention& p = a.p;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / (D / 8);
  const int d = threadIdx.x % (D / 8) * 8;
  const int64_t n = (int64_t)p.tokens * p.n_heads;
  if (i >= n) return;
  const int token = (int)(i / p.n_heads), head = (int)(i % p.n_heads);
  if (p.cu_q && token >= p.cu_q[p.batch]) return;  // behind the last sequence
  float top = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_ml[2 * (s * n + i)]);
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float l = 0.0f;
  f32x4 r0 = {0.0f, 0.0f, 0.0f, 0.0f}, r1 = r0;
  for (int s = 0; s < a.splits; ++s) {
    const float f = hw_exp2(a.part_ml[2 * (s * n + i)] - base);
    l += a.part_ml[2 * (s * n + i) + 1] * f;
    const float* from = a.part + (s * n + i) * D + d;
    r0 += *reinterpret_cast<const f32x4*>(from) * f;
    r1 += *reinterpret_cast<const f32x4*>(from + 4) * f;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / (l * kHeld<E>);
  s16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = E::from_f32((e < 4 ? r0[e % 4] : r1[e % 4]) * inv);
  *reinterpret_cast<s16x8*>(static_cast<short*>(p.out) + (int64_t)token * p.out_row +
                            (int64_t)head * p.out_head + d) = v;
  if (p.lse && d == 0) p.lse[i] = (top + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---- host ---------------------------------------------------------------------------------------

int check(const FcvFp4Attention* p) {
  FCV_CHECK(p, FCV_ERR_INVALID, "null arguments");
  FCV_CHECK(p->dtype == FCV_LM_F16 || p->dtype == FCV_LM_BF16, FCV_ERR_INVALID,
            "dtype must be FCV_LM_F16 or FCV_LM_BF16");
  FCV_CHECK(p->head_dim == 64 || p->head_dim == 128, FCV_ERR_INVALID, "head_dim must be 64 or 128");
  FCV_CHECK(p->tokens >= 0 && p->batch >= 1 && p->n_heads >= 1 && p->n_kv_heads >= 1 &&
                p->n_heads % p->n_kv_heads == 0,
            FCV_ERR_INVALID, "need tokens >= 0, batch >= 1 and query heads a multiple of the key heads");
  FCV_CHECK((int64_t)p->tokens * p->n_heads < (1LL << 26), FCV_ERR_INVALID,
            "too many rows: tokens * n_heads must stay below 2^26");
  FCV_CHECK(p->cu_q || p->tokens % p->batch == 0, FCV_ERR_INVALID,
            "without cu_q the rows must divide by the sequences");
  FCV_CHECK(p->n_pages >= 1 && p->n_pages <= (1 << 24), FCV_ERR_INVALID,
            "n_pages must be in [1, 2^24]");
  FCV_CHECK(p->max_pages >= 1 && p->max_pages <= (1 << 24), FCV_ERR_INVALID,
            "max_pages must be in [1, 2^24]");
  FCV_CHECK(p->max_q >= 1 && p->max_length >= 0, FCV_ERR_INVALID, "need max_q >= 1 and max_length >= 0");
  FCV_CHECK(p->scale > 0.0f && p->scale < __builtin_inff(), FCV_ERR_INVALID,
            "scale must be finite and > 0");
  if (p->tokens == 0) return FCV_OK;
  FCV_CHECK(p->q && p->pages && p->table && p->lengths && p->out, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(aligned(p->q, 16) && aligned(p->out, 16), FCV_ERR_INVALID,
            "q and out must start on 16-byte boundaries");
  FCV_CHECK(stride_fits(p->q_row, p->tokens) && stride_fits(p->q_head, p->n_heads) &&
                stride_fits(p->out_row, p->tokens) && stride_fits(p->out_head, p->n_heads),
            FCV_ERR_INVALID, "strides must be multiples of 8 elements, and not negative");
  FCV_CHECK(pages_fit(p->pages, p->page_stride, p->head_stride, p->n_pages, p->n_kv_heads,
                      p->head_dim),
            FCV_ERR_INVALID, "pages must lie on 16-byte boundaries, none over another");
  FCV_CHECK(p->batch == 1 || p->table_row >= 0, FCV_ERR_INVALID, "negative stride");
  return FCV_OK;
}

struct Plan {
  int64_t row_tiles;
  int splits, pages_per;
};

Plan plan_of(const FcvFp4Attention& p) {
  const int group = p.n_heads / p.n_kv_heads;
  const int64_t all = std::max<int64_t>(((int64_t)std::min(p.max_q, p.tokens) * group + 15) / 16, 1);
  // tiles past a launch's size take turns
  const int64_t tiles = std::min(all, std::max<int64_t>(1, (1 << 22) / ((int64_t)p.batch * p.n_kv_heads)));
  const int64_t blocks = tiles * p.batch * p.n_kv_heads;
  const int64_t most = (int64_t)p.max_pages * kPage;
  const int pages = (int)std::max<int64_t>((std::min<int64_t>(p.max_length, most) + kPage - 1) / kPage, 1);
  const int64_t want = std::max<int64_t>(1, 4 * kCus / blocks);
  const int per = (int)std::max<int64_t>((pages + want - 1) / want, 4);
  return Plan{tiles, (pages + per - 1) / per, per};
}

size_t workspace_bytes(const FcvFp4Attention& p, const Plan& plan) {
  return plan.splits > 1 ? (size_t)plan.splits * p.tokens * p.n_heads * (p.head_dim + 2) * 4 : 0;
}

template <class E, int D>
void launch(const AttendArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.row_tiles * a.p.batch * a.p.n_kv_heads), (unsigned)a.splits);
  hipLaunchKernelGGL((attend_fp4_kernel<E, D>), grid, dim3(256), 0, stream, a);
  if (a.splits > 1) {
    const int64_t threads = (int64_t)a.p.tokens * a.p.n_heads * (D / 8);
    hipLaunchKernelGGL((attend_join_kernel<E, D>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0,
                       stream, a);
  }
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" size_t fcv_fp4_attention_workspace_bytes(const FcvFp4Attention* args) {
  if (fcv::lm::check(args) || args->tokens == 0) return 0;
  return fcv::lm::workspace_bytes(*args, fcv::lm::plan_of(*args));
}

extern "C" int fcv_fp4_attention(const FcvFp4Attention* args, void* workspace, size_t workspace_bytes,
                                 hipStream_t stream) {
  using namespace fcv::lm;
  if (int rc = check(args)) return rc;
  if (args->tokens == 0) return FCV_OK;
  const Plan plan = plan_of(*args);
  const size_t need = fcv::lm::workspace_bytes(*args, plan);
  FCV_CHECK(need == 0 || workspace, FCV_ERR_INVALID, "null workspace");
  FCV_CHECK(workspace_bytes >= need, FCV_ERR_INVALID,
            "workspace too small: need " + std::to_string(need) + " bytes");
  FCV_CHECK(need == 0 || aligned(workspace, 256), FCV_ERR_INVALID, "workspace must be 256-byte aligned");
  FCV_CHECK((int64_t)args->batch * args->n_kv_heads <= (1 << 23), FCV_ERR_INVALID,
            "batch * n_kv_heads is limited to 2^23");
  float* part = static_cast<float*>(workspace);
  const AttendArgs a{*args, args->n_heads / args->n_kv_heads, (int)plan.row_tiles, plan.splits,
                     plan.pages_per, part,
                     part ? part + (size_t)plan.splits * args->tokens * args->n_heads * args->head_dim
                          : nullptr};
  if (args->dtype == FCV_LM_F16)
    args->head_dim == 64 ? launch<Half, 64>(a, stream) : launch<Half, 128>(a, stream);
  else
    args->head_dim == 64 ? launch<Bf16, 64>(a, stream) : launch<Bf16, 128>(a, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}
