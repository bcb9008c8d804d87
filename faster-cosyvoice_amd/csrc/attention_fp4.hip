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
// bf16's values are held at 2^-24 times their size: sums of 2^24 of its largest values do not pass fp32's.  What
// that costs are bits of results below 2^-64.
template <class E>
constexpr float kHeld = std::is_same<E, Bf16>::value ? 0x1p-24f : 1.0f;

constexpr int kTileRows = 128;  // of a workgroup of many rows

struct AttendArgs {
  FcvFp4Attention p;
  int group;                 // query heads of a key head
  int each;                  // rows of every sequence without cu_q
  int row_tiles;             // tiles of 16 rows of a sequence's longest query range
  int splits, pages_per;     // ranges of keys, and the pages of one
  int order_shift;           // of sequence_of, or -1: sequences in their order
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

// The sequence of a workgroup's slot: of every kOrdered sequences the one of that rank by falling length (in
// steps of 2^order_shift; equal ones in their order), so that the longest start first and the short ones fill the
// ends.  Every wave selects it for itself, by ballots: the largest key that more than `rank` of the sequences
// reach, then one of those that have it.
constexpr int kOrdered = 1024, kKeyBits = 8;
__device__ __forceinline__ int sequence_of(const AttendArgs& a, int slot) {
  if (a.order_shift < 0) return slot;
  constexpr int kChunks = kOrdered / 64;
  const int lane = threadIdx.x & 63;
  const int first = slot / kOrdered * kOrdered, count = min(a.p.batch - first, kOrdered);
  int rank = slot - first;
  int key[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    key[c] = -1;
    if (64 * c >= count) continue;
    if (64 * c + lane < count)
      key[c] = min(max(a.p.lengths[first + 64 * c + lane], 0) >> a.order_shift, (1 << kKeyBits) - 1);
  }
  auto reach = [&](int k) {  // how many have a key of k or more
    int n = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (64 * c >= count) break;
      n += __popcll(__ballot(key[c] >= k));
    }
    return n;
  };
  int k = 0;
#pragma unroll
  for (int bit = kKeyBits - 1; bit >= 0; --bit)
    if (reach(k | 1 << bit) > rank) k |= 1 << bit;
  rank -= reach(k + 1);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (64 * c >= count) break;
    const uint64_t those = __ballot(key[c] == k);
    const int n = __popcll(those);
    if (rank < n) {
      const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(those >> 32),
                                                  __builtin_amdgcn_mbcnt_lo((uint32_t)those, 0));
      return first + 64 * c + __builtin_ctzll(__ballot(key[c] == k && below == rank));
    }
    rank -= n;
  }
  return slot;
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

// ROWS 8: the tile has 8 rows, each in two columns, so that one product takes the weights' first parts in
// columns 0 .. 7 and their second parts in 8 .. 15.
template <class E, int D, int ROWS>
__global__ __launch_bounds__(256, 2) void attend_fp4_kernel(const AttendArgs a) {
  using P = Page<D>;
  constexpr int kWaves = 4, kU = D / 32, kJ = D / 32;  // value tiles; steps of 32 of the first product
  __shared__ __attribute__((aligned(16))) float so[kWaves - 1][16][D + 4];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  const FcvFp4Attention& p = a.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 15, blk = lane >> 4;
  int b, first, n;  // the sequence, its first row of q, its queries
  const int kv = blockIdx.x % p.n_kv_heads, tile = blockIdx.x / p.n_kv_heads % a.row_tiles;
  b = sequence_of(a, blockIdx.x / p.n_kv_heads / a.row_tiles);
  // What the whole workgroup asks for first, in one go.  Nothing writes it while the kernel runs: scalar loads.
  typedef const int32_t __attribute__((address_space(4))) * Uniform;
  const Uniform table = (Uniform)(uintptr_t)(p.table + (int64_t)b * p.table_row);
  const Uniform ends = (Uniform)(uintptr_t)(p.cu_q ? p.cu_q + b : p.table);
  const int page_first = blockIdx.y * a.pages_per + wave;
  const int id_first = table[min(page_first, p.max_pages - 1)];
  const int id_second = table[min(page_first + kWaves, p.max_pages - 1)];
  const int keys = ((Uniform)(uintptr_t)p.lengths)[b], end0 = ends[0], end1 = ends[p.cu_q ? 1 : 0];
  if (p.cu_q) {
    first = min(max(end0, 0), p.tokens);
    n = min(max(end1, first), p.tokens) - first;
  } else {
    n = a.each;
    first = b * n;
  }
  const int rows = n * a.group;  // below 2^26
  const int length = min(max(keys, 0), (int)min((int64_t)p.max_pages * kPage, (int64_t)0x7fffffff));
  const uint8_t* pool = p.pages + (int64_t)kv * p.head_stride;

  // a batch whose sequence has more rows than max_q said: the tiles take turns
  for (int row0 = tile * ROWS; row0 < rows; row0 += a.row_tiles * ROWS) {
    const bool there = row0 + (int)(col % ROWS) < rows;
    const int row = min(row0 + (int)(col % ROWS), rows - 1);
    const int token = row / a.group, head = kv * a.group + row - token * a.group;
    const int limit = there ? length - n + token + 1 : 0;  // the row's visible keys
    const int last_token = min(row0 + ROWS - 1, rows - 1) / a.group;
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

    Raw<D> r;
    // 32-bit offsets from a page's address, which all lanes share
    const uint32_t key0 = 16 * (col >> 2) + (col & 3);
    const uint32_t at_k = key0 * P::kKey + blk * (D / 8);
    const uint32_t at_ks = P::kScales + key0 * P::kKeyScales + (D == 128 ? blk : blk >> 1);
    const uint32_t at_v = P::kValues + col * kPage + 16 * blk, at_vs = P::kValueScales + 16 * blk;
    auto load_keys = [&](int id) {
      const uint8_t* page = pool + (int64_t)id * p.page_stride;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if constexpr (D == 128) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(page + (at_k + 4 * t * P::kKey));
#pragma unroll
          for (int j = 0; j < 4; ++j) r.k[t][j] = w[j];
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2*>(page + (at_k + 4 * t * P::kKey));
          r.k[t][0] = w[0];
          r.k[t][1] = w[1];
        }
        r.ks[t] = page[at_ks + 4 * t * P::kKeyScales];
      }
    };
    auto load_values = [&](int id) {
      const uint8_t* page = pool + (int64_t)id * p.page_stride;
#pragma unroll
      for (int u = 0; u < kU; ++u)
        r.v[u] = *reinterpret_cast<const u32x4*>(page + (at_v + 16 * u * kPage));
      r.vs = *reinterpret_cast<const u32x4*>(page + at_vs);
    };
    // page `page`'s number, -1 where it has no keys
    auto checked = [&](int page, int id) { return page < page1 && id < p.n_pages ? id : -1; };
    auto number = [&](int page) { return checked(page, table[min(page, p.max_pages - 1)]); };
    f32x4 s[4];
    auto scores = [&](bool there) {
      // a page that is not there: page 0's bytes with scales of 0, so that its scores are numbers
      const uint32_t keep = there ? ~0u : 0u;
#pragma unroll
      for (int t = 0; t < 4; ++t) r.ks[t] &= keep;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const float ks = scale_of(r.ks[t]);
#pragma unroll
        for (int j = 0; j < kJ; ++j) s[t] = E::mfma16(fp4_octet<E>(r.k[t][j], ks), fq[j], s[t]);
        __builtin_amdgcn_sched_barrier(0);  // conversions of one tile at a time: registers
      }
      if (!there) {  // whatever the queries hold
        asm volatile("");
#pragma unroll
        for (int t = 0; t < 4; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    };
    // `masked`: some rows do not see all of the page's keys
    auto weigh = [&](int page, bool there, auto masked) {
      if constexpr (decltype(masked)::value) {  // hidden keys: no score, and a scale that is a number
        const int seen = limit - page * kPage - 16 * (int)blk;  // the lane's visible keys of its 16
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[t][j] = 4 * t + j < seen ? s[t][j] : -__builtin_inff();
          const int n = min(max(seen - 4 * t, 0), 4);
          r.vs[t] &= n == 4 ? ~0u : (1u << (8 * n)) - 1;
        }
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, s[t][j]);
      top = there ? across_max(top) * scale : -__builtin_inff();
      if (__any(top > m)) {  // seldom, once a few pages have passed
        const float next = fmaxf(m, top);
        const float alpha = next == -__builtin_inff() ? 1.0f : hw_exp2(m - next);
        m = next;
        l *= alpha;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          o[u][0] *= alpha;
          o[u][1] *= alpha;
        }
      }
      const float base = there ? (m == -__builtin_inff() ? 0.0f : m) : __builtin_inff();
      const uint32_t keep = there ? ~0u : 0u;
#pragma unroll
      for (int t = 0; t < 4; ++t) r.vs[t] &= keep;
      uint32_t hi[2][4], lo[2][4];  // the weights of keys 8 st .. + 7 of the lane's 16, in pairs i and i + 4
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float e = hw_exp2(fmaf(s[2 * st + i][j], scale, -base));
            l += e;
            w[i] = e * scale_of((r.vs[2 * st + i] >> (8 * j)) & 255);
          }
          const uint32_t u = bf16_pair(w[0], w[1]);
          const uint32_t v =
              bf16_pair(w[0] - __uint_as_float(u << 16), w[1] - __uint_as_float(u & 0xffff0000u));
          hi[st][j] = ROWS == 8 && col >= 8 ? v : u;
          lo[st][j] = v;
        }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const s16x8 ph = __builtin_bit_cast(s16x8, u32x4{hi[st][0], hi[st][1], hi[st][2], hi[st][3]});
        const s16x8 pl = __builtin_bit_cast(s16x8, u32x4{lo[st][0], lo[st][1], lo[st][2], lo[st][3]});
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          // codes of one element of keys i and i + 4 side by side, as one byte
          const uint32_t w0 = r.v[u][2 * st], w1 = r.v[u][2 * st + 1];
          const uint32_t we = (w0 & 0x0f0f0f0fu) | (w1 << 4 & 0xf0f0f0f0u);
          const uint32_t wo = (w0 >> 4 & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u);
          const s16x8 ve = fp4_octet<Bf16>(we, kHeld<E>), vo = fp4_octet<Bf16>(wo, kHeld<E>);
          o[u][0] = Bf16::mfma16(ve, ph, o[u][0]);
          o[u][1] = Bf16::mfma16(vo, ph, o[u][1]);
          if constexpr (ROWS == 16) {
            o[u][0] = Bf16::mfma16(ve, pl, o[u][0]);
            o[u][1] = Bf16::mfma16(vo, pl, o[u][1]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    // The next page's keys are asked for once this one's are used up, its values likewise (page 0's where there
    // is none: without a branch around the loads the waits for them are exact).
    if (page0 + wave < page1) {
      int id = checked(page_first, id_first), next = checked(page_first + kWaves, id_second);
      load_keys(max(id, 0));
      load_values(max(id, 0));
      // pages that the tile's first row, and with it every other, sees all of; then the others
      const int full = min(page1, max(length - n + row0 / a.group + 1, 0) / kPage);
      int page = page0 + wave;
      auto step = [&](auto masked) {
        const int after = number(page + 2 * kWaves);
        scores(id >= 0);
        load_keys(max(next, 0));
        weigh(page, id >= 0, masked);
        load_values(max(next, 0));
        id = next;
        next = after;
        page += kWaves;
      };
      const bool all_there = row0 + ROWS <= rows;
      while (all_there && page < full) step(std::false_type{});
      while (page < page1) step(std::true_type{});
    }

    if constexpr (ROWS == 8) {  // the two parts' columns
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[u][h][j] += dpp_f<0x128>(o[u][h][j]);  // rotated by 8 in rows of 16
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
      if (there && col < ROWS) {
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

// ---- many rows -------------------------------------------------------------------------------------
//
// 128 rows of a sequence's key head to a workgroup, 32 to a wave (v_mfma_f32_32x32x16).  Each page's codes become
// 16-bit numbers once, in LDS: keys [64][D], values [D][64] in the order of the S^T tiles' rows, so that a
// lane's weights are its right operand again.  Two pages' room: one barrier a page, with the next page's
// conversions beside this one's first product, and a step's weights between the products of the one before.
// m is set kSlack above a row's maximum, and again only where a score passes it, so that few pages scale the sums:
// the row's largest weight lies between 2^-1.75 and 1.  The other tiles' m is the maximum.
//
// Bound: instructions.  4000 tokens of 32 heads of 128 over 8 run at 0.65 PFLOP/s (200 us), 4 texts of 300 to 1024
// behind 4096 keys at 0.60 (210 us), 7000 of 14 heads of 64 over 2 at 0.48 (181 us), in bf16 and fp16 alike.  A
// weight in one 16-bit number, half of the second product, would take 181 instead of 210 us for the texts, but its
// rounding shows where values cancel, and fp16's range does not hold weights times any scale.
//
// A value without a scale (its byte is 255) lies in LDS as zeros, and rows that see it become NaN at their end.
constexpr float kSlack = 1.75f;
template <int D>
__device__ __forceinline__ int key_chunk(int row, int c) {  // 16 rows read at one chunk touch all banks
  return D == 128 ? c ^ (row & 15) : c ^ ((row >> 1) & 7);
}
__device__ __forceinline__ int value_chunk(int row, int c) { return c ^ ((row >> 1) & 7); }

template <class E, int D>
__global__ __launch_bounds__(256, 2) void attend_fp4_tile_kernel(const AttendArgs a) {
  using P = Page<D>;
  constexpr int kRows = kTileRows, kSteps = D / 16, kDT = D / 32;
  // products before the other workgroup's vector instructions: 4 texts of 32 heads of 128 210 -> 204 us, but 7000
  // tokens of 14 of 64 179 -> 186
  constexpr bool kFirst = D == 128;
  __shared__ __attribute__((aligned(16))) short sk[2][kPage * D];
  __shared__ __attribute__((aligned(16))) short sv[2][D * kPage];
  __shared__ __attribute__((aligned(16))) f32x4 svs[2][2][kPage / 8];  // the values' scales, by half waves
  __shared__ __attribute__((aligned(8))) uint32_t without[2][2];  // which keys' values have no scale
  const FcvFp4Attention& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 31, fh = lane >> 5;
  const int kv = blockIdx.x % p.n_kv_heads, turn = blockIdx.x / p.n_kv_heads % a.row_tiles;
  const int b = sequence_of(a, blockIdx.x / p.n_kv_heads / a.row_tiles);
  typedef const int32_t __attribute__((address_space(4))) * Uniform;  // nothing writes these: scalar loads
  const Uniform table = (Uniform)(uintptr_t)(p.table + (int64_t)b * p.table_row);
  int first, n;
  if (p.cu_q) {
    const Uniform ends = (Uniform)(uintptr_t)(p.cu_q + b);
    first = min(max(ends[0], 0), p.tokens);
    n = min(max(ends[1], first), p.tokens) - first;
  } else {
    n = a.each;
    first = b * n;
  }
  const int keys = ((Uniform)(uintptr_t)p.lengths)[b];
  const int rows = n * a.group;  // below 2^24
  const int length = min(max(keys, 0), (int)min((int64_t)p.max_pages * kPage, (int64_t)0x7fffffff));
  const uint8_t* pool = p.pages + (int64_t)kv * p.head_stride;
  const float scale = p.scale * kLog2e;
  // the tiles with the most keys first
  const int tiles = (rows + kRows - 1) / kRows;
  for (int t0 = turn; t0 < tiles; t0 += a.row_tiles) {
    const int row0 = (tiles - 1 - t0) * kRows;
    const int row1 = row0 + 32 * wave;  // the wave's first row
    const bool there = row1 + fr < rows;
    const int row = min(row1 + fr, rows - 1);
    const int token = row / a.group, head = kv * a.group + row - token * a.group;
    const int limit = there ? length - n + token + 1 : 0;  // the row's visible keys
    auto sees = [&](int r) { return min(max(length - n + min(r, rows - 1) / a.group + 1, 0), length); };
    const int reach = row1 < rows ? sees(row1 + 31) : 0;   // of the wave
    const int all_pages = (sees(row0 + kRows - 1) + kPage - 1) / kPage;
    const int page0 = blockIdx.y * a.pages_per;
    int page1 = min(page0 + a.pages_per, all_pages);
    if (blockIdx.y == (unsigned)a.splits - 1) page1 = all_pages;  // and what max_length left out

    s16x8 fq[kSteps];
    {
      const short* q = static_cast<const short*>(p.q) + (int64_t)(first + token) * p.q_row +
                       (int64_t)head * p.q_head + 8 * fh;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) fq[j] = *reinterpret_cast<const s16x8*>(q + 16 * j);
    }
    f32x16 o[kDT];
#pragma unroll
    for (int d = 0; d < kDT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;
    float poison = 1.0f;  // or NaN, of the row

    // a thread's share of a page: D / 4 codes of a key, 16 bytes of a byte row of the values
    uint32_t kw[D / 32], ks, vsw = 0;
    u32x4 vw = {0, 0, 0, 0};
    auto load = [&](int id) {
      const uint8_t* page = pool + (int64_t)max(id, 0) * p.page_stride;
      if constexpr (D == 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(page + (uint32_t)tid * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) kw[j] = w[j];
        ks = page[P::kScales + (uint32_t)tid];
        vw = *reinterpret_cast<const u32x4*>(page + P::kValues + (uint32_t)tid * 16);
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(page + (uint32_t)tid * 8);
        kw[0] = w[0];
        kw[1] = w[1];
        ks = page[P::kScales + (uint32_t)tid / 2];
        if (tid < 128) vw = *reinterpret_cast<const u32x4*>(page + P::kValues + (uint32_t)tid * 16);
      }
      if (tid < kPage / 4)
        vsw = *reinterpret_cast<const uint32_t*>(page + P::kValueScales + (uint32_t)tid * 4);
    };
    auto unpack = [&](int buf) {
      const int key = tid / 4;
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
        *reinterpret_cast<s16x8*>(&sk[buf][key * D + key_chunk<D>(key, tid % 4 * (D / 32) + j) * 8]) =
            fp4_octet<E>(kw[j], scale_of(ks));
      if (D == 128 || tid < 128) {
        // key 8 g + 4 h + j of 16: half h's slot pair j, as codes of one element side by side in a byte
        const int pair = tid / 4, step = tid % 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w0 = vw[h], w1 = vw[2 + h];
          const uint32_t we = (w0 & 0x0f0f0f0fu) | (w1 << 4 & 0xf0f0f0f0u);
          const uint32_t wo = (w0 >> 4 & 0x0f0f0f0fu) | (w1 & 0xf0f0f0f0u);
          *reinterpret_cast<s16x8*>(
              &sv[buf][2 * pair * kPage + value_chunk(2 * pair, 2 * step + h) * 8]) =
              fp4_octet<Bf16>(we, kHeld<E>);
          *reinterpret_cast<s16x8*>(
              &sv[buf][(2 * pair + 1) * kPage + value_chunk(2 * pair + 1, 2 * step + h) * 8]) =
              fp4_octet<Bf16>(wo, kHeld<E>);
        }
      }
      if (tid < kPage / 4) {  // 16 lanes of one row, four keys each
        int byte[4];
        uint32_t bad[4];  // the lanes whose j-th key has no scale
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          byte[j] = vsw >> (8 * j) & 255;
          bad[j] = (uint32_t)__ballot(byte[j] == 255);
          byte[j] = byte[j] == 255 ? 0 : byte[j];
        }
        if (tid == 0) {
          without[buf][0] = bad[0] | bad[1] << 16;
          without[buf][1] = bad[2] | bad[3] << 16;
        }
        svs[buf][tid % 2][tid / 2] =
            f32x4{scale_of(byte[0]), scale_of(byte[1]), scale_of(byte[2]), scale_of(byte[3])};
      }
    };
    f32x16 s[2];
    s16x8 kf[2][2];  // the keys' fragments of four steps
    auto load_kf = [&](int buf, int j) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = 32 * t + fr;
        kf[j % 2][t] =
            *reinterpret_cast<const s16x8*>(&sk[buf][key * D + key_chunk<D>(key, 2 * j + fh) * 8]);
      }
    };
    auto scores = [&](int buf) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[t][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = E::mfma32(kf[j % 2][t], fq[j], s[t]);
        if (j + 2 < kSteps) load_kf(buf, j + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto take = [&](int page, int buf) {
      s16x8 vf[2][kDT];
      auto load_vf = [&](int st) {
#pragma unroll
        for (int d = 0; d < kDT; ++d) {
          const int r = 32 * d + fr;
          vf[st & 1][d] =
              *reinterpret_cast<const s16x8*>(&sv[buf][r * kPage + value_chunk(r, 2 * st + fh) * 8]);
        }
      };
      const u32x2 none = *reinterpret_cast<const u32x2*>(without[buf]);
      if (!__all(limit >= (page + 1) * kPage)) {  // hidden keys have no score
        asm volatile("");  // a branch: the compiler would do this for every page
        const int seen = limit - page * kPage - 4 * fh;
#pragma unroll
        for (int g = 0; g < 8; ++g)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (8 * g + j >= seen) s[g / 4][g % 4 * 4 + j] = -__builtin_inff();
      }
      const uint32_t bad = __builtin_amdgcn_readfirstlane(none[0] | none[1]);
      if (bad != 0) {  // a value without a scale is in LDS as zeros: NaN for the rows that see it
        const int seen = limit - page * kPage;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t lanes = none[j / 2] >> (16 * (j % 2)) & 0xffffu;
          const int n = min(max((seen - j + 3) >> 2, 0), 16);
          if (lanes & ((1u << n) - 1)) poison = __builtin_nanf("");
        }
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[t][e]);
      {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false,
                                                        false);
        top = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) * scale;
      }
      if (__any(top > m)) {
        const float next = top > m ? top + kSlack : m;
        const float shrink = top > m ? hw_exp2(m - next) : 1.0f;  // of the sums
        m = next;
        l *= shrink;
#pragma unroll
        for (int d = 0; d < kDT; ++d) o[d] *= shrink;
      }
      const float base = m == -__builtin_inff() ? 0.0f : m;
      u32x4 hi[2], lo[2];
      auto weights = [&](int st) {  // of 16 keys: words 2 st and 2 st + 1 of the lane's eight
        // the scales of the lane's keys: 8 g + 4 fh + j is element j of vs[g % 2]
        f32x4 vs[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) vs[i] = svs[buf][fh][2 * st + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float w[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int g = 2 * st + i;
            const float e = hw_exp2(fmaf(s[g / 4][g % 4 * 4 + j], scale, -base));
            l += e;
            w[i] = e * vs[i][j];
          }
          const uint32_t u = bf16_pair(w[0], w[1]);
          hi[st & 1][j] = u;
          lo[st & 1][j] =
              bf16_pair(w[0] - __uint_as_float(u << 16), w[1] - __uint_as_float(u & 0xffff0000u));
        }
      };
      load_vf(0);
      weights(0);
      if constexpr (kFirst) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (st < 3) load_vf(st + 1);
        __builtin_amdgcn_sched_barrier(0);
        // this step's products, and between them the next one's weights
#pragma unroll
        for (int d = 0; d < kDT; ++d) {
          o[d] = Bf16::mfma32(vf[st & 1][d], __builtin_bit_cast(s16x8, hi[st & 1]), o[d]);
          o[d] = Bf16::mfma32(vf[st & 1][d], __builtin_bit_cast(s16x8, lo[st & 1]), o[d]);
        }
        if (st < 3) {
          weights(st + 1);
#pragma unroll
          for (int i = 0; i < 2 * kDT; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
            __builtin_amdgcn_sched_group_barrier(0x002, 60 / (2 * kDT), 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    if (page0 < page1) {
      auto number = [&](int page) {
        const int id = table[min(page, p.max_pages - 1)];
        return page < page1 && id < p.n_pages ? id : -1;
      };
      int id = number(page0), next = number(page0 + 1);
      load(id);
      unpack(0);
      load(next);
      for (int page = page0; page < page1; ++page) {
        const int buf = (page - page0) & 1;
        const int after = number(page + 2);
        __syncthreads();  // this page is in LDS, and every wave is through with the one before
        const bool sees_it = id >= 0 && page * kPage < reach;
        if (sees_it)
          for (int j = 0; j < 2; ++j) load_kf(buf, j);
        unpack(buf ^ 1);
        load(after);
        if (sees_it) {
          if constexpr (kFirst) __builtin_amdgcn_s_setprio(1);
          scores(buf);
          if constexpr (kFirst) __builtin_amdgcn_s_setprio(0);
          take(page, buf);
          if constexpr (kFirst) __builtin_amdgcn_s_setprio(0);
        }
        id = next;
        next = after;
      }
    }
    l = swap32_sum(l);
#pragma unroll
    for (int d = 0; d < kDT; ++d) o[d] *= poison;
    if (there) {
      const int64_t at = (int64_t)(first + token) * p.n_heads + head;
      if (a.splits > 1) {
        const int64_t i = (int64_t)blockIdx.y * p.tokens * p.n_heads + at;
#pragma unroll
        for (int d = 0; d < kDT; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(a.part + i * D + 32 * d + 8 * g + 4 * fh) =
                f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
        if (fh == 0) {
          a.part_ml[2 * i] = m;
          a.part_ml[2 * i + 1] = l;
        }
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / (l * kHeld<E>);
        short* to = static_cast<short*>(p.out) + (int64_t)(first + token) * p.out_row +
                    (int64_t)head * p.out_head + 4 * fh;
#pragma unroll
        for (int d = 0; d < kDT; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<s16x4*>(to + 32 * d + 8 * g) =
                s16x4{E::from_f32(o[d][4 * g] * inv), E::from_f32(o[d][4 * g + 1] * inv),
                      E::from_f32(o[d][4 * g + 2] * inv), E::from_f32(o[d][4 * g + 3] * inv)};
        if (p.lse && fh == 0) p.lse[at] = (m + __builtin_amdgcn_logf(l)) * kLn2;
      }
    }
    __syncthreads();  // the next tile's pages go where this one's were
  }
}

// The ranges' sums.  A workgroup has one row's head: a thread 4 elements of every kGroups-th range, in their
// order, and the groups are summed in theirs.
template <class E, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(const AttendArgs a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ __attribute__((aligned(16))) float so[kGroups][D];
  __shared__ float sm[kGroups], sl[kGroups];
  const FcvFp4Attention& p = a.p;
  const int token = blockIdx.x / p.n_heads, head = blockIdx.x - token * p.n_heads;
  if (p.cu_q && token >= p.cu_q[p.batch]) return;  // behind the last sequence
  const int64_t i = blockIdx.x, n = (int64_t)p.tokens * p.n_heads;
  const int g = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = g; s0 < a.splits; s0 += 2 * kGroups) {  // two asked for at once
    float pm[2], pl[2];
    f32x4 po[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int s = s0 + k * kGroups;
      const int64_t at = (s < a.splits ? s : s0) * n + i;
      pm[k] = s < a.splits ? a.part_ml[2 * at] : -__builtin_inff();
      pl[k] = a.part_ml[2 * at + 1];
      po[k] = *reinterpret_cast<const f32x4*>(a.part + at * D + d);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (pm[k] == -__builtin_inff() && pl[k] == 0.0f) continue;  // a range without keys, or none
      if (s0 + k * kGroups >= a.splits) continue;
      const float next = fmaxf(m, pm[k]), base = next == -__builtin_inff() ? 0.0f : next;
      const float f0 = hw_exp2(m - base), f1 = hw_exp2(pm[k] - base);
      m = next;
      l = l * f0 + pl[k] * f1;
      o = o * f0 + po[k] * f1;
    }
  }
  *reinterpret_cast<f32x4*>(&so[g][d]) = o;
  if (d == 0) {
    sm[g] = m;
    sl[g] = l;
  }
  __syncthreads();
  if (g > 0) return;
  float top = m;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) top = fmaxf(top, sm[k]);
  const float base = top == -__builtin_inff() ? 0.0f : top;
  l = 0.0f;
  o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < kGroups; ++k) {
    const float f = hw_exp2(sm[k] - base);
    l += sl[k] * f;
    o += *reinterpret_cast<const f32x4*>(&so[k][d]) * f;
  }
  o *= l == 0.0f ? 0.0f : 1.0f / (l * kHeld<E>);
  *reinterpret_cast<s16x4*>(static_cast<short*>(p.out) + (int64_t)token * p.out_row +
                            (int64_t)head * p.out_head + d) =
      s16x4{E::from_f32(o[0]), E::from_f32(o[1]), E::from_f32(o[2]), E::from_f32(o[3])};
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
  FCV_CHECK((int64_t)p->tokens * p->n_heads < (1LL << 24), FCV_ERR_INVALID,
            "too many rows: tokens * n_heads must stay below 2^24");
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
  int rows;  // of a tile
  int64_t row_tiles;
  int splits, pages_per;
  int order_shift;
};

Plan plan_of(const FcvFp4Attention& p) {
  const int group = p.n_heads / p.n_kv_heads;
  const int64_t most_rows = (int64_t)std::min(p.max_q, p.tokens) * group;
  // Tiles of 128 rows where they fill the card, which takes more of heads of 64, whose pages are short.  Heads of
  // 128, 32 over 8, by tiles of 128 and of 16 rows: 4000 tokens (1000 tiles) 202 and 329 us, 2000 (500) 73 and
  // 96, 8 x 128 behind 4000 keys (256) 119 and 156, 1000 (250) 36 and 36, 4 x 128 behind 2000 (128) 54 and 47.
  // Heads of 64, 14 over 2: 7000 (766) 180 and 230, 20 x 300 behind 3000 keys (680) 163 and 179, 16 x 300 (544)
  // 153 and 135, 8 x 300 (272) 101 and 75, 2000 (220) 55 and 30.
  const int64_t many = (most_rows + kTileRows - 1) / kTileRows * p.batch * p.n_kv_heads;
  const int rows = most_rows <= 8 ? 8 : many < (p.head_dim == 128 ? kCus : 5 * kCus / 2) ? 16 : kTileRows;
  const int64_t all = std::max<int64_t>((most_rows + rows - 1) / rows, 1);
  // tiles past a launch's size take turns
  const int64_t tiles = std::min(all, std::max<int64_t>(1, (1 << 22) / ((int64_t)p.batch * p.n_kv_heads)));
  const int64_t blocks = tiles * p.batch * p.n_kv_heads;
  const int64_t most = (int64_t)p.max_pages * kPage;
  const int pages = (int)std::max<int64_t>((std::min<int64_t>(p.max_length, most) + kPage - 1) / kPage, 1);
  // Ranges of pages: two workgroups a CU; a workgroup's beginning and end cost about 5 us.  32 heads of 128 over
  // 8, single tokens behind 1000 to 7000 keys: 64 sequences (512 workgroups) take 67, 67, 68 and 74 us in one,
  // two, three and four ranges, 24 (192) 46, 38, 34 and 40; 14 over 2 of 64, 64 of 500 to 4000: one, two, four
  // and eight 20, 16, 15.5 and 16.5; one of 7000 keys in ranges of 4, 8 and 16 pages 8.2, 8.8 and 10.6.
  // Up to 16 pages one range: it costs a microsecond there (8.5 instead of 7.6 for 600 keys) and saves a launch.
  // Two where one leaves CUs with half of what others have: 36 sequences (288) 62 us in one and 48 in two,
  // 44 (352) 61 and 48, 48 (384) 63 and 58; but behind 300 to 3000 keys 44 take 31 in one and 38 in two.
  int64_t want = pages <= 16 ? 1 : std::max<int64_t>(1, 2 * kCus / blocks);
  if (blocks > kCus && blocks < 2 * kCus) {
    auto filled = [](int64_t n) { return (double)n / (double)((n + kCus - 1) / kCus * kCus); };
    const double us = (double)blocks * pages * kPage * (p.head_dim + p.head_dim / 32 + 1) / 5.0e6;
    if (us / filled(blocks) - us / filled(2 * blocks) > 22.0) want = 2;
  }
  int per = (int)std::max<int64_t>((pages + want - 1) / want, 4);
  if (rows == kTileRows) {
    // Time in pages of a workgroup that shares its CU; one that has it alone takes 0.63 of it, and a tile's
    // sums of one range cost 0.02.  8 x 128 tokens of 32 heads of 128 over 8 (256 tiles) behind 16000 keys take
    // 430 us in one range, 381, 412 and 393 in two, three and four, behind 4000 keys 119 and 121; 10 x 128 (320)
    // behind 8000 309, 303 and 286; 520 tiles behind 8000 501, 450 and 428, 640 behind 16000 1052, 933 and 958.
    // Tiles whose keys are new ones too have lengths of their own, and the short ones fill the ends.
    const int most_ranges = p.max_q <= p.max_length / 2 ? 3 : 1;
    double best = 0.0;
    for (int s = 1; s <= most_ranges; ++s) {
      const int64_t n = blocks * s, rest = n % (2 * kCus);
      const int each = (pages + s - 1) / s;
      const double time = each * (n / (2 * kCus) + (rest == 0 ? 0.0 : rest <= kCus ? 0.63 : 1.0)) +
                          (s > 1 ? 0.02 * n : 0.0);
      if (s == 1 || time < best) {
        best = time;
        per = each;
      }
    }
  }
  const int splits = (pages + per - 1) / per;
  // The longest sequences first, where their workgroups are long: 64 of 2000 to 8000 keys 84 us in their own
  // order, 76 so; 100 of 1000 to 7000 115 and 96; 30 x 100 to 300 tokens behind 500 to 3000, 14 over 2 of 64,
  // 168 and 131.  It costs a workgroup about a microsecond: 8 of 500 to 7000 in ranges of 14 pages 17.0 and 18.4.
  int shift = -1;
  if (p.batch >= (rows == kTileRows ? 8 : 2) && per >= 32 && blocks * splits > kCus)
    for (shift = 6; pages * (int64_t)kPage >> shift >= 1 << kKeyBits; ++shift) {}
  return Plan{rows, tiles, splits, per, shift};
}

size_t workspace_bytes(const FcvFp4Attention& p, const Plan& plan) {
  return plan.splits > 1 ? (size_t)plan.splits * p.tokens * p.n_heads * (p.head_dim + 2) * 4 : 0;
}

template <class E, int D>
void launch(const AttendArgs& a, int rows, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.row_tiles * a.p.batch * a.p.n_kv_heads), (unsigned)a.splits);
  if (rows == 8)
    hipLaunchKernelGGL((attend_fp4_kernel<E, D, 8>), grid, dim3(256), 0, stream, a);
  else if (rows == 16)
    hipLaunchKernelGGL((attend_fp4_kernel<E, D, 16>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((attend_fp4_tile_kernel<E, D>), grid, dim3(256), 0, stream, a);
  if (a.splits > 1) {
    hipLaunchKernelGGL((attend_join_kernel<E, D>), dim3((unsigned)(a.p.tokens * a.p.n_heads)), dim3(256),
                       0, stream, a);
  }
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" size_t fcv_fp4_attention_workspace_bytes(const FcvFp4Attention* args) {
  if (fcv::lm::check(args) || args->tokens == 0) return 0;
  return fcv::lm::workspace_bytes(*args, fcv::lm::plan_of(*args));
}

extern "C" int fcv_fp4_attention_plan(const FcvFp4Attention* args, int32_t* rows, int32_t* tiles, int32_t* ranges,
                                      int32_t* ordered) {
  if (int rc = fcv::lm::check(args)) return rc;
  FCV_CHECK(rows && tiles && ranges && ordered, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(args->tokens > 0, FCV_ERR_INVALID, "no rows: nothing is launched");
  const fcv::lm::Plan plan = fcv::lm::plan_of(*args);
  *rows = plan.rows;
  *tiles = (int32_t)plan.row_tiles;
  *ranges = plan.splits;
  *ordered = plan.order_shift >= 0;
  return FCV_OK;
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
  const AttendArgs a{*args, args->n_heads / args->n_kv_heads, args->tokens / args->batch,
                     (int)plan.row_tiles, plan.splits,
                     plan.pages_per, plan.order_shift, part,
                     part ? part + (size_t)plan.splits * args->tokens * args->n_heads * args->head_dim
                          : nullptr};
  if (args->dtype == FCV_LM_F16)
    args->head_dim == 64 ? launch<Half, 64>(a, plan.rows, stream) : launch<Half, 128>(a, plan.rows, stream);
  else
    args->head_dim == 64 ? launch<Bf16, 64>(a, plan.rows, stream) : launch<Bf16, 128>(a, plan.rows, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}
