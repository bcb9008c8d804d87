// Attention of a batch whose sequences share one prefix in front of caches of their own.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(t_j - m + shift),  t_j = scale log2(e) q.k_j
// over the prefix's keys and the sequence's own up to the query's, with m the running maximum of t (or
// somewhat below it, see kLag).  The keys are split into parts; each leaves its m, its sum l of p and its
// sum o of p v, and a second launch joins a query's parts in a fixed order:
//   M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
//
// The prefix is read once for the batch: the queries of all sequences that read one key head are the
// rows of one product against it.  A sequence's own keys meet its own queries only.  A batch whose sequences
// append about 128 rows (tokens x heads of a key head) or more each reads prefix and own keys in one pass,
// and so does a call of few keys; these need no join.
//
// Matrix form (v_mfma_f32_32x32x16): S^T = K Q^T puts query l % 32 into lane l with 16 of a tile's
// 32 keys, so that the softmax is per lane (one exchange with lane l ^ 32) and the weights, in two 16-bit
// parts, are the B operand of O^T = V^T P^T as they stand.  V^T's fragments are read from the row-major
// tile by ds_read_b64_tr_b16, which hands each of 16 lanes one column of a 4 x 16 block.
// Keys and values are copied straight into LDS.
//
// Bound and rate, 32 / 8 heads x 128 in bf16:
//   64 queries behind a prompt of 8192 and 200 to 2000 own keys each: 111 to 115 us, 3.0 TB/s of the bytes
//     that have to be read (the own keys alone 90 us, 3.3 TB/s; the prompt alone 38 us: its blocks come first
//     and leave little room beside them).
//   4 texts of 300 to 1024 tokens behind 4096 keys: 397 to 406 us, 0.54 PFLOP/s.  The vector pipe (32
//     exponentials and about 230 other instructions a wave and tile of 64 keys) and the matrix pipe (48
//     products) take their turns rather than overlap: the matrix pipes are busy for 37 % of the cycles, CUs
//     for 74 %, as the last round of tiles is not full.  A tile's scores taken ahead beside the weights of
//     the one before was slower (more registers, or half the tile), and so were fewer keys a barrier.  What
//     costs most are reloads of spilled registers in the key loops: each waits for the copies in flight.
//   A token behind 512 + 100 keys: 10 us on the GPU.
#include <algorithm>
#include <climits>
#include <cmath>

#include "lm.hpp"

namespace fcv {
namespace lm {
namespace {

constexpr int kWaves = 4;
constexpr int kFewRows = 32;    // queries of a row tile whose waves share the keys out
constexpr int kFewKeys = 32;    // keys of a wave's tile there
constexpr int kManyRows = 128;  // queries of a row tile whose waves share its queries out, 32 each
constexpr int kManyKeys = 64;   // keys of a workgroup's tile there
// Rows of all key heads times dims up to which stacked rows of few queries a sequence are taken 32 at a time.
// Above, tiles of 128 need a launch of their own (us, 32 at a time / 128): 16384 rows of 128 dims behind 1024
// keys 89 / 108, 4096 keys 127 / 134, 16384 keys 296 / 266; 32768 rows 164 / 167, 242 / 228, 580 / 500; 32768
// rows of 64 dims behind 4096 keys 110 / 114, 65536 211 / 202.
constexpr int64_t kStackedFew = 1 << 21;
constexpr int kShortKeys = 768;  // prefix and own keys up to which tiles of 32 queries take them all at once
constexpr int kMaxKeys = 1 << 29;  // of the prefix and of a session: their sum and a tile more fit 31 bits
constexpr int kMaxParts = 64;      // lanes of the joining wave
constexpr float kLog2e = 1.4426950408889634f;

// How a call is split.  Parts 0 .. np - 1 are ranges of the prefix for the rows of all sequences
// together, np .. np + no - 1 ranges of a sequence's own keys, or (np = 0, fused) of the prefix and its
// own keys behind one another.
struct Shape {
  bool prefix_many, own_many;  // tiles of 128 rows, else of 32
  bool fused, direct;          // direct: one part, written to the output
  int prefix_tiles, np, prefix_step;
  int own_tiles, no, own_step; // own_step: keys of a range at least (longer caches widen it)
  int64_t prefix_blocks, own_blocks;
  __host__ __device__ int parts() const { return np + no; }
};

struct Args {
  FcvLmAttention p;
  Shape s;
  float* part_o;  // [parts][tokens * n_heads][head_dim]
  float2* part_s; // [parts][tokens * n_heads]: m, l
  float scale2;   // scale * log2(e)
};

// A value that is the same in all lanes, as a scalar.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const short* scalar(const short* p) {
  const uint64_t u = (uint64_t)p;
  return (const short*)((uint64_t)(uint32_t)scalar((int)u) |
                        (uint64_t)(uint32_t)scalar((int)(u >> 32)) << 32);
}

__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ uint32_t lds_base(short* smem) {
  return (uint32_t)scalar((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem);
}

template <int N>
__device__ __forceinline__ void wait_vmem() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// LDS position of 16-byte chunk c of row r.  The keys' reads (16 rows at one chunk index) and the
// transposed reads of values (four rows at four neighbouring chunks) both touch all banks: the row's low
// bits choose the group of four chunks, its next two the chunk in the group.
template <int D>
__device__ __forceinline__ int swz(int r, int c) {
  return D == 64 ? c ^ ((r & 2) << 1 | ((r >> 2) & 3)) : c ^ ((r & 3) << 2 | ((r >> 2) & 3));
}

// The keys and values of one head of the prefix or of one session.
struct Segment {
  const short* k;
  const short* v;
  int64_t k_row, v_row;
};

// A wave's running softmax over its query (lane l % 32): acc[d / 32] holds O^T.
template <int D>
struct State {
  f32x16 acc[D / 32];
  float m, l;
  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
    m = -INFINITY;
    l = 0.0f;
  }
};

// LDS addresses of a tile's fragments, for the tile whose keys (or values) start at byte `base`, a
// multiple of 256.  In swz, a row's bits and a chunk's are joined by exclusive or, so that a lane's
// addresses differ from its first by constants in the low byte and in the instruction's offset.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"  // of the host's pass
typedef __attribute__((address_space(3))) const s16x8* lds16;
typedef __attribute__((address_space(3))) s16x4* lds8;

// K fragment of step ks (16 dims) of keys 32 t .. + 31: lane l holds key 32 t + l % 32, dims 16 ks +
// 8 (l / 32) .. + 7.
template <int D>
struct KeyFragments {
  uint32_t at;
  __device__ __forceinline__ KeyFragments(uint32_t base, int lane)
      : at(base + (lane & 31) * (2 * D) + swz<D>(lane & 31, lane >> 5) * 16) {}
  __device__ __forceinline__ s16x8 get(int t, int ks) const {
    return *(lds16)((at ^ (uint32_t)(ks << 5)) + t * 64 * D);
  }
};

// V^T fragment of step k (16 keys) and dims 32 dt .. + 31: slot j of lane l is value
// [16 k + 8 (j / 4) + 4 (l / 32) + j % 4][32 dt + l % 32], the keys of P's slots.
template <int D>
struct ValueFragments {
  uint32_t at;
  __device__ __forceinline__ ValueFragments(uint32_t base, int lane) {
    const int i = lane & 15, g = lane >> 4, row = (g >> 1) * 4 + (i >> 2);
    at = base + row * (2 * D) + swz<D>(row, (g & 1) * 2 + ((i & 3) >> 1)) * 16 + (i & 1) * 8;
  }
  __device__ __forceinline__ s16x8 get(int k, int dt) const {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds8)((at ^ (uint32_t)(dt << 6)) + k * 32 * D));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds8)((at ^ (uint32_t)(dt << 6 | 32)) + k * 32 * D + 16 * D));  // eight rows on
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

#pragma clang diagnostic pop

// v with zeros in the place of infinities and NaN, whose presence is noted in `found`.
template <class E>
__device__ __forceinline__ s16x8 finite_only(const s16x8& v, uint32_t& found) {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u16x8 size = __builtin_bit_cast(u16x8, v) & (unsigned short)0x7fff;
  const u16x8 past = __builtin_elementwise_sub_sat(size, (u16x8)(unsigned short)(E::kInf - 1));
  const u32x4 p = __builtin_bit_cast(u32x4, past);
  found |= (p[0] | p[1]) | (p[2] | p[3]);
  const u16x8 keep = __builtin_elementwise_min(past, (u16x8)(unsigned short)1) - (unsigned short)1;
  return __builtin_bit_cast(s16x8, __builtin_bit_cast(u16x8, v) & keep);
}

__device__ __forceinline__ bool finite4(const f32x4& o) {
  return fmaf(o[0], 0.0f, o[1] * 0.0f) + fmaf(o[2], 0.0f, o[3] * 0.0f) == 0.0f;
}

// The steps of a tile of 32 KT keys.

// s = K Q^T of the keys at LDS byte sk.
template <class E, int D, int KT>
__device__ __forceinline__ void tile_scores(uint32_t sk, const s16x8 (&qf)[D / 16], int lane,
                                            f32x16 (&s)[KT]) {
  const KeyFragments<D> keys(sk, lane);
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) s[t][e] = 0.0f;
  // sums that do not wait for one another are taken in turn
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int t = 0; t < KT; ++t) s[t] = E::mfma32(keys.get(t, ks), qf[ks], s[t]);
}

// Hides the scores of keys from `limit` (the lane's, from the tile's first key on) and takes the running
// maximum along.
template <class E, int D, int KT>
__device__ __forceinline__ void tile_maximum(f32x16 (&s)[KT], State<D>& st, int lane, int limit,
                                             bool all_visible, float scale2) {
  if (!all_visible) {
    int first = limit - (lane >> 5) * 4;
    asm volatile("" : "+v"(first));  // a branch, not 32 selects in every tile
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        s[t][e] = t * 32 + (e >> 2) * 8 + (e & 3) < first ? s[t][e] : -INFINITY;
  }
  float tops[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) tops[e & 3] = fmaxf(tops[e & 3], s[t][e]);
  const float top = half_max(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))) * scale2;
  if (__any(top > st.m + E::kLag)) {
    const float m_new = top > st.m + E::kLag ? top : st.m;
    // a query that has seen no finite score yet keeps m = -inf (and sums of 0)
    const float corr = hw_exp2(st.m - (m_new == -INFINITY ? 0.0f : m_new));
    st.m = m_new;
    st.l *= corr;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.acc[dt][e] *= corr;
  }
}

// The weights of a lane's scores 8 h .. + 7, and their sums.  The matrix instruction takes 16-bit operands,
// so that a weight goes in as two of them, rounded and rest: together they are off by 2^-16 (bf16) or 2^-22
// (fp16) of it, and a result's error is that of its own rounding.  With the rounded one alone it is 1.4
// times that (2.33e-3 against 1.66e-3 relative L2 for texts in bf16), at 16 products of 48 less a wave and
// tile of 64 keys: texts behind 4096 keys 307 against 393 us, tokens the same time (fp16 up to 6 % more).
template <class E>
__device__ __forceinline__ void weights8(const f32x16& s, int h, float scale2, float shift,
                                         float (&sums)[4], s16x8 (&pf)[2]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef typename E::T2 T2;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const f32x2 w = {hw_exp2(fmaf(s[8 * h + e], scale2, shift)),
                     hw_exp2(fmaf(s[8 * h + e + 1], scale2, shift))};
    sums[e & 3] += w[0];
    sums[(e & 3) + 1] += w[1];
    const T2 r = __builtin_convertvector(w, T2);
    const f32x2 rest = {w[0] - (float)r[0], w[1] - (float)r[1]};
    const s16x2 p0 = __builtin_bit_cast(s16x2, r);
    const s16x2 p1 = __builtin_bit_cast(s16x2, __builtin_convertvector(rest, T2));
    pf[0][e] = p0[0];
    pf[0][e + 1] = p0[1];
    pf[1][e] = p1[0];
    pf[1][e + 1] = p1[1];
  }
}

// O^T += V^T P^T of 16 keys, step k of a tile.  With HIDE, values that are not finite are left out and
// noted in `found`.
template <class E, int D, bool HIDE>
__device__ __forceinline__ void values16(const ValueFragments<D>& values, int k, const s16x8 (&pf)[2],
                                         State<D>& st, uint32_t& found) {
  s16x8 v[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
    v[dt] = values.get(k, dt);
    if (HIDE) v[dt] = finite_only<E>(v[dt], found);
  }
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) st.acc[dt] = E::mfma32(v[dt], pf[n], st.acc[dt]);
}

// Weights and values of a tile of 32 KT keys with the values at LDS byte sv, 16 keys after another: two
// parts of all weights of 64 keys at once are more registers than two workgroups a CU have (456 us for the
// 393 above).
template <class E, int D, int KT, bool HIDE>
__device__ __forceinline__ void tile_steps(const f32x16 (&s)[KT], uint32_t sv, State<D>& st, float scale2,
                                           int lane, uint32_t& found) {
  const ValueFragments<D> values(sv, lane);
  const float shift = E::kShift - (st.m == -INFINITY ? 0.0f : st.m);
  float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 2 * KT; ++k) {
    s16x8 pf[2];
    weights8<E>(s[k / 2], k % 2, scale2, shift, sums, pf);
    values16<E, D, HIDE>(values, k, pf, st, found);
  }
  st.l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
}
template <class E, int D, int KT>
__device__ __forceinline__ void tile_steps(const f32x16 (&s)[KT], uint32_t sv, State<D>& st, float scale2,
                                           int lane, bool hide, uint32_t& found) {
  if (hide)
    tile_steps<E, D, KT, true>(s, sv, st, scale2, lane, found);
  else
    tile_steps<E, D, KT, false>(s, sv, st, scale2, lane, found);
}

// The same of 32 keys, apart, so that the weights do not wait for the values.
template <class E, int D>
__device__ __forceinline__ void tile_weights(const f32x16& s, State<D>& st, float scale2,
                                             s16x8 (&pf)[2][2]) {
  const float shift = E::kShift - (st.m == -INFINITY ? 0.0f : st.m);
  float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  weights8<E>(s, 0, scale2, shift, sums, pf[0]);
  weights8<E>(s, 1, scale2, shift, sums, pf[1]);
  st.l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
}
template <class E, int D>
__device__ __forceinline__ void tile_values(uint32_t sv, const s16x8 (&pf)[2][2], State<D>& st, int lane,
                                            bool hide, uint32_t& found) {
  const ValueFragments<D> values(sv, lane);
  if (hide) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        const s16x8 v = finite_only<E>(values.get(k, dt), found);
#pragma unroll
        for (int n = 0; n < 2; ++n) st.acc[dt] = E::mfma32(v, pf[k][n], st.acc[dt]);
      }
    return;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      const s16x8 v = values.get(k, dt);
#pragma unroll
      for (int n = 0; n < 2; ++n) st.acc[dt] = E::mfma32(v, pf[k][n], st.acc[dt]);
    }
}

// The queries of a row tile: rows first .. first + count - 1 of the (token, head of the group) pairs of
// one key head, token-major from token0 on.
struct Rows {
  int kvh, group, token0, first, count;
  __device__ __forceinline__ int token(int r) const { return token0 + (first + r) / group; }
  __device__ __forceinline__ int head(int r) const { return kvh * group + (first + r) % group; }
};

template <int D>
__device__ __forceinline__ void load_q(const FcvLmAttention& p, const Rows& rows, int r, int hl,
                                       s16x8 (&qf)[D / 16]) {
  const int row = min(r, rows.count - 1);
  const short* q = static_cast<const short*>(p.q) + rows.token(row) * p.q_row + rows.head(row) * p.q_head;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
    qf[ks] = *reinterpret_cast<const s16x8*>(q + ks * 16 + hl * 8);
}

// Copies of one wave: N times 64 / (D / 8) rows, from row `row0` (a multiple of 16) on, of a tile of
// `tile_rows` keys (or values) with a row stride in bytes.  left: rows of the range from the tile's first
// on; rows past it are read as its last one (and get no weight).
template <int D, int N>
__device__ __forceinline__ void copy_rows(const short* tile, uint32_t row_bytes, int tile_rows, int left,
                                          int row0, int lane, uint32_t lds) {
  constexpr int kChunks = D / 8, kRows = 64 / kChunks;
  const int r0 = lane / kChunks;
  const uint32_t chunk = swz<D>(r0, lane % kChunks) * 16;
  if (left >= tile_rows) {
    const char* base = reinterpret_cast<const char*>(scalar(tile)) + (int64_t)row0 * row_bytes;
    const uint32_t row = r0 * row_bytes;
#pragma unroll
    for (int i = 0; i < N; ++i)  // kRows further on, the position's bits 2 and up count i
      lds_dma16(base + (int64_t)(i * kRows) * row_bytes, row + (chunk ^ (uint32_t)swz<D>(i * kRows, 0) * 16),
                lds + i * 1024);
  } else {
    const char* base = reinterpret_cast<const char*>(scalar(tile));
#pragma unroll
    for (int i = 0; i < N; ++i)
      lds_dma16(base, min(row0 + i * kRows + r0, left - 1) * row_bytes +
                          (chunk ^ (uint32_t)swz<D>(i * kRows, 0) * 16), lds + i * 1024);
  }
}

// LDS in elements: the tiles' keys and values ([kWaves][K, V][32][D], or [2][K, V][64][D]), and over them in
// the end [kWaves][32] rows of O (16 bytes apart in their banks) with their m and l behind them, and the
// first keys that mend_tile finds and any_bad's words.
template <int D>
constexpr int pitch() { return D + 4; }
template <int D>
constexpr int lds_elems() { return kWaves * 32 * (pitch<D>() * 2 + 4) + 4 * D + 8; }
template <int D>
__device__ __forceinline__ float2* lds_sums(short* smem) {
  return reinterpret_cast<float2*>(smem + kWaves * 32 * pitch<D>() * 2);
}
template <int D>
__device__ __forceinline__ int* lds_first(short* smem) {
  return reinterpret_cast<int*>(lds_sums<D>(smem) + kWaves * 32);
}

// Whether `bad` holds in any lane of the workgroup, through a word of each wave's in LDS (the library's
// vote costs 64 long requests 5 us); ends in a barrier, and a barrier stands before the next call's words.
template <int D>
__device__ __forceinline__ bool any_bad(short* smem, bool bad) {
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  int* words = lds_first<D>(smem) + 2 * D;
  const bool wave_bad = __any(bad);
  if ((threadIdx.x & 63) == 0) words[threadIdx.x >> 6] = wave_bad;
  __syncthreads();
  const i32x4 v = *reinterpret_cast<const i32x4*>(words);
  return ((v[0] | v[1]) | (v[2] | v[3])) != 0;
}

// A row tile of up to 32 queries against keys [k0, k1) of the prefix and [o0, o1) of the sequence's own; the
// four waves take a range's tiles in turn, each through LDS buffers of its own (no barrier), and are joined
// at the end.  first_pos: the position of the sequence's first new token.  Whether the results need
// mend_tile.
template <class E, int D>
__device__ bool few_rows(const Args& a, short* smem, const Rows& rows, const Segment& prefix, int k0,
                         int k1, const Segment& own, int o0, int o1, int first_pos, int part) {
  const FcvLmAttention& p = a.p;
  if (k0 >= k1 && o0 >= o1 && !a.s.direct) {  // nothing to sum: no weight, no output that the join would read
    if (threadIdx.x < (unsigned)rows.count) {
      const int64_t at = (int64_t)part * p.tokens * p.n_heads +
                         (int64_t)rows.token(threadIdx.x) * p.n_heads + rows.head(threadIdx.x);
      a.part_s[at] = float2{-INFINITY, 0.0f};
    }
    return false;
  }
  constexpr int kCopies = kFewKeys / (512 / D);
  constexpr int kTileElems = kFewKeys * D;
  const int lane = threadIdx.x & 63, ql = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  s16x8 qf[D / 16];
  load_q<D>(p, rows, ql, hl, qf);
  // first own key past the query's view; the wave's smallest decides which tiles need the mask
  const int limit = min(o1, first_pos + rows.token(min(ql, rows.count - 1)) - rows.token0 + 1);
  int low = limit;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) low = min(low, __shfl_xor(low, off, kWave));
  low = scalar(low);

  // a wave's two buffers hold a tile's keys and its values; each is filled again as soon as it was read
  const uint32_t sk = lds_base(smem) + wave * 2 * kTileElems * 2, sv = sk + kTileElems * 2;
  State<D> st;
  st.reset();
  uint32_t found = 0;
#pragma unroll 1
  for (int g = 0; g < 2; ++g) {
    const Segment seg = g == 0 ? prefix : own;
    const int begin = g == 0 ? k0 : o0, end = g == 0 ? k1 : o1;
    const uint32_t k_bytes = (uint32_t)seg.k_row * 2, v_bytes = (uint32_t)seg.v_row * 2;
    auto fetch_k = [&](int kt) {
      copy_rows<D, kCopies>(seg.k + (int64_t)kt * seg.k_row, k_bytes, kFewKeys, end - kt, 0, lane, sk);
    };
    auto fetch_v = [&](int kt) {
      copy_rows<D, kCopies>(seg.v + (int64_t)kt * seg.v_row, v_bytes, kFewKeys, end - kt, 0, lane, sv);
    };
    int kt = begin + wave * kFewKeys;
    if (kt < end) {
      fetch_k(kt);
      fetch_v(kt);
    }
    for (; kt < end; kt += kWaves * kFewKeys) {
      const int next = kt + kWaves * kFewKeys;
      const bool all_visible = kt + kFewKeys <= (g == 0 ? end : low);
      wait_vmem<kCopies>();  // the keys are here, the values may be on their way
      f32x16 scores[1];
      tile_scores<E, D, 1>(sk, qf, lane, scores);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads have returned
      if (next < end) fetch_k(next);
      tile_maximum<E, D, 1>(scores, st, lane, (g == 0 ? end : limit) - kt, all_visible, a.scale2);
      s16x8 pf[2][2];
      tile_weights<E, D>(scores[0], st, a.scale2, pf);
      if (next < end)
        wait_vmem<kCopies>();
      else
        wait_vmem<0>();
      tile_values<E, D>(sv, pf, st, lane, g == 1 && !all_visible, found);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (next < end) fetch_v(next);
    }
  }

  // join the waves: O is [wave][query][dim], four dims of a query a thread
  const float l_wave = half_sum(st.l);
  __syncthreads();  // every wave is done with its buffers
  float* so = reinterpret_cast<float*>(smem);
  float2* ss = lds_sums<D>(smem);  // [kWaves][kFewRows]
  if (ql < rows.count) {
    if (hl == 0) ss[wave * kFewRows + ql] = float2{st.m, l_wave};
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(so + (wave * kFewRows + ql) * pitch<D>() + dt * 32 + g * 8 + hl * 4) =
            f32x4{st.acc[dt][4 * g], st.acc[dt][4 * g + 1], st.acc[dt][4 * g + 2], st.acc[dt][4 * g + 3]};
  }
  __syncthreads();
  const int64_t rows_all = (int64_t)p.tokens * p.n_heads;
  bool bad = found != 0;
  for (int i = threadIdx.x; i < rows.count * (D / 4); i += 256) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ss[w * kFewRows + r].x);
    const float base = m == -INFINITY ? 0.0f : m;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 s = ss[w * kFewRows + r];
      const float f = hw_exp2(s.x - base);
      l = fmaf(s.y, f, l);
      o += *reinterpret_cast<const f32x4*>(so + (w * kFewRows + r) * pitch<D>() + d) * f;
    }
    bad |= !finite4(o);
    if (a.s.direct) {
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      *reinterpret_cast<s16x4*>(static_cast<short*>(p.out) + rows.token(r) * p.out_row +
                                rows.head(r) * p.out_head + d) =
          s16x4{E::from_f32(o[0] * inv), E::from_f32(o[1] * inv), E::from_f32(o[2] * inv),
                E::from_f32(o[3] * inv)};
      if (p.lse && d == 0)
        p.lse[(int64_t)rows.token(r) * p.n_heads + rows.head(r)] =
            (m - E::kShift + log2f(l)) * 0.6931471805599453f;
      continue;
    }
    const int64_t at = part * rows_all + (int64_t)rows.token(r) * p.n_heads + rows.head(r);
    *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = o;
    if (d == 0) a.part_s[at] = float2{m, l};
  }
  return any_bad<D>(smem, bad);  // the next row tile fills the buffers again
}

// A row tile of up to 128 queries, 32 a wave, against keys [k0, k1) of the prefix and [o0, o1) of the
// sequence's own; all waves share a tile of 64 keys in LDS, the next one on its way.
template <class E, int D>
__device__ bool many_rows(const Args& a, short* smem, const Rows& rows, const Segment& prefix, int k0,
                          int k1, const Segment& own, int o0, int o1, int first_pos, int part) {
  constexpr int kCopies = kManyKeys / (512 / D) / kWaves;  // a wave's, of K and of V
  constexpr int kTileElems = kManyKeys * D;
  const FcvLmAttention& p = a.p;
  const int lane = threadIdx.x & 63, ql = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int my = min(wave * 32 + ql, rows.count - 1);

  s16x8 qf[D / 16];
  load_q<D>(p, rows, my, hl, qf);
  const int limit = min(o1, first_pos + rows.token(my) - rows.token0 + 1);
  int low = limit, high = limit;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    low = min(low, __shfl_xor(low, off, kWave));
    high = max(high, __shfl_xor(high, off, kWave));
  }
  low = scalar(low);
  high = scalar(high);

  const int row0 = wave * kCopies * (512 / D);
  const uint32_t lds = lds_base(smem);
  State<D> st;
  st.reset();
  uint32_t found = 0;
  int stage = 0;
#pragma unroll 1
  for (int g = 0; g < 2; ++g) {
    const Segment seg = g == 0 ? prefix : own;
    const int begin = g == 0 ? k0 : o0, end = g == 0 ? k1 : o1;
    if (begin >= end) continue;
    const uint32_t k_bytes = (uint32_t)seg.k_row * 2, v_bytes = (uint32_t)seg.v_row * 2;
    auto fetch = [&](int kt, int to) {
      const uint32_t at = lds + to * 2 * kTileElems * 2 + wave * kCopies * 1024;
      copy_rows<D, kCopies>(seg.k + (int64_t)kt * seg.k_row, k_bytes, kManyKeys, end - kt, row0, lane, at);
      copy_rows<D, kCopies>(seg.v + (int64_t)kt * seg.v_row, v_bytes, kManyKeys, end - kt, row0, lane,
                            at + kTileElems * 2);
    };
    fetch(begin, stage);
    for (int kt = begin; kt < end; kt += kManyKeys, stage ^= 1) {
      wait_vmem<0>();
      // every wave's copies of this tile have landed, and every wave has read the one before
      __syncthreads();
      if (kt + kManyKeys < end) fetch(kt + kManyKeys, stage ^ 1);
      if (g == 1 && kt >= high) continue;  // none of the wave's queries sees the tile
      const uint32_t sk = lds + stage * 2 * kTileElems * 2;
      const bool all_visible = kt + kManyKeys <= (g == 0 ? end : low);
      f32x16 scores[2];
      tile_scores<E, D, 2>(sk, qf, lane, scores);
      tile_maximum<E, D, 2>(scores, st, lane, (g == 0 ? end : limit) - kt, all_visible, a.scale2);
      tile_steps<E, D, 2>(scores, sk + kTileElems * 2, st, a.scale2, lane, g == 1 && !all_visible, found);
    }
  }

  // through LDS, 32 lanes (16 of 64 dims) to a row, so that stores cover whole rows
  const float l = half_sum(st.l);
  __syncthreads();  // every wave is done with the last tile
  float* so = reinterpret_cast<float*>(smem) + wave * 32 * pitch<D>();
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(so + ql * pitch<D>() + dt * 32 + g * 8 + hl * 4) =
          f32x4{st.acc[dt][4 * g], st.acc[dt][4 * g + 1], st.acc[dt][4 * g + 2], st.acc[dt][4 * g + 3]};
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const int d = lane % (D / 4) * 4, mine = wave * 32;
  bool bad = found != 0;
#pragma unroll 4
  for (int q0 = 0; q0 < 32; q0 += 256 / D) {
    const int q = q0 + lane / (D / 4), r = mine + q;
    const float lr = __shfl(l, q, kWave), mr = __shfl(st.m, q, kWave);
    if (r >= rows.count) continue;
    const f32x4 o = *reinterpret_cast<const f32x4*>(so + q * pitch<D>() + d);
    const int token = rows.token(r), head = rows.head(r);
    bad |= !finite4(o);
    if (a.s.direct) {
      const float inv = lr > 0.0f || lr != lr ? 1.0f / lr : 0.0f;
      *reinterpret_cast<s16x4*>(static_cast<short*>(p.out) + token * p.out_row + head * p.out_head + d) =
          s16x4{E::from_f32(o[0] * inv), E::from_f32(o[1] * inv), E::from_f32(o[2] * inv),
                E::from_f32(o[3] * inv)};
      if (p.lse && d == 0)
        p.lse[(int64_t)token * p.n_heads + head] = (mr - E::kShift + log2f(lr)) * 0.6931471805599453f;
    } else {
      const int64_t at = ((int64_t)part * p.tokens + token) * p.n_heads + head;
      *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = o;
      if (d == 0) a.part_s[at] = float2{mr, lr};
    }
  }
  if (hl == 0) lds_sums<D>(smem)[wave * 32 + ql] = float2{st.m, l};  // for mend_tile
  return any_bad<D>(smem, bad);  // the next row tile fills the buffers again
}

// What a workgroup does: a key head's rows of all sequences or of one, against a range of its keys.
struct Work {
  int kvh, group, part, token0, tokens, length, prefix_len;
  int c0, c1;  // the range: keys of the prefix (if it is read here) and the sequence's own behind it
  int first_tile, tiles, stride, tile_rows;
  bool stacked;
  Segment prefix, own;
};

template <bool MANY>
__device__ __forceinline__ Work work_of(const Args& a, uint32_t b) {
  const FcvLmAttention& p = a.p;
  const Shape& s = a.s;
  Work w;
  w.group = p.n_heads / p.n_kv_heads;
  w.stacked = b < (uint32_t)s.prefix_blocks;
  if (!w.stacked) b -= (uint32_t)s.prefix_blocks;
  // key head fastest: the row tiles of one head and range are dealt to one XCD and share its L2
  w.kvh = scalar((int)(b % (uint32_t)p.n_kv_heads));
  b /= (uint32_t)p.n_kv_heads;
  const uint32_t ranges = w.stacked ? s.np : s.no;
  const int range = scalar((int)(b % ranges));
  b /= ranges;

  int slot = 0;
  w.token0 = w.length = 0;
  w.first_tile = (int)b;
  if (w.stacked) {
    w.tokens = p.cu_q ? min(max(p.cu_q[p.batch], 0), p.tokens) : p.tokens;
  } else {
    const int seq = scalar((int)(b % (uint32_t)p.batch));
    w.first_tile = (int)(b / (uint32_t)p.batch);
    if (p.cu_q) {
      w.token0 = min(max(p.cu_q[seq], 0), p.tokens);
      w.tokens = min(max(p.cu_q[seq + 1], w.token0), p.tokens) - w.token0;
    } else {
      w.tokens = p.tokens / p.batch;
      w.token0 = seq * w.tokens;
    }
    slot = p.slots ? p.slots[seq] : seq;
    w.length = min(max(p.lengths[seq], 0), p.capacity);
    if (slot < 0 || slot >= p.sessions) slot = w.length = 0;
  }
  w.prefix = {static_cast<const short*>(p.prefix_k) + w.kvh * p.pk_head,
              static_cast<const short*>(p.prefix_v) + w.kvh * p.pv_head, p.pk_row, p.pv_row};
  w.own = {static_cast<const short*>(p.k_cache) + slot * p.k_session + w.kvh * p.k_head,
           static_cast<const short*>(p.v_cache) + slot * p.v_session + w.kvh * p.v_head, p.k_row, p.v_row};
  w.prefix_len = w.stacked || s.fused ? p.prefix_len : 0;
  const int total = w.prefix_len + w.length;  // at most 2 kMaxKeys
  const int step = w.stacked ? s.prefix_step : max(s.own_step, (total + s.no - 1) / s.no);
  w.c0 = (int)min((int64_t)range * step, (int64_t)total);
  w.c1 = (int)min((int64_t)w.c0 + step, (int64_t)total);
  w.part = w.stacked ? range : s.np + range;
  w.tile_rows = MANY ? kManyRows : kFewRows;
  w.tiles = (w.tokens * w.group + w.tile_rows - 1) / w.tile_rows;
  w.stride = w.stacked ? s.prefix_tiles : s.own_tiles;
  return w;
}

// The rows of one of its tiles, and their keys: [k0, k1) of the prefix, [o0, o1) of the sequence's own.
struct TileWork {
  Rows rows;
  int k0, k1, o0, o1, first_pos;
};

__device__ __forceinline__ TileWork tile_of(const Work& w, int index) {
  TileWork t;
  const int first = index * w.tile_rows;
  t.rows = {w.kvh, w.group, w.token0, first, min(w.tile_rows, w.tokens * w.group - first)};
  t.first_pos = w.length - w.tokens;
  // own keys past the tile's last query are not visited
  const int seen =
      w.stacked ? 0 : min(w.length, t.first_pos + (first + t.rows.count - 1) / w.group + 1);
  t.k0 = min(w.c0, w.prefix_len);
  t.k1 = min(w.c1, w.prefix_len);
  t.o0 = max(w.c0 - w.prefix_len, 0);
  t.o1 = min(max(w.c1 - w.prefix_len, 0), seen);
  return t;
}

// Values that are not finite and that a query sees.  Every visible key has a weight above zero, so an
// infinity among the values is what the row gets, and NaN for NaN or for both infinities.  The products
// do not keep to that: a weight that rounds to zero or whose second part is negative makes NaN of an
// infinity, a row read again behind a range's end has a weight of zero, and masked tiles leave such values
// out.  All of these leave a sum that is not finite, or a note in `found`; the tile's values are then
// looked through, and what each row sees is written over its results (a row whose sum of weights is NaN
// has NaN already).  Seldom runs, takes about as long as the tile itself, and derives all it needs again
// from opaque copies of the kernel's arguments: with what it needs kept from the key loops on, every call
// pays (a token 10.2 to 11.1 us, 64 long requests 108 to 118 us; so 10.1 and 112), and as a function of
// its own it costs small calls 0.6 us.
typedef const __attribute__((address_space(4))) Args* ArgsAt;

template <class E, int D, bool MANY>
__device__ __forceinline__ void mend_tile(ArgsAt at, __attribute__((address_space(3))) short* lds,
                                          uint32_t block, int index) {
  const Args& a = *(const Args*)at;
  const FcvLmAttention& p = a.p;
  short* smem = (short*)lds;
  const Work w = work_of<MANY>(a, block);
  const TileWork t = tile_of(w, index);
  __threadfence();  // the results stand before they are written over
  // first[0][d], first[1][d]: the first own key whose value in dim d is inf or NaN, -inf or NaN; a key of
  // the prefix, which every query sees, stands before all of them
  int* first = lds_first<D>(smem);
  for (int i = threadIdx.x; i < 2 * D; i += 64 * kWaves) first[i] = INT_MAX;
  __syncthreads();
  constexpr int kKeys = 64 * kWaves / (D / 8);  // a step's; 8 dims a thread
  const int d = threadIdx.x % (D / 8) * 8, key0 = threadIdx.x / (D / 8);
  int up[8], down[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) up[e] = down[e] = INT_MAX;
#pragma unroll 1
  for (int g = 0; g < 2; ++g) {
    const short* v = (g == 0 ? w.prefix.v : w.own.v) + d;
    const int64_t v_row = g == 0 ? w.prefix.v_row : w.own.v_row;
    const int end = g == 0 ? t.k1 : t.o1;
#pragma unroll 1
    for (int key = (g == 0 ? t.k0 : t.o0) + key0; key < end; key += 4 * kKeys) {
      s16x8 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)  // four asked for at once; keys past the end are the last one again
        x[u] = *reinterpret_cast<const s16x8*>(v + (int64_t)min(key + u * kKeys, end - 1) * v_row);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = E::to_f32(x[u][e]);
          const int here = g == 0 ? INT_MIN : min(key + u * kKeys, end - 1);
          if (!(f < INFINITY)) up[e] = min(up[e], here);
          if (!(f > -INFINITY)) down[e] = min(down[e], here);
        }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (up[e] != INT_MAX) atomicMin(first + d + e, up[e]);
    if (down[e] != INT_MAX) atomicMin(first + D + d + e, down[e]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < t.rows.count * D; i += 64 * kWaves) {
    const int r = i / D, dim = i % D, token = t.rows.token(r), head = t.rows.head(r);
    const int limit = min(t.o1, t.first_pos + token - w.token0 + 1);  // the first own key past its view
    const bool has_up = first[dim] < limit, has_down = first[D + dim] < limit;
    if (!has_up && !has_down) continue;
    float o = has_up && has_down ? NAN : has_up ? INFINITY : -INFINITY;
    if (a.s.direct) {
      const float2* ss = lds_sums<D>(smem) + r;  // of the row, or of each wave's share of its keys
#pragma unroll
      for (int k = 0; k < (MANY ? 1 : kWaves); ++k)
        if (ss[k * kFewRows].y != ss[k * kFewRows].y) o = NAN;
      static_cast<short*>(p.out)[token * p.out_row + head * p.out_head + dim] = E::from_f32(o);
    } else {
      a.part_o[(((int64_t)w.part * p.tokens + token) * p.n_heads + head) * D + dim] = o;
    }
  }
  __syncthreads();  // the next row tile fills the buffers again
}

// The blocks of the stacked rows first, then the sequences'; a launch has those of one kind of tile.
// (Both kinds in one kernel need more registers than two workgroups a CU have; few queries of 64 dims leave
// room for three.)
template <class E, int D, bool MANY>
__global__ __launch_bounds__(256, D == 64 && !MANY ? 3 : 2) void prefix_attention_kernel(const Args a) {
  __shared__ __attribute__((aligned(1024))) short smem[lds_elems<D>()];
  const Work w = work_of<MANY>(a, blockIdx.x);
  for (int i = scalar(w.first_tile); i < w.tiles; i += w.stride) {
    const int index = w.tiles - 1 - i;  // the last tiles see the most keys and go first
    const TileWork t = tile_of(w, index);
    bool bad;
    if constexpr (MANY)
      bad = many_rows<E, D>(a, smem, t.rows, w.prefix, t.k0, t.k1, w.own, t.o0, t.o1, t.first_pos, w.part);
    else
      bad = few_rows<E, D>(a, smem, t.rows, w.prefix, t.k0, t.k1, w.own, t.o0, t.o1, t.first_pos, w.part);
    if (bad) {
      // opaque, so that nothing of what it derives is shared with the code above and kept until here
      ArgsAt args = (ArgsAt)__builtin_amdgcn_kernarg_segment_ptr();
      uint32_t block = blockIdx.x;
      asm volatile("" : "+s"(args), "+s"(block));
      mend_tile<E, D, MANY>(args, (__attribute__((address_space(3))) short*)smem, block, index);
    }
  }
}

// o + v w; what a row saw that is not finite stays, however small the part's weight.
__device__ __forceinline__ float add_part(float v, float w, float o) {
  return fabsf(v) < INFINITY ? fmaf(v, w, o) : o + v;
}

// Joins the parts of each (token, head): W waves to a row, each its share of the parts, eight at a time;
// lane l holds dims 2 l, 2 l + 1 (of 128) or l.
template <class E, int D, int W>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  __shared__ float sums[4][D];
  static_assert(kMaxParts == kWave, "a lane to a part");
  const FcvLmAttention& p = a.p;
  const int live = p.cu_q ? min(max(p.cu_q[p.batch], 0), p.tokens) : p.tokens;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = wave % W;
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + wave / W;
  if (row >= (int64_t)live * p.n_heads) return;  // W = 4: the whole workgroup
  const int parts = a.s.parts();
  const int64_t rows_all = (int64_t)p.tokens * p.n_heads;
  float2 part = {-INFINITY, 0.0f};
  if (lane < parts) part = a.part_s[lane * rows_all + row];
  float top = part.x;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  const float f = hw_exp2(part.x - (top == -INFINITY ? 0.0f : top));
  const float l = wave_sum(part.y * f);
  float2 o = {0.0f, 0.0f};
  // a part without keys (a range that a short sequence does not reach) was not written
  const uint64_t live_parts = __ballot(part.x != -INFINITY);
  for (int i0 = mine; i0 < parts; i0 += 8 * W) {
    float2 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * W;
      v[u] = float2{0.0f, 0.0f};
      if (i < parts && (live_parts >> i & 1)) {
        const float* src = a.part_o + (i * rows_all + row) * D;
        if (D == 128)
          v[u] = reinterpret_cast<const float2*>(src)[lane];
        else
          v[u].x = src[lane];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * W;
      if (i >= parts) break;
      const float w = __shfl(f, i, kWave);
      o.x = add_part(v[u].x, w, o.x);
      if (D == 128) o.y = add_part(v[u].y, w, o.y);
    }
  }
  if constexpr (W > 1) {
    if (D == 128)
      reinterpret_cast<float2*>(sums[wave])[lane] = o;
    else
      sums[wave][lane] = o.x;
    __syncthreads();
    if (wave != 0) return;
    o = float2{0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (D == 128) {
        const float2 v = reinterpret_cast<const float2*>(sums[w])[lane];
        o.x += v.x;
        o.y += v.y;
      } else {
        o.x += sums[w][lane];
      }
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const int token = (int)(row / p.n_heads), head = (int)(row % p.n_heads);
  short* out = static_cast<short*>(p.out) + token * p.out_row + head * p.out_head;
  if (D == 128) {
    const uint32_t lo = (uint16_t)E::from_f32(o.x * inv), hi = (uint16_t)E::from_f32(o.y * inv);
    reinterpret_cast<uint32_t*>(out)[lane] = lo | hi << 16;
  } else {
    out[lane] = E::from_f32(o.x * inv);
  }
  if (p.lse && lane == 0) p.lse[row] = (top - E::kShift + log2f(l)) * 0.6931471805599453f;
}

// ---- host ---------------------------------------------------------------------------------------

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

Shape shape_of(const FcvLmAttention& p) {
  Shape s{};
  const int group = p.n_heads / p.n_kv_heads;
  const int64_t seq_rows = std::min<int64_t>(p.max_q, std::max(p.tokens, 1)) * group;
  const int64_t all_rows = (int64_t)p.tokens * group;
  const int max_length = std::min(std::max(p.max_length, 1), p.capacity);
  // Keys of a range.  With r ranges a block's chain of tiles takes tile_us * tiles / r and the join about
  // 0.1 us a part plus the part's bytes, written and read at 4 TB/s; the sum is least at the root of the
  // quotient.  Beyond `full` blocks more ranges only wait for others.
  const float part_us = 0.1f + (float)p.tokens * p.n_heads * p.head_dim * 8.0f / 4.0e6f;
  auto cut = [&](int keys, int unit, float tile_us, int64_t blocks, int64_t full, int most) {
    const float best = std::sqrt((float)ceil_div(keys, unit) * tile_us / part_us);
    const int64_t want = std::min<int64_t>({(int64_t)best, std::max<int64_t>(full / blocks, 1), most});
    return ceil_div(ceil_div(keys, std::max<int64_t>(want, 1)), unit) * unit;
  };
  s.own_many = seq_rows > kFewRows;
  // A sequence with at least a tile of rows of its own may read the prompt with them, which saves the join.
  // But each of a batch's sequences reads it then, in whole tiles: their tiles (at most a ragged one a
  // sequence more than the stacked rows have) against the join's two parts.  A round of 512 tiles takes
  // 3.9 us a 64 keys of 128 dims, 0.46 of that with one a CU or less.  64 requests of 32 / 8 heads, one of
  // them with 512 new tokens and 63 with one: behind 8192 keys 667 us, stacked 184, behind 64 keys 85,
  // stacked 89; 8 of them with 512 tokens: behind 8192 keys 1087, stacked 940, behind 512 keys 171, stacked
  // 225; 16 of 33 tokens: behind 2048 keys 79, stacked 69, behind 512 keys 38, stacked 43.
  // Nor is anything stacked where all keys are few: one launch and no join (a token behind 512 + 100 keys
  // 17 -> 13 us with the host's share; on the GPU alone even at about that many keys).
  const int64_t stacked_tiles = ceil_div(all_rows, kManyRows);
  const int64_t fused_tiles =
      std::min<int64_t>((int64_t)p.batch * ceil_div(seq_rows, kManyRows), stacked_tiles + p.batch);
  const float per_round = 2.0f * kCus / (float)p.n_kv_heads;  // tiles of one key head
  const float rounds = std::max((float)fused_tiles / per_round, 0.46f) - (float)stacked_tiles / per_round;
  const float again_us =
      rounds * (float)ceil_div(p.prefix_len, kManyKeys) * 3.9f * (float)p.head_dim / 128.0f;
  const bool own_reads = seq_rows >= kManyRows && again_us <= 3.0f + 2.0f * (part_us - 0.1f);
  const bool short_keys = !s.own_many && p.prefix_len + (int64_t)max_length <= kShortKeys;
  s.fused = p.prefix_len == 0 || own_reads || (p.batch == 1 && s.own_many) || short_keys;
  if (!s.fused) {
    s.prefix_many = s.own_many || (int64_t)p.tokens * p.n_heads * p.head_dim > kStackedFew;
    s.prefix_tiles = ceil_div(all_rows, s.prefix_many ? kManyRows : kFewRows);
    s.prefix_step = cut(p.prefix_len, s.prefix_many ? kManyKeys : kWaves * kFewKeys, 0.6f,
                        (int64_t)s.prefix_tiles * p.n_kv_heads, 2 * kCus, 32);
    s.np = ceil_div(p.prefix_len, s.prefix_step);
    s.prefix_blocks = (int64_t)s.prefix_tiles * p.n_kv_heads * s.np;
  }
  s.own_tiles = std::max(1, ceil_div(seq_rows, s.own_many ? kManyRows : kFewRows));
  const int keys = (s.fused ? p.prefix_len : 0) + max_length;
  const int64_t blocks = (int64_t)s.own_tiles * p.n_kv_heads * p.batch;
  // sequences differ in length: their ranges are dealt out in several rounds where they are short
  s.own_step = s.own_many ? cut(keys, kManyKeys, 0.6f, blocks, 2 * kCus, 32)
                          : cut(keys, kWaves * kFewKeys, 1.2f, blocks, 8 * kCus, 32);
  if (short_keys) s.own_step = keys;
  s.no = ceil_div(keys, s.own_step);
  s.own_blocks = blocks * s.no;
  s.direct = s.parts() == 1;
  return s;
}

int64_t sums_bytes(const FcvLmAttention& p, const Shape& s) {
  if (s.direct) return 0;
  return ((int64_t)s.parts() * p.tokens * p.n_heads * 8 + 255) / 256 * 256;
}

int check(const FcvLmAttention* p) {
  FCV_CHECK(p, FCV_ERR_INVALID, "null arguments");
  FCV_CHECK(p->dtype == FCV_LM_F16 || p->dtype == FCV_LM_BF16, FCV_ERR_INVALID,
            "dtype must be FCV_LM_F16 or FCV_LM_BF16");
  FCV_CHECK(p->head_dim == 64 || p->head_dim == 128, FCV_ERR_INVALID, "head_dim must be 64 or 128");
  FCV_CHECK(p->n_kv_heads >= 1 && p->n_heads >= 1 && p->n_heads <= 4096 &&
                p->n_heads % p->n_kv_heads == 0,
            FCV_ERR_INVALID, "n_heads must be a multiple of n_kv_heads, up to 4096");
  FCV_CHECK(p->tokens >= 0 && p->batch >= 1 && (int64_t)p->tokens * p->n_heads < (1LL << 26),
            FCV_ERR_INVALID, "need batch >= 1 and tokens * n_heads in [0, 2^26)");
  FCV_CHECK(p->cu_q || p->tokens % p->batch == 0, FCV_ERR_INVALID,
            "without cu_q every sequence has tokens / batch queries: not a whole number");
  FCV_CHECK(p->prefix_len >= 0 && p->prefix_len <= kMaxKeys, FCV_ERR_INVALID,
            "prefix_len must be in [0, 2^29]");
  FCV_CHECK(p->sessions >= 1 && p->capacity >= 1 && p->capacity <= kMaxKeys, FCV_ERR_INVALID,
            "the caches need at least one session and a capacity in [1, 2^29]");
  FCV_CHECK(p->slots || p->batch <= p->sessions, FCV_ERR_INVALID,
            "without slots the batch must not pass the sessions");
  FCV_CHECK(p->max_q >= 1 && p->max_length >= 0, FCV_ERR_INVALID, "need max_q >= 1 and max_length >= 0");
  FCV_CHECK(p->scale > 0.0f && p->scale < __builtin_inff(), FCV_ERR_INVALID,
            "scale must be positive and finite");
  const int64_t rows_of_keys[][2] = {{p->k_row, p->capacity}, {p->v_row, p->capacity},
                                     {p->pk_row, p->prefix_len}, {p->pv_row, p->prefix_len}};
  const int64_t others[][2] = {{p->q_row, p->tokens},        {p->q_head, p->n_heads},
                               {p->out_row, p->tokens},      {p->out_head, p->n_heads},
                               {p->pk_head, p->n_kv_heads},  {p->pv_head, p->n_kv_heads},
                               {p->k_session, p->sessions},  {p->k_head, p->n_kv_heads},
                               {p->v_session, p->sessions},  {p->v_head, p->n_kv_heads}};
  for (const auto& v : rows_of_keys)
    FCV_CHECK(stride_fits(v[0], v[1]), FCV_ERR_INVALID, "strides must be multiples of 8 elements, >= 0");
  for (const auto& v : others)
    FCV_CHECK(stride_fits(v[0], v[1]), FCV_ERR_INVALID, "strides must be multiples of 8 elements, >= 0");
  for (const auto& v : rows_of_keys)
    FCV_CHECK(v[1] <= 1 || v[0] < (1LL << 24), FCV_ERR_INVALID,
              "a key's row stride must be below 2^24 elements");
  if (p->tokens == 0) return FCV_OK;
  FCV_CHECK(p->q && p->k_cache && p->v_cache && p->lengths && p->out, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(p->prefix_len == 0 || (p->prefix_k && p->prefix_v), FCV_ERR_INVALID, "null prefix");
  FCV_CHECK(aligned(p->q, 16) && aligned(p->out, 16) && aligned(p->k_cache, 16) &&
                aligned(p->v_cache, 16) && aligned(p->prefix_k, 16) && aligned(p->prefix_v, 16),
            FCV_ERR_INVALID, "q, out, the prefix and the caches must start on 16-byte boundaries");
  FCV_CHECK((p->n_heads == 1 || p->out_head >= p->head_dim) &&
                (p->tokens == 1 || p->out_row >= p->head_dim),
            FCV_ERR_INVALID, "rows of out overlap");
  const Shape s = shape_of(*p);
  FCV_CHECK(s.prefix_blocks + s.own_blocks <= (1 << 23), FCV_ERR_INVALID,
            "the batch is too large for one call: split it");
  return FCV_OK;
}

template <class E, int D>
void launch_tiles(bool many, const Args& a, int64_t blocks, hipStream_t stream) {
  if (many)
    hipLaunchKernelGGL((prefix_attention_kernel<E, D, true>), dim3((unsigned)blocks), dim3(256), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((prefix_attention_kernel<E, D, false>), dim3((unsigned)blocks), dim3(256), 0,
                       stream, a);
}

template <class E, int D>
void launch(const Args& a, hipStream_t stream) {
  if (a.s.np == 0 || a.s.prefix_many == a.s.own_many) {
    launch_tiles<E, D>(a.s.own_many, a, a.s.prefix_blocks + a.s.own_blocks, stream);
  } else {
    launch_tiles<E, D>(a.s.prefix_many, a, a.s.prefix_blocks, stream);
    Args own = a;
    own.s.prefix_blocks = 0;
    launch_tiles<E, D>(a.s.own_many, own, a.s.own_blocks, stream);
  }
  if (a.s.direct) return;
  // a workgroup to a row where there are more parts than one wave asks for at once
  const int64_t rows = (int64_t)a.p.tokens * a.p.n_heads;
  if (a.s.parts() > 8)
    hipLaunchKernelGGL((join_kernel<E, D, 4>), dim3((unsigned)rows), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((join_kernel<E, D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a);
}

size_t workspace_bytes(const FcvLmAttention& p, const Shape& s) {
  if (s.direct) return 0;
  return (size_t)(sums_bytes(p, s) + (int64_t)s.parts() * p.tokens * p.n_heads * p.head_dim * 4);
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" size_t fcv_lm_prefix_attention_workspace_bytes(const FcvLmAttention* args) {
  if (fcv::lm::check(args) || args->tokens == 0) return 0;
  return fcv::lm::workspace_bytes(*args, fcv::lm::shape_of(*args));
}

extern "C" int fcv_lm_prefix_attention(const FcvLmAttention* args, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  using namespace fcv::lm;
  if (int rc = check(args)) return rc;
  if (args->tokens == 0) return FCV_OK;
  Args a{*args, shape_of(*args), nullptr, nullptr, args->scale * kLog2e};
  const size_t need = fcv::lm::workspace_bytes(*args, a.s);
  FCV_CHECK(need == 0 || workspace, FCV_ERR_INVALID, "null workspace");
  FCV_CHECK(workspace_bytes >= need, FCV_ERR_INVALID,
            "workspace too small: need " + std::to_string(need) + " bytes");
  FCV_CHECK(need == 0 || aligned(workspace, 256), FCV_ERR_INVALID,
            "workspace must be 256-byte aligned");
  if (need) {
    a.part_s = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums_bytes(*args, a.s));
  }
  const bool half = args->dtype == FCV_LM_F16;
  if (args->head_dim == 64)
    half ? launch<Half, 64>(a, stream) : launch<Bf16, 64>(a, stream);
  else
    half ? launch<Half, 128>(a, stream) : launch<Bf16, 128>(a, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}
