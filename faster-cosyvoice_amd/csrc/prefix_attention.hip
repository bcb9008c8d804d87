// Attention of a batch whose sequences share one prefix in front of caches of their own.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(t_j - max t + shift),  t_j = scale log2(e) q.k_j
// over the prefix's keys and the sequence's own up to the query's.  The keys are split into parts;
// each leaves its maximum m, its sum l and its unnormalised output, and a second launch joins a
// query's parts in a fixed order:  M = max m,  out = sum 2^(m - M) o / sum 2^(m - M) l.
//
// The prefix is read once for the batch: the queries of all sequences that read one key head are the
// rows of one product against it.  A sequence's own keys meet its own queries only.
//
// Matrix form (v_mfma_f32_32x32x16): S^T = K Q^T puts query l % 32 into lane l with 16 of a tile's
// 32 keys, so that the softmax is per lane (one exchange with lane l ^ 32) and the weights, rounded
// to 16 bits, are the B operand of O^T = V^T P^T as they stand.  V^T's fragments are read from the
// row-major tile by ds_read_b64_tr_b16, which hands each of 16 lanes one column of a 4 x 16 block.
#include <algorithm>

#include "lm.hpp"

namespace fcv {
namespace lm {
namespace {

constexpr int kRows = 32;   // queries of a row tile
constexpr int kKeys = 32;   // keys of a wave's tile
constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

// How a call is split.  Parts 0 .. np - 1 are ranges of the prefix, np .. np + no - 1 of a
// sequence's own keys.
struct Shape {
  int prefix_tiles, np;      // row tiles over the whole batch; ranges of the prefix
  int own_tiles, no;         // row tiles of a sequence; ranges of its keys
  int prefix_step, own_step; // keys of a range (own_step at least: longer caches widen it)
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

__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int N>
__device__ __forceinline__ void wait_vmem() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// LDS position of 16-byte chunk c of row r: 16 consecutive rows read at one chunk index, and the
// 4 x 16 blocks of the transposed reads, spread over all banks.
template <int D>
__device__ __forceinline__ int swz(int r, int c) {
  return D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15);
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

// V^T fragment of MFMA step st (16 keys) and dims 32 dt .. + 31: slot j of lane l is value
// [16 st + 8 (j / 4) + 4 (l / 32) + j % 4][32 dt + l % 32], the keys of P's slots.
template <int D>
__device__ __forceinline__ s16x8 v_fragment(const short* sv, int lane, int st, int dt) {
  const int i = lane & 15, g = lane >> 4;
  const int row = st * 16 + (g >> 1) * 4 + (i >> 2);
  const int chunk = dt * 4 + (g & 1) * 2 + ((i & 3) >> 1);
  typedef __attribute__((address_space(3))) s16x4* lds4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds4)(sv + row * D + swz<D>(row, chunk) * 8 + (i & 1) * 4));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds4)(sv + (row + 8) * D + swz<D>(row + 8, chunk) * 8 + (i & 1) * 4));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// One tile of 32 keys from LDS.  `limit` (per lane) is the first key of the tile that the lane's
// query does not see; all_visible says that no lane has one.
template <class E, int D>
__device__ __forceinline__ void tile32(const short* sk, const short* sv, const s16x8 (&qf)[D / 16],
                                       State<D>& st, int lane, int limit, bool all_visible,
                                       float scale2) {
  const int ql = lane & 31, hl = lane >> 5;
  f32x16 s;
#pragma unroll
  for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const s16x8 kf =
        *reinterpret_cast<const s16x8*>(sk + ql * D + swz<D>(ql, ks * 2 + hl) * 8);
    s = E::mfma32(kf, qf[ks], s);
  }
  if (!all_visible) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      s[e] = (e >> 2) * 8 + hl * 4 + (e & 3) < limit ? s[e] : -INFINITY;
  }
  float top = s[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
  const float m_new = fmaxf(st.m, half_max(top) * scale2);
  // a query that has seen no finite score yet keeps m = -inf and subtracts 0
  const float base = m_new == -INFINITY ? 0.0f : m_new;
  const float corr = hw_exp2(st.m - base);
  const float shift = E::kShift - base;
  st.m = m_new;
  float sum = 0.0f;
  s16x8 pf[2];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float w = hw_exp2(fmaf(s[e], scale2, shift));
    sum += w;
    // 16-bit weights (relative error 2^-9 bf16, 2^-12 fp16, each with its own sign): what the
    // matrix instruction takes; the sum keeps the unrounded ones
    pf[e >> 3][e & 7] = E::from_f32(w);
  }
  st.l = fmaf(st.l, corr, sum);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
#pragma unroll
    for (int e = 0; e < 16; ++e) st.acc[dt][e] *= corr;
    s16x8 vf[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) vf[k] = v_fragment<D>(sv, lane, k, dt);
    if (!all_visible) {
      // 0 * inf and 0 * NaN: a value that is not finite is taken out of the product and given to
      // the queries that see its key
      bool bad = false;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) bad |= (vf[k][e] & E::kInf) == E::kInf;
      if (__any(bad)) {
        f32x16 up, down, nan;
#pragma unroll
        for (int e = 0; e < 16; ++e) up[e] = down[e] = nan[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          s16x8 seen, is_up = {}, is_down = {}, is_nan = {};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int key = k * 16 + (e >> 2) * 8 + hl * 4 + (e & 3);
            seen[e] = key < limit ? E::kOne : (short)0;
            const short b = vf[k][e];
            if ((b & E::kInf) != E::kInf) continue;
            if ((b & 0x7fff) != E::kInf) is_nan[e] = E::kOne;
            else if (b < 0) is_down[e] = E::kOne;
            else is_up[e] = E::kOne;
            vf[k][e] = 0;
          }
          up = E::mfma32(is_up, seen, up);
          down = E::mfma32(is_down, seen, down);
          nan = E::mfma32(is_nan, seen, nan);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (nan[e] > 0.0f) st.acc[dt][e] += NAN;
          if (up[e] > 0.0f) st.acc[dt][e] += INFINITY;
          if (down[e] > 0.0f) st.acc[dt][e] -= INFINITY;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) st.acc[dt] = E::mfma32(vf[k], pf[k], st.acc[dt]);
  }
}

// A row tile of up to 32 queries against keys [k0, k1) of a segment; the four waves take the range's
// tiles in turn, each through LDS buffers of its own (no barrier), and are joined at the end.
//
// first_row .. first_row + n_rows - 1 are (token, head of the group) pairs, token-major; own: query i
// of the tile's tokens sees keys up to first_pos + its token.
template <class E, int D>
__device__ void few_rows(const Args& a, short* smem, int kvh, int token0, int first_row, int n_rows,
                         const Segment& seg, int k0, int k1, bool own, int first_pos, int part) {
  constexpr int kChunks = D / 8;                     // 16-byte chunks of a row
  constexpr int kCopyRows = 64 / kChunks;            // rows of one copy
  constexpr int kCopies = kKeys / kCopyRows;         // copies of a K or V tile
  constexpr int kTileElems = kKeys * D;
  const FcvLmAttention& p = a.p;
  const int group = p.n_heads / p.n_kv_heads;
  const int lane = threadIdx.x & 63, ql = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const int my_row = first_row + min(ql, n_rows - 1);
  const int my_token = token0 + my_row / group, my_head = kvh * group + my_row % group;
  s16x8 qf[D / 16];
  {
    const short* q = static_cast<const short*>(p.q) + my_token * p.q_row + my_head * p.q_head;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
      qf[ks] = *reinterpret_cast<const s16x8*>(q + ks * 16 + hl * 8);
  }
  // first key past the query's view; the wave's smallest decides which tiles need the mask
  const int limit = own ? min(k1, first_pos + my_row / group + 1) : k1;
  int low = limit;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) low = min(low, __shfl_xor(low, off, kWave));

  short* ring = smem + wave * 4 * kTileElems;
  const uint32_t ring_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)ring;
  const int copy_row = lane / kChunks, copy_pos = lane % kChunks;
  auto fetch = [&](int kt, int stage) {
    const short* kb = seg.k + (int64_t)kt * seg.k_row;
    const short* vb = seg.v + (int64_t)kt * seg.v_row;
    const uint32_t at = ring_lds + stage * 2 * kTileElems * 2;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = i * kCopyRows + copy_row;
      // keys past the range are read as its last one and get no weight
      const uint32_t key = (uint32_t)(min(kt + r, k1 - 1) - kt);
      const uint32_t chunk = (uint32_t)swz<D>(r, copy_pos) * 16;
      lds_dma16(kb, key * (uint32_t)(seg.k_row * 2) + chunk, at + i * 1024);
      lds_dma16(vb, key * (uint32_t)(seg.v_row * 2) + chunk, at + kTileElems * 2 + i * 1024);
    }
  };

  State<D> st;
  st.reset();
  int kt = k0 + wave * kKeys, stage = 0;
  if (kt < k1) fetch(kt, 0);
  for (; kt < k1; kt += kWaves * kKeys, stage ^= 1) {
    const int next = kt + kWaves * kKeys;
    if (next < k1) {
      fetch(next, stage ^ 1);
      wait_vmem<2 * kCopies>();
    } else {
      wait_vmem<0>();
    }
    const short* sk = ring + stage * 2 * kTileElems;
    tile32<E, D>(sk, sk + kTileElems, qf, st, lane, limit - kt, kt + kKeys <= low, a.scale2);
    // the tile's reads have returned before its buffer is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  // join the waves: O is [wave][dim][query], a lane's own column
  const auto lr = __builtin_amdgcn_permlane32_swap(__float_as_uint(st.l), __float_as_uint(st.l), false, false);
  const float l_wave = __uint_as_float(lr[0]) + __uint_as_float(lr[1]);
  __syncthreads();  // every wave is done with its buffers
  float* so = reinterpret_cast<float*>(smem);        // [kWaves][D][kRows]
  float2* ss = reinterpret_cast<float2*>(so + kWaves * D * kRows);  // [kWaves][kRows]
  if (hl == 0) ss[wave * kRows + ql] = float2{st.m, l_wave};
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int d = dt * 32 + (e >> 2) * 8 + hl * 4 + (e & 3);
      so[(wave * D + d) * kRows + ql] = st.acc[dt][e];
    }
  __syncthreads();
  const int64_t rows_all = (int64_t)p.tokens * p.n_heads;
  for (int i = threadIdx.x; i < n_rows * D; i += 256) {
    const int r = i / D, d = i % D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ss[w * kRows + r].x);
    const float base = m == -INFINITY ? 0.0f : m;
    float o = 0.0f, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 s = ss[w * kRows + r];
      const float f = hw_exp2(s.x - base);
      l = fmaf(s.y, f, l);
      o = fmaf(so[(w * D + d) * kRows + r], f, o);
    }
    const int row = first_row + r;
    const int64_t at = (int64_t)part * rows_all + (int64_t)(token0 + row / group) * p.n_heads +
                       kvh * group + row % group;
    a.part_o[at * D + d] = o;
    if (d == 0) a.part_s[at] = float2{m, l};
  }
  __syncthreads();  // the next row tile fills the buffers again
}

template <class E, int D>
__global__ __launch_bounds__(256) void prefix_attention_kernel(const Args a) {
  __shared__ __attribute__((aligned(1024))) short smem[kWaves * 4 * kKeys * D + kWaves * kRows * 4];
  const FcvLmAttention& p = a.p;
  const Shape& s = a.s;
  const int group = p.n_heads / p.n_kv_heads;
  int64_t b = blockIdx.x;
  if (b < s.prefix_blocks) {
    // key head fastest: the row tiles of one head and range are dealt to one XCD and share its L2
    const int kvh = (int)(b % p.n_kv_heads);
    b /= p.n_kv_heads;
    const int part = (int)(b % s.np), tile = (int)(b / s.np);
    const int live = p.cu_q ? min(max(p.cu_q[p.batch], 0), p.tokens) : p.tokens;
    const int first = tile * kRows, rows = min(kRows, live * group - first);
    if (rows <= 0) return;
    const int k0 = part * s.prefix_step, k1 = min(k0 + s.prefix_step, p.prefix_len);
    const Segment seg = {static_cast<const short*>(p.prefix_k) + kvh * p.pk_head,
                         static_cast<const short*>(p.prefix_v) + kvh * p.pv_head, p.pk_row, p.pv_row};
    few_rows<E, D>(a, smem, kvh, 0, first, rows, seg, k0, k1, false, 0, part);
    return;
  }
  b -= s.prefix_blocks;
  const int kvh = (int)(b % p.n_kv_heads);
  b /= p.n_kv_heads;
  const int range = (int)(b % s.no);
  b /= s.no;
  const int seq = (int)(b % p.batch), tile0 = (int)(b / p.batch);
  int t0, t1;
  if (p.cu_q) {
    t0 = min(max(p.cu_q[seq], 0), p.tokens);
    t1 = min(max(p.cu_q[seq + 1], t0), p.tokens);
  } else {
    const int n = p.tokens / p.batch;
    t0 = seq * n;
    t1 = t0 + n;
  }
  const int slot = p.slots ? p.slots[seq] : seq;
  int length = min(max(p.lengths[seq], 0), p.capacity);
  if (slot < 0 || slot >= p.sessions) length = 0;
  const int step = max(s.own_step, (length + s.no - 1) / s.no);
  const int k0 = min(range * step, length), k1 = min(k0 + step, length);
  const Segment seg = {
      static_cast<const short*>(p.k_cache) + (length ? slot * p.k_session : 0) + kvh * p.k_head,
      static_cast<const short*>(p.v_cache) + (length ? slot * p.v_session : 0) + kvh * p.v_head,
      p.k_row, p.v_row};
  const int n_rows = (t1 - t0) * group;
  for (int first = tile0 * kRows; first < n_rows; first += s.own_tiles * kRows)
    few_rows<E, D>(a, smem, kvh, t0, first, min(kRows, n_rows - first), seg, k0, k1, true,
                   length - (t1 - t0), s.np + range);
}

// Joins the parts of each (token, head): one wave to a row, lane l holds dims 2 l, 2 l + 1.
template <class E, int D>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  const FcvLmAttention& p = a.p;
  const int live = p.cu_q ? min(max(p.cu_q[p.batch], 0), p.tokens) : p.tokens;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)live * p.n_heads) return;
  const int lane = threadIdx.x & 63, parts = a.s.parts();
  const int64_t rows_all = (int64_t)p.tokens * p.n_heads;
  float2 mine = {-INFINITY, 0.0f};
  if (lane < parts) mine = a.part_s[lane * rows_all + row];
  float top = mine.x;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  const float base = top == -INFINITY ? 0.0f : top;
  const float f = hw_exp2(mine.x - base);
  const float l = wave_sum(mine.y * f);
  float o0 = 0.0f, o1 = 0.0f;
  for (int i = 0; i < parts; ++i) {
    const float w = __shfl(f, i, kWave);
    const float* o = a.part_o + (i * rows_all + row) * D;
    if (D == 128) {
      const float2 v = reinterpret_cast<const float2*>(o)[lane];
      o0 = fmaf(v.x, w, o0);
      o1 = fmaf(v.y, w, o1);
    } else {
      o0 = fmaf(o[lane], w, o0);
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  const int token = (int)(row / p.n_heads), head = (int)(row % p.n_heads);
  short* out = static_cast<short*>(p.out) + token * p.out_row + head * p.out_head;
  if (D == 128) {
    const uint32_t lo = (uint16_t)E::from_f32(o0 * inv), hi = (uint16_t)E::from_f32(o1 * inv);
    reinterpret_cast<uint32_t*>(out)[lane] = lo | hi << 16;
  } else {
    out[lane] = E::from_f32(o0 * inv);
  }
  if (p.lse && lane == 0) p.lse[row] = (top - E::kShift + log2f(l)) * 0.6931471805599453f;
}

// ---- host ---------------------------------------------------------------------------------------

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

Shape shape_of(const FcvLmAttention& p) {
  Shape s{};
  const int group = p.n_heads / p.n_kv_heads;
  s.prefix_tiles = ceil_div((int64_t)p.tokens * group, kRows);
  if (p.prefix_len > 0) {
    const int blocks = s.prefix_tiles * p.n_kv_heads;
    const int want = std::max(1, std::min({ceil_div(2 * kCus, blocks), ceil_div(p.prefix_len, 256), 32}));
    s.prefix_step = ceil_div(ceil_div(p.prefix_len, want), kWaves * kKeys) * kWaves * kKeys;
    s.np = ceil_div(p.prefix_len, s.prefix_step);
  }
  s.own_tiles = std::max(1, ceil_div((int64_t)p.max_q * group, kRows));
  s.no = std::max(1, std::min(ceil_div(p.max_length, 256), 32));
  s.own_step = ceil_div(std::max(1, p.max_length), s.no);
  s.prefix_blocks = (int64_t)s.prefix_tiles * p.n_kv_heads * s.np;
  s.own_blocks = (int64_t)s.own_tiles * p.n_kv_heads * s.no * p.batch;
  return s;
}

int64_t sums_bytes(const FcvLmAttention& p, const Shape& s) {
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
  FCV_CHECK(p->prefix_len >= 0 && p->prefix_len <= (1 << 30), FCV_ERR_INVALID,
            "prefix_len must be in [0, 2^30]");
  FCV_CHECK(p->sessions >= 1 && p->capacity >= 1 && p->capacity <= (1 << 30), FCV_ERR_INVALID,
            "the caches need at least one session and a capacity in [1, 2^30]");
  FCV_CHECK(p->slots || p->batch <= p->sessions, FCV_ERR_INVALID,
            "without slots the batch must not pass the sessions");
  FCV_CHECK(p->max_q >= 1 && p->max_length >= 0, FCV_ERR_INVALID, "need max_q >= 1 and max_length >= 0");
  FCV_CHECK(p->scale > 0.0f && p->scale < __builtin_inff(), FCV_ERR_INVALID,
            "scale must be positive and finite");
  const int64_t strides[] = {p->q_row, p->q_head, p->out_row, p->out_head, p->pk_row, p->pk_head,
                             p->pv_row, p->pv_head, p->k_session, p->k_row, p->k_head, p->v_session,
                             p->v_row, p->v_head};
  for (int64_t v : strides)
    FCV_CHECK(v >= 0 && v % 8 == 0, FCV_ERR_INVALID, "strides must be multiples of 8 elements, >= 0");
  FCV_CHECK(std::max({p->k_row, p->v_row, p->pk_row, p->pv_row}) < (1LL << 24), FCV_ERR_INVALID,
            "a key's row stride must be below 2^24 elements");
  if (p->tokens == 0) return FCV_OK;
  FCV_CHECK(p->q && p->k_cache && p->v_cache && p->lengths && p->out, FCV_ERR_INVALID, "null argument");
  FCV_CHECK(p->prefix_len == 0 || (p->prefix_k && p->prefix_v), FCV_ERR_INVALID, "null prefix");
  FCV_CHECK(aligned(p->q, 16) && aligned(p->out, 16) && aligned(p->k_cache, 16) &&
                aligned(p->v_cache, 16) && aligned(p->prefix_k, 16) && aligned(p->prefix_v, 16),
            FCV_ERR_INVALID, "q, out, the prefix and the caches must start on 16-byte boundaries");
  const Shape s = shape_of(*p);
  FCV_CHECK(s.prefix_blocks + s.own_blocks <= (1 << 23), FCV_ERR_INVALID,
            "the batch is too large for one call: split it");
  return FCV_OK;
}

template <class E, int D>
void launch(const Args& a, hipStream_t stream) {
  const unsigned blocks = (unsigned)(a.s.prefix_blocks + a.s.own_blocks);
  hipLaunchKernelGGL((prefix_attention_kernel<E, D>), dim3(blocks), dim3(256), 0, stream, a);
  const int64_t rows = (int64_t)a.p.tokens * a.p.n_heads;
  hipLaunchKernelGGL((join_kernel<E, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a);
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" size_t fcv_lm_prefix_attention_workspace_bytes(const FcvLmAttention* args) {
  if (fcv::lm::check(args) || args->tokens == 0) return 0;
  const fcv::lm::Shape s = fcv::lm::shape_of(*args);
  return (size_t)(fcv::lm::sums_bytes(*args, s) +
                  (int64_t)s.parts() * args->tokens * args->n_heads * args->head_dim * 4);
}

extern "C" int fcv_lm_prefix_attention(const FcvLmAttention* args, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  using namespace fcv::lm;
  if (int rc = check(args)) return rc;
  if (args->tokens == 0) return FCV_OK;
  const size_t need = fcv_lm_prefix_attention_workspace_bytes(args);
  FCV_CHECK(need == 0 || workspace, FCV_ERR_INVALID, "null workspace");
  FCV_CHECK(workspace_bytes >= need, FCV_ERR_INVALID,
            "workspace too small: need " + std::to_string(need) + " bytes");
  FCV_CHECK(aligned(workspace, 256), FCV_ERR_INVALID, "workspace must be 256-byte aligned");
  Args a{*args, shape_of(*args), nullptr, nullptr, args->scale * kLog2e};
  a.part_s = static_cast<float2*>(workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + sums_bytes(*args, a.s));
  const bool half = args->dtype == FCV_LM_F16;
  if (args->head_dim == 64)
    half ? launch<Half, 64>(a, stream) : launch<Bf16, 64>(a, stream);
  else
    half ? launch<Half, 128>(a, stream) : launch<Bf16, 128>(a, stream);
  FCV_HIP(hipGetLastError());
  return FCV_OK;
}
