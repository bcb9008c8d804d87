// The norm and rotation of a head in fp32, shared by the operators that append to a cache (qk_norm_rope.hip,
// kv_fp4.hip).
//
// A head takes D / 16 lanes, each with two 16-byte chunks.  A lane's chunks are j and j + R / 16 inside the
// rotated part, so that both members of a pair (i, i + R / 2) are in one lane (pairs (2 i, 2 i + 1) are
// inside a chunk anyway), and 2 j, 2 j + 1 behind it: no exchange but the sum of squares over 4 or 8
// neighbouring lanes.
#pragma once

#include "lm.hpp"

namespace fcv {
namespace lm {
namespace {

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

// The chunks c0 and c1 of lane j of a head of token `token`, as bits, normed by w (NULL: not) and rotated by
// p's tables, rounded once.  `turned`: the chunks are in the rotated part.
template <class E, int D, class P>
__device__ __forceinline__ void norm_rotate(const P& p, uint32_t token, const void* w, bool turned, int c0,
                                            int c1, s16x8& x0, s16x8& x1) {
  constexpr int L = D / 16;
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

}  // namespace
}  // namespace lm
}  // namespace fcv
