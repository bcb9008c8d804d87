// Copies of a cache's pages: the forks and compactions of a scheduler, in all layers.
//
// Bound: bandwidth (a page is read once and written once; of a fork the one source comes from cache).
// Split: a workgroup has one piece of one page in one layer.  The page numbers travel as kernel
// arguments: no copy to the device, nothing that the host has to keep, and a captured graph holds them.
#include <algorithm>
#include <cstring>
#include <new>
#include <string>
#include <vector>

#include "fp4.hpp"

namespace fcv {
namespace lm {
namespace {

constexpr int kThreads = 256, kMoves = 256;  // page pairs of a launch
constexpr int kDeep = 4, kPiece = kThreads * 16 * kDeep;

struct Moves {
  int32_t src[kMoves], dst[kMoves];
};

template <bool kWide>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(char* pages, int64_t layer_stride,
                                                              int64_t page_stride, int64_t page_bytes,
                                                              const Moves moves) {
  char* layer = pages + (int64_t)blockIdx.z * layer_stride;
  const char* src = layer + (int64_t)moves.src[blockIdx.y] * page_stride;
  char* dst = layer + (int64_t)moves.dst[blockIdx.y] * page_stride;
  if constexpr (kWide) {
    const int64_t at = (int64_t)blockIdx.x * kPiece + threadIdx.x * 16;
    u32x4 v[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (at + i * kThreads * 16 < page_bytes)
        v[i] = *reinterpret_cast<const u32x4*>(src + at + i * kThreads * 16);
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (at + i * kThreads * 16 < page_bytes)
        *reinterpret_cast<u32x4*>(dst + at + i * kThreads * 16) = v[i];
  } else {
    const int64_t end = min(page_bytes, ((int64_t)blockIdx.x + 1) * kPiece);
    for (int64_t i = (int64_t)blockIdx.x * kPiece + threadIdx.x; i < end; i += kThreads) dst[i] = src[i];
  }
}

}  // namespace
}  // namespace lm
}  // namespace fcv

extern "C" int fcv_copy_pages(void* pages, int32_t layers, int64_t layer_stride, int32_t n_pages,
                              int64_t page_stride, int64_t page_bytes, const int32_t* src_host,
                              const int32_t* dst_host, int32_t count, hipStream_t stream) {
  using namespace fcv::lm;
  FCV_CHECK(layers >= 0 && n_pages >= 0 && count >= 0, FCV_ERR_INVALID, "negative count");
  FCV_CHECK(layers <= 65535, FCV_ERR_INVALID, "at most 65535 layers");
  FCV_CHECK(page_bytes >= 0 && page_bytes <= (1LL << 36), FCV_ERR_INVALID, "page_bytes out of range");
  if (count == 0) return FCV_OK;
  FCV_CHECK(src_host && dst_host, FCV_ERR_INVALID, "null page lists");
  try {
    std::vector<int32_t> written(dst_host, dst_host + count);
    std::sort(written.begin(), written.end());
    for (int i = 0; i < count; ++i)
      FCV_CHECK(src_host[i] >= 0 && src_host[i] < n_pages && dst_host[i] >= 0 && dst_host[i] < n_pages,
                FCV_ERR_INVALID, "a page is outside the pool of " + std::to_string(n_pages));
    const auto twice = std::adjacent_find(written.begin(), written.end());
    FCV_CHECK(twice == written.end(), FCV_ERR_INVALID,
              "page " + std::to_string(*twice) + " is a destination twice");
    for (int i = 0; i < count; ++i)
      FCV_CHECK(!std::binary_search(written.begin(), written.end(), src_host[i]), FCV_ERR_INVALID,
                "page " + std::to_string(src_host[i]) + " is both a source and a destination");
  } catch (const std::bad_alloc&) {
    return fcv::fail(FCV_ERR_RUNTIME, "out of host memory");
  }
  if (layers == 0 || page_bytes == 0) return FCV_OK;
  FCV_CHECK(pages, FCV_ERR_INVALID, "null pages");
  FCV_CHECK(page_stride >= page_bytes && page_stride <= (1LL << 40), FCV_ERR_INVALID,
            "pages overlap, or lie too far apart");
  FCV_CHECK(layers == 1 ||
                (layer_stride >= page_bytes && layer_stride <= (1LL << 46) &&
                 (layer_stride >= (n_pages - 1) * page_stride + page_bytes ||
                  page_stride >= (layers - 1) * layer_stride + page_bytes)),
            FCV_ERR_INVALID, "layers overlap, or lie too far apart");
  const bool wide = aligned(pages, 16) && page_stride % 16 == 0 && page_bytes % 16 == 0 &&
                    (layers == 1 || layer_stride % 16 == 0);
  const int64_t pieces = (page_bytes + kPiece - 1) / kPiece;
  for (int first = 0; first < count; first += kMoves) {
    const int n = std::min(kMoves, count - first);
    Moves moves;
    std::memcpy(moves.src, src_host + first, n * sizeof(int32_t));
    std::memcpy(moves.dst, dst_host + first, n * sizeof(int32_t));
    const dim3 grid((unsigned)pieces, (unsigned)n, (unsigned)layers);
    if (wide)
      hipLaunchKernelGGL(copy_pages_kernel<true>, grid, dim3(kThreads), 0, stream,
                         static_cast<char*>(pages), layer_stride, page_stride, page_bytes, moves);
    else
      hipLaunchKernelGGL(copy_pages_kernel<false>, grid, dim3(kThreads), 0, stream,
                         static_cast<char*>(pages), layer_stride, page_stride, page_bytes, moves);
    FCV_HIP(hipGetLastError());
  }
  return FCV_OK;
}
