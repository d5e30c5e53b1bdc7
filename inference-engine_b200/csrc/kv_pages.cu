// Copies pages of a paged KV cache: page dst[i] <- page src[i] in every layer's
// K and V cache, with one launch for all of them.
//
// Pure data movement: each moved page is read and written once, so the floor is
// 2 * pages * page bytes at the copy bandwidth.  A CTA moves 16 KB of one page of one
// cache (256 threads x four 16-byte vectors, all loaded before the first store);
// eight are resident on an SM, 128 KB of loads in flight.  220 pages of 32 KB in 64
// caches take 140 us, 6.6 TB/s; CTAs that stay and stride over the units took 160, as
// each waits for its own stores before it loads again.
//
// The page numbers and the cache addresses travel as kernel parameters (up to
// 32,764 bytes): no device copy of the lists, nothing whose lifetime the
// caller has to keep, and the call can be captured in a graph.  Longer lists
// take several launches.  The host rejects a page that is written twice, or
// both read and written, so no order of the copies matters.
#include <algorithm>
#include <new>

#include "common.cuh"

namespace ie {
namespace page_detail {

constexpr int kThreads = 256;
constexpr int kPer = 4;
constexpr int kCaches = 256;      // caches of one launch
constexpr int kFewPairs = 200;    // parameters below 4 KB
constexpr int kManyPairs = 3700;

template <int N>
struct Params {
  void* cache[kCaches];
  int32_t src[N], dst[N];
  int32_t caches, pairs;
  int64_t page_elems;             // elements of the copy type in a page
  int32_t pieces;                 // units of a page
};

template <typename E, int N>
__global__ void __launch_bounds__(kThreads)
copy_pages_kernel(const __grid_constant__ Params<N> p) {
  const int64_t per_cache = (int64_t)p.pairs * p.pieces;
  const int64_t units = per_cache * p.caches;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = (int)(u / per_cache);
    const int rest = (int)(u - c * per_cache);
    const int pair = rest / p.pieces, piece = rest - pair * p.pieces;
    E* base = static_cast<E*>(p.cache[c]);
    const E* src = base + p.src[pair] * p.page_elems;
    E* dst = base + p.dst[pair] * p.page_elems;
    const int64_t e0 = (int64_t)piece * (kThreads * kPer) + threadIdx.x;
    E v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (e0 + i * kThreads < p.page_elems) v[i] = src[e0 + i * kThreads];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (e0 + i * kThreads < p.page_elems) dst[e0 + i * kThreads] = v[i];
  }
}

template <typename E, int N>
int launch(void* const* caches, int ncaches, int64_t page_bytes, const int32_t* src,
           const int32_t* dst, int64_t n, cudaStream_t s) {
  Params<N> p;
  p.page_elems = page_bytes / (int64_t)sizeof(E);
  p.pieces = (int32_t)((p.page_elems + kThreads * kPer - 1) / (kThreads * kPer));
  for (int c0 = 0; c0 < ncaches; c0 += kCaches) {
    p.caches = std::min(kCaches, ncaches - c0);
    for (int c = 0; c < p.caches; ++c) p.cache[c] = caches[c0 + c];
    for (int64_t i0 = 0; i0 < n; i0 += N) {
      p.pairs = (int32_t)std::min<int64_t>(N, n - i0);
      std::copy(src + i0, src + i0 + p.pairs, p.src);
      std::copy(dst + i0, dst + i0 + p.pairs, p.dst);
      const int64_t units = (int64_t)p.caches * p.pairs * p.pieces;
      const int grid = (int)std::min<int64_t>(units, 0x7FFFFFFF);
      copy_pages_kernel<E, N><<<grid, kThreads, 0, s>>>(p);
      if (int rc = launch_status("copy_pages_kernel")) return rc;
    }
  }
  return IE_OK;
}

template <typename E>
int launch(void* const* caches, int ncaches, int64_t page_bytes, const int32_t* src,
           const int32_t* dst, int64_t n, cudaStream_t s) {
  return n <= kFewPairs ? launch<E, kFewPairs>(caches, ncaches, page_bytes, src, dst, n, s)
                        : launch<E, kManyPairs>(caches, ncaches, page_bytes, src, dst, n, s);
}

}  // namespace page_detail
}  // namespace ie

using namespace ie;

extern "C" int ie_copy_pages(void* const* caches, int32_t ncaches, int64_t page_bytes,
                             int64_t num_pages, const int32_t* src, const int32_t* dst,
                             int64_t n, void* stream) {
  IE_CHECK(ncaches >= 0 && n >= 0, "copy_pages: negative count");
  IE_CHECK(num_pages >= 0 && num_pages <= 0x7FFFFFFF, "copy_pages: %lld pages",
           (long long)num_pages);
  IE_CHECK(page_bytes > 0 && page_bytes % 2 == 0 && page_bytes <= (1ll << 28),
           "copy_pages: a page of %lld bytes", (long long)page_bytes);
  if (ncaches == 0 || n == 0) return IE_OK;
  IE_CHECK(caches && src && dst, "copy_pages: null pointer");
  bool wide = page_bytes % 16 == 0;
  for (int32_t c = 0; c < ncaches; ++c) {
    IE_CHECK(caches[c], "copy_pages: cache %d is null", c);
    const auto at = reinterpret_cast<uintptr_t>(caches[c]);
    IE_CHECK(at % 2 == 0, "copy_pages: cache %d is not aligned to its type", c);
    wide = wide && at % 16 == 0;
  }
  // one mark per page: 1 read, 2 written
  uint8_t few[4096];
  uint8_t* mark = few;
  if (num_pages > (int64_t)sizeof(few)) {
    mark = new (std::nothrow) uint8_t[num_pages];
    if (!mark) return set_error(IE_ERR_CUDA, "copy_pages: out of host memory");
  }
  std::fill(mark, mark + num_pages, (uint8_t)0);
  int rc = IE_OK;
  for (int64_t i = 0; i < n && !rc; ++i) {
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages)
      rc = set_error(IE_ERR_INVALID, "copy_pages: copy %lld is %d -> %d of %lld pages",
                     (long long)i, src[i], dst[i], (long long)num_pages);
    else
      mark[src[i]] |= 1;
  }
  for (int64_t i = 0; i < n && !rc; ++i) {
    if (mark[dst[i]])
      rc = set_error(IE_ERR_INVALID, "copy_pages: page %d is written and %s", dst[i],
                     mark[dst[i]] & 2 ? "written again" : "read");
    mark[dst[i]] |= 2;
  }
  if (mark != few) delete[] mark;
  if (rc) return rc;
  cudaStream_t s = as_stream(stream);
  if (wide) return page_detail::launch<uint4>(caches, ncaches, page_bytes, src, dst, n, s);
  return page_detail::launch<uint16_t>(caches, ncaches, page_bytes, src, dst, n, s);
}
