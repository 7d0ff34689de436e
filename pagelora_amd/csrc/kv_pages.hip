// Pages copied within a paged KV pool, in every layer (gfx950):
//   page dst[i] <- page src[i].
// The pages are few enough to name in the kernel's arguments: no list is
// uploaded, and nothing outlives the call.  A workgroup copies kBytes of one
// page of one layer, all its loads in flight before its stores, both past the
// caches.  Bound by HBM: 256 pages of 64 KiB in 36 layers 214 us, 5.7 TB/s read and
// written; one page 3.2 us, a launch's latency.
#include <vector>

#include "pl_common.h"

namespace pl {
namespace pages {

constexpr int kThreads = 256;
constexpr int kLoads = 4;                       // 16-byte loads of a thread
constexpr int kBytes = kThreads * kLoads * 16;  // of a workgroup
constexpr int kPairs = 448;                     // pages named by one launch (3.5 KiB of arguments)

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct Args {
  char* cache;
  int64_t layer_stride, page_stride, page_bytes;  // bytes
  int pieces;                                     // workgroups per page
  int32_t src[kPairs], dst[kPairs];
};

__global__ __launch_bounds__(kThreads) void copy_kernel(Args A) {
  const int pair = blockIdx.x / A.pieces, piece = blockIdx.x % A.pieces;
  char* layer = A.cache + (int64_t)blockIdx.y * A.layer_stride;
  const char* from = layer + (int64_t)A.src[pair] * A.page_stride;
  char* to = layer + (int64_t)A.dst[pair] * A.page_stride;
  const int64_t at = (int64_t)piece * kBytes + threadIdx.x * 16;
  u32x4 x[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    if (at + i * kThreads * 16 < A.page_bytes) x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + at + i * kThreads * 16));
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    if (at + i * kThreads * 16 < A.page_bytes) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(to + at + i * kThreads * 16));
}

}  // namespace pages
}  // namespace pl

using namespace pl;

extern "C" int pl_kv_copy_pages(void* cache, int64_t layer_stride, int64_t page_stride, int64_t page_elements,
                                int num_layers, int64_t num_pages, const int32_t* src_h, const int32_t* dst_h, int n,
                                int dtype, void* stream) {
  if (n < 0 || num_layers < 0 || page_elements < 0) return fail(PL_ERR_INVALID, "n, num_layers and page_elements must be >= 0");
  if (dtype != PL_DTYPE_F32 && dtype != PL_DTYPE_F16 && dtype != PL_DTYPE_BF16)
    return fail(PL_ERR_UNSUPPORTED, "dtype %d", dtype);
  if (n == 0 || num_layers == 0 || page_elements == 0) return ok();
  if (!cache || !src_h || !dst_h) return fail(PL_ERR_INVALID, "null pointer argument");
  if (num_pages <= 0 || num_pages > INT32_MAX) return fail(PL_ERR_INVALID, "num_pages must be in [1, 2^31)");
  const int eb = dtype_bytes(dtype), per = 16 / eb;
  if (layer_stride % per || page_stride % per || page_elements % per)
    return fail(PL_ERR_INVALID, "strides and page_elements must be multiples of %d elements", per);
  if (page_elements > page_stride && num_pages > 1)
    return fail(PL_ERR_INVALID, "pages of %lld elements overlap at a stride of %lld", (long long)page_elements,
                (long long)page_stride);
  if ((uintptr_t)cache % 16) return fail(PL_ERR_INVALID, "cache must be 16-byte aligned");
  // a launch has less than 2^32 threads per dimension
  const int64_t pieces = page_elements > (1ll << 40) ? 1 << 24 : (page_elements * eb + pages::kBytes - 1) / pages::kBytes;
  if (num_layers > 65535 || pieces * pages::kPairs >= (1 << 24))
    return fail(PL_ERR_UNSUPPORTED, "%d layers or pages of %lld elements are too many", num_layers,
                (long long)page_elements);
  for (int i = 0; i < n; ++i)
    if (src_h[i] < 0 || src_h[i] >= num_pages || dst_h[i] < 0 || dst_h[i] >= num_pages)
      return fail(PL_ERR_INVALID, "copy %d: page %d to page %d is outside the %lld-page pool", i, src_h[i], dst_h[i],
                  (long long)num_pages);
  auto clash = [&](int i, bool source) {
    return fail(PL_ERR_INVALID, "copy %d: page %d is %s", i, dst_h[i], source ? "also a source" : "written twice");
  };
  if ((int64_t)n * n <= num_pages) {
    for (int i = 0; i < n; ++i)
      for (int j = 0; j < n; ++j)
        if (dst_h[i] == src_h[j] || (j < i && dst_h[i] == dst_h[j])) return clash(i, dst_h[i] == src_h[j]);
  } else {
    try {
      std::vector<uint8_t> role((size_t)num_pages, 0);  // 1: some copy reads the page, 2: one writes it
      for (int i = 0; i < n; ++i) role[src_h[i]] = 1;
      for (int i = 0; i < n; ++i) {
        if (role[dst_h[i]]) return clash(i, role[dst_h[i]] == 1);
        role[dst_h[i]] = 2;
      }
    } catch (...) {
      return fail(PL_ERR_INVALID, "no host memory to check the copies of a %lld-page pool", (long long)num_pages);
    }
  }
  pages::Args a{};
  a.cache = (char*)cache;
  a.layer_stride = layer_stride * eb;
  a.page_stride = page_stride * eb;
  a.page_bytes = page_elements * eb;
  a.pieces = (int)pieces;
  for (int i0 = 0; i0 < n; i0 += pages::kPairs) {
    const int m = n - i0 < pages::kPairs ? n - i0 : pages::kPairs;
    for (int i = 0; i < m; ++i) {
      a.src[i] = src_h[i0 + i];
      a.dst[i] = dst_h[i0 + i];
    }
    hipLaunchKernelGGL(pages::copy_kernel, dim3((unsigned)(m * a.pieces), num_layers), dim3(pages::kThreads), 0,
                       (hipStream_t)stream, a);
    PL_LAUNCH_CHECK("kv copy_kernel");
  }
  return ok();
}
