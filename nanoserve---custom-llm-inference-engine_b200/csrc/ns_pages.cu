// ns_pages.cu -- pages of a cache: copies between pages of many pools
// (ns_pages_copy), and token histories out of pages (ns_paged_history_gather).
//
// Both only move bytes.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <string>
#include <vector>

#include "../../include/nanoserve_sampler.h"

namespace ns {
int fail(int code, const std::string& msg);

namespace pages {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 148 * 8;
constexpr int kMaxPools = 64;

// The page numbers and pools of one launch travel as kernel parameters: no
// staging buffer to wait for, and a captured launch keeps its own copy.
template <int kPairs>
struct CopyPlan {
  NsPagePool pool[kMaxPools];
  int32_t src[kPairs], dst[kPairs];
  int32_t pools, pairs;
};

// Unit of all page sizes, strides and bases of the plan: 16 bytes, or 1.
template <int kPairs, typename Unit>
__global__ void __launch_bounds__(kThreads) copy_kernel(const __grid_constant__ CopyPlan<kPairs> p) {
  for (int k = 0; k < p.pools; ++k) {
    const int64_t units = p.pool[k].page_bytes / (int64_t)sizeof(Unit);
    const int64_t stride = p.pool[k].page_stride / (int64_t)sizeof(Unit);
    Unit* base = static_cast<Unit*>(p.pool[k].base);
    const int64_t total = units * p.pairs;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
      const int j = (int)(i / units);
      const int64_t u = i % units;
      base[p.dst[j] * stride + u] = base[p.src[j] * stride + u];
    }
  }
}

template <int kPairs>
cudaError_t launch(const NsPagePool* pools, int num_pools, const int64_t* src, const int64_t* dst, int count,
                   bool wide, cudaStream_t st) {
  CopyPlan<kPairs> p;
  p.pools = num_pools;
  p.pairs = count;
  int64_t bytes = 0;
  for (int k = 0; k < num_pools; ++k) {
    p.pool[k] = pools[k];
    bytes = std::max(bytes, pools[k].page_bytes * count);
  }
  for (int j = 0; j < count; ++j) p.src[j] = (int32_t)src[j], p.dst[j] = (int32_t)dst[j];
  const int64_t blocks = (bytes / (wide ? 16 : 1) + kThreads - 1) / kThreads;
  const int grid = (int)std::min<int64_t>(blocks, kMaxBlocks);
  if (wide) copy_kernel<kPairs, uint4><<<grid, kThreads, 0, st>>>(p);
  else copy_kernel<kPairs, uint8_t><<<grid, kThreads, 0, st>>>(p);
  return cudaGetLastError();
}

// Empty where the plan is sound, else what is wrong with it.
std::string check_plan(int64_t num_pages, const int64_t* src, const int64_t* dst, int64_t count) {
  for (int64_t j = 0; j < count; ++j)
    if (src[j] < 0 || src[j] >= num_pages || dst[j] < 0 || dst[j] >= num_pages)
      return "page outside [0, " + std::to_string(num_pages) + "): " + std::to_string(src[j]) + " -> " +
             std::to_string(dst[j]);
  std::vector<int64_t> d(dst, dst + count);
  std::sort(d.begin(), d.end());
  for (int64_t j = 1; j < count; ++j)
    if (d[j] == d[j - 1]) return "page " + std::to_string(d[j]) + " is a destination twice";
  for (int64_t j = 0; j < count; ++j)
    if (std::binary_search(d.begin(), d.end(), src[j]))
      return "page " + std::to_string(src[j]) + " is both a source and a destination";
  return "";
}

__global__ void __launch_bounds__(kThreads)
    gather_kernel(const int32_t* __restrict__ pool, int64_t num_pages, int page_size, const int32_t* __restrict__ pages,
                  int64_t num_table, const int64_t* __restrict__ page_offsets, const int64_t* __restrict__ offsets,
                  int rows, int32_t* __restrict__ ids, int64_t num_ids, uint32_t* status) {
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t o0 = offsets[r], n = offsets[r + 1] - o0;
    const int64_t t0 = page_offsets[r], tn = page_offsets[r + 1] - t0;
    bool bad = n < 0 || o0 < 0 || o0 + n > num_ids;
    for (int64_t j = threadIdx.x; j < n; j += kThreads) {
      const int64_t at = o0 + j;
      if (at < 0 || at >= num_ids) continue;
      const int64_t t = j / page_size;
      int32_t id = -1;
      if (t < tn && t0 + t >= 0 && t0 + t < num_table) {
        const int64_t page = pages[t0 + t];
        if (page >= 0 && page < num_pages) id = pool[page * page_size + j % page_size];
        else bad = true;
      } else {
        bad = true;
      }
      ids[at] = id;
    }
    if (bad && status) atomicOr(status, NS_STATUS_BAD_POOL_RANGE);
  }
}

}  // namespace pages
}  // namespace ns

extern "C" {

int ns_pages_copy(const NsPagePool* pools, int32_t num_pools, int64_t num_pages, const int64_t* src,
                  const int64_t* dst, int64_t count, void* stream) {
  using namespace ns;
  if (num_pools < 0 || num_pages < 0 || count < 0)
    return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: num_pools, num_pages or count < 0");
  if (num_pages > 0x7fffffff) return fail(NS_ERR_UNSUPPORTED, "ns_pages_copy: more than 2^31 - 1 pages");
  if (num_pools == 0 || count == 0) return NS_OK;
  if (!pools || !src || !dst) return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: null pointer");
  bool wide = true;
  for (int32_t k = 0; k < num_pools; ++k) {
    if (!pools[k].base || pools[k].page_bytes <= 0 || pools[k].page_stride < pools[k].page_bytes)
      return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: pool " + std::to_string(k) +
                                          " has no base, no bytes or pages that overlap");
    wide = wide && (reinterpret_cast<uintptr_t>(pools[k].base) | (uint64_t)pools[k].page_bytes |
                    (uint64_t)pools[k].page_stride) % 16 == 0;
  }
  try {
    const std::string wrong = pages::check_plan(num_pages, src, dst, count);
    if (!wrong.empty()) return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: " + wrong);
  } catch (const std::bad_alloc&) {
    return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: out of host memory");
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  constexpr int kSmall = 128, kLarge = 3500;
  for (int32_t k = 0; k < num_pools; k += pages::kMaxPools) {
    const int np = std::min<int32_t>(pages::kMaxPools, num_pools - k);
    for (int64_t j = 0; j < count; j += kLarge) {
      const int n = (int)std::min<int64_t>(kLarge, count - j);
      const cudaError_t e = n <= kSmall ? pages::launch<kSmall>(pools + k, np, src + j, dst + j, n, wide, st)
                                        : pages::launch<kLarge>(pools + k, np, src + j, dst + j, n, wide, st);
      if (e != cudaSuccess) return fail(NS_ERR_CUDA, std::string("ns_pages_copy launch: ") + cudaGetErrorString(e));
    }
  }
  return NS_OK;
}

int ns_paged_history_gather(const int32_t* pool, int64_t num_pages, int32_t page_size, const int32_t* table,
                            int64_t num_table_pages, const int64_t* page_offsets, const int64_t* offsets,
                            int32_t num_rows, int32_t* out_ids, int64_t num_ids, uint32_t* status, void* stream) {
  using namespace ns;
  if (num_rows < 0 || num_pages < 0 || num_table_pages < 0 || num_ids < 0)
    return fail(NS_ERR_INVALID_ARG, "ns_paged_history_gather: num_rows, num_pages, num_table_pages or num_ids < 0");
  if (page_size <= 0) return fail(NS_ERR_INVALID_ARG, "ns_paged_history_gather: page_size must be positive");
  if (num_rows == 0 || num_ids == 0) return NS_OK;
  if (!page_offsets || !offsets || !out_ids || (!pool && num_pages > 0) || (!table && num_table_pages > 0))
    return fail(NS_ERR_INVALID_ARG, "ns_paged_history_gather: null device pointer");
  const int grid = std::min(num_rows, pages::kMaxBlocks);
  pages::gather_kernel<<<grid, pages::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      pool, num_pages, page_size, table, num_table_pages, page_offsets, offsets, num_rows, out_ids, num_ids, status);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return fail(NS_ERR_CUDA, std::string("ns_paged_history_gather launch: ") + cudaGetErrorString(e));
  return NS_OK;
}

}  // extern "C"
