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

// out[p] for every position p of the CSR array: a warp owns kChunk consecutive
// positions, so that a few long rows and many short ones spread alike.  It finds
// the row of its first position by a 32-way search of the offsets and walks over
// the row ends inside the chunk; then every lane has, for each of its positions
// (32 apart), the row and the place in it, and loads a page number and the id.
// The chain of dependent loads (search, ends, page table, page) is what a warp
// waits for, and integer work is what the GPU spends, so places are 32-bit.
constexpr int kEach = 16;  // positions per lane
constexpr int kBatch = 8;  // of these, in flight at a time
constexpr int kChunk = kEach * 32;
constexpr int kEndBits = 9;  // kChunk = 2^9; the rows that end in a chunk fit into the other 23 bits
constexpr int kMaxRows = 1 << 22;
static_assert(kChunk == 1 << kEndBits, "places in a chunk");

struct GatherArgs {
  const int32_t* pool;
  int64_t num_pages;
  int page_size;
  const int32_t* pages;
  int64_t num_table;
  const int64_t *page_offsets, *offsets;
  int rows;
  int32_t* ids;
  int64_t num_ids;
  uint32_t* status;
};

__global__ void __launch_bounds__(kThreads) gather_kernel(const __grid_constant__ GatherArgs a) {
  const int lane = threadIdx.x % 32;
  bool bad = false;
  // every row's range, whatever the walk below makes of it
  for (int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * kThreads) {
    const int64_t o = __ldg(a.offsets + r), e = __ldg(a.offsets + r + 1);
    bad |= o < 0 || e < o || e > a.num_ids || e - o > 0x7fffffff;
  }
  const int64_t first = ((int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kChunk;
  const int64_t begin = __ldg(a.offsets), end = min(__ldg(a.offsets + a.rows), a.num_ids);
  if (first < end) {
    // the number of rows that end at or before `first`
    int row = 0;
    for (int n = a.rows; n > 0;) {
      const int step = (n + 31) / 32;
      const int at = row + (lane + 1) * step - 1;
      const int c = __popc(__ballot_sync(0xffffffffu, at < row + n && __ldg(a.offsets + at + 1) <= first));
      const int left = n - c * step;
      row += c * step;
      n = min(step - 1, left);
    }
    const int64_t here = __ldg(a.offsets + min(row, a.rows));  // row's first position
    // per position: the rows that end in the chunk up to it, and the last such end (from `first`)
    uint32_t walked[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) walked[k] = 0;
    for (int base = row; base < a.rows; base += 32) {
      const int64_t ends = __ldg(a.offsets + min(base + lane, a.rows - 1) + 1) - first;
      const uint32_t inside = __ballot_sync(0xffffffffu, ends >= 0 && ends < kChunk && base + lane < a.rows);
      const int n = __popc(inside & ~(inside + 1u));  // leading run of ends in the chunk
      // of a whole window of empty rows only the last counts
      const int from = n == 32 && __shfl_sync(0xffffffffu, (int)ends, 0) == __shfl_sync(0xffffffffu, (int)ends, 31) ? 31 : 0;
      for (int k = from; k < n; ++k) {
        const int e = __shfl_sync(0xffffffffu, (int)ends, k);
        const uint32_t w = ((uint32_t)(base + k + 1 - row) << kEndBits) | (uint32_t)e;
#pragma unroll
        for (int q = 0; q < kEach; ++q)
          if (e <= q * 32 + lane) walked[q] = w;
      }
      if (n < 32) break;
    }
    const int64_t before = first - here;  // places of `row` before the chunk
    const uint32_t size = (uint32_t)a.page_size;
    const int shift = (size & (size - 1)) == 0 ? 31 - __clz(size) : -1;
#pragma unroll
    for (int k0 = 0; k0 < kEach; k0 += kBatch) {
      int id[kBatch];
      int64_t at[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int pos = (k0 + k) * 32 + lane;
        const uint32_t w = walked[k0 + k];
        const int r = row + (int)(w >> kEndBits);
        const int64_t j64 = w ? pos - (int)(w & (kChunk - 1)) : before + pos;
        const bool here_ = r < a.rows && first + pos < end && first + pos >= begin && j64 >= 0 && j64 <= 0x7fffffff;
        const uint32_t j = here_ ? (uint32_t)j64 : 0u;
        const uint32_t t = shift >= 0 ? j >> shift : j / size;
        const int64_t table = here_ ? __ldg(a.page_offsets + r) + t : 0;
        const bool listed = here_ && table < __ldg(a.page_offsets + r + 1) && table >= 0 && table < a.num_table;
        const int64_t page = listed ? __ldg(a.pages + table) : -1;
        at[k] = page >= 0 && page < a.num_pages ? page * size + (j - t * size) : here_ ? -1 : -2;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) id[k] = at[k] >= 0 ? __ldg(a.pool + at[k]) : -1;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (at[k] > -2) a.ids[first + (k0 + k) * 32 + lane] = id[k];
        bad |= at[k] == -1;
      }
    }
  }
  if (bad && a.status) atomicOr(a.status, NS_STATUS_BAD_POOL_RANGE);
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
  if (num_rows > pages::kMaxRows) return fail(NS_ERR_UNSUPPORTED, "ns_paged_history_gather: more than 2^22 rows");
  const int64_t per_block = pages::kChunk * (pages::kThreads / 32);
  const int64_t blocks = (num_ids + per_block - 1) / per_block;
  if (blocks > 0x7fffffff) return fail(NS_ERR_UNSUPPORTED, "ns_paged_history_gather: num_ids is too large");
  const pages::GatherArgs g = {pool, num_pages, page_size, table, num_table_pages, page_offsets, offsets,
                               num_rows, out_ids, num_ids, status};
  pages::gather_kernel<<<(unsigned)blocks, pages::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return fail(NS_ERR_CUDA, std::string("ns_paged_history_gather launch: ") + cudaGetErrorString(e));
  return NS_OK;
}

}  // extern "C"
