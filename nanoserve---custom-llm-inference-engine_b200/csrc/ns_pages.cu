// ns_pages.cu -- pages of a cache: copies between pages of many pools
// (ns_pages_copy), and token histories out of pages (ns_paged_history_gather).
//
// Both only move bytes.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <exception>
#include <string>
#include <vector>

#include "../../include/nanoserve_sampler.h"

namespace ns {
int fail(int code, const std::string& msg);

namespace pages {

constexpr int kThreads = 256;
constexpr int kMaxPools = 64;

// 300 pages of 32 KB in 16 pools (315 MB read and written) take 52 us, 49 at the
// 6446 GB/s of a copy; 32 pages 8 us, of which the launch is most.  Long lists are
// bound by the host's check of them: 87 thousand pages of 64 bytes take about 200 us, 140
// of them the check (68 us on the device as launches of 3500 pages).  Pages that are
// off the 16-byte grid move in smaller units: the 300 pages take 96 us where all
// sizes, strides and addresses are multiples of 4 bytes, 371 where they are not.
// A block copies kUnits units of one pool: the pool's moved pages one after the
// other, cut into equal pieces, so that small pages share a block and large ones
// are spread.  A thread has its four loads in flight together.
constexpr int kPerThread = 4;
constexpr int kUnits = kThreads * kPerThread;

struct CopyPool {
  char* base;
  int64_t stride;   // bytes between pages
  int64_t blocks;   // of the pools up to and with this one
  uint32_t units;   // of a page
  uint32_t unit;    // bytes: 16, 4 or 1
};

// The page numbers and pools of one launch travel as kernel parameters: no
// staging buffer to wait for, and a captured launch keeps its own copy.
template <int kPairs>
struct CopyPlan {
  static constexpr bool kChecked = true;
  CopyPool pool[kMaxPools];
  int32_t src[kPairs], dst[kPairs];
  int32_t pairs;
};

// Longer lists lie in device memory, and are checked as they are read.
struct ListedPlan {
  static constexpr bool kChecked = false;
  CopyPool pool[kMaxPools];
  const int32_t *src, *dst;
  int32_t pairs;
  int32_t num_pages;
  uint32_t* status;
};

template <typename Unit, typename Plan>
__device__ __forceinline__ void copy_block(const Plan& p, const CopyPool& pool, int64_t block) {
  const int64_t first = block * kUnits;
  const int page = (int)(first / pool.units);  // the first of the block's pages
  const uint32_t skip = (uint32_t)(first - (int64_t)page * pool.units);
  const Unit* from[kPerThread];
  Unit* to[kPerThread];
  Unit v[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const uint32_t u = skip + k * kThreads + threadIdx.x;  // below 2^32: a page has at most 2^31 units
    const uint32_t j = page + u / pool.units, at = u % pool.units;
    to[k] = nullptr;
    if (j < (uint32_t)p.pairs) {
      const int32_t src = p.src[j], dst = p.dst[j];
      if constexpr (!Plan::kChecked) {
        if ((uint32_t)src >= (uint32_t)p.num_pages || (uint32_t)dst >= (uint32_t)p.num_pages) {
          if (p.status) atomicOr(p.status, NS_STATUS_BAD_POOL_RANGE);
          continue;
        }
      }
      from[k] = reinterpret_cast<const Unit*>(pool.base + src * pool.stride) + at;
      to[k] = reinterpret_cast<Unit*>(pool.base + dst * pool.stride) + at;
      v[k] = __ldcs(from[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kPerThread; ++k)
    if (to[k]) __stcs(to[k], v[k]);
}

template <typename Plan>
__global__ void __launch_bounds__(kThreads) copy_kernel(const __grid_constant__ Plan p) {
  int k = 0;
  while ((int64_t)blockIdx.x >= p.pool[k].blocks) ++k;
  const CopyPool& pool = p.pool[k];
  const int64_t block = blockIdx.x - (k ? p.pool[k - 1].blocks : 0);
  if (pool.unit == 16) copy_block<uint4>(p, pool, block);
  else if (pool.unit == 4) copy_block<uint32_t>(p, pool, block);
  else copy_block<uint8_t>(p, pool, block);
}

// Fills in the pools of a launch of `count` pairs and enqueues it; says how many
// of the pools fitted into it (at least one).
template <typename Plan>
cudaError_t launch(Plan& p, const NsPagePool* pools, int num_pools, int64_t count, cudaStream_t st, int* taken) {
  p.pairs = (int32_t)count;
  int64_t blocks = 0;
  int k = 0;
  for (; k < std::min(num_pools, kMaxPools); ++k) {
    const NsPagePool& q = pools[k];
    const uint64_t grid = reinterpret_cast<uintptr_t>(q.base) | (uint64_t)q.page_bytes | (uint64_t)q.page_stride;
    const uint32_t unit = grid % 16 == 0 ? 16 : grid % 4 == 0 ? 4 : 1;
    const int64_t units = q.page_bytes / unit, more = (units * count + kUnits - 1) / kUnits;
    if (k > 0 && blocks + more > 0x7fffffff) break;
    blocks += more;
    p.pool[k] = {static_cast<char*>(q.base), q.page_stride, blocks, (uint32_t)units, unit};
  }
  *taken = k;
  void* args[] = {&p};
  return cudaLaunchKernel(reinterpret_cast<const void*>(copy_kernel<Plan>), dim3((unsigned)blocks), dim3(kThreads), args, 0, st);
}

template <int kPairs>
cudaError_t launch_pairs(const NsPagePool* pools, int num_pools, const int64_t* src, const int64_t* dst, int count,
                         cudaStream_t st) {
  CopyPlan<kPairs> p;
  for (int j = 0; j < count; ++j) p.src[j] = (int32_t)src[j], p.dst[j] = (int32_t)dst[j];
  for (int k = 0, taken = 0; k < num_pools; k += taken) {
    const cudaError_t e = launch(p, pools + k, num_pools - k, count, st, &taken);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

thread_local std::vector<uint64_t> marks;  // a bit per page, all clear between calls

// What is wrong with a plan, in loops that only note it.  `mark` has a bit per page.
struct Wrong {
  bool outside, twice, both;
};
Wrong look(uint64_t* __restrict__ mark, int64_t num_pages, const int64_t* __restrict__ src,
           const int64_t* __restrict__ dst, int64_t count) {
  const uint64_t last = (uint64_t)num_pages - 1;
  uint64_t sign = 0;  // the top bit: of a page, or of its distance to the last one
  for (int64_t j = 0; j < count; ++j) {
    const uint64_t s = (uint64_t)src[j], d = (uint64_t)dst[j];
    sign |= s | d | (last - s) | (last - d);
  }
  if (sign >> 63) return {true, false, false};
  uint64_t twice = 0, both = 0;
  for (int64_t j = 0; j < count; ++j) {
    const uint64_t was = mark[dst[j] >> 6], bit = 1ull << (dst[j] & 63);
    mark[dst[j] >> 6] = was | bit;
    twice |= was & bit;
  }
  for (int64_t j = 0; j < count; ++j) both |= mark[src[j] >> 6] >> (src[j] & 63);
  return {false, twice != 0, (both & 1) != 0};
}

// Empty where the plan is sound, else what is wrong with it.
std::string check_plan(int64_t num_pages, const int64_t* src, const int64_t* dst, int64_t count) {
  // a compaction's plan: both lists ascend, and every destination is below every source
  if (src[0] > dst[count - 1] && dst[0] >= 0 && src[count - 1] < num_pages) {
    int64_t j = 1;
    while (j < count && dst[j - 1] < dst[j] && src[j - 1] <= src[j]) ++j;
    if (j == count) return "";
  }
  const size_t words = (size_t)(num_pages + 63) / 64;
  if (marks.size() < words) marks.resize(words, 0);
  uint64_t* mark = marks.data();
  const auto marked = [&](int64_t p) { return mark[p >> 6] >> (p & 63) & 1; };
  const Wrong wrong = look(mark, num_pages, src, dst, count);
  if (wrong.outside)
    for (int64_t j = 0;; ++j)
      if (src[j] < 0 || src[j] >= num_pages || dst[j] < 0 || dst[j] >= num_pages)
        return "page outside [0, " + std::to_string(num_pages) + "): " + std::to_string(src[j]) + " -> " +
               std::to_string(dst[j]);
  const auto clear = [&] {
    if ((size_t)count > words) std::fill(mark, mark + words, 0);
    else
      for (int64_t j = 0; j < count; ++j) mark[dst[j] >> 6] = 0;
  };
  if (!wrong.twice && !wrong.both) {
    clear();
    return "";
  }
  int64_t at = 0;
  if (!wrong.twice) {
    while (!marked(src[at])) ++at;
    clear();
    return "page " + std::to_string(src[at]) + " is both a source and a destination";
  }
  clear();
  for (; !marked(dst[at]); ++at) mark[dst[at] >> 6] |= 1ull << (dst[at] & 63);
  clear();
  return "page " + std::to_string(dst[at]) + " is a destination twice";
}

// out[p] for every position p of the CSR array: a warp owns kEach * 32 consecutive
// positions, so that a few long rows and many short ones spread alike.  It finds
// the row of its first position by a 32-way search of the offsets; then its lanes
// fetch what 32 rows from there need, one each, and leave it in shared memory, and
// every lane looks up, for each of its positions (32 apart), its row, the page
// number and the id.  Runs of empty rows are skipped by another search.  What is
// spent is integer work and the latency of that chain of loads: places are 32-bit,
// and four positions per lane are in flight.
//
// 9.4 M ids in pages of 16 take 31 us (78 MB: 12 at the 6446 GB/s of a copy), the
// same for pages in order, with issue slots 57% and L1 60% busy.  A block per row took
// 57 us, a warp that takes the rows of its chunk one after the other 62.

// A row as its positions in a chunk see it: position pos is place p = pos + shift
// of the row (counted from the first page that the tables hold), on page
// list[p / page_size] if that is below `pages`.
struct __align__(16) RowPages {
  const int32_t* list;
  uint32_t pages;
  int shift;
};

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
  uint32_t row_pages;  // of 2^31 ids
  uint32_t* status;
};

// kPow2: the page size is a power of two.  kEach: positions per lane.
template <bool kPow2, int kEach>
__global__ void __launch_bounds__(kThreads, 6) gather_kernel(const __grid_constant__ GatherArgs a) {
  constexpr int kChunk = kEach * 32, kBatch = kEach < 4 ? kEach : 4;
  __shared__ RowPages s_rows[kThreads / 32][32];
  const int lane = threadIdx.x % 32;
  bool bad = false;
  // every row's range, whatever the walk below makes of it
  for (int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * kThreads) {
    const int64_t o = __ldg(a.offsets + r), e = __ldg(a.offsets + r + 1);
    bad |= o < 0 || e < o || e > a.num_ids || e - o > 0x7fffffff;
  }
  const int64_t first = ((int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kChunk;
  const int64_t end = min(__ldg(a.offsets + a.rows), a.num_ids);
  if (first < end) {
    // the first row, from `row` on, that ends behind position `pos`
    const auto find = [&](int row, int64_t pos) {
      for (int n = a.rows - row; n > 0;) {
        const int step = (n + 31) / 32;
        const int at = row + (lane + 1) * step - 1;
        const int c = __popc(__ballot_sync(0xffffffffu, at < row + n && __ldg(a.offsets + at + 1) <= pos));
        const int left = n - c * step;
        row += c * step;
        n = min(step - 1, left);
      }
      return row;
    };
    const uint32_t size = (uint32_t)a.page_size;
    const int bits = 31 - __clz(size);
    const uint32_t num_pages = (uint32_t)min(a.num_pages, (int64_t)0x80000000);  // page numbers are 31 bits
    int32_t* out = a.ids + first + lane;
    RowPages* rows = s_rows[threadIdx.x / 32];
    for (int base = find(0, first); base < a.rows;) {
      const int r = min(base + lane, a.rows - 1);
      const int64_t o = __ldg(a.offsets + r) - first, e = __ldg(a.offsets + r + 1) - first;
      const int64_t table = __ldg(a.page_offsets + r), table_end = min(__ldg(a.page_offsets + r + 1), a.num_table);
      const int64_t held = max(table, (int64_t)0);
      const int64_t shift = (int64_t)(0 - (uint64_t)o - ((uint64_t)held - (uint64_t)table) * size);
      // Page offsets may be any 64-bit numbers: `far` says where a difference of them could wrap around into the
      // tables.  A place before its row's table is negative: as 32 bits without a sign it is behind the pages of
      // 2^31 ids, which are all that a row may have.  (16384 rows take 30.8 us, as without the two; with the smaller
      // number of pages for all rows, in place of a choice, 32.3.)
      const bool far = table_end < 0 || (int)(table >> 32) < -1;
      const uint32_t most = table < 0 ? a.row_pages : 0x7fffffffu;
      RowPages mine;
      mine.list = a.pages + held;
      mine.pages = !far && o <= e && shift > -0x40000000 && shift < 0x7fffffff - kChunk
                       ? (uint32_t)max((int64_t)0, min(table_end - held, (int64_t)most)) : 0u;
      mine.shift = (int)shift;
      __syncwarp();
      rows[lane] = mine;
      __syncwarp();
      // the window's positions, and the rows that end among them
      const int n = min(32, a.rows - base);
      const int64_t all = __shfl_sync(0xffffffffu, e, n - 1);
      const int from = (int)max((int64_t)0, min(__shfl_sync(0xffffffffu, o, 0), (int64_t)kChunk));
      const int to = (int)max((int64_t)0, min(min(all, end - first), (int64_t)kChunk));
      const int ends = __popc(__ballot_sync(0xffffffffu, e < kChunk) & (uint32_t)((1ull << n) - 1));
      const int e32 = (int)max((int64_t)-1, min(e, (int64_t)kChunk));
      base += 32;
      if (to <= from) {  // empty rows: there may be many
        if (all >= kChunk) break;
        base = find(base, first + max(all, (int64_t)0));
        continue;
      }
      uint32_t at[(kEach + 3) / 4] = {};  // a byte per position: which of the window's rows it is in
      for (int k = 0; k < min(ends, n - 1); ++k) {
        const int x = __shfl_sync(0xffffffffu, e32, k);
#pragma unroll
        for (int q = 0; q < kEach; ++q)
          if (x <= q * 32 + lane) at[q / 4] += 1u << (q % 4 * 8);
      }
#pragma unroll
      for (int k0 = 0; k0 < kEach; k0 += kBatch) {
        uint32_t rest[kBatch], id[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int pos = (k0 + k) * 32 + lane;
          const RowPages p = rows[(at[(k0 + k) / 4] >> ((k0 + k) % 4 * 8)) & 0xffu];
          const uint32_t place = (uint32_t)(pos + p.shift);
          const uint32_t t = kPow2 ? place >> bits : place / size;
          rest[k] = kPow2 ? place & (size - 1) : place - t * size;
          id[k] = pos >= from && pos < to && t < p.pages ? (uint32_t)__ldg(p.list + t) : ~0u;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (id[k] < num_pages) id[k] = (uint32_t)__ldg(a.pool + ((uint64_t)id[k] * size + rest[k]));
          else id[k] = ~0u, rest[k] = ~0u;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int pos = (k0 + k) * 32 + lane;
          if (pos >= from && pos < to) {
            out[(k0 + k) * 32] = (int32_t)id[k];
            bad |= rest[k] == ~0u;
          }
        }
      }
      if (all >= kChunk) break;
    }
  }
  if (bad && a.status) atomicOr(a.status, NS_STATUS_BAD_POOL_RANGE);
}

int check_pools(const NsPagePool* pools, int32_t num_pools, int64_t num_pages, int64_t count) {
  if (num_pools < 0 || num_pages < 0 || count < 0)
    return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: num_pools, num_pages or count < 0");
  if (num_pages > 0x7fffffff) return fail(NS_ERR_UNSUPPORTED, "ns_pages_copy: more than 2^31 - 1 pages");
  if (num_pools == 0 || count == 0) return NS_OK;
  if (!pools) return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: null pointer");
  for (int32_t k = 0; k < num_pools; ++k) {
    if (!pools[k].base || pools[k].page_bytes <= 0 || pools[k].page_stride < pools[k].page_bytes)
      return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: pool " + std::to_string(k) +
                                          " has no base, no bytes or pages that overlap");
    if (pools[k].page_bytes > 0x7fffffff)
      return fail(NS_ERR_UNSUPPORTED, "ns_pages_copy: pages of more than 2^31 - 1 bytes");
    if (count > (int64_t{0x7fffffff} * kUnits) / pools[k].page_bytes)  // its blocks, of kUnits bytes at least, in 31 bits
      return fail(NS_ERR_UNSUPPORTED, "ns_pages_copy: more than 2^41 bytes of a pool");
  }
  return NS_OK;
}

}  // namespace pages
}  // namespace ns

extern "C" {

int ns_pages_check(int64_t num_pages, const int64_t* src, const int64_t* dst, int64_t count) {
  using namespace ns;
  if (num_pages < 0 || count < 0) return fail(NS_ERR_INVALID_ARG, "ns_pages_check: num_pages or count < 0");
  if (count == 0) return NS_OK;
  if (!src || !dst) return fail(NS_ERR_INVALID_ARG, "ns_pages_check: null pointer");
  try {
    const std::string wrong = pages::check_plan(num_pages, src, dst, count);
    if (!wrong.empty()) return fail(NS_ERR_INVALID_ARG, "ns_pages_copy: " + wrong);
  } catch (const std::exception&) {  // of the marks: num_pages bits
    pages::marks.clear();
    return fail(NS_ERR_UNSUPPORTED, "ns_pages_copy: out of host memory");
  }
  return NS_OK;
}

int ns_pages_copy(const NsPagePool* pools, int32_t num_pools, int64_t num_pages, const int64_t* src,
                  const int64_t* dst, int64_t count, void* stream) {
  using namespace ns;
  int rc = pages::check_pools(pools, num_pools, num_pages, count);
  if (rc != NS_OK || num_pools == 0 || count == 0) return rc;
  rc = ns_pages_check(num_pages, src, dst, count);
  if (rc != NS_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  constexpr int kSmall = 64, kMiddle = 512, kLarge = 3500;  // the parameters of a launch have 32764 bytes
  for (int64_t j = 0; j < count; j += kLarge) {
    const int n = (int)std::min<int64_t>(kLarge, count - j);
    const auto launch = n <= kSmall    ? pages::launch_pairs<kSmall>
                        : n <= kMiddle ? pages::launch_pairs<kMiddle>
                                       : pages::launch_pairs<kLarge>;
    const cudaError_t e = launch(pools, num_pools, src + j, dst + j, n, st);
    if (e != cudaSuccess) return fail(NS_ERR_CUDA, std::string("ns_pages_copy launch: ") + cudaGetErrorString(e));
  }
  return NS_OK;
}

int ns_pages_copy_listed(const NsPagePool* pools, int32_t num_pools, int64_t num_pages, const int32_t* src,
                         const int32_t* dst, int64_t count, uint32_t* status, void* stream) {
  using namespace ns;
  const int rc = pages::check_pools(pools, num_pools, num_pages, count);
  if (rc != NS_OK || num_pools == 0 || count == 0) return rc;
  if (!src || !dst) return fail(NS_ERR_INVALID_ARG, "ns_pages_copy_listed: null pointer");
  if (count > 0x7fffffff) return fail(NS_ERR_UNSUPPORTED, "ns_pages_copy_listed: more than 2^31 - 1 pages");
  pages::ListedPlan p;
  p.src = src, p.dst = dst, p.status = status, p.num_pages = (int32_t)num_pages;
  for (int k = 0, taken = 0; k < num_pools; k += taken) {
    const cudaError_t e = pages::launch(p, pools + k, num_pools - k, count, static_cast<cudaStream_t>(stream), &taken);
    if (e != cudaSuccess)
      return fail(NS_ERR_CUDA, std::string("ns_pages_copy_listed launch: ") + cudaGetErrorString(e));
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
  if (num_rows > 1 << 30)  // the search's row numbers stay in 32 bits
    return fail(NS_ERR_UNSUPPORTED, "ns_paged_history_gather: more than 2^30 rows");
  if (!page_offsets || !offsets || !out_ids || (!pool && num_pages > 0) || (!table && num_table_pages > 0))
    return fail(NS_ERR_INVALID_ARG, "ns_paged_history_gather: null device pointer");
  // A warp's search costs as much as several of its positions: sixteen per lane where there are warps enough to
  // fill the GPU (9.4 M ids: 31 us against 37 with eight), eight where there are not (278 K ids: 5.5 us
  // against 6.1).  Where rows have fewer than eight ids, a warp of more positions would walk through many rows, 32 at
  // a time: one position per lane (16384 rows of 0 or 1 ids 56 us with eight, 8 with one; of 3 to 5 ids 12, 6; of 8
  // to 10 ids 8 with eight).
  const bool many = num_ids >= (int64_t)148 * 48 * 32 * 16, few = num_ids / 8 < num_rows;
  const int64_t per_block = pages::kThreads * (few ? 1 : many ? 16 : 8);
  const int64_t blocks = (num_ids + per_block - 1) / per_block;
  if (blocks > 0x7fffffff) return fail(NS_ERR_UNSUPPORTED, "ns_paged_history_gather: num_ids is too large");
  const pages::GatherArgs g = {pool, num_pages, page_size, table, num_table_pages, page_offsets, offsets,
                               num_rows, out_ids, num_ids, 0x7fffffffu / (uint32_t)page_size + 1, status};
  const bool pow2 = (page_size & (page_size - 1)) == 0;
  const auto kernel = few    ? (pow2 ? pages::gather_kernel<true, 1> : pages::gather_kernel<false, 1>)
                      : many ? (pow2 ? pages::gather_kernel<true, 16> : pages::gather_kernel<false, 16>)
                             : (pow2 ? pages::gather_kernel<true, 8> : pages::gather_kernel<false, 8>);
  kernel<<<(unsigned)blocks, pages::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(g);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return fail(NS_ERR_CUDA, std::string("ns_paged_history_gather launch: ") + cudaGetErrorString(e));
  return NS_OK;
}

}  // extern "C"
