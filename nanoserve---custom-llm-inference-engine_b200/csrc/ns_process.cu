// ns_process.cu -- penalties for repeated tokens, biases and grammar masks on
// logits (ns_process_logits).
//
// For every row, with seen(v) and c(v) counted from the row's history:
//   x = seen ? (x < 0 ? x * rp : x / rp) : x
//   x = x - freq * c - pres  where c > 0
//   x = x + bias             where the row has one
//   x = -inf                 where the row's mask bit is 0
//
// Two kernels.  tile_kernel writes whole rows (or, in place, what a mask
// forbids): a block owns a tile of vocabulary ids of one row.
// sparse_kernel serves calls in place without masks, which change only the ids
// that a history or a bias names: a block owns a row (or a part of its ids).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "ns_device.cuh"

namespace ns {
int fail(int code, const std::string& msg);

namespace proc {

constexpr int kMostThreads = 512;  // of a block of tile_kernel
// Most ids of a tile, and ids of it that are listed: three blocks of the largest tiles share an SM's memory.
template <typename In>
constexpr int kTile = sizeof(In) == 4 ? 12032 : 16384;
template <typename In>
constexpr int kHits = sizeof(In) == 4 ? 1280 : 4096;
constexpr int kPre = 4;       // history entries per thread that are in flight at a time
constexpr uint32_t kMaxTries = 1u << 22;

// Word of one vocabulary id: occurrences after the prompt in the low bits.
constexpr uint32_t kInPrompt = 1u << 31;
constexpr uint32_t kBias = 1u << 30;
constexpr uint32_t kBiasTwice = 1u << 29;
constexpr uint32_t kCount = kBiasTwice - 1;
constexpr int64_t kMaxRowIds = 1 << 28;  // a row's counts fit below the flag bits
// An entry of an id that a row biases twice looks for a later one, work that grows with the product of the list and
// the vocabulary: 65536 ids twice each take 0.15 s (in place 0.29), and the 2^28 entries that a history may have would
// take many minutes.
constexpr int64_t kMaxRowBiases = 1 << 18;

__device__ __forceinline__ float load_f(const float* p) { return *p; }
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// [o[row], o[row+1]) of an array of `total` entries; empty (and flagged) where
// it leaves the array or has more than `most`.
__device__ __forceinline__ int row_range(const int64_t* o, int row, int64_t total, int64_t most, int64_t* first,
                                         uint32_t* bad) {
  const int64_t a = __ldg(o + row), b = __ldg(o + row + 1);
  *first = a;
  if (a >= 0 && b >= a && b <= total && b - a <= most) return (int)(b - a);
  *first = 0;
  *bad |= NS_STATUS_BAD_ROW_RANGE;
  return 0;
}

struct Penalty {
  float rep, pres, freq;
};

__device__ __forceinline__ float penalised(float x, uint32_t w, const Penalty& p) {
  const uint32_t c = w & kCount;
  if ((w & (kInPrompt | kCount)) && p.rep != 1.0f) x = x < 0.0f ? __fmul_rn(x, p.rep) : __fdiv_rn(x, p.rep);
  if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(p.freq, (float)c)), p.pres);
  return x;
}

// What one row asks for.
struct RowWork {
  Penalty pen;
  const int32_t *hist, *bias;
  const float* value;
  int hn, bn, prompt;
  uint32_t bad;
};

__device__ __forceinline__ RowWork row_work(const NsProcessArgs& a, int row) {
  RowWork r;
  r.bad = 0;
  r.pen.rep = a.repetition_penalty ? __ldg(a.repetition_penalty + row) : 1.0f;
  r.pen.pres = a.presence_penalty ? __ldg(a.presence_penalty + row) : 0.0f;
  r.pen.freq = a.frequency_penalty ? __ldg(a.frequency_penalty + row) : 0.0f;
  int64_t h0 = 0, b0 = 0;
  r.hn = a.history_offsets ? row_range(a.history_offsets, row, a.num_history_ids, kMaxRowIds, &h0, &r.bad) : 0;
  r.bn = a.bias_offsets ? row_range(a.bias_offsets, row, a.num_biases, kMaxRowBiases, &b0, &r.bad) : 0;
  r.prompt = a.prompt_lens ? __ldg(a.prompt_lens + row) : 0;
  if (r.pen.rep == 1.0f && r.pen.pres == 0.0f && r.pen.freq == 0.0f) r.hn = 0;  // nothing would change
  r.hist = a.history_ids + h0;
  r.bias = a.bias_ids + b0;
  r.value = a.bias_values + b0;
  return r;
}

// A row's first ids, kBlock apart, on their way to registers while the block
// clears its table: four history entries and one bias per thread.
template <int kBlock>
struct FirstIds {
  int hist[kPre], bias;
  float value;
  __device__ __forceinline__ explicit FirstIds(const RowWork& r) {
#pragma unroll
    for (int u = 0; u < kPre; ++u) {
      const int j = threadIdx.x + u * kBlock;
      hist[u] = j < r.hn ? __ldg(r.hist + j) : -1;
    }
    bias = (int)threadIdx.x < r.bn ? __ldg(r.bias + threadIdx.x) : -1;
    value = (int)threadIdx.x < r.bn ? __ldg(r.value + threadIdx.x) : 0.0f;
  }
};

// f(j, id) for all history entries of the row, kPre loads in flight.
template <int kBlock, typename F>
__device__ __forceinline__ void for_history(const RowWork& r, const FirstIds<kBlock>& first, F f) {
  int v[kPre];
#pragma unroll
  for (int u = 0; u < kPre; ++u) v[u] = first.hist[u];
  for (int j = threadIdx.x; j < r.hn;) {
    int next[kPre];
#pragma unroll
    for (int u = 0; u < kPre; ++u) {
      const int k = j + (kPre + u) * kBlock;
      next[u] = k < r.hn ? __ldg(r.hist + k) : -1;
    }
#pragma unroll
    for (int u = 0; u < kPre; ++u)
      if (j + u * kBlock < r.hn) f(j + u * kBlock, v[u]);
    j += kPre * kBlock;
#pragma unroll
    for (int u = 0; u < kPre; ++u) v[u] = next[u];
  }
}

// f(j, id, value) for all biases of the row.
template <int kBlock, typename F>
__device__ __forceinline__ void for_biases(const RowWork& r, const FirstIds<kBlock>& first, F f) {
  if ((int)threadIdx.x < r.bn) f((int)threadIdx.x, first.bias, first.value);
  for (int j = threadIdx.x + kBlock; j < r.bn; j += kBlock) f(j, __ldg(r.bias + j), __ldg(r.value + j));
}

// Entry j is the row's last for its id (asked only where an id has several).
__device__ __forceinline__ bool last_entry(const RowWork& r, int j, int v) {
  for (int k = j + 1; k < r.bn; ++k)
    if (__ldg(r.bias + k) == v) return false;
  return true;
}

// Bits [i, i + 32) of a mask in shared memory, one word longer than its bits.
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* mask, int i) {
  return __funnelshift_r(mask[i >> 5], mask[(i >> 5) + 1], i & 31);
}
__host__ __device__ constexpr int mask_bytes(int width) { return (width / 128 + 1) * 16; }  // of a tile's mask and a word, in 16s

// Bulk copy of `bytes` (multiple of 16, both addresses 16-byte aligned) from this
// CTA's shared memory to global memory, and the wait until it has been read.
__device__ __forceinline__ void bulk_s2g(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;" ::"l"(dst),
               "r"(smem_addr(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_s2g_wait() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

__device__ __forceinline__ bool wait_for(uint64_t* bar) {
  for (uint32_t i = 0; i < kMaxTries; ++i)
    if (mbar_try_wait(bar, 0)) return true;
  return false;
}

// A tile's ids have 16 bits each in shared memory: occurrences after the prompt
// in the low 13 (an id that comes near their end makes the block start over with
// 32 bits), then bits for the prompt and for biases.
constexpr uint32_t kHalfCount = 0x1fffu, kHalfMost = 7000, kHalfBiasTwice = 0x2000u, kHalfBias = 0x4000u,
                   kHalfPrompt = 0x8000u;
static_assert(kTile<float> <= 32 * kMostThreads && kTile<__nv_bfloat16> <= 32 * kMostThreads, "a mask word each");
static_assert(kHalfMost + kMostThreads < kHalfCount, "the count is noticed before it overflows");
__device__ __forceinline__ uint32_t widen(uint32_t h) {
  return (h & kHalfCount) | (h & kHalfBiasTwice ? kBiasTwice : 0u) | (h & kHalfBias ? kBias : 0u) |
         (h & kHalfPrompt ? kInPrompt : 0u);
}

// One tile of one row.  The tile is brought into shared memory by a bulk copy
// while the block counts the row's history ids that fall into it, 16 bits per id
// in shared memory, and lists the ids it meets first.  Then each listed id's logit
// is recomputed where it lies, what a mask forbids is overwritten, and the tile
// leaves through a bulk copy (or, with another type, through registers).
//
// 256 rows of 128256 fp32 with histories of about 1088 take 45 us (263.9 MB at the
// 6446 GB/s of a copy: 41), without histories 43; 2048 rows of 50257 under masks
// 153 us (130; 160 with the mask read where it lies); 64 bf16 rows into fp32 under masks,
// histories of about 2300, 18 us (8; 21 replayed from a graph, and 25 with the mask
// read where it lies).  In place under masks, which only overwrites what they forbid, element
// by element, the 256 rows take 56 us (8), in bf16 43 (4).
// Bulk copies need no registers and few instructions; what is left is a block's chain of
// dependent loads (offsets, ids, the tile) and barriers, about 6 us during which three
// blocks have 144 KB on their way on each SM.  Reading and writing through registers, with
// the named ids corrected in global memory afterwards, took 88 us (histories) and 51 us
// (none): the corrections are partial writes to lines that are on their way out.  A hash
// table in place of 16 bits per id took 53 us.
template <typename In, typename Out, bool kInPlace, int kThreads>
__global__ void __launch_bounds__(kThreads, 1536 / kThreads) tile_kernel(const __grid_constant__ NsProcessArgs a, int tiles, int width) {
  constexpr bool kSame = sizeof(In) == sizeof(Out);
  constexpr int kVec = 16 / sizeof(In);
  extern __shared__ __align__(128) unsigned char smem[];
  uint32_t* words = reinterpret_cast<uint32_t*>(smem);  // width 16-bit words
  uint16_t* hits = reinterpret_cast<uint16_t*>(smem + width * 2);
  __shared__ uint64_t bar;
  __shared__ int s_hits, s_over;
  const int tid = threadIdx.x;
  const int row = blockIdx.x / tiles;
  const int v0 = (blockIdx.x % tiles) * width;
  const int n = min(width, a.vocab_size - v0);
  uint32_t bad = 0;

  int64_t src = row;
  if (a.sample_indices) {
    src = __ldg(a.sample_indices + row);
    if (src < 0 || src >= a.num_logit_rows) {
      bad |= NS_STATUS_BAD_SAMPLE_INDEX;
      src = 0;
    }
  }
  const In* in = static_cast<const In*>(a.logits) + src * a.logits_row_stride + v0;
  Out* out = static_cast<Out*>(a.out) + (int64_t)row * a.out_row_stride + v0;
  // the tile in shared memory, at the same offset to the 16-byte grid as in global memory
  const int skew = (int)(reinterpret_cast<uintptr_t>(in) & 15);
  uint32_t* s_mask = reinterpret_cast<uint32_t*>(smem + width * 2 + kHits<In> * 2);
  In* x = reinterpret_cast<In*>(smem + width * 2 + kHits<In> * 2 + mask_bytes(width) + skew);
  const int head = min(n, (16 - skew) % 16 / (int)sizeof(In));  // elements before the first 16-byte boundary
  const int body = (n - head) / kVec * kVec;
  if (!kInPlace) {
    if (tid == 0) {
      mbar_init(&bar, 1);
      fence_mbar_init();
      mbar_arrive_expect_tx(&bar, body * sizeof(In));
      if (body) bulk_g2s(x + head, in + head, body * sizeof(In), &bar);
    }
    if (tid < head) x[tid] = in[tid];
    if (tid < n - head - body) x[head + body + tid] = in[head + body + tid];
  }

  const RowWork r = row_work(a, row);
  bad |= r.bad;
  const FirstIds<kThreads> first(r);
  const uint32_t* mask = nullptr;
  if (a.allowed) {
    const int m = a.allowed_rows ? __ldg(a.allowed_rows + row) : row;
    if (m >= a.num_masks) bad |= NS_STATUS_BAD_MASK_ROW;
    else if (m >= 0) mask = reinterpret_cast<const uint32_t*>(a.allowed) + m * a.mask_stride + v0 / 32;
  }
  const int mask_words = (n + 31) / 32;
  const uint32_t mask_word = mask && tid < mask_words ? __ldg(mask + tid) : 0u;
  const auto allowed = [&](int i) { return !mask || ((s_mask[i >> 5] >> (i & 31)) & 1u); };
  const bool counted = r.hn || r.bn;  // the same in all threads

  const auto half = [&](uint32_t i) { return (words[i >> 1] >> ((i & 1) * 16)) & 0xffffu; };
  const auto clear = [&] {  // a width is a multiple of 32
    for (int i = tid; i < width / 8; i += kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  };
  // Every bias entry of ids [p0, p0 + pn) of the tile: or(i, bit) sets a bit of id p0 + i and gives what was there.
  const auto count_biases = [&](int p0, int pn, uint32_t bias, uint32_t twice, auto set) {
    for_biases(r, first, [&](int, int v, float) {
      if ((uint32_t)v >= (uint32_t)a.vocab_size) bad |= NS_STATUS_BAD_TOKEN_ID;
      const uint32_t i = (uint32_t)(v - v0 - p0);
      if (i < (uint32_t)pn && (set(i, bias) & bias)) set(i, twice);
    });
  };
  // The results of the biased ids (one entry of each computes it).
  const auto fix_biased = [&](auto get, auto put, int p0, int pn, auto word) {
    for_biases(r, first, [&](int j, int v, float value) {
      const uint32_t i = (uint32_t)(v - v0 - p0);
      if (i >= (uint32_t)pn) return;
      const uint32_t w = word(i);
      if (!(w & kBiasTwice) || last_entry(r, j, v))
        put(p0 + (int)i, __fadd_rn(penalised(get(p0 + (int)i), w, r.pen), value));
    });
  };
  // All ids of the tile that a penalty or a bias names.  `put` is where their results go: into the tile, before
  // it is written; or, where the tile keeps another type or is not there, to the output.
  const auto fix = [&](auto get, auto put) {
    const auto history = [&](int i, uint32_t w) {
      if (w && !(w & kBias)) put(i, penalised(get(i), w, r.pen));
    };
    if (!s_over) {
      const int nh = s_hits;
      if (nh <= kHits<In>)
        for (int h = tid; h < nh; h += kThreads) history(hits[h], widen(half(hits[h])));
      else
        for (int i = tid; i < n; i += kThreads) history(i, widen(half(i)));
      fix_biased(get, put, 0, n, [&](uint32_t i) { return widen(half(i)); });
      return;
    }
    const int part = width / 2;  // ids that the same memory holds in 32 bits
    for (int p0 = 0; p0 < n; p0 += part) {
      const int pn = min(part, n - p0);
      __syncthreads();
      clear();
      __syncthreads();
      for_history(r, first, [&](int j, int v) {
        const uint32_t i = (uint32_t)(v - v0 - p0);
        if (i >= (uint32_t)pn) return;
        if (j < r.prompt) atomicOr(&words[i], kInPrompt);
        else atomicAdd(&words[i], 1u);
      });
      count_biases(p0, pn, kBias, kBiasTwice, [&](uint32_t i, uint32_t bit) { return atomicOr(&words[i], bit); });
      __syncthreads();
      for (int i = tid; i < pn; i += kThreads) history(p0 + i, words[i]);
      fix_biased(get, put, p0, pn, [&](uint32_t i) { return words[i]; });
    }
  };

  if (counted) {
    if (tid == 0) s_hits = s_over = 0;
    clear();
    __syncthreads();
    for_history(r, first, [&](int j, int v) {
      if ((uint32_t)v >= (uint32_t)a.vocab_size) bad |= NS_STATUS_BAD_HISTORY_ID;
      const uint32_t i = (uint32_t)(v - v0);
      if (i >= (uint32_t)n) return;
      const int sh = (i & 1) * 16;
      const uint32_t was = (j < r.prompt ? atomicOr(&words[i >> 1], kHalfPrompt << sh) : atomicAdd(&words[i >> 1], 1u << sh)) >> sh;
      if (!(was & (kHalfPrompt | kHalfCount))) {
        const int h = atomicAdd(&s_hits, 1);
        if (h < kHits<In>) hits[h] = (uint16_t)i;
      }
      if ((was & kHalfCount) >= kHalfMost) s_over = 1;
    });
    count_biases(0, n, kHalfBias, kHalfBiasTwice, [&](uint32_t i, uint32_t bit) {
      const int sh = (i & 1) * 16;
      return atomicOr(&words[i >> 1], bit << sh) >> sh;
    });
  }
  if (mask) {
    if (tid < mask_words) s_mask[tid] = mask_word;
    if (tid == 0) s_mask[mask_words] = 0;
  }
  __syncthreads();  // also: the barrier is initialised, the tile's ends are there
  if (!kInPlace && !wait_for(&bar)) {
    if (tid == 0 && a.status) atomicOr(a.status, NS_STATUS_WAIT_TIMEOUT);
    wait_for(&bar);  // the copy may still land
    return;
  }

  if constexpr (kInPlace) {
    if (mask)
      for (int i = tid; i < n; i += kThreads)
        if (!allowed(i)) store_f(out + i, -INFINITY);
    if (counted)
      fix([&](int i) { return load_f(in + i); },
          [&](int i, float y) {
            if (allowed(i)) store_f(out + i, y);
          });
  } else if constexpr (kSame) {
    if (counted) {
      fix([&](int i) { return load_f(x + i); }, [&](int i, float y) { store_f(x + i, y); });
      fence_proxy_async_smem();
      __syncthreads();
    }
    const bool aligned = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    if (!aligned) {
      for (int i = tid; i < n; i += kThreads) {
        if (allowed(i)) out[i] = x[i];
        else store_f(out + i, -INFINITY);
      }
    } else {
      if (mask) {
        constexpr uint32_t kAll = (1u << kVec) - 1;
        for (int i = head + tid * kVec; i < head + body; i += kThreads * kVec) {
          const uint32_t bits = mask_bits(s_mask, i);
          if ((bits & kAll) == kAll) continue;
          uint4 y = *reinterpret_cast<const uint4*>(x + i);
          uint32_t* w = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (sizeof(In) == 4) {
              if (!((bits >> e) & 1u)) w[e] = 0xff800000u;
            } else {
              if (!((bits >> (2 * e)) & 1u)) w[e] = (w[e] & 0xffff0000u) | 0xff80u;
              if (!((bits >> (2 * e + 1)) & 1u)) w[e] = (w[e] & 0xffffu) | 0xff800000u;
            }
          }
          *reinterpret_cast<uint4*>(x + i) = y;
        }
        fence_proxy_async_smem();
        __syncthreads();
      }
      if (tid == 0 && body) bulk_s2g(out + head, x + head, body * sizeof(Out));
      const int e = tid < head ? tid : tid - head < n - head - body ? body + tid : -1;  // the ends
      if (e >= 0) {
        if (allowed(e)) out[e] = x[e];
        else store_f(out + e, -INFINITY);
      }
      if (tid == 0) bulk_s2g_wait();  // shared memory is read before the block ends
    }
  } else {
    // bf16 in, fp32 out: four elements at a time along the output's 16-byte grid, so that neighbours write
    // neighbouring sectors (183 rows of 101344 ids, or of 101341 whose input and output lie differently to the
    // grid, take 25 us; eight along the tile's took 6 % longer for the first and more than twice as long for the second)
    const auto one = [&](int i) { store_f(out + i, allowed(i) ? load_f(x + i) : -INFINITY); };
    const int before = min(n, (int)(-reinterpret_cast<uintptr_t>(out) & 15) / 4);
    const int many = (n - before) / 4 * 4;
    const bool wide = (reinterpret_cast<uintptr_t>(x + before) & 7) == 0;
    for (int i = before + tid * 4; i < before + many; i += kThreads * 4) {
      const uint32_t bits = mask ? mask_bits(s_mask, i) : ~0u;
      float f[4];
      if (wide) {
        const uint2 y = *reinterpret_cast<const uint2*>(x + i);
        f[0] = __uint_as_float(y.x << 16), f[1] = __uint_as_float(y.x & 0xffff0000u);
        f[2] = __uint_as_float(y.y << 16), f[3] = __uint_as_float(y.y & 0xffff0000u);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = load_f(x + i + e);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!((bits >> e) & 1u)) f[e] = -INFINITY;
      *reinterpret_cast<float4*>(out + i) = make_float4(f[0], f[1], f[2], f[3]);
    }
    if (tid < before) one(tid);
    if (tid < n - before - many) one(before + many + tid);
    if (counted) {
      __syncthreads();
      fix([&](int i) { return load_f(x + i); },
          [&](int i, float y) {
            if (allowed(i)) store_f(out + i, y);
          });
    }
  }
  if (bad && a.status) atomicOr(a.status, bad);
}

// Ids and their words in shared memory, open addressing.  `ids` holds id + 1, 0
// for a free slot.
struct Table {
  uint32_t *ids, *words;
  uint32_t mask;  // slots - 1

  // v's slot, taken if it has none; -1 where `tries` slots in a row are others'
  __device__ __forceinline__ int slot(uint32_t v, int tries) const {
    uint32_t s = (v * 2654435761u) >> 12;  // golden ratio
    for (int k = 0; k < tries; ++k, ++s) {
      s &= mask;
      uint32_t was = *reinterpret_cast<volatile uint32_t*>(ids + s);
      if (was == 0) was = atomicCAS(ids + s, 0u, v + 1);
      if (was == 0 || was == v + 1) return (int)s;
    }
    return -1;
  }
};
// In place and without masks only the ids that a history or a bias names
// change.  Block `row` counts its row's ids in a hash table in shared memory (open
// addressing, at most half full) and recomputes each once.  Rows with more ids
// than the table takes are left to the kHelpers blocks behind: every one finds
// these rows, and they share out their ranges of kRange ids, one word per id.
//
// 256 rows of 128256 fp32 with histories of about 1088 ids take 20 us, all rows'
// blocks resident at once: about half is the 278 thousand scattered reads and
// writes of logits (a run without them took 8 to 11), the rest the longest rows' chain
// of table accesses.
constexpr int kSparseThreads = 512;
constexpr int kRowSlots = 8192;  // most slots of a row's table, a power of two
constexpr int kRange = 2 * kRowSlots;
constexpr int kHelpers = 32;

template <typename T>
__global__ void __launch_bounds__(kSparseThreads, 2) sparse_kernel(const __grid_constant__ NsProcessArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  uint32_t* words = reinterpret_cast<uint32_t*>(smem);  // kRowSlots words and as many ids, or kRange words
  uint32_t* ids = words + kRowSlots;
  __shared__ uint32_t s_long[kSparseThreads / 32];
  __shared__ int s_rows[kSparseThreads];
  const int tid = threadIdx.x, lane = tid % 32;
  const uint32_t V = (uint32_t)a.vocab_size;
  uint32_t bad = 0;

  if ((int)blockIdx.x < a.num_rows) {
    const int row = blockIdx.x;
    const RowWork r = row_work(a, row);
    bad |= r.bad;
    if (r.hn + r.bn > kRowSlots / 2) return;  // a long row
    T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_row_stride;
    const FirstIds<kSparseThreads> first(r);
    int slots = 256;
    while (slots < 2 * (r.hn + r.bn)) slots *= 2;
    for (int i = tid; i < slots; i += kSparseThreads) words[i] = ids[i] = 0;
    __syncthreads();
    const Table table{ids, words, (uint32_t)slots - 1};
    const auto slot_of = [&](uint32_t v) { return table.slot(v, slots); };  // found: the table is at most half full
    for_history(r, first, [&](int j, int v) {
      if ((uint32_t)v >= V) {
        bad |= NS_STATUS_BAD_HISTORY_ID;
        return;
      }
      const uint32_t s = slot_of(v);
      if (j < r.prompt) atomicOr(&words[s], kInPrompt);
      else atomicAdd(&words[s], 1u);
    });
    for_biases(r, first, [&](int, int v, float) {
      if ((uint32_t)v >= V) {
        bad |= NS_STATUS_BAD_TOKEN_ID;
        return;
      }
      const uint32_t s = slot_of(v);
      if (atomicOr(&words[s], kBias) & kBias) atomicOr(&words[s], kBiasTwice);
    });
    const float biased = (uint32_t)first.bias < V ? load_f(out + first.bias) : 0.0f;  // on its way
    __syncthreads();
    for (int i = tid; i < slots; i += 4 * kSparseThreads) {
      uint32_t v[4], w[4];
      float y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = i + u * kSparseThreads;
        v[u] = s < slots ? ids[s] : 0;
        w[u] = v[u] ? words[s] : 0;
        if (w[u] & kBias) v[u] = 0;
        y[u] = v[u] ? load_f(out + (v[u] - 1)) : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (v[u]) store_f(out + (v[u] - 1), penalised(y[u], w[u], r.pen));
    }
    for_biases(r, first, [&](int j, int v, float value) {
      if ((uint32_t)v >= V) return;
      const uint32_t w = words[slot_of(v)];
      if (!(w & kBiasTwice) || last_entry(r, j, v))
        store_f(out + v, __fadd_rn(penalised(j == tid ? biased : load_f(out + v), w, r.pen), value));
    });
  } else {
    const int ranges = (a.vocab_size - 1) / kRange + 1;
    int64_t item = 0;  // of all rows' ranges, in order
    for (int base = 0; base < a.num_rows; base += kSparseThreads) {
      bool is_long = false;
      if (base + tid < a.num_rows) {
        const RowWork r = row_work(a, base + tid);
        is_long = r.hn + r.bn > kRowSlots / 2;
      }
      const uint32_t vote = __ballot_sync(0xffffffffu, is_long);
      if (lane == 0) s_long[tid / 32] = vote;
      if (!__syncthreads_or(is_long)) continue;
      int before = __popc(vote & ((1u << lane) - 1)), rows = 0;
      for (int w = 0; w < kSparseThreads / 32; ++w) {
        if (w < tid / 32) before += __popc(s_long[w]);
        rows += __popc(s_long[w]);
      }
      if (is_long) s_rows[before] = base + tid;
      __syncthreads();
      for (int k = 0; k < rows * ranges; ++k, ++item) {
        if (item % kHelpers != (int)blockIdx.x - a.num_rows) continue;
        const int row = s_rows[k / ranges], v0 = (k % ranges) * kRange;
        const uint32_t n = min(kRange, a.vocab_size - v0);
        const RowWork r = row_work(a, row);
        bad |= r.bad;
        const FirstIds<kSparseThreads> first(r);
        T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_row_stride + v0;
        for (int i = tid; i < kRange; i += kSparseThreads) words[i] = 0;
        __syncthreads();
        for_history(r, first, [&](int j, int v) {
          if ((uint32_t)v >= V) bad |= NS_STATUS_BAD_HISTORY_ID;
          const uint32_t i = (uint32_t)(v - v0);
          if (i >= n) return;
          if (j < r.prompt) atomicOr(&words[i], kInPrompt);
          else atomicAdd(&words[i], 1u);
        });
        for_biases(r, first, [&](int, int v, float) {
          if ((uint32_t)v >= V) bad |= NS_STATUS_BAD_TOKEN_ID;
          const uint32_t i = (uint32_t)(v - v0);
          if (i < n && (atomicOr(&words[i], kBias) & kBias)) atomicOr(&words[i], kBiasTwice);
        });
        __syncthreads();
        for (uint32_t i = tid; i < n; i += kSparseThreads) {
          const uint32_t w = words[i];
          if (w && !(w & kBias)) store_f(out + i, penalised(load_f(out + i), w, r.pen));
        }
        for_biases(r, first, [&](int j, int v, float value) {
          const uint32_t i = (uint32_t)(v - v0);
          if (i >= n) return;
          const uint32_t w = words[i];
          if (!(w & kBiasTwice) || last_entry(r, j, v))
            store_f(out + i, __fadd_rn(penalised(load_f(out + i), w, r.pen), value));
        });
        __syncthreads();  // words may be cleared
      }
      __syncthreads();  // s_long and s_rows may be written
    }
  }
  if (bad && a.status) atomicOr(a.status, bad);
}

// Dynamic shared memory above 48 KB has to be allowed once per device and kernel.
template <auto kernel>
cudaError_t allow_smem(int bytes) {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

// A block of tile_kernel has one thread per word of its tile's mask at least.
template <typename In, typename Out, bool kInPlace, int kThreads>
cudaError_t launch_block(const NsProcessArgs& a, unsigned blocks, int tiles, int width, cudaStream_t st) {
  const auto bytes = [](int w) {
    return w * 2 + kHits<In> * 2 + mask_bytes(w) + (kInPlace ? 0 : w * (int)sizeof(In) + 16);
  };
  const cudaError_t e = allow_smem<tile_kernel<In, Out, kInPlace, kThreads>>(bytes(std::min(kTile<In>, 32 * kThreads)));
  if (e != cudaSuccess) return e;
  tile_kernel<In, Out, kInPlace, kThreads><<<blocks, kThreads, bytes(width), st>>>(a, tiles, width);
  return cudaGetLastError();
}

template <typename In, typename Out, bool kInPlace>
cudaError_t launch_tiles(const NsProcessArgs& a, cudaStream_t st) {
  // Every tile of a row reads the row's history and waits for its loads in turn, so a row has as few tiles as
  // possible; where all blocks fit on the GPU at once, as many as do.  (256 rows of 128256 fp32 with histories
  // of about 1088: 46 us in 11 tiles, 62 in 21; 1024 rows of bf16: 89 us in 8 tiles, 106 in 11.)  All tiles are of
  // one width, a multiple of 32: a tile starts on a mask word.
  const int64_t least = (a.vocab_size - 1) / kTile<In> + 1;
  const int64_t fit = std::min<int64_t>(148 * 3 / a.num_rows, a.vocab_size / 2048);
  const int64_t wanted = std::max(least, fit);
  const int width = (int)((a.vocab_size + wanted - 1) / wanted + 31) / 32 * 32;
  const int tiles = (a.vocab_size - 1) / width + 1;
  const unsigned blocks = (unsigned)(tiles * (int64_t)a.num_rows);
  // Narrow tiles get small blocks, more of them on an SM: a block's time is its chain of loads and barriers, and more
  // rows then wait at a time.  Where all blocks are resident anyway and have long histories to count, the count
  // wants the threads.  (4000 fp32 rows of 2500 ids, masks, histories of 150: 45 us with 512 threads, 28 with 256,
  // 23 with 128; of 8192 ids 60, 50 with 256; 8 rows of 2500 with histories of 800: 6.1 and 6.2, of 3000: 6.2 and
  // 10.5.)
  const bool narrow = blocks > 148 * 3 || a.num_history_ids <= (int64_t)a.num_rows * 1024;
  if (narrow && width <= 32 * 128) return launch_block<In, Out, kInPlace, 128>(a, blocks, tiles, width, st);
  if (narrow && width <= 32 * 256) return launch_block<In, Out, kInPlace, 256>(a, blocks, tiles, width, st);
  return launch_block<In, Out, kInPlace, 512>(a, blocks, tiles, width, st);
}

template <typename T>
cudaError_t launch_in_place(const NsProcessArgs& a, cudaStream_t st) {
  if (a.allowed) return launch_tiles<T, T, true>(a, st);
  // rows longer than the table are possible only where there are that many ids
  const bool longer = a.num_history_ids + a.num_biases > kRowSlots / 2;
  const cudaError_t e = allow_smem<sparse_kernel<T>>(kRange * 4);
  if (e != cudaSuccess) return e;
  sparse_kernel<T><<<a.num_rows + (longer ? kHelpers : 0), kSparseThreads, kRange * 4, st>>>(a);
  return cudaGetLastError();
}

}  // namespace proc
}  // namespace ns

extern "C" int ns_process_logits(const NsProcessArgs* args, void* stream) {
  using namespace ns;
  if (!args) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: args is NULL");
  const NsProcessArgs& a = *args;
  if (a.num_rows < 0) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: num_rows < 0");
  if (a.num_rows == 0) return NS_OK;
  if (!a.logits || !a.out) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: logits and out are required");
  if (a.logits_dtype != NS_DTYPE_F32 && a.logits_dtype != NS_DTYPE_BF16)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: logits_dtype must be NS_DTYPE_F32 or NS_DTYPE_BF16");
  if (a.out_dtype != NS_DTYPE_F32 && a.out_dtype != a.logits_dtype)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: out_dtype must be NS_DTYPE_F32 or the logits' type");
  if (a.vocab_size <= 0) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: vocab_size must be positive");
  if (a.logits_row_stride < 0) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: logits_row_stride < 0");
  if (a.num_rows > 1 && a.out_row_stride < a.vocab_size)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: out_row_stride < vocab_size");
  if (a.num_logit_rows <= 0) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: num_logit_rows must be positive");
  if (!a.sample_indices && a.num_logit_rows < a.num_rows)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: fewer logits rows than num_rows and no sample_indices");
  if (a.num_history_ids < 0 || a.num_biases < 0)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: num_history_ids / num_biases < 0");
  if (a.history_offsets && a.num_history_ids > 0 && !a.history_ids)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: history_offsets given without history_ids");
  if (a.bias_offsets && a.num_biases > 0 && (!a.bias_ids || !a.bias_values))
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: bias_offsets given without bias_ids and bias_values");
  if (a.allowed && (a.num_masks < 0 || a.mask_stride < (a.vocab_size - 1) / 32 + 1))
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: num_masks < 0 or mask_stride < (vocab_size + 31) / 32");
  if (a.allowed && !a.allowed_rows && a.num_masks < a.num_rows)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: fewer masks than num_rows and no allowed_rows");
  if (a.reserved != 0) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: reserved must be 0");
  const int64_t blocks = ((a.vocab_size - 1) / proc::kTile<float> + (int64_t)1) * a.num_rows;
  if (blocks > 1 << 30)  // row numbers and their windows stay in 32 bits
    return fail(NS_ERR_UNSUPPORTED, "ns_process_logits: num_rows * vocab_size is too large");

  const int64_t in_size = a.logits_dtype == NS_DTYPE_F32 ? 4 : 2, out_size = a.out_dtype == NS_DTYPE_F32 ? 4 : 2;
  const uintptr_t i0 = reinterpret_cast<uintptr_t>(a.logits), o0 = reinterpret_cast<uintptr_t>(a.out);
  if (i0 % in_size || o0 % out_size)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: logits / out not aligned to their element");
  const uintptr_t i1 = i0 + ((a.num_logit_rows - 1) * a.logits_row_stride + a.vocab_size) * in_size;
  const uintptr_t o1 = o0 + ((a.num_rows - 1) * a.out_row_stride + a.vocab_size) * out_size;
  const bool in_place = i0 == o0 && in_size == out_size && !a.sample_indices &&
                        (a.num_rows == 1 || a.logits_row_stride == a.out_row_stride);
  if (!in_place && i0 < o1 && o0 < i1)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: out overlaps the logits without being the same rows");

  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  using bf16 = __nv_bfloat16;
  if (a.logits_dtype == NS_DTYPE_F32)
    e = in_place ? proc::launch_in_place<float>(a, st) : proc::launch_tiles<float, float, false>(a, st);
  else if (a.out_dtype == NS_DTYPE_F32)
    e = proc::launch_tiles<bf16, float, false>(a, st);
  else
    e = in_place ? proc::launch_in_place<bf16>(a, st) : proc::launch_tiles<bf16, bf16, false>(a, st);
  if (e != cudaSuccess) return fail(NS_ERR_CUDA, std::string("ns_process_logits launch: ") + cudaGetErrorString(e));
  return NS_OK;
}
