// ns_logprobs.cu -- log-probabilities of given tokens, their ranks, and the
// n largest of each row (ns_token_logprobs).
//
//   L = m + log(sum_v exp(x_v - m)),  logprob = (x_t - m) - log(sum)
//   rank = 1 + #{v : x_v > x_t}
//   top n: larger logits first, equal ones by ascending id
//
// One pass over the logits gives every sum: a cluster of C blocks takes a row
// (C by the number of rows, so that few rows still fill the GPU), each block a
// contiguous slice of it, each thread every 256th (or 128th) 16-byte vector of the
// slice (its bucket).  A thread keeps the maxima of its batches, its sum of
// exponentials over a reference that follows the maximum in steps, and its count
// of larger logits.  The n largest are then in few batches: those whose maximum
// reaches a bound that n buckets reach.  Only these are read again (out of L2);
// the elements that reach the bound are ranked by counting (or, where ties make
// them many, through sorted lists), within the block and then, through
// distributed shared memory, within the cluster.
//
// Measured on a B200 (V = 128256; the logits' bytes at the 6446 GB/s of a copy in
// brackets): 4096 bf16 rows, top 1: 176 us (163) in short runs, 187 in a loop of
// seconds under the power cap; 256 fp32 rows, top 20: 33 us (20); 8 fp32 rows,
// top 5: 10 us (0.6).  Large batches are bound by the loads,
// with the exponential units two thirds busy; a few hundred rows are one wave of
// blocks, whose search for the top tokens (about 6 us after the 20 us of loads)
// nothing overlaps: four blocks a row in place of two took 42 us, as each block
// pays for its own.  Eight rows are bound by the launch and the chain of barriers.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>
#include <type_traits>

#include "ns_device.cuh"

namespace ns {
int fail(int code, const std::string& msg);

namespace lp {

constexpr int kMaxCluster = 8;     // the portable limit
constexpr float kLag = 8.0f;       // the reference follows the maximum in steps of at least this
constexpr float kHuge = 0x1p100f;  // beyond it the fused argument of the exponential could overflow
constexpr int kEntries = 32;       // maxima that a thread keeps
constexpr int kListed = 512;       // entries that are read again
constexpr int kCands = 256;        // candidates that are ranked by counting
typedef unsigned long long u64;

// Larger value first, then smaller id, as one key to maximise; -0 counts as 0, and
// masked elements (-inf) have key 0: they are the last to be taken, by id.
__device__ __forceinline__ uint32_t value_key(float x) { return x == -INFINITY ? 0u : f2key(x + 0.0f); }
__device__ __forceinline__ u64 top_key(float x, int v) {
  return x == -INFINITY ? 0ull : ((u64)f2key(x + 0.0f) << 32) | (uint32_t)~v;
}
__device__ __forceinline__ int top_id(u64 k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float top_value(u64 k) { return key2f((uint32_t)(k >> 32)); }

// Two floats in a register pair: one instruction works on both.
__device__ __forceinline__ u64 pack2(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(u64 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <typename In>
struct Row;

template <>
struct Row<float> {
  static constexpr int kVec = 4;
  static constexpr int kUnroll = 6;  // 16-byte loads in flight per thread
  __device__ static float one(const float* p) { return __ldg(p); }
  struct Vec {
    float4 v;
    __device__ void load(const float* p) { v = __ldg(reinterpret_cast<const float4*>(p)); }
    __device__ float get(int e) const { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; }
    __device__ u64 two(int i) const { return i ? pack2(v.z, v.w) : pack2(v.x, v.y); }
  };
  // NaN-propagating maximum of a batch
  template <int N>
  __device__ static float max_of(const Vec (&b)[N]) {
    float m = b[0].v.x;
#pragma unroll
    for (int u = 0; u < N; ++u) m = fmax_nan(fmax_nan(fmax_nan(m, b[u].v.x), fmax_nan(b[u].v.y, b[u].v.z)), b[u].v.w);
    return m;
  }
  struct Count {
    float t;
    int n = 0;
    __device__ explicit Count(float x) : t(x) {}
    template <int N>
    __device__ void add(const Vec (&b)[N]) {
#pragma unroll
      for (int u = 0; u < N; ++u) n += (b[u].v.x > t) + (b[u].v.y > t) + (b[u].v.z > t) + (b[u].v.w > t);
    }
    __device__ int total() const { return n; }
  };
};

template <>
struct Row<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static constexpr int kUnroll = 8;
  __device__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  struct Vec {
    uint32_t w[4];
    __device__ void load(const __nv_bfloat16* p) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
    __device__ float get(int e) const { return __uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16); }
    __device__ u64 two(int i) const { return pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)); }
    __device__ __nv_bfloat162 pair(int i) const { return reinterpret_cast<const __nv_bfloat162*>(w)[i]; }
  };
  template <int N>
  __device__ static float max_of(const Vec (&b)[N]) {
    __nv_bfloat162 m = b[0].pair(0);
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __hmax2_nan(m, b[u].pair(i));
    return fmax_nan(__low2float(m), __high2float(m));
  }
  // Two at a time: a comparison gives 1 or 0 per half, and bf16 counts exactly up to 256.
  struct Count {
    __nv_bfloat162 t, part;
    int n = 0, batches = 0;
    __device__ explicit Count(float x) : t(__float2bfloat162_rn(x)), part(__float2bfloat162_rn(0.0f)) {}
    template <int N>
    __device__ void add(const Vec (&b)[N]) {
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) part = __hadd2(part, __hgt2(b[u].pair(i), t));
      if (++batches == 256 / (4 * kUnroll)) flush();
    }
    __device__ void flush() {
      n += (int)(__low2float(part) + __high2float(part));
      part = __float2bfloat162_rn(0.0f);
      batches = 0;
    }
    __device__ int total() {
      flush();
      return n;
    }
  };
};

// A thread's running sum of exp(x - ref): with c = RN(log2 e) and
// hi + lo = ref * c exactly (an FMA gives lo), exp(x - ref) =
// 2^(fma(x, c, -hi)) * 2^-lo, so an element costs one FMA, one exponential and
// one addition, and the factor 2^-lo is applied once.  The argument is rounded
// once and the error of c only scales with x - ref.  (The exponential units take
// eight cycles for a warp's 32 elements, what the loop issues for bf16 elements
// about six; taking a quarter of the exponentials as polynomials on the FMA pipe made
// 4096 bf16 rows slower, 196 us against 191.)
struct Sum {
  float ref = -INFINITY, hi = 0.0f, lo = 0.0f, s = 0.0f;

  template <typename R, int N>
  __device__ __forceinline__ void add(const typename R::Vec (&b)[N], float bm) {
    if (!(bm <= ref + kLag)) move(bm);
    if (ref == -INFINITY) return;  // only -inf so far
    float p = 0.0f;
    if (fabsf(ref) < kHuge) {
      const u64 c = pack2(kLog2e, kLog2e), h = pack2(-hi, -hi);
      u64 q = 0;
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < R::kVec / 2; ++e) {
          const u64 arg = fma2(b[u].two(e), c, h);
          const float2 x = unpack2(arg);
          q = add2(q, pack2(ex2_approx(x.x), ex2_approx(x.y)));
        }
      const float2 x = unpack2(q);
      p = x.x + x.y;
    } else {
      for (int u = 0; u < N; ++u)
        for (int e = 0; e < R::kVec; ++e) p += exp_shifted(b[u].get(e), ref);
    }
    s += p;
  }
  __device__ void move(float m) {
    const float old = over(m);
    ref = m;
    const bool fused = fabsf(m) < kHuge;
    hi = fused ? __fmul_rn(m, kLog2e) : 0.0f;
    lo = fused ? __fmaf_rn(m, kLog2e, -hi) : 0.0f;
    s = old * ex2_approx(lo);
  }
  // the sum over another reference (>= -inf)
  __device__ float over(float m) const {
    return ref == -INFINITY ? 0.0f : s * ex2_approx(-lo) * exp_shifted(ref, m);
  }
};

// The 32 largest of two descending lists, one key per lane, descending.
__device__ __forceinline__ u64 merge_lists(u64 a, u64 b, int lane) {
  const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
  u64 c = a > r ? a : r;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const u64 p = __shfl_xor_sync(0xffffffffu, c, o);
    c = ((lane & o) != 0) == (p < c) ? p : c;
  }
  return c;
}

// Puts key c (the same in every lane) into the list.
__device__ __forceinline__ u64 insert(u64 list, u64 c, int lane) {
  const int at = __popc(__ballot_sync(0xffffffffu, list > c));
  const u64 up = __shfl_up_sync(0xffffffffu, list, 1);
  return lane < at ? list : lane == at ? c : up;
}

struct Part {  // a block's sums over its slice
  double sum;  // of exp(x - max)
  float max;
  int count;
};

// kThreads: 256, or less where a block takes a whole short row (then without a cluster).
template <typename In, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logprob_kernel(const NsLogprobArgs a, int clusters) {
  constexpr int kWarps = kThreads / 32, kMaxCluster = kThreads < 256 ? 1 : lp::kMaxCluster;
  static_assert(kMaxCluster == 1 || kMaxCluster * NS_MAX_TOP_LOGPROBS <= kThreads, "a thread ranks one key");
  const int C = kMaxCluster == 1 ? 1 : clusters;
  using R = Row<In>;
  using Vec = typename R::Vec;
  constexpr int kVec = R::kVec, kUnroll = R::kUnroll;
  __shared__ float s_max[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ int s_cnt[kWarps];
  __shared__ uint32_t s_entry[kEntries][kThreads];
  __shared__ uint32_t s_few[kWarps];
  __shared__ uint16_t s_list[kListed];
  __shared__ int s_listed, s_cands;
  __shared__ u64 s_best[kThreads];  // sorted keys: the warps', then the block's, then the row's
  __shared__ u64 s_cand[kCands];
  __shared__ u64 s_remote[kMaxCluster * NS_MAX_TOP_LOGPROBS];  // the other blocks' keys and parts
  __shared__ Part s_part[kMaxCluster];
  if (C > 1) cluster_arrive_relaxed();  // this block runs: its shared memory may be written
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int row = blockIdx.x / C, rank = blockIdx.x % C;
  const int V = a.vocab_size, n = a.top_n;

  uint32_t bad = 0;
  int64_t src = row;
  if (a.sample_indices) {
    src = __ldg(a.sample_indices + row);
    if (src < 0 || src >= a.num_logit_rows) {
      bad |= NS_STATUS_BAD_SAMPLE_INDEX;
      src = 0;
    }
  }
  const In* x = static_cast<const In*>(a.logits) + src * a.logits_row_stride;
  const int64_t t = a.ids_dtype == NS_OUT_I64 ? __ldg(static_cast<const int64_t*>(a.token_ids) + row)
                                              : (int64_t)__ldg(static_cast<const int32_t*>(a.token_ids) + row);
  const bool tok_ok = t >= 0 && t < V;
  if (!tok_ok) bad |= NS_STATUS_BAD_TOKEN_ID;
  const float xt = tok_ok ? R::one(x + t) : 0.0f;

  // the row: up to kVec - 1 elements before the first 16-byte boundary, vectors, and as many behind the last
  const int head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(In));
  const int vecs = (V - head) / kVec;
  const int tail = V - head - vecs * kVec;
  const int lo = (int)((int64_t)vecs * rank / C), hi = (int)((int64_t)vecs * (rank + 1) / C);
  const In* xv = x + head;

  // Batches of kUnroll vectors per thread, then what is left of its vectors.  The key of each batch's (or, in
  // long slices, of each `group` batches') maximum stays in shared memory; the one largest element alone is
  // found well enough from the maximum of all.
  const int batches = (hi - lo + kUnroll * kThreads - 1) / (kUnroll * kThreads);
  const int group = n > 1 ? (batches + kEntries - 1) / kEntries : batches;
  Sum sum;
  typename R::Count count(xt);
  float m = -INFINITY;
  uint32_t bucket = 0, entry = 0;  // keys of maxima: this thread's, and the current entry's (0: nothing)
  int entries = 0, in_entry = 0;
  const auto note = [&](float bm) {
    entry = max(entry, value_key(bm));
    if (++in_entry == group) {
      s_entry[entries++][tid] = entry;
      bucket = max(bucket, entry);
      entry = 0, in_entry = 0;
    }
  };
  int i = lo + tid;
  const auto take = [&](auto size) {  // the next vectors of the bucket, that many at once; their maximum
    constexpr int N = decltype(size)::value;
    Vec b[N];
#pragma unroll
    for (int u = 0; u < N; ++u) b[u].load(xv + (int64_t)(i + u * kThreads) * kVec);
    i += N * kThreads;
    const float bm = R::max_of(b);
    count.add(b);
    sum.template add<R>(b, bm);
    return bm;
  };
  while (i + (kUnroll - 1) * kThreads < hi) {
    const float bm = take(std::integral_constant<int, kUnroll>{});
    m = fmax_nan(m, bm);
    if (n > 1) note(bm);
  }
  float rest = -INFINITY;
  const bool some = i < hi;
  if (i + (kUnroll / 2 - 1) * kThreads < hi) rest = take(std::integral_constant<int, kUnroll / 2>{});
  while (i < hi) rest = fmax_nan(rest, take(std::integral_constant<int, 1>{}));
  m = fmax_nan(m, rest);
  if (n == 1 && lo + tid < hi) {
    entry = value_key(m);
  } else if (n > 1 && some) {
    entry = max(entry, value_key(rest));
  }
  if (n > 0) {
    if (entry) s_entry[entries++][tid] = entry;  // (one without a key is behind all others)
    bucket = max(bucket, entry);
  }
  int cnt = count.total();
  // the elements off the 16-byte grid: one each for threads of the first block
  const int odd = rank == 0 && tid < head + tail ? (tid < head ? tid : V - tail + tid - head) : -1;
  u64 odd_key = 0;
  if (odd >= 0) {
    const float y = R::one(x + odd);
    odd_key = top_key(y, odd);
    cnt += y > xt;
    if (!(y <= sum.ref + kLag)) sum.move(fmax_nan(m, y));
    m = fmax_nan(m, y);
    if (y > -INFINITY) sum.s += exp_shifted(y, sum.ref) * ex2_approx(sum.lo);
  }

  // block maximum and count
  float bm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) bm = fmax_nan(bm, __shfl_xor_sync(0xffffffffu, bm, o));
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  if (n > 0) {
    // the q-th largest bucket maximum of the warp, q = ceil(n / kWarps)
    uint32_t left = bucket, few = 0;
    for (int q = 0; q < n; q += kWarps) {
      few = __reduce_max_sync(0xffffffffu, left);
      if (__ffs(__ballot_sync(0xffffffffu, left == few)) - 1 == lane) left = 0;
    }
    if (lane == 0) s_few[warp] = few;
    if (tid == 0) s_listed = s_cands = 0;
  }
  if (lane == 0) s_max[warp] = bm, s_cnt[warp] = cnt;
  __syncthreads();
  bm = s_max[0], cnt = s_cnt[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) bm = fmax_nan(bm, s_max[w]), cnt += s_cnt[w];
  const double part = warp_dsum((double)sum.over(bm));
  if (lane == 0) s_sum[warp] = part;

  if (n > 0) {
    // n buckets reach the least of the warps' q-th maxima, so the n largest elements reach it too: list the
    // entries that do, and read them again
    uint32_t bound = s_few[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) bound = n == 1 ? max(bound, s_few[w]) : min(bound, s_few[w]);
    if (n > 1 && bound == 0) {
      // A warp has fewer buckets with anything in them than it should: the largest bound with 16 low bits of zero
      // that n of all buckets reach (0 if there are fewer), bit by bit.
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t higher = bound | 1u << bit;
        if (__syncthreads_count(bucket >= higher) >= n) bound = higher;
      }
    }
    if (bucket && bucket >= bound)
      for (int e = 0; e < entries; ++e)
        if (s_entry[e][tid] && s_entry[e][tid] >= bound) {
          const int k = atomicAdd(&s_listed, 1);
          if (k < kListed) s_list[k] = (uint16_t)(e * kThreads + tid);
        }
    const float least = bound ? key2f(bound) : -INFINITY;
    if (odd_key && (uint32_t)(odd_key >> 32) >= bound) s_cand[atomicAdd(&s_cands, 1)] = odd_key;
    if (tid < 32) s_best[tid] = 0;  // a slice with fewer elements leaves zeros
    __syncthreads();
    const int listed = s_listed;
    if (listed <= kListed)
      for (int q = tid; q < listed * group * kUnroll; q += kThreads) {
        const int e = s_list[q / (group * kUnroll)];
        const int j = lo + (e / kThreads * group * kUnroll + q % (group * kUnroll)) * kThreads + e % kThreads;
        if (j >= hi) continue;
        Vec y;
        y.load(xv + (int64_t)j * kVec);
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (y.get(k) >= least && y.get(k) > -INFINITY) {
            const int c = atomicAdd(&s_cands, 1);
            if (c < kCands) s_cand[c] = top_key(y.get(k), head + j * kVec + k);
          }
      }
    __syncthreads();
    const int nc = s_cands;
    if (listed <= kListed && nc <= kCands) {
      // few candidates: each counts the larger ones, and the best n take their places
      for (int c = tid; c < nc; c += kThreads) {
        const u64 mine = s_cand[c];
        int place = 0;
        for (int j = 0; j < nc; ++j) place += s_cand[j] > mine;
        if (place < n) s_best[place] = mine;
      }
    } else {
      // many equal or close ones: sorted lists, one per warp, merged.  A bucket whose best possible key
      // cannot enter its warp's list is not read.
      u64 list = 0;
      for (uint32_t take = __ballot_sync(0xffffffffu, odd_key != 0); take; take &= take - 1)
        list = insert(list, __shfl_sync(0xffffffffu, odd_key, __ffs(take) - 1), lane);
      for (uint32_t left = __ballot_sync(0xffffffffu, bucket && bucket >= bound); left; left &= left - 1) {
        const int owner = __ffs(left) - 1;
        const int first = lo + warp * 32 + owner;  // the bucket's first vector
        const u64 best = ((u64)__shfl_sync(0xffffffffu, bucket, owner) << 32) | (uint32_t)~(head + first * kVec);
        u64 nth = __shfl_sync(0xffffffffu, list, n - 1);
        if (best <= nth) continue;
        for (int j = first; j < hi; j += 32 * kThreads) {
          const int at = j + lane * kThreads;
          Vec b;
          if (at < hi) b.load(xv + (int64_t)at * kVec);
#pragma unroll
          for (int q = 0; q < kVec; ++q) {
            const u64 key = at < hi ? top_key(b.get(q), head + at * kVec + q) : 0;
            for (uint32_t take = __ballot_sync(0xffffffffu, key > nth); take; take &= take - 1) {
              const u64 c = __shfl_sync(0xffffffffu, key, __ffs(take) - 1);
              if (c > nth) {
                list = insert(list, c, lane);
                nth = __shfl_sync(0xffffffffu, list, n - 1);
              }
            }
          }
        }
      }
      s_best[tid] = list;
#pragma unroll
      for (int s = 1; s < kWarps; s <<= 1) {
        __syncthreads();
        if (warp % (2 * s) == 0) {
          list = merge_lists(list, s_best[(warp + s) * 32 + lane], lane);
          s_best[tid] = list;
        }
      }
    }
  }
  __syncthreads();
  Part p;
  p.sum = 0.0, p.max = bm, p.count = cnt;
  if (warp == 0) {
    for (int w = 0; w < kWarps; ++w) p.sum += s_sum[w];
  }
  if (C > 1) {
    // every block's part and list to the first block of the cluster
    cluster_wait();
    if (warp == 0 && rank != 0) {
      const uint32_t to = dsmem_map(smem_addr(&s_part[rank]), 0);
      if (lane == 0) {
        dsmem_st_f64(to + offsetof(Part, sum), p.sum);
        dsmem_st_f32(to + offsetof(Part, max), p.max);
        dsmem_st_u32(to + offsetof(Part, count), (uint32_t)p.count);
      }
      if (lane < n) dsmem_st_u64(dsmem_map(smem_addr(&s_remote[(rank - 1) * n + lane]), 0), s_best[lane]);
    }
    cluster_sync();
    if (rank != 0) return;
    if (n > 0) {
      // each of the blocks' best counts the larger ones
      const u64 mine = tid < n ? s_best[tid] : tid < C * n ? s_remote[tid - n] : 0;
      int place = 0;
      for (int j = 0; j < n; ++j) place += s_best[j] > mine;
      for (int j = 0; j < (C - 1) * n; ++j) place += s_remote[j] > mine;
      __syncthreads();
      if (mine && place < n) s_best[place] = mine;
      __syncthreads();
    }
  }
  if (warp != 0) return;
  const u64 list = lane < n ? s_best[lane] : 0;
  float top = p.max;
  for (int c = 1; c < C; ++c) top = fmax_nan(top, s_part[c].max), p.count += s_part[c].count;
  const bool uniform = !(fabsf(top) < INFINITY);  // NaN, +inf, or only -inf
  double total = p.max == -INFINITY ? 0.0 : p.sum * (double)exp_shifted(p.max, top);
  for (int c = 1; c < C; ++c)
    if (s_part[c].max != -INFINITY) total += s_part[c].sum * (double)exp_shifted(s_part[c].max, top);
  const float logsum = logf(uniform ? (float)V : (float)total);
  if (lane == 0) {
    a.out_logprobs[row] = !tok_ok ? __int_as_float(0x7fc00000) : uniform ? -logsum : (xt - top) - logsum;
    a.out_ranks[row] = !tok_ok ? 0 : uniform ? 1 : 1 + p.count;
    if (bad && a.status) atomicOr(a.status, bad);
  }
  // Where fewer than n tokens are not masked, the masked ones follow by id: among the first 64 ids (or all)
  // there are enough of them.
  const int found = __popc(__ballot_sync(0xffffffffu, list != 0));
  int masked = 0;
  if (found < n && !uniform) {
    const uint32_t m0 = __ballot_sync(0xffffffffu, lane < V && R::one(x + lane) == -INFINITY);
    const uint32_t m1 = __ballot_sync(0xffffffffu, lane + 32 < V && R::one(x + lane + 32) == -INFINITY);
    const int k = lane - found + 1;  // the k-th masked id
    masked = k <= __popc(m0) ? (int)__fns(m0, 0, max(k, 1)) : 32 + (int)__fns(m1, 0, k - __popc(m0));
  }
  if (lane < n) {
    const int64_t at = (int64_t)row * n + lane;
    const int id = uniform ? lane : list ? top_id(list) : masked;
    if (a.ids_dtype == NS_OUT_I64) static_cast<int64_t*>(a.out_top_ids)[at] = id;
    else static_cast<int32_t*>(a.out_top_ids)[at] = id;
    a.out_top_logprobs[at] = uniform ? -logsum : list ? (top_value(list) - top) - logsum : -INFINITY;
  }
}

template <typename In>
cudaError_t launch(const NsLogprobArgs& a, cudaStream_t st) {
  // Blocks per row: as many as bring about two per SM onto the GPU.  (Top 20 in us with 1, 2, 4 blocks: 256 fp32
  // rows 42, 33, 42; 1024 bf16 rows 64, 83, 115; with 2, 4, 8: 64 fp32 rows 26, 21, 21, 8 rows 18, 15, 13.5.)
  int C = 1;
  while (C < kMaxCluster && (int64_t)a.num_rows * C < 148 * 2 && a.vocab_size / C >= 4096) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.num_rows * C), 1, 1);
  // Threads per block: where the rows fill the GPU more than once, blocks of 128 have eight rows of an SM in flight
  // in place of four, and one row's search and barriers run beside the others' loads; the longest rows and few
  // ones want the larger block.  (Top 20 in us with 256, 128 threads: 4000 bf16 rows of 1000 ids 42, 26, of 16000
  // 80, 53, of 128256 199, 188; 4000 fp32 rows of 128256 335, 338; 400 fp32 rows of 1000 9.0, 8.2, of 50000 24,
  // 29.  64 threads: 29, 67, 244, 443 for the 4000 rows.)
  const int64_t row_bytes = (int64_t)a.vocab_size * (int)sizeof(In);
  const bool small = C == 1 && (row_bytes <= 16384 || (a.num_rows > 148 * 4 && row_bytes <= 262144));
  cfg.blockDim = dim3(small ? 128 : 256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, small ? logprob_kernel<In, 128> : logprob_kernel<In, 256>, a, C);
}

}  // namespace lp
}  // namespace ns

extern "C" int ns_token_logprobs(const NsLogprobArgs* args, void* stream) {
  using namespace ns;
  if (!args) return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: args is NULL");
  const NsLogprobArgs& a = *args;
  if (a.num_rows < 0) return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: num_rows < 0");
  if (a.num_rows == 0) return NS_OK;
  if (!a.logits || !a.token_ids || !a.out_logprobs || !a.out_ranks)
    return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: logits, token_ids, out_logprobs and out_ranks are required");
  if (a.logits_dtype != NS_DTYPE_F32 && a.logits_dtype != NS_DTYPE_BF16)
    return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: logits_dtype must be NS_DTYPE_F32 or NS_DTYPE_BF16");
  if (a.ids_dtype != NS_OUT_I64 && a.ids_dtype != NS_OUT_I32)
    return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: ids_dtype must be NS_OUT_I64 or NS_OUT_I32");
  if (a.vocab_size <= 0) return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: vocab_size must be positive");
  if (a.logits_row_stride < 0) return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: logits_row_stride < 0");
  if (a.num_logit_rows <= 0) return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: num_logit_rows must be positive");
  if (!a.sample_indices && a.num_logit_rows < a.num_rows)
    return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: fewer logits rows than num_rows and no sample_indices");
  if (a.top_n < 0 || a.top_n > NS_MAX_TOP_LOGPROBS || a.top_n > a.vocab_size)
    return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: top_n must be between 0 and min(vocab_size, " +
                                        std::to_string(NS_MAX_TOP_LOGPROBS) + ")");
  if (a.top_n > 0 && (!a.out_top_ids || !a.out_top_logprobs))
    return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: out_top_ids and out_top_logprobs are required for top_n > 0");
  if (a.reserved != 0) return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: reserved must be 0");
  if (reinterpret_cast<uintptr_t>(a.logits) % (a.logits_dtype == NS_DTYPE_F32 ? 4 : 2))
    return fail(NS_ERR_INVALID_ARG, "ns_token_logprobs: logits not aligned to their element");

  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      a.logits_dtype == NS_DTYPE_F32 ? lp::launch<float>(a, st) : lp::launch<__nv_bfloat16>(a, st);
  if (e != cudaSuccess) return fail(NS_ERR_CUDA, std::string("ns_token_logprobs launch: ") + cudaGetErrorString(e));
  return NS_OK;
}
