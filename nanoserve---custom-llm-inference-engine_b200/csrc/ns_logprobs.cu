// ns_logprobs.cu -- log-probabilities of given tokens, their ranks, and the
// n largest of each row (ns_token_logprobs).
//
//   L = m + log(sum_v exp(x_v - m)),  logprob = (x_t - m) - log(sum)
//   rank = 1 + #{v : x_v > x_t}
//   top n: larger logits first, equal ones by ascending id
//
// One pass over the logits gives every sum: a cluster of C blocks takes a row
// (C by the number of rows, so that few rows still fill the GPU), each block a
// contiguous slice of it, each thread every 256th 16-byte vector of the slice
// (its bucket).  A thread keeps its bucket's maximum, its sum of exponentials
// over a reference that follows the maximum in steps, and its count of larger
// logits.  The n largest are then in few buckets: those whose maximum reaches
// the n-th largest bucket maximum.  Only these are read again (out of L2); the
// elements that reach the bound are ranked by counting (or, where ties make
// them many, through sorted lists), within the block and then, through
// distributed shared memory, within the cluster.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "ns_device.cuh"

namespace ns {
int fail(int code, const std::string& msg);

namespace lp {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;         // 16-byte loads in flight per thread
constexpr int kMaxCluster = 8;     // the portable limit
constexpr float kLag = 8.0f;       // the reference follows the maximum in steps of at least this
constexpr float kHuge = 0x1p100f;  // beyond it the fused argument of the exponential could overflow
constexpr int kCands = 256;        // candidates that are ranked by counting
typedef unsigned long long u64;
static_assert(kMaxCluster * NS_MAX_TOP_LOGPROBS <= kThreads, "the cluster's lists fit into s_list");

// Larger value first, then smaller id, as one key to maximise; -0 counts as 0.
// No logit's key is 0.
__device__ __forceinline__ u64 top_key(float x, int v) {
  return ((u64)f2key(x + 0.0f) << 32) | (uint32_t)~v;
}
__device__ __forceinline__ int top_id(u64 k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float top_value(u64 k) { return key2f((uint32_t)(k >> 32)); }

template <typename In>
struct Row;

template <>
struct Row<float> {
  static constexpr int kVec = 4;
  __device__ static float one(const float* p) { return __ldg(p); }
  struct Vec {
    float4 v;
    __device__ void load(const float* p) { v = __ldg(reinterpret_cast<const float4*>(p)); }
    __device__ float get(int e) const { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; }
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
  __device__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  struct Vec {
    uint32_t w[4];
    __device__ void load(const __nv_bfloat16* p) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
    __device__ float get(int e) const { return __uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16); }
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
// once and the error of c only scales with x - ref.
struct Sum {
  float ref = -INFINITY, hi = 0.0f, lo = 0.0f, s = 0.0f;

  template <typename R, int N>
  __device__ __forceinline__ void add(const typename R::Vec (&b)[N], float bm) {
    if (!(bm <= ref + kLag)) move(bm);
    if (ref == -INFINITY) return;  // only -inf so far
    float p = 0.0f;
    if (fabsf(ref) < kHuge) {
#pragma unroll
      for (int u = 0; u < N; ++u) {
        float q = 0.0f;
#pragma unroll
        for (int e = 0; e < R::kVec; ++e) q += ex2_approx(__fmaf_rn(b[u].get(e), kLog2e, -hi));
        p += q;
      }
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

template <typename In>
__global__ void __launch_bounds__(kThreads, 4) logprob_kernel(const NsLogprobArgs a, int C) {
  using R = Row<In>;
  using Vec = typename R::Vec;
  constexpr int kVec = R::kVec;
  __shared__ float s_max[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ int s_cnt[kWarps];
  __shared__ uint32_t s_few[kWarps], s_bound;
  __shared__ int s_buckets, s_cands;
  __shared__ u64 s_list[kThreads];  // buckets, then sorted keys
  __shared__ u64 s_cand[kCands];
  __shared__ Part s_part[kMaxCluster];
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

  Sum sum;
  typename R::Count count(xt);
  float m = -INFINITY;
  int i = lo + tid;
  for (; i + (kUnroll - 1) * kThreads < hi; i += kUnroll * kThreads) {
    Vec b[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) b[u].load(xv + (int64_t)(i + u * kThreads) * kVec);
    const float bm = R::max_of(b);
    m = fmax_nan(m, bm);
    count.add(b);
    sum.template add<R>(b, bm);
  }
  for (; i < hi; i += kThreads) {
    Vec b[1];
    b[0].load(xv + (int64_t)i * kVec);
    const float bm = R::max_of(b);
    m = fmax_nan(m, bm);
    count.add(b);
    sum.template add<R>(b, bm);
  }
  // this thread's bucket: vectors lo + tid, lo + tid + kThreads, ...
  const uint32_t bucket = lo + tid < hi ? f2key(m + 0.0f) : 0u;
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
    if (tid == 0) s_buckets = s_cands = 0;
  }
  if (lane == 0) s_max[warp] = bm, s_cnt[warp] = cnt;
  __syncthreads();
  bm = s_max[0], cnt = s_cnt[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) bm = fmax_nan(bm, s_max[w]), cnt += s_cnt[w];
  const double part = warp_dsum((double)sum.over(bm));
  if (lane == 0) s_sum[warp] = part;

  if (n > 0) {
    // n buckets reach the least of the warps' q-th maxima: list the buckets that do, and find the
    // n-th largest maximum (0 if there are fewer) among them
    uint32_t few = s_few[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) few = n == 1 ? max(few, s_few[w]) : min(few, s_few[w]);
    if (bucket && bucket >= few) s_list[atomicAdd(&s_buckets, 1)] = ((u64)bucket << 32) | (uint32_t)tid;
    if (tid == 0) s_bound = few;
    __syncthreads();
    const int nb = s_buckets;
    if (n > 1 && tid < nb) {
      const uint32_t mine = (uint32_t)(s_list[tid] >> 32);
      int more = 0, same = 0;
      for (int j = 0; j < nb; ++j) {
        const uint32_t k = (uint32_t)(s_list[j] >> 32);
        more += k > mine, same += k == mine;
      }
      if (more < n && n <= more + same) s_bound = mine;  // one value, whoever writes it
    }
    __syncthreads();
    // every element that reaches the bound is in one of these buckets: read them again
    const u64 bound = (u64)s_bound << 32;
    const int chunks = (hi - lo + 32 * kThreads - 1) / (32 * kThreads);
    const int items = nb * chunks;
    for (int k = warp; k < items; k += kWarps * kUnroll) {
      Vec b[kUnroll];
      int at[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int item = k + u * kWarps;
        at[u] = -1;
        if (item < items) {
          const u64 e = s_list[item / chunks];
          const int j = lo + (int)(uint32_t)e + ((item % chunks) * 32 + lane) * kThreads;
          if (e >= bound && j < hi) at[u] = j;
        }
        if (at[u] >= 0) b[u].load(xv + (int64_t)at[u] * kVec);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (at[u] < 0) continue;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const u64 key = top_key(b[u].get(e), head + at[u] * kVec + e);
          if (key >= bound) {
            const int c = atomicAdd(&s_cands, 1);
            if (c < kCands) s_cand[c] = key;
          }
        }
      }
    }
    if (odd_key >= bound && odd_key) {
      const int c = atomicAdd(&s_cands, 1);
      if (c < kCands) s_cand[c] = odd_key;
    }
    __syncthreads();
    const int nc = s_cands;
    u64 mine = 0;
    int place = 32;
    if (nc <= kCands) {
      // few candidates: each counts the larger ones
      if (tid < nc) {
        mine = s_cand[tid];
        place = 0;
        for (int j = 0; j < nc; ++j) place += s_cand[j] > mine;
      }
    } else {
      // many equal or close ones: sorted lists, one per warp, merged.  A bucket whose best possible key
      // cannot enter its warp's list is not read.
      u64 list = 0;
      for (uint32_t take = __ballot_sync(0xffffffffu, odd_key != 0); take; take &= take - 1)
        list = insert(list, __shfl_sync(0xffffffffu, odd_key, __ffs(take) - 1), lane);
      for (int k = warp; k < nb; k += kWarps) {
        const u64 e = s_list[k];
        if (e < bound) continue;
        const int first = lo + (int)(uint32_t)e;  // the bucket's first vector
        u64 nth = __shfl_sync(0xffffffffu, list, n - 1);
        if (((e >> 32 << 32) | (uint32_t)~(head + first * kVec)) <= nth) continue;
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
      __syncthreads();  // the buckets have been read
      s_list[tid] = list;
#pragma unroll
      for (int s = 1; s < kWarps; s <<= 1) {
        __syncthreads();
        if (warp % (2 * s) == 0) {
          list = merge_lists(list, s_list[(warp + s) * 32 + lane], lane);
          s_list[tid] = list;
        }
      }
      if (warp == 0) mine = list, place = lane;
    }
    // the block's best n, in order; a slice with fewer elements leaves zeros
    __syncthreads();
    if (tid < 32) s_list[tid] = 0;
    __syncthreads();
    if (place < n) s_list[place] = mine;
  }
  __syncthreads();
  Part p;
  p.sum = 0.0, p.max = bm, p.count = cnt;
  if (warp == 0) {
    for (int w = 0; w < kWarps; ++w) p.sum += s_sum[w];
  }
  if (C > 1) {
    // every block's part and list to the first block of the cluster
    cluster_sync();  // every block of the cluster runs and is done with its lists
    if (warp == 0 && rank != 0) {
      const uint32_t to = dsmem_map(smem_addr(&s_part[rank]), 0);
      if (lane == 0) {
        dsmem_st_f64(to + offsetof(Part, sum), p.sum);
        dsmem_st_f32(to + offsetof(Part, max), p.max);
        dsmem_st_u32(to + offsetof(Part, count), (uint32_t)p.count);
      }
      if (lane < n) dsmem_st_u64(dsmem_map(smem_addr(&s_list[rank * n + lane]), 0), s_list[lane]);
    }
    cluster_sync();
    if (rank != 0) return;
    if (n > 0) {
      // each of the blocks' best counts the larger ones
      const u64 mine = tid < C * n ? s_list[tid] : 0;
      int place = 0;
      for (int j = 0; j < C * n; ++j) place += s_list[j] > mine;
      __syncthreads();
      if (mine && place < n) s_list[place] = mine;
      __syncthreads();
    }
  }
  if (warp != 0) return;
  const u64 list = lane < n ? s_list[lane] : 0;
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
  if (lane < n) {
    const int64_t at = (int64_t)row * n + lane;
    const int id = uniform ? lane : top_id(list);
    if (a.ids_dtype == NS_OUT_I64) static_cast<int64_t*>(a.out_top_ids)[at] = id;
    else static_cast<int32_t*>(a.out_top_ids)[at] = id;
    a.out_top_logprobs[at] = uniform ? -logsum : (top_value(list) - top) - logsum;
  }
}

template <typename In>
cudaError_t launch(const NsLogprobArgs& a, cudaStream_t st) {
  int C = 1;
  while (C < kMaxCluster && (int64_t)a.num_rows * C < 148 * 2 && a.vocab_size / C >= 4096) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.num_rows * C), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logprob_kernel<In>, a, C);
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
