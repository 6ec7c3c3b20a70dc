// ns_logprobs.cu -- log-probabilities of given tokens, their ranks, and the
// n largest of each row (ns_token_logprobs).
//
//   L = m + log(sum_v exp(x_v - m)),  logprob = (x_t - m) - log(sum)
//   rank = 1 + #{v : x_v > x_t}
//   top n: larger logits first, equal ones by ascending id
//
// One block per row.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "ns_device.cuh"

namespace ns {
int fail(int code, const std::string& msg);

namespace lp {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ float load_f(const float* p) { return *p; }
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Larger value first, then smaller id, as one key to maximise; -0 counts as 0.
__device__ __forceinline__ unsigned long long top_key(float x, int v) {
  return ((unsigned long long)f2key(x + 0.0f) << 32) | (uint32_t)~v;
}
__device__ __forceinline__ int top_id(unsigned long long k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float top_value(unsigned long long k) { return key2f((uint32_t)(k >> 32)); }

template <typename In>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const NsLogprobArgs a) {
  __shared__ float s_max[kWarps];
  __shared__ double s_sum[kWarps];
  __shared__ int s_cnt[kWarps];
  __shared__ unsigned long long s_key[kWarps], s_best;
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int V = a.vocab_size;
  uint32_t bad = 0;
  int64_t src = row;
  if (a.sample_indices) {
    src = a.sample_indices[row];
    if (src < 0 || src >= a.num_logit_rows) {
      bad |= NS_STATUS_BAD_SAMPLE_INDEX;
      src = 0;
    }
  }
  const In* x = static_cast<const In*>(a.logits) + src * a.logits_row_stride;
  const int64_t t = a.ids_dtype == NS_OUT_I64 ? static_cast<const int64_t*>(a.token_ids)[row]
                                              : static_cast<const int32_t*>(a.token_ids)[row];
  const bool tok_ok = t >= 0 && t < V;
  if (!tok_ok) bad |= NS_STATUS_BAD_TOKEN_ID;
  const float xt = tok_ok ? load_f(x + t) : 0.0f;

  float m = -INFINITY;
  int cnt = 0;
  for (int v = tid; v < V; v += kThreads) {
    const float y = load_f(x + v);
    m = fmax_nan(m, y);
    cnt += y > xt;
  }
  for (int o = 16; o; o >>= 1) {
    m = fmax_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
  }
  if (lane == 0) s_max[warp] = m, s_cnt[warp] = cnt;
  __syncthreads();
  m = s_max[0], cnt = s_cnt[0];
  for (int w = 1; w < kWarps; ++w) m = fmax_nan(m, s_max[w]), cnt += s_cnt[w];
  const bool uniform = !(fabsf(m) < INFINITY);  // NaN, +inf, or only -inf

  double sum = 0.0;
  if (!uniform)
    for (int v = tid; v < V; v += kThreads) sum += (double)exp_shifted(load_f(x + v), m);
  sum = warp_dsum(sum);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kWarps; ++w) sum += s_sum[w];
  const float logsum = uniform ? logf((float)V) : (float)log(sum);

  if (tid == 0) {
    a.out_logprobs[row] = !tok_ok ? __int_as_float(0x7fc00000) : uniform ? -logsum : (xt - m) - logsum;
    a.out_ranks[row] = !tok_ok ? 0 : uniform ? 1 : 1 + cnt;
    if (bad && a.status) atomicOr(a.status, bad);
  }

  unsigned long long below = ~0ull;
  for (int j = 0; j < a.top_n; ++j) {
    unsigned long long best = 0;
    if (!uniform)
      for (int v = tid; v < V; v += kThreads) {
        const unsigned long long k = top_key(load_f(x + v), v);
        if (k < below && k > best) best = k;
      }
    for (int o = 16; o; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) s_key[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kWarps; ++w) best = s_key[w] > best ? s_key[w] : best;
      s_best = best;
      const int64_t at = (int64_t)row * a.top_n + j;
      const int id = uniform ? j : top_id(best);
      if (a.ids_dtype == NS_OUT_I64) static_cast<int64_t*>(a.out_top_ids)[at] = id;
      else static_cast<int32_t*>(a.out_top_ids)[at] = id;
      a.out_top_logprobs[at] = uniform ? -logsum : (top_value(best) - m) - logsum;
    }
    __syncthreads();
    below = s_best;
  }
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
  if (a.logits_dtype == NS_DTYPE_F32)
    lp::logprob_kernel<float><<<a.num_rows, lp::kThreads, 0, st>>>(a);
  else
    lp::logprob_kernel<__nv_bfloat16><<<a.num_rows, lp::kThreads, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(NS_ERR_CUDA, std::string("ns_token_logprobs launch: ") + cudaGetErrorString(e));
  return NS_OK;
}
