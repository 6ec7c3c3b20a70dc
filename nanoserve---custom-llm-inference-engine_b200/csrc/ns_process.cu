// ns_process.cu -- penalties for repeated tokens, biases and grammar masks on
// logits (ns_process_logits).
//
// For every row, with seen(v) and c(v) counted from the row's history:
//   x = seen ? (x < 0 ? x * rp : x / rp) : x
//   x = x - freq * c - pres  where c > 0
//   x = x + bias             where the row has one
//   x = -inf                 where the row's mask bit is 0
//
// A block owns one tile of kTile vocabulary ids of one row.  It counts the
// row's history ids that fall into its tile in shared memory (one 32-bit word
// per id: the count, a bit for the prompt, bits for biases), copies the tile
// through (masked), and then recomputes the few ids that a penalty or a bias
// names from the input.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "ns_device.cuh"

namespace ns {
int fail(int code, const std::string& msg);

namespace proc {

constexpr int kThreads = 256;
constexpr int kTile = 8192;  // multiple of 32: a tile starts on a mask word

// Word of one vocabulary id: occurrences after the prompt in the low bits.
constexpr uint32_t kInPrompt = 1u << 31;
constexpr uint32_t kBias = 1u << 30;
constexpr uint32_t kBiasTwice = 1u << 29;
constexpr uint32_t kCount = kBiasTwice - 1;
constexpr int64_t kMaxRowIds = 1 << 28;  // a row's counts fit below the flag bits

template <typename T>
__device__ __forceinline__ float load_f(const T* p);
template <>
__device__ __forceinline__ float load_f<float>(const float* p) {
  return *p;
}
template <>
__device__ __forceinline__ float load_f<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}
__device__ __forceinline__ void store_f(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// [o[row], o[row+1]) of an array of `total` entries; empty (and flagged) where
// it leaves the array or is too long to count.
__device__ __forceinline__ int row_range(const int64_t* o, int row, int64_t total, int64_t* first, uint32_t* bad) {
  const int64_t a = o[row], b = o[row + 1];
  *first = a;
  if (a >= 0 && b >= a && b <= total && b - a <= kMaxRowIds) return (int)(b - a);
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

template <typename In, typename Out, bool kInPlace>
__global__ void __launch_bounds__(kThreads) process_kernel(const NsProcessArgs a, int tiles) {
  __shared__ uint32_t words[kTile];
  const int tid = threadIdx.x;
  const int row = blockIdx.x / tiles;
  const int v0 = (blockIdx.x % tiles) * kTile;
  const int n = min(kTile, a.vocab_size - v0);
  uint32_t bad = 0;

  int64_t src = row;
  if (a.sample_indices) {
    src = a.sample_indices[row];
    if (src < 0 || src >= a.num_logit_rows) {
      bad |= NS_STATUS_BAD_SAMPLE_INDEX;
      src = 0;
    }
  }
  const In* in = static_cast<const In*>(a.logits) + src * a.logits_row_stride + v0;
  Out* out = static_cast<Out*>(a.out) + (int64_t)row * a.out_row_stride + v0;

  const uint32_t* mask = nullptr;
  if (a.allowed) {
    const int m = a.allowed_rows ? a.allowed_rows[row] : row;
    if (m >= a.num_masks) bad |= NS_STATUS_BAD_MASK_ROW;
    else if (m >= 0) mask = reinterpret_cast<const uint32_t*>(a.allowed) + m * a.mask_stride + v0 / 32;
  }

  Penalty pen;
  pen.rep = a.repetition_penalty ? a.repetition_penalty[row] : 1.0f;
  pen.pres = a.presence_penalty ? a.presence_penalty[row] : 0.0f;
  pen.freq = a.frequency_penalty ? a.frequency_penalty[row] : 0.0f;
  const bool counts = a.history_offsets && !(pen.rep == 1.0f && pen.pres == 0.0f && pen.freq == 0.0f);
  int64_t h0 = 0, b0 = 0;
  const int hn = counts ? row_range(a.history_offsets, row, a.num_history_ids, &h0, &bad) : 0;
  const int bn = a.bias_offsets ? row_range(a.bias_offsets, row, a.num_biases, &b0, &bad) : 0;
  const int32_t* hist = a.history_ids + h0;
  const int32_t* bias = a.bias_ids + b0;
  const int prompt = a.prompt_lens ? a.prompt_lens[row] : 0;

  if (hn || bn) {
    for (int i = tid; i < n; i += kThreads) words[i] = 0;
    __syncthreads();
    for (int j = tid; j < hn; j += kThreads) {
      const int v = hist[j];
      if ((uint32_t)v >= (uint32_t)a.vocab_size) bad |= NS_STATUS_BAD_HISTORY_ID;
      const uint32_t i = (uint32_t)(v - v0);
      if (i < (uint32_t)n) {
        if (j < prompt) atomicOr(&words[i], kInPrompt);
        else atomicAdd(&words[i], 1u);
      }
    }
    for (int j = tid; j < bn; j += kThreads) {
      const int v = bias[j];
      if ((uint32_t)v >= (uint32_t)a.vocab_size) bad |= NS_STATUS_BAD_TOKEN_ID;
      const uint32_t i = (uint32_t)(v - v0);
      if (i < (uint32_t)n && (atomicOr(&words[i], kBias) & kBias)) atomicOr(&words[i], kBiasTwice);
    }
  }
  if (!kInPlace || mask) {
    for (int i = tid; i < n; i += kThreads) {
      const bool ok = !mask || ((mask[i >> 5] >> (i & 31)) & 1u);
      if (!ok) store_f(out + i, -INFINITY);
      else if (!kInPlace) store_f(out + i, load_f(in + i));
    }
  }
  if (hn || bn) {
    __syncthreads();
    // biased ids first: the row's last entry for an id takes its word
    for (int j = tid; j < bn; j += kThreads) {
      const uint32_t i = (uint32_t)(bias[j] - v0);
      if (i >= (uint32_t)n) continue;
      const uint32_t w = words[i];
      if (!(w & kBias)) continue;  // taken by the id's last entry
      if (w & kBiasTwice) {
        bool last = true;
        for (int k = j + 1; k < bn && last; ++k) last = bias[k] != bias[j];
        if (!last) continue;
      }
      words[i] = 0;
      if (mask && !((mask[i >> 5] >> (i & 31)) & 1u)) continue;
      store_f(out + i, __fadd_rn(penalised(load_f(in + i), w, pen), a.bias_values[b0 + j]));
    }
    __syncthreads();
    for (int j = tid; j < hn; j += kThreads) {
      const uint32_t i = (uint32_t)(hist[j] - v0);
      if (i >= (uint32_t)n) continue;
      const uint32_t w = atomicExch(&words[i], 0u);
      if (!w) continue;  // another occurrence, or a bias, has done it
      if (mask && !((mask[i >> 5] >> (i & 31)) & 1u)) continue;
      store_f(out + i, penalised(load_f(in + i), w, pen));
    }
  }
  if (bad && a.status) atomicOr(a.status, bad);
}

template <typename In, typename Out, bool kInPlace>
cudaError_t launch(const NsProcessArgs& a, cudaStream_t st) {
  const int tiles = (a.vocab_size + kTile - 1) / kTile;
  process_kernel<In, Out, kInPlace><<<(unsigned)(tiles * (int64_t)a.num_rows), kThreads, 0, st>>>(a, tiles);
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
  if (a.allowed && (a.num_masks < 0 || a.mask_stride < (a.vocab_size + 31) / 32))
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: num_masks < 0 or mask_stride < (vocab_size + 31) / 32");
  if (a.allowed && !a.allowed_rows && a.num_masks < a.num_rows)
    return fail(NS_ERR_INVALID_ARG, "ns_process_logits: fewer masks than num_rows and no allowed_rows");
  if (a.reserved != 0) return fail(NS_ERR_INVALID_ARG, "ns_process_logits: reserved must be 0");
  const int64_t blocks = (int64_t)((a.vocab_size + proc::kTile - 1) / proc::kTile) * a.num_rows;
  if (blocks > 0x7fffffff) return fail(NS_ERR_UNSUPPORTED, "ns_process_logits: num_rows * vocab_size is too large");

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
    e = in_place ? proc::launch<float, float, true>(a, st) : proc::launch<float, float, false>(a, st);
  else if (a.out_dtype == NS_DTYPE_F32)
    e = proc::launch<bf16, float, false>(a, st);
  else
    e = in_place ? proc::launch<bf16, bf16, true>(a, st) : proc::launch<bf16, bf16, false>(a, st);
  if (e != cudaSuccess) return fail(NS_ERR_CUDA, std::string("ns_process_logits launch: ") + cudaGetErrorString(e));
  return NS_OK;
}
