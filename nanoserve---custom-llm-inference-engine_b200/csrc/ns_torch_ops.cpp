// ns_torch_ops.cpp -- registers torch.ops.nanoserve_b200.* over the C ABI.
//
// A thin adapter: each op checks devices/dtypes, turns tensors into raw
// pointers, fills the argument struct (NsSampleArgs and its like) and calls
// the C entry point on the current CUDA stream of the tensors' device.
// No math happens here; the kernels live in libnanoserve_sampler.so.
//
// ``sample`` alone needs a workspace: each (device, stream) gets its own workspace (NsSampleArgs.workspace),
// zeroed once when it is allocated through torch's caching allocator and
// left zero by every call, so calls on different streams never share one.
// Warm a stream up before capturing a graph on it, so that the graph does
// not hold the workspace's first zeroing.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <mutex>
#include <tuple>
#include <unordered_map>
#include <vector>

#include "../../include/nanoserve_sampler.h"

namespace {

struct Workspace {
  at::Tensor t;
  bool zero_pending = false;  // made during a stream capture: its zeroing ran only inside the graph
};
std::mutex g_ws_mu;
// never destroyed: the tensors must not be freed after the CUDA context at exit
auto* g_ws = new std::unordered_map<uint64_t, Workspace>();

at::Tensor workspace_for(const at::Device& dev, cudaStream_t stream, int64_t bytes) {
  const uint64_t key = (uint64_t)reinterpret_cast<uintptr_t>(stream) * 64u + (uint64_t)dev.index();
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  TORCH_CHECK(cudaStreamIsCapturing(stream, &cap) == cudaSuccess, "cudaStreamIsCapturing failed");
  const bool capturing = cap != cudaStreamCaptureStatusNone;
  std::lock_guard<std::mutex> lk(g_ws_mu);
  auto it = g_ws->find(key);
  if (it != g_ws->end() && it->second.t.numel() >= bytes) {
    Workspace& w = it->second;
    if (w.zero_pending && !capturing) {
      // a graph made it and may never have been replayed: zero it before this eager call
      TORCH_CHECK(cudaMemsetAsync(w.t.data_ptr(), 0, (size_t)w.t.numel(), stream) == cudaSuccess,
                  "cudaMemsetAsync of the sampler workspace failed");
      w.zero_pending = false;
    }
    return w.t;
  }
  // zeroed on the current stream, the one the kernel is enqueued on (inside a
  // capture the zeroing becomes a node of the graph)
  Workspace w;
  w.t = at::zeros({bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
  w.zero_pending = capturing;
  (*g_ws)[key] = w;
  return w.t;
}

const void* opt_ptr(const c10::optional<at::Tensor>& t) {
  return (t.has_value() && t->defined()) ? t->data_ptr() : nullptr;
}

void check_cuda(const at::Tensor& t, const at::Device& dev, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void check_opt(const c10::optional<at::Tensor>& t, const at::Device& dev, const char* name, at::ScalarType st) {
  if (!t.has_value() || !t->defined()) return;
  check_cuda(*t, dev, name);
  TORCH_CHECK(t->scalar_type() == st, name, " has dtype ", t->scalar_type(), ", expected ", st);
}

// A kernel has written t: autograd's graphs that saved it notice, as after torch's own in-place operations.  (Tensors
// made in inference mode have no version.)
void wrote(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void wrote(const c10::optional<at::Tensor>& t) {
  if (t.has_value() && t->defined()) wrote(*t);
}

// sample(logits, sample_indices, row_params, history_offsets, history_ids,
//        uniforms, philox_seed, philox_offset, row_offset, out,
//        out_penalized, out_filtered, out_probs, status, row_order, kernel) -> ()
void sample_op(const at::Tensor& logits, const c10::optional<at::Tensor>& sample_indices,
               const at::Tensor& row_params, const c10::optional<at::Tensor>& history_offsets,
               const c10::optional<at::Tensor>& history_ids, const c10::optional<at::Tensor>& uniforms,
               int64_t philox_seed, int64_t philox_offset, int64_t row_offset, at::Tensor& out,
               const c10::optional<at::Tensor>& out_penalized, const c10::optional<at::Tensor>& out_filtered,
               const c10::optional<at::Tensor>& out_probs, const c10::optional<at::Tensor>& status,
               const c10::optional<at::Tensor>& row_order, int64_t kernel) {
  TORCH_CHECK(logits.dim() == 2, "logits must be 2-D [rows, vocab]");
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK(logits.stride(1) == 1, "logits rows must be contiguous");
  TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
              "logits must be float32 or bfloat16");
  const at::Device dev = logits.device();
  c10::cuda::CUDAGuard guard(dev);
  check_cuda(row_params, dev, "row_params");
  TORCH_CHECK(row_params.scalar_type() == at::kByte && row_params.numel() % (int64_t)sizeof(NsRowParams) == 0,
              "row_params must be uint8 with a multiple of ", sizeof(NsRowParams), " bytes");
  const int64_t S = row_params.numel() / (int64_t)sizeof(NsRowParams);
  check_cuda(out, dev, "out");
  TORCH_CHECK(out.numel() == S, "out must have one element per row");
  TORCH_CHECK(out.scalar_type() == at::kLong || out.scalar_type() == at::kInt, "out must be int64 or int32");
  check_opt(sample_indices, dev, "sample_indices", at::kLong);
  check_opt(history_offsets, dev, "history_offsets", at::kLong);
  check_opt(history_ids, dev, "history_ids", at::kInt);
  check_opt(uniforms, dev, "uniforms", at::kFloat);
  check_opt(out_penalized, dev, "out_penalized", at::kFloat);
  check_opt(out_filtered, dev, "out_filtered", at::kFloat);
  check_opt(out_probs, dev, "out_probs", at::kFloat);
  check_opt(status, dev, "status", at::kInt);
  check_opt(row_order, dev, "row_order", at::kInt);
  if (row_order.has_value() && row_order->defined())
    TORCH_CHECK(row_order->numel() == S, "row_order must have one element per row");
  if (sample_indices.has_value() && sample_indices->defined())
    TORCH_CHECK(sample_indices->numel() == S, "sample_indices must have one element per row");
  if (uniforms.has_value() && uniforms->defined())
    TORCH_CHECK(uniforms->numel() == S, "uniforms must have one element per row");
  if (history_offsets.has_value() && history_offsets->defined())
    TORCH_CHECK(history_offsets->numel() == S + 1, "history_offsets must have rows+1 elements");
  const int64_t V = logits.size(1);
  for (const auto* t : {&out_penalized, &out_filtered, &out_probs})
    if (t->has_value() && (*t)->defined())
      TORCH_CHECK((*t)->numel() == S * V, "debug outputs must be [rows, vocab]");

  NsSampleArgs a = {};
  a.logits = logits.data_ptr();
  a.logits_dtype = logits.scalar_type() == at::kFloat ? NS_DTYPE_F32 : NS_DTYPE_BF16;
  a.vocab_size = (int32_t)V;
  a.num_logit_rows = logits.size(0);
  // a single-row tensor may report any stride for its size-1 dimension
  a.logits_row_stride = logits.size(0) == 1 ? V : logits.stride(0);
  a.num_rows = (int32_t)S;
  a.out_dtype = out.scalar_type() == at::kLong ? NS_OUT_I64 : NS_OUT_I32;
  a.sample_indices = static_cast<const int64_t*>(opt_ptr(sample_indices));
  a.row_params = static_cast<const NsRowParams*>(row_params.data_ptr());
  a.history_offsets = static_cast<const int64_t*>(opt_ptr(history_offsets));
  a.history_ids = static_cast<const int32_t*>(opt_ptr(history_ids));
  a.uniforms = static_cast<const float*>(opt_ptr(uniforms));
  a.philox_seed = (uint64_t)philox_seed;
  a.philox_offset = (uint64_t)philox_offset;
  a.row_offset = row_offset;
  a.out_tokens = out.data_ptr();
  a.out_penalized = static_cast<float*>(const_cast<void*>(opt_ptr(out_penalized)));
  a.out_filtered = static_cast<float*>(const_cast<void*>(opt_ptr(out_filtered)));
  a.out_probs = static_cast<float*>(const_cast<void*>(opt_ptr(out_probs)));
  a.status = static_cast<uint32_t*>(const_cast<void*>(opt_ptr(status)));
  a.row_order = static_cast<const int32_t*>(opt_ptr(row_order));
  a.kernel = (int32_t)kernel;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int64_t ws_bytes = ns_workspace_bytes((int32_t)S);
  const at::Tensor ws = workspace_for(dev, stream, ws_bytes);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = ws.numel();
  const int rc = ns_sample(&a, stream);
  TORCH_CHECK(rc == NS_OK, "ns_sample failed (", rc, "): ", ns_last_error());
  wrote(out);
  for (const auto* t : {&out_penalized, &out_filtered, &out_probs, &status}) wrote(*t);
}

void check_no_grad(const at::Tensor& t, const char* op) {
  TORCH_CHECK(!t.requires_grad() || !c10::GradMode::is_enabled(), op,
              " has no gradient: call it under torch.no_grad() or on detached tensors");
}

bool given(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined(); }

void check_size(const c10::optional<at::Tensor>& t, int64_t n, const char* name) {
  if (given(t)) TORCH_CHECK(t->numel() == n, name, " must have ", n, " elements, it has ", t->numel());
}

// fp32 or bf16 rows; returns NS_DTYPE_*
int32_t check_rows(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (no CPU fallback)");
  TORCH_CHECK_VALUE(t.dim() == 2, name, " must be [rows, vocab]");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " rows must be contiguous");
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, " must be float32 or bfloat16");
  TORCH_CHECK(t.size(1) > 0 && t.size(1) <= INT32_MAX, name, " must have between 1 and 2^31 - 1 columns");
  return t.scalar_type() == at::kFloat ? NS_DTYPE_F32 : NS_DTYPE_BF16;
}

template <typename T>
T* opt_data(const c10::optional<at::Tensor>& t) {
  return static_cast<T*>(const_cast<void*>(opt_ptr(t)));
}

// process_logits_(logits, sample_indices, history_offsets, history_ids, prompt_lens, repetition_penalty,
//   presence_penalty, frequency_penalty, bias_offsets, bias_ids, bias_values, allowed, allowed_rows, status, out) -> ()
void process_logits_into(const at::Tensor& logits, const c10::optional<at::Tensor>& sample_indices,
                       const c10::optional<at::Tensor>& history_offsets, const c10::optional<at::Tensor>& history_ids,
                       const c10::optional<at::Tensor>& prompt_lens,
                       const c10::optional<at::Tensor>& repetition_penalty,
                       const c10::optional<at::Tensor>& presence_penalty,
                       const c10::optional<at::Tensor>& frequency_penalty,
                       const c10::optional<at::Tensor>& bias_offsets, const c10::optional<at::Tensor>& bias_ids,
                       const c10::optional<at::Tensor>& bias_values, const c10::optional<at::Tensor>& allowed,
                       const c10::optional<at::Tensor>& allowed_rows, const c10::optional<at::Tensor>& status,
                       at::Tensor& out) {
  NsProcessArgs a = {};
  a.logits_dtype = check_rows(logits, "logits");
  check_no_grad(logits, "process_logits");
  a.out_dtype = check_rows(out, "out");
  const at::Device dev = logits.device();
  c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK(out.device() == dev, "out must be on ", dev);
  const int64_t S = out.size(0), V = logits.size(1);
  TORCH_CHECK(S <= INT32_MAX, "out has too many rows");
  TORCH_CHECK(out.size(1) == V, "out must have the logits' columns");
  TORCH_CHECK(given(sample_indices) || logits.size(0) == S, "out must have one row per row of logits");
  check_opt(sample_indices, dev, "sample_indices", at::kLong);
  check_opt(history_offsets, dev, "history_offsets", at::kLong);
  check_opt(history_ids, dev, "history_ids", at::kInt);
  check_opt(prompt_lens, dev, "prompt_lens", at::kInt);
  check_opt(repetition_penalty, dev, "repetition_penalty", at::kFloat);
  check_opt(presence_penalty, dev, "presence_penalty", at::kFloat);
  check_opt(frequency_penalty, dev, "frequency_penalty", at::kFloat);
  check_opt(bias_offsets, dev, "bias_offsets", at::kLong);
  check_opt(bias_ids, dev, "bias_ids", at::kInt);
  check_opt(bias_values, dev, "bias_values", at::kFloat);
  check_opt(allowed_rows, dev, "allowed_rows", at::kInt);
  check_opt(status, dev, "status", at::kInt);
  check_size(sample_indices, S, "sample_indices");
  check_size(history_offsets, S + 1, "history_offsets");
  check_size(prompt_lens, S, "prompt_lens");
  check_size(repetition_penalty, S, "repetition_penalty");
  check_size(presence_penalty, S, "presence_penalty");
  check_size(frequency_penalty, S, "frequency_penalty");
  check_size(bias_offsets, S + 1, "bias_offsets");
  check_size(allowed_rows, S, "allowed_rows");
  check_size(status, 1, "status");
  TORCH_CHECK(given(history_offsets) == given(history_ids), "history_offsets and history_ids go together");
  TORCH_CHECK(given(bias_offsets) == given(bias_ids) && given(bias_ids) == given(bias_values),
              "bias_offsets, bias_ids and bias_values go together");
  if (given(bias_ids)) check_size(bias_values, bias_ids->numel(), "bias_values");
  TORCH_CHECK(given(allowed) || !given(allowed_rows), "allowed_rows given without allowed");
  if (given(allowed)) {
    TORCH_CHECK(allowed->is_cuda() && allowed->device() == dev, "allowed must be on ", dev);
    TORCH_CHECK(allowed->scalar_type() == at::kInt && allowed->dim() == 2 && allowed->size(1) >= (V + 31) / 32 &&
                    allowed->stride(1) == 1,
                "allowed must be int32 [masks, at least ", (V + 31) / 32, " words], its rows contiguous");
    TORCH_CHECK(allowed->size(0) <= INT32_MAX, "allowed has too many rows");
    TORCH_CHECK(allowed->size(0) <= 1 || allowed->stride(0) >= (V + 31) / 32, "allowed's rows overlap");
    TORCH_CHECK(given(allowed_rows) || allowed->size(0) == S, "allowed must have one row per row, or allowed_rows");
    a.allowed = static_cast<const int32_t*>(allowed->data_ptr());
    a.mask_stride = std::max<int64_t>(allowed->stride(0), (V + 31) / 32);
    a.num_masks = (int32_t)allowed->size(0);
  }
  if (S == 0) return;
  a.logits = logits.data_ptr();
  a.vocab_size = (int32_t)V;
  a.num_logit_rows = logits.size(0);
  a.logits_row_stride = logits.size(0) == 1 ? V : logits.stride(0);
  a.num_rows = (int32_t)S;
  a.sample_indices = opt_data<const int64_t>(sample_indices);
  a.history_offsets = opt_data<const int64_t>(history_offsets);
  a.history_ids = opt_data<const int32_t>(history_ids);
  a.num_history_ids = given(history_ids) ? history_ids->numel() : 0;
  a.prompt_lens = opt_data<const int32_t>(prompt_lens);
  a.repetition_penalty = opt_data<const float>(repetition_penalty);
  a.presence_penalty = opt_data<const float>(presence_penalty);
  a.frequency_penalty = opt_data<const float>(frequency_penalty);
  a.bias_offsets = opt_data<const int64_t>(bias_offsets);
  a.bias_ids = opt_data<const int32_t>(bias_ids);
  a.bias_values = opt_data<const float>(bias_values);
  a.num_biases = given(bias_ids) ? bias_ids->numel() : 0;
  a.allowed_rows = opt_data<const int32_t>(allowed_rows);
  a.out = out.data_ptr();
  a.out_row_stride = S == 1 ? V : out.stride(0);
  a.status = opt_data<uint32_t>(status);
  const int rc = ns_process_logits(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  TORCH_CHECK(rc == NS_OK, "ns_process_logits failed (", rc, "): ", ns_last_error());
  wrote(status);
}

void process_logits_into_op(const at::Tensor& logits, const c10::optional<at::Tensor>& sample_indices,
                            const c10::optional<at::Tensor>& history_offsets,
                            const c10::optional<at::Tensor>& history_ids,
                            const c10::optional<at::Tensor>& prompt_lens,
                            const c10::optional<at::Tensor>& repetition_penalty,
                            const c10::optional<at::Tensor>& presence_penalty,
                            const c10::optional<at::Tensor>& frequency_penalty,
                            const c10::optional<at::Tensor>& bias_offsets,
                            const c10::optional<at::Tensor>& bias_ids, const c10::optional<at::Tensor>& bias_values,
                            const c10::optional<at::Tensor>& allowed, const c10::optional<at::Tensor>& allowed_rows,
                            const c10::optional<at::Tensor>& status, at::Tensor& out) {
  check_no_grad(out, "process_logits");
  process_logits_into(logits, sample_indices, history_offsets, history_ids, prompt_lens, repetition_penalty,
                      presence_penalty, frequency_penalty, bias_offsets, bias_ids, bias_values, allowed, allowed_rows,
                      status, out);
  wrote(out);
}

// Rows whose elements are next to each other (a copy of columns that are not).
at::Tensor packed_rows(const at::Tensor& t) {
  return t.dim() == 2 && t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
}

// process_logits(logits, ..., status, out_dtype) -> a new tensor
at::Tensor process_logits_op(const at::Tensor& given_logits, const c10::optional<at::Tensor>& sample_indices,
                             const c10::optional<at::Tensor>& history_offsets,
                             const c10::optional<at::Tensor>& history_ids,
                             const c10::optional<at::Tensor>& prompt_lens,
                             const c10::optional<at::Tensor>& repetition_penalty,
                             const c10::optional<at::Tensor>& presence_penalty,
                             const c10::optional<at::Tensor>& frequency_penalty,
                             const c10::optional<at::Tensor>& bias_offsets,
                             const c10::optional<at::Tensor>& bias_ids, const c10::optional<at::Tensor>& bias_values,
                             const c10::optional<at::Tensor>& allowed, const c10::optional<at::Tensor>& allowed_rows,
                             const c10::optional<at::Tensor>& status, c10::optional<at::ScalarType> out_dtype) {
  const at::Tensor logits = packed_rows(given_logits);
  check_rows(logits, "logits");
  TORCH_CHECK_VALUE(!out_dtype || *out_dtype == logits.scalar_type() || *out_dtype == at::kFloat,
                    "out_dtype must be the logits' type or float32");
  const int64_t S = given(sample_indices) ? sample_indices->numel() : logits.size(0);
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor out = at::empty({S, logits.size(1)}, logits.options().dtype(out_dtype.value_or(logits.scalar_type())));
  process_logits_into(logits, sample_indices, history_offsets, history_ids, prompt_lens, repetition_penalty,
                      presence_penalty, frequency_penalty, bias_offsets, bias_ids, bias_values, allowed, allowed_rows,
                      status, out);
  return out;
}

// token_logprobs(logits, sample_indices, token_ids, top_n, status) -> (logprobs, ranks, top_ids, top_logprobs)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs_op(
    const at::Tensor& given_logits, const c10::optional<at::Tensor>& sample_indices,
    const at::Tensor& given_ids, int64_t n, const c10::optional<at::Tensor>& status) {
  const at::Tensor logits = packed_rows(given_logits), token_ids = given_ids.contiguous();
  NsLogprobArgs a = {};
  a.logits_dtype = check_rows(logits, "logits");
  check_no_grad(logits, "token_logprobs");
  const at::Device dev = logits.device();
  c10::cuda::CUDAGuard guard(dev);
  check_cuda(token_ids, dev, "token_ids");
  TORCH_CHECK(token_ids.scalar_type() == at::kLong || token_ids.scalar_type() == at::kInt,
              "token_ids must be int64 or int32");
  const int64_t S = token_ids.numel(), V = logits.size(1);
  TORCH_CHECK(S <= INT32_MAX, "token_ids has too many elements");
  TORCH_CHECK(given(sample_indices) || logits.size(0) == S, "token_ids must have one element per row of logits");
  check_opt(sample_indices, dev, "sample_indices", at::kLong);
  check_size(sample_indices, S, "sample_indices");
  check_opt(status, dev, "status", at::kInt);
  check_size(status, 1, "status");
  TORCH_CHECK_VALUE(n >= 0 && n <= NS_MAX_TOP_LOGPROBS && n <= V, "top_n must be between 0 and min(vocab, ",
                    NS_MAX_TOP_LOGPROBS, "), got ", n);
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor out_logprobs = at::empty({S}, f32), out_ranks = at::empty({S}, f32.dtype(at::kInt));
  at::Tensor out_top_ids = at::empty({S, n}, token_ids.options()), out_top_logprobs = at::empty({S, n}, f32);
  const auto result = std::make_tuple(out_logprobs, out_ranks, out_top_ids, out_top_logprobs);
  if (S == 0) return result;
  a.logits = logits.data_ptr();
  a.vocab_size = (int32_t)V;
  a.num_logit_rows = logits.size(0);
  a.logits_row_stride = logits.size(0) == 1 ? V : logits.stride(0);
  a.num_rows = (int32_t)S;
  a.ids_dtype = token_ids.scalar_type() == at::kLong ? NS_OUT_I64 : NS_OUT_I32;
  a.sample_indices = opt_data<const int64_t>(sample_indices);
  a.token_ids = token_ids.data_ptr();
  a.top_n = (int32_t)n;
  a.out_logprobs = static_cast<float*>(out_logprobs.data_ptr());
  a.out_ranks = static_cast<int32_t*>(out_ranks.data_ptr());
  a.out_top_ids = out_top_ids.data_ptr();
  a.out_top_logprobs = static_cast<float*>(out_top_logprobs.data_ptr());
  a.status = opt_data<uint32_t>(status);
  const int rc = ns_token_logprobs(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  TORCH_CHECK(rc == NS_OK, "ns_token_logprobs failed (", rc, "): ", ns_last_error());
  wrote(status);
  return result;
}

constexpr int64_t kLongList = 3500;  // what ns_pages_copy takes in one launch

// copy_pages(pools, src, dst) -> (): src and dst are CPU int64 lists of pages
void copy_pages_op(at::TensorList pools, const at::Tensor& src, const at::Tensor& dst) {
  TORCH_CHECK(src.device().is_cpu() && dst.device().is_cpu() && src.scalar_type() == at::kLong &&
                  dst.scalar_type() == at::kLong && src.is_contiguous() && dst.is_contiguous(),
              "src and dst must be contiguous int64 CPU tensors");
  TORCH_CHECK_VALUE(src.numel() == dst.numel(), src.numel(), " source pages and ", dst.numel(), " destination pages");
  if (pools.empty()) return;
  const at::Device dev = pools[0].device();
  TORCH_CHECK(dev.is_cuda(), "copy_pages needs CUDA pools (no CPU fallback)");
  const int64_t num_pages = pools[0].dim() > 0 ? pools[0].size(0) : 0;
  std::vector<NsPagePool> p;
  p.reserve(pools.size());
  for (const at::Tensor& t : pools) {
    TORCH_CHECK(t.is_cuda() && t.device() == dev, "pools must be CUDA tensors on one device");
    check_no_grad(t, "copy_pages");
    TORCH_CHECK(t.dim() > 0 && t.size(0) == num_pages, "pools must have the same number of pages (dimension 0)");
    int64_t elems = 1;
    bool packed = true;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
      packed = packed && (t.size(d) == 1 || t.stride(d) == elems);
      elems *= t.size(d);
    }
    TORCH_CHECK(packed, "each page of a pool must be contiguous");
    const int64_t stride = num_pages > 1 ? t.stride(0) : elems;
    TORCH_CHECK(num_pages <= 1 || stride >= elems, "a pool's pages overlap");
    if (elems == 0 || num_pages == 0) continue;
    p.push_back({t.data_ptr(), stride * (int64_t)t.element_size(), elems * (int64_t)t.element_size()});
  }
  if (p.empty()) {
    TORCH_CHECK(num_pages > 0 || src.numel() == 0, "page outside an empty pool");
    return;
  }
  c10::cuda::CUDAGuard guard(dev);
  const int64_t n = src.numel();
  const int64_t *s = static_cast<const int64_t*>(src.data_ptr()), *d = static_cast<const int64_t*>(dst.data_ptr());
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (n > kLongList)
    TORCH_CHECK(cudaStreamIsCapturing(stream, &cap) == cudaSuccess, "cudaStreamIsCapturing failed");
  int rc;
  if (n > kLongList && cap == cudaStreamCaptureStatusNone && num_pages <= INT32_MAX) {
    rc = ns_pages_check(num_pages, s, d, n);
    if (rc == NS_OK) {
      // one copy of the lists (both allocators keep what is in flight) in place of a launch for each few thousand
      const at::Tensor host = at::empty({2, n}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
      host[0].copy_(src.view({n}));
      host[1].copy_(dst.view({n}));
      const at::Tensor lists = host.to(dev, /*non_blocking=*/true);
      const int32_t* l = static_cast<const int32_t*>(lists.data_ptr());
      rc = ns_pages_copy_listed(p.data(), (int32_t)p.size(), num_pages, l, l + n, n, nullptr, stream);
    }
  } else {
    rc = ns_pages_copy(p.data(), (int32_t)p.size(), num_pages, s, d, n, stream);
  }
  TORCH_CHECK_VALUE(rc != NS_ERR_INVALID_ARG, ns_last_error());
  TORCH_CHECK(rc == NS_OK, "ns_pages_copy failed (", rc, "): ", ns_last_error());
  if (n > 0)
    for (const at::Tensor& t : pools) wrote(t);
}

// paged_history_gather(pool, pages, page_offsets, history_offsets, out, status) -> ()
void paged_history_gather_op(const at::Tensor& pool, const at::Tensor& pages, const at::Tensor& page_offsets,
                             const at::Tensor& history_offsets, at::Tensor& out,
                             const c10::optional<at::Tensor>& status) {
  TORCH_CHECK(pool.is_cuda(), "pool must be a CUDA tensor (no CPU fallback)");
  const at::Device dev = pool.device();
  c10::cuda::CUDAGuard guard(dev);
  check_opt(pool, dev, "pool", at::kInt);
  check_opt(pages, dev, "pages", at::kInt);
  check_opt(page_offsets, dev, "page_offsets", at::kLong);
  check_opt(history_offsets, dev, "history_offsets", at::kLong);
  check_opt(out, dev, "out", at::kInt);
  check_opt(status, dev, "status", at::kInt);
  check_size(status, 1, "status");
  TORCH_CHECK(pool.dim() == 2 && pool.size(1) > 0 && pool.size(1) <= INT32_MAX, "pool must be [pages, page_size]");
  TORCH_CHECK(history_offsets.numel() >= 1 && history_offsets.numel() <= INT32_MAX,
              "history_offsets must have rows+1 elements");
  TORCH_CHECK(page_offsets.numel() == history_offsets.numel(), "page_offsets must have rows+1 elements");
  const int rc = ns_paged_history_gather(
      static_cast<const int32_t*>(pool.data_ptr()), pool.size(0), (int32_t)pool.size(1),
      static_cast<const int32_t*>(pages.data_ptr()), pages.numel(), static_cast<const int64_t*>(page_offsets.data_ptr()),
      static_cast<const int64_t*>(history_offsets.data_ptr()), (int32_t)(history_offsets.numel() - 1),
      static_cast<int32_t*>(out.data_ptr()), out.numel(), opt_data<uint32_t>(status),
      c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  TORCH_CHECK(rc == NS_OK, "ns_paged_history_gather failed (", rc, "): ", ns_last_error());
  wrote(out);
  wrote(status);
}

}  // namespace

TORCH_LIBRARY(nanoserve_b200, m) {
  m.def(
      "sample(Tensor logits, Tensor? sample_indices, Tensor row_params, Tensor? history_offsets, "
      "Tensor? history_ids, Tensor? uniforms, int philox_seed, int philox_offset, int row_offset, "
      "Tensor(a!) out, Tensor(b!)? out_penalized, Tensor(c!)? out_filtered, Tensor(d!)? out_probs, "
      "Tensor(e!)? status, Tensor? row_order=None, int kernel=0) -> ()");
  m.def(
      "process_logits(Tensor logits, Tensor? sample_indices, Tensor? history_offsets, Tensor? history_ids, "
      "Tensor? prompt_lens, Tensor? repetition_penalty, Tensor? presence_penalty, Tensor? frequency_penalty, "
      "Tensor? bias_offsets, Tensor? bias_ids, Tensor? bias_values, Tensor? allowed, Tensor? allowed_rows, "
      "Tensor(a!)? status=None, ScalarType? out_dtype=None) -> Tensor");
  m.def(
      "process_logits_(Tensor logits, Tensor? sample_indices, Tensor? history_offsets, Tensor? history_ids, "
      "Tensor? prompt_lens, Tensor? repetition_penalty, Tensor? presence_penalty, Tensor? frequency_penalty, "
      "Tensor? bias_offsets, Tensor? bias_ids, Tensor? bias_values, Tensor? allowed, Tensor? allowed_rows, "
      "Tensor(a!)? status, Tensor(b!) out) -> ()");
  m.def(
      "token_logprobs(Tensor logits, Tensor? sample_indices, Tensor token_ids, int top_n, Tensor(a!)? status=None) "
      "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("copy_pages(Tensor(a!)[] pools, Tensor src, Tensor dst) -> ()");
  m.def(
      "paged_history_gather(Tensor pool, Tensor pages, Tensor page_offsets, Tensor history_offsets, "
      "Tensor(a!) out, Tensor(b!)? status=None) -> ()");
}

// CPU tensors get the ops' own message
TORCH_LIBRARY_IMPL(nanoserve_b200, CPU, m) {
  m.impl("process_logits", &process_logits_op);
  m.impl("process_logits_", &process_logits_into_op);
  m.impl("token_logprobs", &token_logprobs_op);
  m.impl("copy_pages", &copy_pages_op);
  m.impl("paged_history_gather", &paged_history_gather_op);
}

// these have no gradient and say so themselves, and say what they wrote: no autograd layer to go through
TORCH_LIBRARY_IMPL(nanoserve_b200, Autograd, m) {
  for (const char* op : {"process_logits", "process_logits_", "token_logprobs", "copy_pages", "paged_history_gather"})
    m.impl(op, torch::CppFunction::makeFallthrough());
}

TORCH_LIBRARY_IMPL(nanoserve_b200, CUDA, m) {
  m.impl("sample", &sample_op);
  m.impl("process_logits", &process_logits_op);
  m.impl("process_logits_", &process_logits_into_op);
  m.impl("token_logprobs", &token_logprobs_op);
  m.impl("copy_pages", &copy_pages_op);
  m.impl("paged_history_gather", &paged_history_gather_op);
}
