// Python bindings of the operators beside the sync: token log probabilities (wb_logprobs.cu) and
// the optimizer kernels (wb_optim.cu).  Argument checks live here: everything a kernel relies on
// (types, sizes, strides, devices) is checked on the host before a launch, and a call that does not
// fit raises ValueError.  Outputs and scratch come from torch's allocator on the current stream of
// the tensors' device, and the kernels run on that stream, so calls on different streams share nothing.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <limits>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "wb_learn.h"
#include "wb_logprobs.h"
#include "wb_optim.h"

namespace py = pybind11;

namespace {

using at::Tensor;

[[noreturn]] void bad(const std::string& what) { throw std::invalid_argument(what); }

void check(cudaError_t e, const char* what) {
  if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

uint32_t float_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return wb::DT_BF16;
    case at::kHalf: return wb::DT_F16;
    case at::kFloat: return wb::DT_F32;
    default: return 0;
  }
}

std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
  return s + "]";
}

// Why a tensor's memory may not be read as its values, or null.  Wrappers of other tensors (DTensor, what
// torch.func hands to a function) and lazy zeros have no memory of their own, some an address of 0; a
// forward mode derivative would be lost without a word.
const char* unfit(const Tensor& t, bool dual) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet kWrappers({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::FuncTorchBatched,
                                           DispatchKey::FuncTorchGradWrapper, DispatchKey::Batched, DispatchKey::ZeroTensor});
  if (t.key_set().has_any(kWrappers) || t.layout() != at::kStrided)
    return " is a sparse tensor or a wrapper (DTensor, a transform's): give the plain local tensor (to_local())";
  if (const int64_t n = t.numel()) {
    size_t bytes = (size_t)(t.storage_offset() + n) * t.itemsize();
    if (!t.is_non_overlapping_and_dense()) bytes = at::detail::computeStorageNbytes(t.sizes(), t.strides(), t.itemsize(), t.storage_offset());
    if (bytes > t.storage().nbytes()) return " has less memory than its shape asks for: its storage was released";
  }
  if (t.is_neg()) return " is negated lazily, its memory holds other values: give resolve_neg() of it";
  if (dual && t._fw_grad(0).defined()) return " carries a derivative of forward mode, which is not implemented: give the primal";
  return nullptr;
}

// Whether forward mode derivatives can be about: asked once a call, since asking a view for its own takes 25 ns.
bool duals() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

int sm_count(int device) {
  static std::array<int, 64> known{};          // one attribute query per device; the value never changes
  int v = device < 64 ? known[device] : 0;
  if (!v) {
    check(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device), "cudaDeviceGetAttribute");
    if (device < 64) known[device] = v;
  }
  return v;
}

// -- token log probabilities ----------------------------------------------------------------------
// The leading dimensions as (outer, inner) with one stride each: any tensor of up to two leading
// dimensions, and more where they merge.
struct Lead { int64_t outer = 1, inner = 1, s_outer = 0, s_inner = 0; };

std::optional<Lead> lead_of(const Tensor& t, int64_t dims) {
  std::vector<std::pair<int64_t, int64_t>> d;      // (size, stride), merged
  for (int64_t k = 0; k < dims; ++k) {
    const int64_t n = t.size(k), s = t.stride(k);
    if (n == 1) continue;
    if (!d.empty() && d.back().second == n * s) d.back() = {d.back().first * n, s};
    else d.push_back({n, s});
  }
  if (d.size() > 2) return std::nullopt;
  Lead l;
  if (d.size() == 2) l.outer = d[0].first, l.s_outer = d[0].second;
  if (!d.empty()) l.inner = d.back().first, l.s_inner = d.back().second;
  return l;
}

struct LogprobOptions {
  int64_t vocab = 0, ignore_index = -100;
  double temperature = 1.0;
  int64_t top_k = 0;
};

wb::LogprobRows rows_of(const Tensor& logits, const Tensor& tokens, const LogprobOptions& o, Tensor& tokens_kept) {
  const int64_t lead = logits.dim() - 1;
  auto l = lead_of(logits, lead);
  if (!l) bad("token_logprobs: logits of shape " + shape_of(logits) + " have more than two leading dimensions that do not "
              "merge into one; pass a tensor of two leading dimensions");
  wb::LogprobRows in{};
  // the tokens follow the logits' split of the rows; where their own strides do not, a packed copy does
  tokens_kept = tokens;
  auto t = lead_of(tokens, lead);
  if (!t || t->inner != l->inner || t->outer != l->outer) {
    if (t && t->outer == 1) {
      t->outer = l->outer, t->s_outer = l->inner * t->s_inner, t->inner = l->inner;   // one stride: any split
    } else {
      tokens_kept = tokens.contiguous();
      t = Lead{l->outer, l->inner, l->inner, 1};
    }
  }
  in.logits = logits.const_data_ptr();
  in.tokens = tokens_kept.const_data_ptr();
  in.stride_outer = l->s_outer;
  in.stride_inner = l->s_inner;
  in.tok_outer = t->s_outer;
  in.tok_inner = t->s_inner;
  in.rows = (uint32_t)tokens.numel();
  in.inner = (uint32_t)std::max<int64_t>(l->inner, 1);
  in.vocab = (uint32_t)o.vocab;
  in.dtype = float_code(logits.scalar_type());
  in.tokens_i32 = tokens.scalar_type() == at::kInt;
  in.inv_temp = (float)(1.0 / o.temperature);
  in.ignore_index = o.ignore_index;
  return in;
}

struct LogprobResult { Tensor logprobs, entropy, stats, top_logprobs, top_ids; };

LogprobResult run_logprobs(const Tensor& logits, const Tensor& tokens, const LogprobOptions& o, bool stats) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  LogprobResult r;
  r.logprobs = at::empty(tokens.sizes(), f32);
  r.entropy = at::empty(tokens.sizes(), f32);
  wb::LogprobOut out{};
  if (stats) {
    r.stats = at::empty({tokens.numel(), 2}, f32);
    out.stats = r.stats.mutable_data_ptr<float>();
  }
  if (o.top_k) {
    auto shape = tokens.sizes().vec();
    shape.push_back(o.top_k);
    r.top_logprobs = at::empty(shape, f32);
    r.top_ids = at::empty(shape, f32.dtype(at::kLong));
    out.top_logprobs = r.top_logprobs.mutable_data_ptr<float>();
    out.top_ids = r.top_ids.mutable_data_ptr<int64_t>();
  }
  out.logprobs = r.logprobs.mutable_data_ptr<float>();
  out.entropy = r.entropy.mutable_data_ptr<float>();
  out.top_k = (int)o.top_k;
  if (tokens.numel() == 0) return r;
  Tensor kept;
  const wb::LogprobRows in = rows_of(logits, tokens, o, kept);
  check(wb::launch_token_logprobs(in, out, sm_count(logits.device().index()), c10::cuda::getCurrentCUDAStream()), "token_logprobs launch");
  return r;
}

// A gradient over the rows as one stride (autograd hands expanded ones).
Tensor row_grad(const Tensor& g, const float*& ptr, int64_t& stride) {
  if (!g.defined()) return g;
  Tensor t = g.to(at::kFloat).resolve_neg();             // the engine may hand a lazily negated one; both leave an ordinary one alone
  auto l = lead_of(t, t.dim());
  if (!l || l->outer != 1) {
    t = t.contiguous();
    l = lead_of(t, t.dim());
  }
  ptr = t.const_data_ptr<float>();
  stride = l->s_inner;
  return t;
}

[[noreturn]] void replaced() {
  throw std::runtime_error("token_logprobs: a hook brought a saved tensor back on another device or in another shape or type");
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const Tensor& tokens,
                                                int64_t vocab, double temperature, int64_t top_k, int64_t ignore_index) {
    const LogprobOptions o{vocab, ignore_index, temperature, top_k};
    LogprobResult r = run_logprobs(logits, tokens, o, true);
    ctx->save_for_backward({logits, tokens, r.stats, r.entropy});
    ctx->saved_data["rows"] = tokens.numel();
    ctx->saved_data["cols"] = logits.size(-1);
    ctx->saved_data["vocab"] = vocab;
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->set_materialize_grads(false);
    if (!top_k) return {r.logprobs, r.entropy};
    ctx->mark_non_differentiable({r.top_logprobs, r.top_ids});
    return {r.logprobs, r.entropy, r.top_logprobs, r.top_ids};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled())
      throw std::runtime_error("token_logprobs: the gradient has no second derivative (create_graph=True)");
    const auto saved = ctx->get_saved_variables();
    // Hooks on saved tensors may have brought other ones back.
    const Tensor &tokens = saved[1], stats = saved[2].contiguous(), entropy = saved[3].contiguous();
    const Tensor logits = saved[0].size(-1) > 1 && saved[0].stride(-1) != 1 ? saved[0].contiguous() : saved[0];
    for (const Tensor* x : {&logits, &tokens, &stats, &entropy})
      if (unfit(*x, false) || !x->is_cuda() || x->device() != logits.device()) replaced();
    for (const Tensor& g : grads)
      if (g.defined() && g.device() != logits.device()) replaced();
    if (!float_code(logits.scalar_type()) || logits.dim() != tokens.dim() + 1 || tokens.sizes() != logits.sizes().slice(0, tokens.dim()) ||
        logits.size(-1) != ctx->saved_data["cols"].toInt() || (tokens.scalar_type() != at::kLong && tokens.scalar_type() != at::kInt) ||
        tokens.numel() != ctx->saved_data["rows"].toInt() || stats.scalar_type() != at::kFloat || entropy.scalar_type() != at::kFloat ||
        stats.numel() != 2 * tokens.numel() || entropy.numel() != tokens.numel())
      replaced();
    const LogprobOptions o{ctx->saved_data["vocab"].toInt(), ctx->saved_data["ignore_index"].toInt(),
                           ctx->saved_data["temperature"].toDouble(), 0};
    const c10::cuda::CUDAGuard guard(logits.device());
    Tensor grad = at::empty(logits.sizes(), logits.options());
    if (tokens.numel()) {
      wb::LogprobGrad g{};
      const Tensor a = row_grad(grads[0], g.g_logprobs, g.g_logprobs_stride);
      const Tensor b = row_grad(grads[1], g.g_entropy, g.g_entropy_stride);
      g.stats = stats.const_data_ptr<float>();
      g.entropy = entropy.const_data_ptr<float>();
      g.grad = grad.mutable_data_ptr();
      g.cols = (uint32_t)logits.size(-1);
      Tensor kept;
      const wb::LogprobRows in = rows_of(logits, tokens, o, kept);
      check(wb::launch_token_logprobs_grad(in, g, c10::cuda::getCurrentCUDAStream()), "token_logprobs gradient launch");
    }
    return {grad, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

py::tuple token_logprobs(const Tensor& logits, const Tensor& tokens, const std::optional<int64_t>& columns, double temperature,
                         int64_t top_k, int64_t ignore_index) {
  for (const Tensor* x : {&logits, &tokens})
    if (const char* why = unfit(*x, duals())) bad(std::string("token_logprobs: an argument") + why);
  if (logits.dim() < 1) bad("token_logprobs: logits need a vocabulary dimension");
  const int64_t cols = logits.size(-1), vocab = columns.value_or(cols);
  if (!float_code(logits.scalar_type())) bad("token_logprobs: logits must be bfloat16, float16 or float32");
  if (tokens.scalar_type() != at::kLong && tokens.scalar_type() != at::kInt) bad("token_logprobs: tokens must be int64 or int32");
  if (tokens.sizes() != logits.sizes().slice(0, logits.dim() - 1))
    bad("token_logprobs: tokens of shape " + shape_of(tokens) + " do not match logits of shape " + shape_of(logits));
  if (vocab < 1 || vocab > cols) bad("token_logprobs: vocab must be between 1 and the logits' " + std::to_string(cols) + " columns");
  if (cols > wb::kLogprobMaxColumns || tokens.numel() >= std::numeric_limits<int32_t>::max())
    bad("token_logprobs: at most 2^30 columns and 2^31 - 2 rows");
  if (!(temperature >= 1e-30 && temperature <= 1e30)) bad("token_logprobs: the temperature must be between 1e-30 and 1e30");
  if (top_k < 0 || top_k > wb::kLogprobMaxTop || top_k > vocab)
    bad("token_logprobs: top_k must be between 0 and " + std::to_string(std::min<int64_t>(wb::kLogprobMaxTop, vocab)));
  if (top_k && vocab > wb::kLogprobMaxTopVocab)
    bad("token_logprobs: alternatives (top_k) of at most " + std::to_string(wb::kLogprobMaxTopVocab) + " columns");
  if (cols > 1 && logits.stride(-1) != 1) bad("token_logprobs: the logits' last dimension must be contiguous");
  if (!logits.is_cuda() || !tokens.is_cuda() || logits.device() != tokens.device())
    bad("token_logprobs: logits and tokens must be CUDA tensors of one device");
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    auto r = TokenLogprobs::apply(logits, tokens, vocab, temperature, top_k, ignore_index);
    return top_k ? py::make_tuple(r[0], r[1], r[2], r[3]) : py::make_tuple(r[0], r[1], py::none(), py::none());
  }
  LogprobResult r = run_logprobs(logits, tokens, {vocab, ignore_index, temperature, top_k}, false);
  return top_k ? py::make_tuple(r.logprobs, r.entropy, r.top_logprobs, r.top_ids)
               : py::make_tuple(r.logprobs, r.entropy, py::none(), py::none());
}

// -- sum of squares, norm -------------------------------------------------------------------------
// A tensor whose elements fill one stretch of memory without holes, in any order of dimensions.
bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense(); }

// Partial sums of squares of tensors that were checked; `dev`: where they are.
Tensor partial_sums(std::vector<wb::NormTensor>& t, const at::TensorOptions& f64, int sms) {
  Tensor partial = at::empty({(int64_t)std::max<uint64_t>(wb::partial_sums_size((uint32_t)t.size(), sms), 1)}, f64);
  uint32_t n = 0;
  check(wb::launch_partial_sums(t.data(), (uint32_t)t.size(), partial.mutable_data_ptr<double>(), &n, sms, c10::cuda::getCurrentCUDAStream()),
        "gradient norm launch");
  return partial.narrow(0, 0, n);
}

wb::NormTensor norm_tensor(const Tensor& x) {
  return {reinterpret_cast<uint64_t>(x.const_data_ptr()), (uint64_t)x.numel(), float_code(x.scalar_type()), 0};
}

// The norm of the tensors of a dict or a sequence (None entries left out), and the buffer whose
// first element is the sum of their squares.
py::tuple sum_squares(const py::object& tensors) {
  std::vector<wb::NormTensor> t;
  const Tensor* first = nullptr;
  const bool dual = duals();
  auto add = [&](PyObject* o) {
    if (o == Py_None) return;
    if (!THPVariable_Check(o)) throw py::type_error("grad_norm: not a tensor");
    const Tensor& x = THPVariable_Unpack(o);
    if (!first) first = &x;
    if (const char* why = unfit(x, dual)) bad(std::string("grad_norm: a tensor") + why);
    if (!x.is_cuda() || x.device() != first->device()) bad("grad_norm: all tensors must be CUDA tensors of one device");
    if (!float_code(x.scalar_type())) bad("grad_norm: tensors must be bfloat16, float16 or float32");
    if (!dense(x)) bad("grad_norm: a tensor of shape " + shape_of(x) + " has holes or overlaps in memory");
    if (x.numel()) t.push_back(norm_tensor(x));
  };
  if (PyDict_Check(tensors.ptr())) {
    PyObject *key = nullptr, *value = nullptr;
    Py_ssize_t pos = 0;
    t.reserve((size_t)PyDict_Size(tensors.ptr()));
    while (PyDict_Next(tensors.ptr(), &pos, &key, &value)) add(value);
  } else {
    for (const py::handle h : py::reinterpret_borrow<py::sequence>(tensors)) add(h.ptr());
  }
  if (!first) bad("grad_norm: no tensors");
  const c10::cuda::CUDAGuard guard(first->device());
  const auto f64 = first->options().dtype(at::kDouble).requires_grad(false);
  const int sms = sm_count(first->device().index());
  Tensor buffer = at::empty({1 + (int64_t)wb::partial_sums_size((uint32_t)t.size(), sms)}, f64), norm = at::empty({}, f64.dtype(at::kFloat));
  double* sum_sq = buffer.mutable_data_ptr<double>();
  uint32_t n = 0;
  const auto stream = c10::cuda::getCurrentCUDAStream();
  check(wb::launch_partial_sums(t.data(), (uint32_t)t.size(), sum_sq + 1, &n, sms, stream), "grad_norm launch");
  check(wb::launch_norm(sum_sq + 1, n, sum_sq, norm.mutable_data_ptr<float>(), stream), "grad_norm launch");
  return py::make_tuple(norm, buffer);
}

// -- AdamW ----------------------------------------------------------------------------------------
// The parameters and flat state buffers of one optimizer, its resident tables and its step.
struct AdamWProgram {
  std::vector<std::string> names;
  std::vector<Tensor> params;
  std::vector<uint64_t> ptrs, offsets;
  struct Shape { int64_t numel; at::ScalarType type; std::vector<int64_t> sizes, strides; };
  std::vector<Shape> shapes;       // as they were given: a parameter's `data` may be set to another tensor
  std::vector<float> decay;
  std::vector<uint32_t> chunk_start;
  Tensor tables, chunks, clock, m, v, m_scale, v_scale, master;
  std::vector<uint64_t> grads;
  std::vector<c10::cuda::CUDAStream> streams;      // that the allocator knows of
  int64_t total = 0;
  uint32_t chunk = wb::kAdamTile;
  double beta1, beta2, eps;
  bool fp8;
  at::Device dev{at::kCPU};
  int sms = 0;

  AdamWProgram(std::vector<std::string> names_, std::vector<Tensor> params_, std::vector<double> decay_, double b1, double b2, double eps_,
               bool fp8_, bool with_master)
      : names(std::move(names_)), params(std::move(params_)), beta1(b1), beta2(b2), eps(eps_), fp8(fp8_) {
    if (params.empty()) bad("AdamW: no parameters");
    dev = params[0].device();
    bool narrow = false;
    uint64_t n_chunks = 0;
    for (size_t i = 0; i < params.size(); ++i) {
      check_param(params[i], names[i]);
      narrow |= params[i].scalar_type() != at::kFloat;
      shapes.push_back({params[i].numel(), params[i].scalar_type(), params[i].sizes().vec(), params[i].strides().vec()});
      offsets.push_back((uint64_t)total);
      decay.push_back((float)decay_[i]);
      total += (params[i].numel() + wb::kStateBlock - 1) / wb::kStateBlock * wb::kStateBlock;
    }
    const c10::cuda::CUDAGuard guard(dev);
    sms = sm_count(dev.index());
    // A work item: one tile with fp32 states (a clipped step over 1.45M parameters: 14.5 us with one, 19.1 with
    // eight; over 436M 2417 and 2375, on another GPU the other way).  8-bit states overlap their loads within
    // an item: eight tiles, as long as every SM gets 32 items (604M parameters: 1620 us with one, 1280 with
    // eight; 24M at odd addresses: 95 with one, 112 with eight).
    chunk = fp8 ? 8 * wb::kAdamTile : wb::kAdamTile;
    while (chunk > wb::kAdamTile && total < (int64_t)sms * 32 * chunk) chunk /= 2;
    for (const Tensor& p : params) {
      chunk_start.push_back((uint32_t)n_chunks);
      n_chunks += ((uint64_t)p.numel() + chunk - 1) / chunk;
      if (n_chunks >= 0x7fffffffull) bad("AdamW: too many elements");
    }
    chunk_start.push_back((uint32_t)n_chunks);
    if (with_master && !narrow) bad("AdamW: master weights need 16-bit parameters");
    check_disjoint();
    const auto f32 = params[0].options().dtype(at::kFloat).requires_grad(false);
    if (fp8) {
      m = at::zeros({total}, f32.dtype(at::kFloat8_e4m3fn));
      v = at::zeros({total}, f32.dtype(at::kFloat8_e4m3fn));
      m_scale = at::ones({total / wb::kStateBlock}, f32);
      v_scale = at::ones({total / wb::kStateBlock}, f32);
    } else {
      m = at::zeros({total}, f32);
      v = at::zeros({total}, f32);
    }
    if (with_master) master = at::zeros({total}, f32);
    clock = at::zeros({(int64_t)sizeof(wb::AdamClock)}, f32.dtype(at::kByte));
    set_step(0);
    std::vector<wb::AdamChunk> ch;
    ch.reserve(n_chunks);
    for (uint32_t i = 0; i < params.size(); ++i)
      for (uint32_t c = 0; c < chunk_start[i + 1] - chunk_start[i]; ++c) ch.push_back({i, c});
    chunks = upload(ch.data(), ch.size() * sizeof(wb::AdamChunk));
    upload_tensors();
    if (with_master) read_master();
    settle();
  }

  // Tables and states are written on the current stream; steps may run on any other.
  void settle() const {
    const c10::cuda::CUDAGuard guard(dev);
    check(cudaStreamSynchronize(c10::cuda::getCurrentCUDAStream()), "AdamW set-up");
  }

  void check_param(const Tensor& p, const std::string& name) const {
    if (const char* why = unfit(p, duals())) bad("AdamW: " + name + why);
    if (!p.is_cuda() || p.device() != dev) bad("AdamW: " + name + " is not on the CUDA device of the first parameter");
    if (!float_code(p.scalar_type())) bad("AdamW: " + name + " must be bfloat16, float16 or float32");
    if (!dense(p)) bad("AdamW: " + name + " has holes or overlaps in memory; give the whole parameter, not a view of part of it");
  }

  void check_disjoint() const {
    std::vector<std::pair<uint64_t, size_t>> at_;
    for (size_t i = 0; i < params.size(); ++i)
      if (params[i].numel()) at_.push_back({reinterpret_cast<uint64_t>(params[i].const_data_ptr()), i});
    std::sort(at_.begin(), at_.end());
    for (size_t k = 1; k < at_.size(); ++k)
      if (at_[k - 1].first + params[at_[k - 1].second].nbytes() > at_[k].first)
        bad("AdamW: " + names[at_[k - 1].second] + " and " + names[at_[k].second] + " share memory: give a tied parameter once");
  }

  Tensor upload(const void* p, size_t bytes) const {
    const c10::cuda::CUDAGuard guard(dev);
    Tensor host = at::empty({(int64_t)std::max<size_t>(bytes, 16)}, at::TensorOptions().dtype(at::kByte));
    std::memcpy(host.mutable_data_ptr(), p, bytes);
    return host.to(dev);
  }

  // The parameters' rows, into one table for the optimizer's life: captured steps hold its address.
  void upload_tensors() {
    std::vector<wb::AdamTensor> t;
    ptrs.clear();
    for (size_t i = 0; i < params.size(); ++i) {
      ptrs.push_back(reinterpret_cast<uint64_t>(params[i].const_data_ptr()));
      t.push_back({ptrs[i], (uint64_t)params[i].numel(), offsets[i], float_code(params[i].scalar_type()), decay[i]});
    }
    const c10::cuda::CUDAGuard guard(dev);
    const size_t bytes = t.size() * sizeof(wb::AdamTensor);
    if (!tables.defined()) tables = at::empty({(int64_t)bytes}, f32_options().dtype(at::kByte));
    check(cudaMemcpyAsync(tables.mutable_data_ptr(), t.data(), bytes, cudaMemcpyHostToDevice, c10::cuda::getCurrentCUDAStream()),
          "AdamW set-up");
    settle();
  }

  // A tensor's slice of a flat state buffer, in the order of the parameter's memory.
  Tensor slice(const Tensor& flat, size_t i) const {
    return at::as_strided(flat, shapes[i].sizes, shapes[i].strides, (int64_t)offsets[i]);
  }

  // The master weights from the parameters' present values.
  void read_master() {
    if (!master.defined()) bad("AdamW.read_master: there are no master weights");
    const c10::cuda::CUDAGuard guard(dev);
    at::NoGradGuard no_grad;
    for (size_t i = 0; i < params.size(); ++i) slice(master, i).copy_(params[i].detach());
  }

  void set_step(int64_t step) {
    wb::AdamClock c{};
    c.step = step;
    c.b1t = std::pow(beta1, (double)step);
    c.b2t = std::pow(beta2, (double)step);
    Tensor host = at::empty({(int64_t)sizeof(c)}, at::TensorOptions().dtype(at::kByte));
    std::memcpy(host.mutable_data_ptr(), &c, sizeof(c));
    clock.copy_(host);
    settle();
  }

  int64_t get_step() const {
    wb::AdamClock c;
    Tensor host = clock.cpu();
    std::memcpy(&c, host.const_data_ptr(), sizeof(c));
    return c.step;
  }

  // Parameters at new addresses (their memory was released and allocated again).
  void rebind(const std::vector<Tensor>& p) {
    if (p.size() != params.size()) bad("AdamW.rebind: another number of parameters");
    for (size_t i = 0; i < p.size(); ++i) {
      check_param(p[i], names[i]);
      if (p[i].sizes() != at::IntArrayRef(shapes[i].sizes) || p[i].strides() != at::IntArrayRef(shapes[i].strides) || p[i].scalar_type() != shapes[i].type)
        bad("AdamW.rebind: " + names[i] + " has another shape, stride or type");
    }
    auto before = params;
    params = p;
    try {
      check_disjoint();
    } catch (...) {
      params = before;
      throw;
    }
    const c10::cuda::CUDAGuard guard(dev);
    check(cudaDeviceSynchronize(), "AdamW.rebind");       // steps in flight on any stream read the old table
    upload_tensors();
  }

  // Collects the gradients of this step, and what the norm reads of them.
  void collect(const py::object& src, std::vector<wb::NormTensor>* normed) {
    grads.assign(params.size(), 0);
    Py_ssize_t found = 0;
    const bool dict = !src.is_none(), dual = duals();
    if (dict && !PyDict_Check(src.ptr())) throw py::type_error("AdamW.step: gradients are a dict of name -> tensor, or None for the parameters' .grad");
    for (size_t i = 0; i < params.size(); ++i) {
      const Tensor& p = params[i];
      if (reinterpret_cast<uint64_t>(p.const_data_ptr()) != ptrs[i])
        throw std::runtime_error("AdamW.step: " + names[i] + " moved in memory; call rebind()");
      if (p.numel() != shapes[i].numel || p.scalar_type() != shapes[i].type || !dense(p))
        throw std::runtime_error("AdamW.step: " + names[i] + " has another size or type than at the constructor; call rebind() with what it was");
      const Tensor* g = nullptr;
      if (dict) {
        PyObject* o = PyDict_GetItemWithError(src.ptr(), py_names[i].ptr());
        if (!o && PyErr_Occurred()) throw py::error_already_set();
        if (o) {
          ++found;
          if (o != Py_None) {
            if (!THPVariable_Check(o)) throw py::type_error("AdamW.step: the gradient of " + names[i] + " is not a tensor");
            g = &THPVariable_Unpack(o);
          }
        }
      } else {
        g = &p.grad();
      }
      if (!g || !g->defined()) continue;
      if (const char* why = unfit(*g, dual)) bad("AdamW.step: the gradient of " + names[i] + why);
      if (!g->is_cuda() || g->device() != dev) bad("AdamW.step: the gradient of " + names[i] + " is on another device");
      if (g->sizes() != p.sizes()) bad("AdamW.step: the gradient of " + names[i] + " has shape " + shape_of(*g) + ", not " + shape_of(p));
      if (g->scalar_type() != p.scalar_type() && g->scalar_type() != at::kFloat)
        bad("AdamW.step: the gradient of " + names[i] + " must have the parameter's type or float32");
      if (g->strides() != p.strides() && !same_order(*g, p))
        bad("AdamW.step: the gradient of " + names[i] + " has another memory layout than the parameter");
      if (!g->numel()) continue;
      grads[i] = reinterpret_cast<uint64_t>(g->const_data_ptr()) | (g->scalar_type() != p.scalar_type() ? 1u : 0u);
      if (normed) normed->push_back(norm_tensor(*g));
    }
    if (dict && found != PyDict_Size(src.ptr())) bad("AdamW.step: the gradients name a tensor that is not one of the parameters");
  }

  // Strides may differ in dimensions of size 1.
  static bool same_order(const Tensor& g, const Tensor& p) {
    for (int64_t d = 0; d < p.dim(); ++d)
      if (p.size(d) != 1 && g.stride(d) != p.stride(d)) return false;
    return true;
  }

  std::vector<py::str> py_names;

  // The sum of squares of this step's gradients, before a reduction over ranks.
  Tensor grad_sum_sq(const py::object& src) {
    std::vector<wb::NormTensor> t;
    collect(src, &t);
    const c10::cuda::CUDAGuard guard(dev);
    const auto f64 = f32_options().dtype(at::kDouble);
    const Tensor partial = partial_sums(t, f64, sms);
    Tensor sum_sq = at::empty({}, f64), norm = at::empty({}, f32_options());
    check(wb::launch_norm(partial.const_data_ptr<double>(), (uint32_t)partial.numel(), sum_sq.mutable_data_ptr<double>(),
                          norm.mutable_data_ptr<float>(), c10::cuda::getCurrentCUDAStream()),
          "gradient norm launch");
    return sum_sq;
  }

  // max_norm > 0: clip, by the given sum of squares or by these gradients' own.
  py::object step(const py::object& src, double lr, const std::optional<Tensor>& lr_dev, const std::optional<Tensor>& sum_sq, double max_norm) {
    const bool clip = max_norm > 0;
    std::vector<wb::NormTensor> t;
    if (clip && !sum_sq) t.reserve(params.size());
    collect(src, clip && !sum_sq ? &t : nullptr);
    const c10::cuda::CUDAGuard guard(dev);
    wb::AdamArgs a{};
    if (lr_dev) {
      if (const char* why = unfit(*lr_dev, duals())) bad(std::string("AdamW.step: lr") + why);
      if (lr_dev->numel() != 1 || lr_dev->device() != dev || (lr_dev->scalar_type() != at::kFloat && lr_dev->scalar_type() != at::kDouble))
        bad("AdamW.step: lr is a number, or a float32 or float64 tensor of one element on the parameters' device");
      a.lr_ptr = lr_dev->const_data_ptr();
      a.lr_f64 = lr_dev->scalar_type() == at::kDouble;
    }
    Tensor norm, partial;
    if (clip) {
      if (sum_sq) partial = *sum_sq;
      else partial = partial_sums(t, f32_options().dtype(at::kDouble), sms);
      norm = at::empty({}, f32_options());
      a.partial = partial.const_data_ptr<double>();
      a.n_partial = (uint32_t)partial.numel();
      a.norm = norm.mutable_data_ptr<float>();
    }
    a.tensors = reinterpret_cast<const wb::AdamTensor*>(tables.const_data_ptr());
    a.chunks = reinterpret_cast<const wb::AdamChunk*>(chunks.const_data_ptr());
    a.n_tensors = (uint32_t)params.size();
    a.chunk = chunk;
    a.master = master.defined() ? master.mutable_data_ptr<float>() : nullptr;
    a.m = m.mutable_data_ptr();
    a.v = v.mutable_data_ptr();
    a.m_scale = fp8 ? m_scale.mutable_data_ptr<float>() : nullptr;
    a.v_scale = fp8 ? v_scale.mutable_data_ptr<float>() : nullptr;
    a.clock = reinterpret_cast<wb::AdamClock*>(clock.mutable_data_ptr());
    a.beta1 = beta1;
    a.beta2 = beta2;
    a.lr = lr;
    a.eps = eps;
    a.max_norm = max_norm;
    const auto stream = c10::cuda::getCurrentCUDAStream();
    used_on(stream);
    check(wb::launch_adamw(a, grads.data(), chunk_start.data(), sms, stream), "AdamW launch");
    for (size_t i = 0; i < params.size(); ++i)          // autograd sees the change of those that took part
      if (grads[i] && !params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
    return norm.defined() ? py::cast(norm) : py::none();
  }

  // Steps may run on any stream.  The allocator is told of each stream once, so that an optimizer released
  // behind its last step leaves its memory to others only when that step has run.
  void used_on(const c10::cuda::CUDAStream& stream) {
    if (std::find(streams.begin(), streams.end(), stream) != streams.end()) return;
    for (const Tensor& t : {tables, chunks, clock, m, v, m_scale, v_scale, master})
      if (t.defined()) t.record_stream(stream.unwrap());
    streams.push_back(stream);
  }

  at::TensorOptions f32_options() const { return params[0].options().dtype(at::kFloat).requires_grad(false); }
};

}  // namespace

namespace wb {

void bind_learn(py::module_& m) {
  m.def("token_logprobs", &token_logprobs, "log probabilities of tokens, entropy and alternatives");
  m.def("sum_squares", &sum_squares, "sum of squares of many tensors and its root (device scalars)");
  py::class_<AdamWProgram>(m, "AdamWProgram")
      .def(py::init([](std::vector<std::string> names, std::vector<Tensor> params, std::vector<double> decay, double b1, double b2,
                       double eps, bool fp8, bool master) {
        if (names.size() != params.size() || names.size() != decay.size()) bad("AdamW: names, parameters and decays must match");
        auto p = std::make_unique<AdamWProgram>(std::move(names), std::move(params), std::move(decay), b1, b2, eps, fp8, master);
        for (const auto& n : p->names) p->py_names.emplace_back(n);
        return p;
      }))
      .def("step", &AdamWProgram::step)
      .def("grad_sum_sq", &AdamWProgram::grad_sum_sq)
      .def("rebind", &AdamWProgram::rebind)
      .def("read_master", [](AdamWProgram& p) {
        const c10::cuda::CUDAGuard guard(p.dev);
        check(cudaDeviceSynchronize(), "AdamW.read_master");     // steps in flight on any stream
        p.read_master();
        p.settle();
      })
      .def("slice", [](const AdamWProgram& p, const Tensor& flat, size_t i) { return p.slice(flat, i); })
      .def_property("step_count", &AdamWProgram::get_step, &AdamWProgram::set_step)
      .def_readonly("total", &AdamWProgram::total)
      .def_readonly("exp_avg", &AdamWProgram::m)
      .def_readonly("second", &AdamWProgram::v)
      .def_readonly("exp_avg_scale", &AdamWProgram::m_scale)
      .def_readonly("second_scale", &AdamWProgram::v_scale)
      .def_readonly("master", &AdamWProgram::master);
}

}  // namespace wb
