// step_bind.cpp -- the training-step operators (include/suika_step.h) on
// torch tensors, part of the host extension: argument checks, outputs and
// workspaces from torch's caching allocator, and the library's calls on the
// device's current stream.

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/DynamicTypes.h>

#include <cstdint>
#include <exception>
#include <string>
#include <unordered_map>
#include <vector>

#include "host_errors.h"
#include "suika_step.h"

namespace py = pybind11;

namespace {

using suika_host::check;
using suika_host::plan_error;

std::string indexed(const char* what, size_t i) { return std::string(what) + "[" + std::to_string(i) + "]"; }

int32_t float_code(const at::Tensor& t, const std::string& what) {
  switch (t.scalar_type()) {
    case at::kFloat: return SR_DT_F32;
    case at::kBFloat16: return SR_DT_BF16;
    case at::kHalf: return SR_DT_F16;
    default: plan_error(what + ": dtype " + c10::toString(t.scalar_type()) + ", not float32, bfloat16 or float16");
  }
}

hipStream_t stream_of(const at::Device& device) {
  static PyObject* current = [] {
    py::object f = py::module_::import("torch._C").attr("_cuda_getCurrentRawStream");
    return f.release().ptr();
  }();
  py::object s = py::reinterpret_steal<py::object>(PyObject_CallFunction(current, "i", int(device.index())));
  if (!s) throw py::error_already_set();
  return reinterpret_cast<hipStream_t>(PyLong_AsUnsignedLongLong(s.ptr()));
}

// What the call writes through raw pointers counts as written for autograd.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const at::Tensor& tensor_of(PyObject* o, const std::string& what) {
  if (!THPVariable_Check(o)) plan_error(what + ": not a tensor");
  return THPVariable_Unpack(o);
}

// Whether a tensor's storage holds its elements: it does not once it was
// released (forcefully_free_tensor), and then a view's address is its offset
// alone.
bool stored(const at::Tensor& t) {
  const int64_t n = t.numel();
  if (n == 0) return true;
  if (!t.has_storage()) return false;
  uint64_t end = uint64_t(t.storage_offset()) + 1;
  if (t.is_contiguous()) end += uint64_t(n) - 1;
  else
    for (int64_t d = 0; d < t.dim(); ++d) end += uint64_t((t.size(d) - 1) * t.stride(d));
  return end * t.dtype().itemsize() <= t.storage().nbytes();
}

void check_stored(const at::Tensor& t, const char* what) {
  if (!stored(t)) plan_error(std::string(what) + ": its storage has been released");
}

// These operators have no forward-mode derivatives: a tangent would be lost.
void check_tangent(const at::Tensor& t, const char* what) {
  if (t._fw_grad(0).defined()) plan_error(std::string(what) + ": forward-mode derivatives are not supported");
}

// Whether a tensor is what check_dense wants, but for its storage.
bool dense(const at::Tensor& t, const c10::optional<at::Device>& device) {
  return t.layout() == at::kStrided && t.is_cuda() && device && t.device() == *device && t.is_contiguous();
}

// A dense tensor on the GPU; `device` is set by the first one.
void check_dense(const at::Tensor& t, const std::string& what, c10::optional<at::Device>& device) {
  if (t.layout() != at::kStrided || !t.is_cuda()) plan_error(what + " is on " + t.device().str() + ", not a dense tensor on the GPU");
  if (!device) device = t.device();
  if (t.device() != *device) plan_error(what + " is on " + t.device().str() + ", not on " + device->str());
  if (!t.is_contiguous()) plan_error(what + " is not contiguous");
  if (!stored(t)) plan_error(what + ": its storage has been released");
}

// The tensors of a list; None stands for a tensor that is not there.
class Fast {
 public:
  Fast(py::handle list, const char* what) {
    seq_ = py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), "a sequence of tensors is wanted"));
    if (!seq_) {
      PyErr_Clear();
      plan_error(std::string(what) + ": a sequence of tensors is wanted");
    }
  }
  size_t size() const { return size_t(PySequence_Fast_GET_SIZE(seq_.ptr())); }
  PyObject* operator[](size_t i) const { return PySequence_Fast_GET_ITEM(seq_.ptr(), Py_ssize_t(i)); }

 private:
  py::object seq_;
};

sr_array array_of(const at::Tensor& t, const std::string& what) {
  return {t.data_ptr(), uint64_t(t.numel()), float_code(t, what), 0};
}

at::Device current_device() {
  const c10::impl::VirtualGuardImpl impl(at::kCUDA);
  if (impl.deviceCount() == 0) plan_error("no GPU");
  return impl.getDevice();
}

at::TensorOptions on(const at::Device& device, at::ScalarType type) {
  return at::TensorOptions().device(device).dtype(type);
}

// The memory that a sum of squares takes: the sum, and the parts of it.
struct SumWork {
  at::Tensor memory;
  uint64_t bytes = 0;      // of the parts

  SumWork(const std::vector<sr_array>& a, const at::Device& device) {
    check(sr_square_sum_workspace(a.data(), int32_t(a.size()), &bytes), "sr_square_sum");
    memory = at::empty({int64_t(bytes) + 16}, on(device, at::kByte));
  }
  double* sum() const { return static_cast<double*>(memory.data_ptr()); }
  void* parts() const { return static_cast<char*>(memory.data_ptr()) + 16; }
};

// Launches the sum of squares into `into`, or into memory of its own.
void square_sum_into(const std::vector<sr_array>& a, const at::Device& device, double* into, float* norm) {
  const SumWork work(a, device);
  check(sr_square_sum(a.data(), int32_t(a.size()), 0, work.parts(), work.bytes, into ? into : work.sum(), norm,
                      stream_of(device)),
        "sr_square_sum");
}

// The norm that gradients are clipped by: of a given sum, or of `grads`, with
// the memory for it.
sr_norm norm_of(const double* given, const std::vector<sr_array>& grads, const at::Device& device, float* norm,
                c10::optional<SumWork>& work) {
  if (given) return {given, nullptr, nullptr, 0, norm};
  work.emplace(grads, device);
  return {nullptr, work->sum(), work->parts(), work->bytes, norm};
}

std::vector<sr_array> arrays_of(const Fast& list, const char* what, c10::optional<at::Device>& device) {
  std::vector<sr_array> a;
  a.reserve(list.size());
  for (size_t i = 0; i < list.size(); ++i) {
    if (list[i] == Py_None) continue;
    const std::string name = indexed(what, i);
    const at::Tensor& t = tensor_of(list[i], name);
    check_dense(t, name, device);
    check_tangent(t, what);
    a.push_back(array_of(t, name));
  }
  return a;
}

at::Tensor grad_square_sum(py::object grads) {
  c10::optional<at::Device> device;
  const Fast list(grads, "grads");
  const std::vector<sr_array> a = arrays_of(list, "grads", device);
  if (!device) device = current_device();
  const c10::DeviceGuard guard(*device);
  at::Tensor out = at::empty({}, on(*device, at::kDouble));
  square_sum_into(a, *device, out.data_ptr<double>(), nullptr);
  return out;
}

at::Tensor grad_norm(py::object grads) {
  c10::optional<at::Device> device;
  const Fast list(grads, "grads");
  const std::vector<sr_array> a = arrays_of(list, "grads", device);
  if (!device) device = current_device();
  const c10::DeviceGuard guard(*device);
  at::Tensor norm = at::empty({}, on(*device, at::kFloat));
  square_sum_into(a, *device, nullptr, norm.data_ptr<float>());
  return norm;
}

// A caller's sum of squares (one float64 on the device); null where it is None.
const double* given_sum(py::handle square_sum, const at::Device& device) {
  if (square_sum.is_none()) return nullptr;
  const at::Tensor& t = tensor_of(square_sum.ptr(), "square_sum");
  if (t.scalar_type() != at::kDouble || t.numel() != 1 || t.device() != device)
    plan_error("square_sum: one float64 on " + device.str() + " is wanted");
  check_stored(t, "square_sum");
  return t.data_ptr<double>();
}

at::Tensor clip_grads(py::object grads, double max_norm, py::object outs, py::object square_sum) {
  c10::optional<at::Device> device;
  const Fast list(grads, "grads");
  std::vector<sr_array> src, dst;
  std::vector<at::Tensor> to;
  const bool in_place = outs.is_none();
  const Fast out_list(in_place ? py::object(py::list()) : outs, "out");
  if (!in_place && out_list.size() != list.size())
    plan_error("out has " + std::to_string(out_list.size()) + " tensors, grads " + std::to_string(list.size()));
  for (size_t i = 0; i < list.size(); ++i) {
    if (list[i] == Py_None) continue;
    const std::string name = indexed("grads", i);
    const at::Tensor& t = tensor_of(list[i], name);
    check_dense(t, name, device);
    check_tangent(t, "grads");
    src.push_back(array_of(t, name));
    if (in_place) {
      to.push_back(t);
      continue;
    }
    const std::string out_name = indexed("out", i);
    const at::Tensor& o = tensor_of(out_list[i], out_name);
    check_dense(o, out_name, device);
    if (o.sizes() != t.sizes()) plan_error(out_name + ": shape differs from the gradient's");
    dst.push_back(array_of(o, out_name));
    to.push_back(o);
  }
  if (!device) device = current_device();
  const c10::DeviceGuard guard(*device);
  const double* sum = given_sum(square_sum, *device);
  at::Tensor norm = at::empty({}, on(*device, at::kFloat));
  c10::optional<SumWork> work;
  const sr_norm by = norm_of(sum, src, *device, norm.data_ptr<float>(), work);
  check(sr_clip_norm(src.data(), in_place ? nullptr : dst.data(), int32_t(src.size()), float(max_norm), &by,
                     stream_of(*device)),
        "sr_clip_norm");
  for (const at::Tensor& t : to) written(t);
  return norm;
}

// The state that an optimizer steps: the tensors, in the order of its names.
class AdamWState {
 public:
  // `steps`: how many updates each parameter has had.
  AdamWState(py::object weight, py::object exp_avg, py::object exp_avg_sq, py::object param, std::vector<std::string> names,
             std::vector<int64_t> steps)
      : names_(std::move(names)) {
    const Fast w(weight, "weight"), m(exp_avg, "exp_avg"), v(exp_avg_sq, "exp_avg_sq"), p(param, "param");
    if (w.size() != names_.size() || m.size() != w.size() || v.size() != w.size() || p.size() != w.size())
      plan_error("state: lists of different lengths");
    for (size_t i = 0; i < names_.size(); ++i) {
      weight_.push_back(tensor_of(w[i], names_[i] + "/weight"));
      exp_avg_.push_back(tensor_of(m[i], names_[i] + "/exp_avg"));
      exp_avg_sq_.push_back(tensor_of(v[i], names_[i] + "/exp_avg_sq"));
      param_.push_back(p[i] == Py_None ? at::Tensor() : tensor_of(p[i], names_[i] + "/param"));
      check_fields(i);
    }
    // names of one tensor count its updates together
    std::unordered_map<const void*, size_t> first;
    for (size_t i = 0; i < names_.size(); ++i)
      counted_.push_back(first.emplace(weight_[i].unsafeGetTensorImpl(), i).first->second);
    set_steps(std::move(steps));
  }

  std::vector<int64_t> steps() const {
    std::vector<int64_t> all;
    for (size_t i : counted_) all.push_back(steps_[i]);
    return all;
  }
  void set_steps(std::vector<int64_t> steps) {
    if (steps.size() != names_.size()) plan_error("steps: one of each parameter is wanted");
    steps_ = std::move(steps);
  }

  // One update; the gradients' norm, or None without clipping.
  py::object step(py::object grads, double lr, double beta1, double beta2, double eps,
                  double weight_decay, py::object max_norm, py::object square_sum) {
    const Fast list(grads, "grads");
    if (list.size() != names_.size())
      plan_error("grads: " + std::to_string(list.size()) + " tensors for a state of " + std::to_string(names_.size()));
    std::vector<sr_adamw_tensor> tensors;
    std::vector<sr_array> arrays;
    std::vector<int64_t> numbers;
    tensors.reserve(names_.size());
    numbers.reserve(names_.size());
    for (size_t i = 0; i < names_.size(); ++i) {
      if (list[i] == Py_None) continue;
      if (!THPVariable_Check(list[i])) plan_error("gradient of " + names_[i] + ": not a tensor");
      const at::Tensor& g = THPVariable_Unpack(list[i]);
      const at::Tensor &w = weight_[i], &m = exp_avg_[i], &v = exp_avg_sq_[i], &p = param_[i];
      check_fields(i);
      if (g.layout() != at::kStrided || !g.is_contiguous() || g.device() != w.device() || g.sizes() != w.sizes())
        plan_error("gradient of " + names_[i] + ": a dense tensor like the weight on " + w.device().str() + " is wanted");
      const at::ScalarType gt = g.scalar_type();
      if (gt != at::kFloat && gt != at::kBFloat16)
        plan_error("gradient of " + names_[i] + ": dtype " + c10::toString(gt) + ", not float32 or bfloat16");
      if (!stored(g)) plan_error("gradient of " + names_[i] + ": its storage has been released");
      const int32_t gc = gt == at::kFloat ? SR_DT_F32 : SR_DT_BF16;
      tensors.push_back({w.data_ptr(), m.data_ptr(), v.data_ptr(), p.defined() ? p.data_ptr() : nullptr, g.data_ptr(),
                         uint64_t(w.numel()), w.scalar_type() == at::kFloat ? SR_DT_F32 : SR_DT_BF16,
                         m.scalar_type() == at::kFloat ? SR_DT_F32 : SR_DT_BF16, gc, 0});
      numbers.push_back(steps_[counted_[i]] + 1);
      if (!max_norm.is_none() && square_sum.is_none()) arrays.push_back({g.data_ptr(), uint64_t(g.numel()), gc, 0});
    }
    const at::Device device = device_ ? *device_ : current_device();
    const c10::DeviceGuard guard(device);
    sr_adamw_options o{lr, beta1, beta2, eps, weight_decay, 1, 0.0};     // the tensors have their own numbers
    c10::optional<SumWork> work;
    sr_norm by{};
    at::Tensor norm;
    if (!max_norm.is_none()) {
      o.max_norm = max_norm.cast<double>();
      const double* sum = given_sum(square_sum, device);
      norm = at::empty({}, on(device, at::kFloat));
      by = norm_of(sum, arrays, device, norm.data_ptr<float>(), work);
    } else if (!square_sum.is_none()) {
      plan_error("square_sum is given without max_norm");
    }
    check(sr_adamw_norm(tensors.data(), numbers.data(), int32_t(tensors.size()), &o,
                        max_norm.is_none() ? nullptr : &by, stream_of(device)),
          "sr_adamw_norm");
    for (size_t i = 0; i < names_.size(); ++i) {
      if (list[i] == Py_None) continue;
      ++steps_[counted_[i]];
      for (const at::Tensor* t : {&weight_[i], &exp_avg_[i], &exp_avg_sq_[i], &param_[i]})
        if (t->defined()) written(*t);
    }
    if (!norm.defined()) return py::none();
    return py::cast(norm);
  }

 private:
  // The fields of parameter i as they are now: a tensor's memory, shape and type
  // can be replaced (`.data`, set_) or its storage released since the state was
  // taken, and the kernels go by the weight's size.
  void check_fields(size_t i) {
    const at::Tensor &w = weight_[i], &m = exp_avg_[i], &v = exp_avg_sq_[i], &p = param_[i];
    const struct { const at::Tensor& t; const char* what; } field[4] = {
        {w, "weight"}, {m, "exp_avg"}, {v, "exp_avg_sq"}, {p, "param"}};
    for (const auto& f : field) {
      if (!f.t.defined()) continue;
      if (!dense(f.t, device_)) check_dense(f.t, names_[i] + "/" + f.what, device_);     // says what is wrong
      if (!stored(f.t)) plan_error(names_[i] + ": a field's storage has been released");
      if (f.t.sizes() != w.sizes()) plan_error(names_[i] + ": fields of different shapes");
    }
    const at::ScalarType wt = w.scalar_type(), mt = m.scalar_type();
    if (wt != at::kFloat && wt != at::kBFloat16)
      plan_error(names_[i] + ": weight of dtype " + c10::toString(wt) + ", not float32 or bfloat16");
    if ((mt != at::kFloat && mt != at::kBFloat16) || v.scalar_type() != mt)
      plan_error(names_[i] + ": moments are both float32 or both bfloat16");
    if (p.defined() && (wt != at::kFloat || p.scalar_type() != at::kBFloat16))
      plan_error(names_[i] + ": a master weight is float32 and its param bfloat16");
  }

  std::vector<std::string> names_;
  std::vector<at::Tensor> weight_, exp_avg_, exp_avg_sq_, param_;
  std::vector<size_t> counted_;     // the first parameter that has this one's weight
  std::vector<int64_t> steps_;      // updates so far, of counted_[i]
  c10::optional<at::Device> device_;
};

// ------------------------------------------------------------- vocabulary shard

int32_t index_code(const at::Tensor& t, const char* what) {
  if (t.scalar_type() == at::kLong) return SR_DT_I64;
  if (t.scalar_type() == at::kInt) return SR_DT_I32;
  plan_error(std::string(what) + ": dtype " + c10::toString(t.scalar_type()) + ", not int64 or int32");
}

// A tensor of rows of dense elements, all of one distance from the next: that
// distance, in elements.
uint64_t row_stride(const at::Tensor& t, const std::string& what) {
  if (t.layout() != at::kStrided || t.dim() < 1) plan_error(what + ": a dense tensor of rows is wanted");
  if (!stored(t)) plan_error(what + ": its storage has been released");
  const int64_t cols = t.size(-1);
  if (t.is_contiguous()) return uint64_t(cols);
  int64_t distance = cols, next = -1;     // from row to row; what an outer dimension's stride has to be
  bool ok = t.stride(-1) == 1 || cols <= 1;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) <= 1) continue;
    if (next < 0) distance = t.stride(d);
    else if (t.stride(d) != next) ok = false;
    next = t.stride(d) * t.size(d);
  }
  if (!ok || distance < cols)
    plan_error(what + ": rows of dense elements, one distance apart, are wanted, not strides of " +
               c10::str(t.strides()));
  return uint64_t(distance);
}

void check_device(const at::Tensor& t, const char* what, const at::Device& device) {
  if (t.device() != device) plan_error(std::string(what) + " is on " + t.device().str() + ", not on " + device.str());
}

sr_embedding_shape embedding_shape(const at::Tensor& tokens, int32_t dtype, int64_t rows, int64_t cols, double scale,
                                   int64_t vocab_start) {
  if (!tokens.is_cuda() || !tokens.is_contiguous()) plan_error("tokens: a contiguous tensor on the GPU is wanted");
  check_stored(tokens, "tokens");
  return {tokens.data_ptr(), index_code(tokens, "tokens"), dtype,         uint64_t(tokens.numel()), uint64_t(rows),
          uint64_t(cols),    vocab_start,                  float(scale), 0};
}

at::Tensor vocab_embedding(const at::Tensor& tokens, const at::Tensor& weight, double scale, int64_t vocab_start,
                           const c10::optional<at::Tensor>& out) {
  if (weight.dim() != 2) plan_error("weight: rows x columns are wanted");
  const int64_t rows = weight.size(0), cols = weight.size(1);
  const sr_embedding_shape s =
      embedding_shape(tokens, float_code(weight, "weight"), rows, cols, scale, vocab_start);
  check_device(weight, "weight", tokens.device());
  check_tangent(weight, "weight");
  const uint64_t stride = row_stride(weight, "weight");
  const c10::DeviceGuard guard(tokens.device());
  std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
  shape.push_back(cols);
  if (out) {
    check_device(*out, "out", tokens.device());
    if (out->sizes() != at::IntArrayRef(shape) || !out->is_contiguous() || out->scalar_type() != weight.scalar_type())
      plan_error("out: a contiguous tensor of the tokens' shape and the weight's columns and dtype is wanted");
    check_stored(*out, "out");
  }
  at::Tensor to = out ? *out : at::empty(shape, on(tokens.device(), weight.scalar_type()));
  check(sr_embedding(&s, weight.data_ptr(), stride, to.data_ptr(), stream_of(tokens.device())), "sr_embedding");
  if (out) written(to);
  return to;
}

at::Tensor vocab_embedding_grad(const at::Tensor& tokens, const at::Tensor& grad_output, int64_t rows, double scale,
                                int64_t vocab_start, py::object dtype, const c10::optional<at::Tensor>& out,
                                bool accumulate) {
  if (grad_output.dim() != tokens.dim() + 1 || grad_output.sizes().slice(0, tokens.dim()) != tokens.sizes())
    plan_error("grad_output: a tensor of the tokens' shape and the columns is wanted");
  if (rows < 0) plan_error("rows: " + std::to_string(rows));
  const int64_t cols = grad_output.size(-1);
  const sr_embedding_shape s =
      embedding_shape(tokens, float_code(grad_output, "grad_output"), rows, cols, scale, vocab_start);
  check_device(grad_output, "grad_output", tokens.device());
  check_tangent(grad_output, "grad_output");
  const uint64_t stride = row_stride(grad_output, "grad_output");
  const c10::DeviceGuard guard(tokens.device());
  at::Tensor to;
  if (out) {
    to = *out;
    check_device(to, "out", tokens.device());
    if (to.dim() != 2 || to.size(0) != rows || to.size(1) != cols || !to.is_contiguous())
      plan_error("out: a contiguous tensor of rows x columns is wanted");
    check_stored(to, "out");
    if (!dtype.is_none() && torch::python::detail::py_object_to_dtype(dtype) != to.scalar_type())
      plan_error("out is of another dtype than the one asked for");
  } else {
    if (accumulate) plan_error("accumulate goes with out");
    const at::ScalarType type =
        dtype.is_none() ? grad_output.scalar_type() : torch::python::detail::py_object_to_dtype(dtype);
    to = at::empty({rows, cols}, on(tokens.device(), type));
  }
  const int32_t code = float_code(to, "the gradient");
  uint64_t need = 0;
  check(sr_embedding_grad_workspace(&s, &need), "sr_embedding_grad");
  const at::Tensor work = at::empty({int64_t(need)}, on(tokens.device(), at::kByte));
  check(sr_embedding_grad(&s, grad_output.data_ptr(), stride, to.data_ptr(), code, accumulate, work.data_ptr(), need,
                          stream_of(tokens.device())),
        "sr_embedding_grad");
  if (out) written(to);
  return to;
}

sr_logprob_shape logprob_shape(const at::Tensor& logits, const at::Tensor& targets, const c10::optional<int64_t>& vocab) {
  if (logits.dim() != targets.dim() + 1 || logits.sizes().slice(0, targets.dim()) != targets.sizes())
    plan_error("logits: a tensor of the targets' shape and the columns is wanted");
  if (!logits.is_cuda() || !targets.is_contiguous()) plan_error("logits on the GPU and contiguous targets are wanted");
  check_device(targets, "targets", logits.device());
  check_stored(targets, "targets");
  check_tangent(logits, "logits");
  const int64_t columns = logits.size(-1), v = vocab ? *vocab : columns;
  if (v < 1 || v > columns)
    plan_error("a vocabulary of " + std::to_string(v) + " in " + std::to_string(columns) + " columns");
  return {logits.data_ptr(), targets.data_ptr(), index_code(targets, "targets"), float_code(logits, "logits"),
          uint64_t(targets.numel()), uint64_t(columns), uint64_t(v), row_stride(logits, "logits")};
}

py::tuple token_logprobs(const at::Tensor& logits, const at::Tensor& targets, int64_t top,
                         const c10::optional<int64_t>& vocab) {
  const sr_logprob_shape s = logprob_shape(logits, targets, vocab);
  if (top < 0 || top > SR_LOGPROB_MAX_TOP || uint64_t(top) > s.vocab)
    plan_error("top " + std::to_string(top) + " of a vocabulary of " + std::to_string(s.vocab) + " (at most " +
               std::to_string(SR_LOGPROB_MAX_TOP) + ")");
  const at::Device device = logits.device();
  const c10::DeviceGuard guard(device);
  const at::TensorOptions f32 = on(device, at::kFloat);
  at::Tensor logprob = at::empty(targets.sizes(), f32), entropy = at::empty(targets.sizes(), f32),
             lse = at::empty(targets.sizes(), f32), lse_low = at::empty(targets.sizes(), f32), best, index, work;
  if (top) {
    std::vector<int64_t> shape(targets.sizes().begin(), targets.sizes().end());
    shape.push_back(top);
    best = at::empty(shape, f32);
    index = at::empty(shape, on(device, at::kLong));
  }
  uint64_t need = 0;
  check(sr_logprob_workspace(&s, int32_t(top), &need), "sr_logprob");
  if (need) work = at::empty({int64_t(need)}, on(device, at::kByte));
  check(sr_logprob_pair(&s, int32_t(top), logprob.data_ptr<float>(), entropy.data_ptr<float>(), lse.data_ptr<float>(),
                        lse_low.data_ptr<float>(), top ? best.data_ptr<float>() : nullptr,
                        top ? index.data_ptr<int64_t>() : nullptr, need ? work.data_ptr() : nullptr, need,
                        stream_of(device)),
        "sr_logprob_pair");
  if (!top) return py::make_tuple(logprob, entropy, lse, py::none(), py::none(), lse_low);
  return py::make_tuple(logprob, entropy, lse, best, index, lse_low);
}

const float* row_values(const at::Tensor& t, const char* what, const at::Tensor& targets) {
  check_device(t, what, targets.device());
  if (t.scalar_type() != at::kFloat || t.sizes() != targets.sizes() || !t.is_contiguous())
    plan_error(std::string(what) + ": a contiguous float32 tensor of the targets' shape is wanted");
  check_stored(t, what);
  check_tangent(t, what);
  return t.data_ptr<float>();
}

at::Tensor token_logprobs_grad(const at::Tensor& logits, const at::Tensor& targets, const at::Tensor& lse,
                               const at::Tensor& entropy, const c10::optional<at::Tensor>& grad_logprob,
                               const c10::optional<at::Tensor>& grad_entropy, const c10::optional<int64_t>& vocab,
                               const c10::optional<at::Tensor>& out, const c10::optional<at::Tensor>& lse_low) {
  const sr_logprob_shape s = logprob_shape(logits, targets, vocab);
  const float* l = row_values(lse, "lse", targets);
  const float* low = lse_low ? row_values(*lse_low, "lse_low", targets) : nullptr;
  const float* h = row_values(entropy, "entropy", targets);
  const float* gl = grad_logprob ? row_values(*grad_logprob, "grad_logprob", targets) : nullptr;
  const float* gh = grad_entropy ? row_values(*grad_entropy, "grad_entropy", targets) : nullptr;
  const c10::DeviceGuard guard(logits.device());
  if (out) {
    check_device(*out, "out", logits.device());
    if (out->sizes() != logits.sizes() || out->scalar_type() != logits.scalar_type())
      plan_error("out: a tensor of the logits' shape and dtype is wanted");
  }
  at::Tensor to = out ? *out : at::empty(logits.sizes(), on(logits.device(), logits.scalar_type()));
  const uint64_t stride = row_stride(to, "out");
  if (lse_low)
    check(sr_logprob_pair_grad(&s, l, low, h, gl, gh, to.data_ptr(), stride, stream_of(logits.device())),
          "sr_logprob_pair_grad");
  else
    check(sr_logprob_grad(&s, l, h, gl, gh, to.data_ptr(), stride, stream_of(logits.device())), "sr_logprob_grad");
  if (out) written(to);
  return to;
}

// --------------------------------------------------------- feed-forward block

int32_t activation_code(const std::string& name) {
  if (name == "silu") return SR_ACT_SILU;
  if (name == "gelu") return SR_ACT_GELU;
  if (name == "gelu_tanh") return SR_ACT_GELU_TANH;
  plan_error("activation: " + name + ", not silu, gelu or gelu_tanh");
}

// A block's tensors; x and what has its shape may have any number of dimensions.
sr_ffn_shape ffn_shape(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up, const at::Tensor& down,
                       const std::string& activation) {
  const struct { const at::Tensor& t; const char* what; } all[4] = {{x, "x"}, {gate, "gate"}, {up, "up"}, {down, "down"}};
  if (x.dim() < 1) plan_error("x: rows of hidden elements are wanted");
  if (!x.is_cuda()) plan_error("x is on " + x.device().str() + ", not on the GPU");
  for (const auto& a : all) {
    check_device(a.t, a.what, x.device());
    check_tangent(a.t, a.what);
    if (a.t.scalar_type() != x.scalar_type())
      plan_error(std::string(a.what) + ": dtype " + c10::toString(a.t.scalar_type()) + ", x has " +
                 c10::toString(x.scalar_type()));
  }
  const int32_t dtype = float_code(x, "x");
  for (int i = 1; i < 4; ++i)
    if (all[i].t.dim() != 2) plan_error(std::string(all[i].what) + ": a matrix is wanted");
  const int64_t hidden = x.size(-1), ffn = gate.size(0);
  if (gate.size(1) != hidden || up.size(0) != ffn || up.size(1) != hidden || down.size(0) != hidden || down.size(1) != ffn)
    plan_error("gate and up of ffn x hidden and down of hidden x ffn are wanted, not " + c10::str(gate.sizes()) + ", " +
               c10::str(up.sizes()) + " and " + c10::str(down.sizes()) + " for " + std::to_string(hidden));
  int64_t tokens = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) tokens *= x.size(d);
  return {x.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), uint64_t(tokens), uint64_t(hidden), uint64_t(ffn),
          row_stride(x, "x"), row_stride(gate, "gate"), row_stride(up, "up"), row_stride(down, "down"), dtype,
          activation_code(activation)};
}

py::tuple gated_ffn(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up, const at::Tensor& down,
                    const std::string& activation, bool keep) {
  const sr_ffn_shape s = ffn_shape(x, gate, up, down, activation);
  const c10::DeviceGuard guard(x.device());
  const at::TensorOptions like = on(x.device(), x.scalar_type());
  uint64_t need = 0;
  check(sr_ffn_workspace(&s, keep, &need), "sr_ffn");
  const at::Tensor out = at::empty(x.sizes(), like), work = at::empty({int64_t(need)}, on(x.device(), at::kByte));
  at::Tensor a, b;
  if (keep) {
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = int64_t(s.ffn);
    a = at::empty(shape, on(x.device(), at::kFloat));
    b = at::empty(shape, on(x.device(), at::kFloat));
  }
  check(sr_ffn(&s, out.data_ptr(), keep ? a.data_ptr<float>() : nullptr, keep ? b.data_ptr<float>() : nullptr,
               work.data_ptr(), need,
               stream_of(x.device())),
        "sr_ffn");
  if (!keep) return py::make_tuple(out);
  return py::make_tuple(out, a, b);
}

py::tuple gated_ffn_grad(const at::Tensor& x, const at::Tensor& gate, const at::Tensor& up, const at::Tensor& down,
                         const at::Tensor& kept_gate, const at::Tensor& kept_up, const at::Tensor& grad_output,
                         const std::string& activation, const std::vector<bool>& wanted) {
  const sr_ffn_shape s = ffn_shape(x, gate, up, down, activation);
  if (wanted.size() != 4) plan_error("wanted: one of each of x, gate, up and down");
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = int64_t(s.ffn);
  const struct { const at::Tensor& t; const char* what; at::IntArrayRef shape; at::ScalarType type; } given[3] = {
      {kept_gate, "kept_gate", shape, at::kFloat},
      {kept_up, "kept_up", shape, at::kFloat},
      {grad_output, "grad_output", x.sizes(), x.scalar_type()}};
  for (const auto& g : given) {
    check_device(g.t, g.what, x.device());
    check_tangent(g.t, g.what);
    if (g.t.scalar_type() != g.type || g.t.sizes() != g.shape)
      plan_error(std::string(g.what) + ": " + c10::str(g.shape) + " of " + c10::toString(g.type) + " is wanted, not " +
                 c10::str(g.t.sizes()) + " of " + c10::toString(g.t.scalar_type()));
  }
  for (const at::Tensor* t : {&kept_gate, &kept_up}) {
    if (!t->is_contiguous()) plan_error("kept_gate and kept_up: contiguous tensors are wanted");
    check_stored(*t, "kept_gate or kept_up");
  }
  const uint64_t stride = row_stride(grad_output, "grad_output");
  const c10::DeviceGuard guard(x.device());
  const at::Tensor* like[4] = {&x, &gate, &up, &down};
  at::Tensor grad[4];
  void* to[4] = {};
  // an empty tensor has no address: what is wanted of it is nothing
  for (int i = 0; i < 4; ++i) {
    if (!wanted[i]) continue;
    grad[i] = at::empty(like[i]->sizes(), on(x.device(), x.scalar_type()));
    to[i] = grad[i].data_ptr();
  }
  const sr_ffn_grads g{to[0], to[1], to[2], to[3]};
  uint64_t need = 0;
  check(sr_ffn_grad_workspace(&s, grad_output.data_ptr(), stride, &g, &need), "sr_ffn_grad");
  const at::Tensor work = at::empty({int64_t(need)}, on(x.device(), at::kByte));
  check(sr_ffn_grad(&s, kept_gate.data_ptr<float>(), kept_up.data_ptr<float>(), grad_output.data_ptr(), stride, &g, work.data_ptr(), need,
                    stream_of(x.device())),
        "sr_ffn_grad");
  py::tuple out(4);
  for (int i = 0; i < 4; ++i) out[i] = wanted[i] ? py::cast(grad[i]) : py::none();
  return out;
}

// ------------------------------------------------------- orthogonal matrices

// A sum over ranks by a Python callable, on views of the call's workspace.  What
// it raises comes back once the library has returned.
class Reduce {
 public:
  explicit Reduce(py::object callable) : callable_(std::move(callable)) {}

  void over(const at::Tensor& work) { work_ = work; }
  sr_reduce function() const { return callable_.is_none() ? nullptr : &Reduce::call; }
  // The library's status, or what the callable raised.
  void check_call(int rc, const char* what) {
    if (raised_) {
      std::exception_ptr e = raised_;
      raised_ = nullptr;
      std::rethrow_exception(e);
    }
    check(rc, what);
  }

 private:
  static int call(void* context, void* data, uint64_t count, int32_t dtype, hipStream_t) {
    Reduce& self = *static_cast<Reduce*>(context);
    try {
      const bool wide = dtype == SR_DT_F64;
      const int64_t at = static_cast<char*>(data) - static_cast<char*>(self.work_.data_ptr());
      const at::Tensor bytes = self.work_.narrow(0, at, int64_t(count) * (wide ? 8 : 4));
      self.callable_(bytes.view(wide ? at::kDouble : at::kFloat));
      return 0;
    } catch (...) {
      self.raised_ = std::current_exception();
      return 1;
    }
  }

  py::object callable_;
  at::Tensor work_;
  std::exception_ptr raised_;
};

int32_t split_code(py::handle dim, const std::string& what) {
  if (dim.is_none()) return -1;
  if (!PyLong_Check(dim.ptr())) plan_error(what + ": None, 0 or 1 is wanted");
  const int64_t d = PyLong_AsLongLong(dim.ptr());
  if (d != 0 && d != 1) {
    PyErr_Clear();
    plan_error(what + ": None, 0 or 1 is wanted");
  }
  return int32_t(d);
}

sr_matrix matrix_of(const at::Tensor& t, const std::string& what, int32_t split, c10::optional<at::Device>& device) {
  if (!t.is_cuda()) plan_error(what + " is on " + t.device().str() + ", not on the GPU");
  if (!device) device = t.device();
  if (t.device() != *device) plan_error(what + " is on " + t.device().str() + ", not on " + device->str());
  if (t.dim() != 2) plan_error(what + ": a matrix is wanted, not " + c10::str(t.sizes()));
  const uint64_t stride = row_stride(t, what);
  return {t.data_ptr(), uint64_t(t.size(0)), uint64_t(t.size(1)), stride, float_code(t, what), split};
}

py::list orthogonalize(py::object matrices, py::object outs, py::object splits, int32_t steps,
                       const std::vector<double>& coefficients, double eps, py::object all_reduce) {
  c10::optional<at::Device> device;
  const Fast list(matrices, "matrices");
  const bool fresh = outs.is_none();
  const Fast out_list(fresh ? py::object(py::list()) : outs, "out"),
      split_list(splits.is_none() ? py::object(py::list()) : splits, "split");
  if (!fresh && out_list.size() != list.size())
    plan_error("out has " + std::to_string(out_list.size()) + " tensors, matrices " + std::to_string(list.size()));
  if (!splits.is_none() && split_list.size() != list.size())
    plan_error("split has " + std::to_string(split_list.size()) + " entries, matrices " + std::to_string(list.size()));
  std::vector<sr_matrix> src, dst;
  std::vector<at::Tensor> to;
  for (size_t i = 0; i < list.size(); ++i) {
    const std::string name = indexed("matrices", i);
    const at::Tensor& t = tensor_of(list[i], name);
    check_tangent(t, name.c_str());
    src.push_back(matrix_of(t, name, splits.is_none() ? -1 : split_code(split_list[i], indexed("split", i)), device));
    if (fresh) continue;
    const std::string out_name = indexed("out", i);
    const at::Tensor& o = tensor_of(out_list[i], out_name);
    check_tangent(o, out_name.c_str());
    dst.push_back(matrix_of(o, out_name, -1, device));
    if (o.sizes() != t.sizes()) plan_error(out_name + ": shape differs from the matrix's");
    to.push_back(o);
  }
  if (!device) device = current_device();
  const c10::DeviceGuard guard(*device);
  if (fresh) {
    for (size_t i = 0; i < list.size(); ++i) {
      const at::Tensor& t = THPVariable_Unpack(list[i]);
      to.push_back(at::empty(t.sizes(), on(*device, t.scalar_type())));
      dst.push_back({to[i].data_ptr(), src[i].rows, src[i].cols, src[i].cols, src[i].dtype, -1});
    }
  }
  Reduce reduce(all_reduce);
  const sr_newton_schulz ns{steps, 0, coefficients.data(), eps, reduce.function(), &reduce};
  uint64_t need = 0;
  check(sr_orthogonalize_workspace(src.data(), dst.data(), int32_t(src.size()), &ns, &need), "sr_orthogonalize");
  const at::Tensor work = at::empty({int64_t(need)}, on(*device, at::kByte));
  reduce.over(work);
  const int rc = sr_orthogonalize(src.data(), dst.data(), int32_t(src.size()), &ns, work.data_ptr(), need, stream_of(*device));
  if (!fresh)
    for (const at::Tensor& t : to) written(t);
  reduce.check_call(rc, "sr_orthogonalize");
  py::list out;
  for (const at::Tensor& t : to) out.append(t);
  return out;
}

// The matrices that Muon steps, in the order of their names.
class MuonState {
 public:
  MuonState(py::object weight, py::object exp_avg, py::object param, std::vector<std::string> names,
            std::vector<int32_t> split, std::vector<double> scale)
      : names_(std::move(names)), split_(std::move(split)), scale_(std::move(scale)) {
    const Fast w(weight, "weight"), m(exp_avg, "exp_avg"), p(param, "param");
    if (w.size() != names_.size() || m.size() != w.size() || p.size() != w.size() || split_.size() != w.size() ||
        scale_.size() != w.size())
      plan_error("state: lists of different lengths");
    for (size_t i = 0; i < names_.size(); ++i) {
      weight_.push_back(tensor_of(w[i], names_[i] + "/weight"));
      exp_avg_.push_back(tensor_of(m[i], names_[i] + "/exp_avg"));
      param_.push_back(p[i] == Py_None ? at::Tensor() : tensor_of(p[i], names_[i] + "/param"));
      check_fields(i);
      shapes_.push_back(weight_[i].sizes().vec());
    }
  }

  py::object step(py::object grads, double lr, double momentum, bool nesterov, double weight_decay, int32_t steps,
                  const std::vector<double>& coefficients, double eps, py::object max_norm, py::object square_sum,
                  py::object all_reduce) {
    const Fast list(grads, "grads");
    if (list.size() != names_.size())
      plan_error("grads: " + std::to_string(list.size()) + " tensors for a state of " + std::to_string(names_.size()));
    std::vector<sr_muon_tensor> tensors;
    std::vector<sr_array> arrays;
    std::vector<size_t> stepped;
    for (size_t i = 0; i < names_.size(); ++i) {
      if (list[i] == Py_None) continue;
      const at::Tensor& g = tensor_of(list[i], "gradient of " + names_[i]);
      const at::Tensor &w = weight_[i], &m = exp_avg_[i], &p = param_[i];
      check_fields(i);
      if (w.sizes() != at::IntArrayRef(shapes_[i])) plan_error(names_[i] + ": another shape than the state was taken with");
      if (g.layout() != at::kStrided || !g.is_contiguous() || g.device() != w.device() || g.sizes() != w.sizes())
        plan_error("gradient of " + names_[i] + ": a dense tensor like the weight on " + w.device().str() + " is wanted");
      const at::ScalarType gt = g.scalar_type();
      if (gt != at::kFloat && gt != at::kBFloat16)
        plan_error("gradient of " + names_[i] + ": dtype " + c10::toString(gt) + ", not float32 or bfloat16");
      if (!stored(g)) plan_error("gradient of " + names_[i] + ": its storage has been released");
      check_tangent(g, "grads");
      tensors.push_back({w.data_ptr(), m.data_ptr(), p.defined() ? p.data_ptr() : nullptr, g.data_ptr(), uint64_t(w.size(0)),
                         uint64_t(w.size(1)), scale_[i], float_code(w, names_[i]), float_code(m, names_[i]),
                         float_code(g, names_[i]), split_[i], 0});
      arrays.push_back(array_of(g, names_[i]));
      stepped.push_back(i);
    }
    const at::Device device = device_ ? *device_ : current_device();
    const c10::DeviceGuard guard(device);
    Reduce reduce(all_reduce);
    const sr_newton_schulz ns{steps, 0, coefficients.data(), eps, reduce.function(), &reduce};
    sr_muon_options o{lr, weight_decay, momentum, nesterov, 0, 0.0, nullptr};
    c10::optional<SumWork> work;
    at::Tensor norm;
    const double* given = nullptr;
    if (!max_norm.is_none()) {
      o.max_norm = max_norm.cast<double>();
      given = given_sum(square_sum, device);
      // each rank would clip its part of a matrix by a factor of its own
      for (const sr_muon_tensor& t : tensors)
        if (t.split >= 0 && !given) plan_error("max_norm: matrices that are split want the square_sum of all ranks");
      norm = at::empty({}, on(device, at::kFloat));
      if (!given) work.emplace(arrays, device);
      o.square_sum = given ? given : work->sum();
    } else if (!square_sum.is_none()) {
      plan_error("square_sum is given without max_norm");
    }
    // all checks, before the sum of squares is launched
    uint64_t need = 0;
    check(sr_muon_workspace(tensors.data(), int32_t(tensors.size()), &o, &ns, &need), "sr_muon");
    const at::Tensor memory = at::empty({int64_t(need)}, on(device, at::kByte));
    reduce.over(memory);
    if (work)
      check(sr_square_sum(arrays.data(), int32_t(arrays.size()), 1, work->parts(), work->bytes, work->sum(),
                          norm.data_ptr<float>(), stream_of(device)),
            "sr_square_sum");
    else if (given)
      check(sr_clip(nullptr, nullptr, 0, given, float(o.max_norm), norm.data_ptr<float>(), stream_of(device)), "sr_clip");
    const int rc = sr_muon(tensors.data(), int32_t(tensors.size()), &o, &ns, memory.data_ptr(), need, stream_of(device));
    for (size_t i : stepped)
      for (const at::Tensor* t : {&weight_[i], &exp_avg_[i], &param_[i]})
        if (t->defined()) written(*t);
    reduce.check_call(rc, "sr_muon");
    if (!norm.defined()) return py::none();
    return py::cast(norm);
  }

 private:
  // The fields as they are now, as AdamWState checks them.
  void check_fields(size_t i) {
    const at::Tensor &w = weight_[i], &m = exp_avg_[i], &p = param_[i];
    const struct { const at::Tensor& t; const char* what; } field[3] = {{w, "weight"}, {m, "exp_avg"}, {p, "param"}};
    for (const auto& f : field) {
      if (!f.t.defined()) continue;
      if (!dense(f.t, device_)) check_dense(f.t, names_[i] + "/" + f.what, device_);     // says what is wrong
      if (!stored(f.t)) plan_error(names_[i] + ": a field's storage has been released");
      if (f.t.sizes() != w.sizes()) plan_error(names_[i] + ": fields of different shapes");
    }
    const at::ScalarType wt = w.scalar_type(), mt = m.scalar_type();
    if (w.dim() != 2) plan_error(names_[i] + ": a matrix is wanted, not " + c10::str(w.sizes()));
    if (wt != at::kFloat && wt != at::kBFloat16)
      plan_error(names_[i] + ": weight of dtype " + c10::toString(wt) + ", not float32 or bfloat16");
    if (mt != at::kFloat && mt != at::kBFloat16)
      plan_error(names_[i] + ": exp_avg of dtype " + c10::toString(mt) + ", not float32 or bfloat16");
    if (p.defined() && (wt != at::kFloat || p.scalar_type() != at::kBFloat16))
      plan_error(names_[i] + ": a master weight is float32 and its param bfloat16");
  }

  std::vector<std::string> names_;
  std::vector<int32_t> split_;
  std::vector<double> scale_;
  std::vector<at::Tensor> weight_, exp_avg_, param_;
  std::vector<std::vector<int64_t>> shapes_;      // what split and scale were formed for
  c10::optional<at::Device> device_;
};

}  // namespace

namespace suika_host {

void bind_step(py::module_& m) {
  m.def("grad_square_sum", &grad_square_sum, py::arg("grads"));
  m.def("grad_norm", &grad_norm, py::arg("grads"));
  m.def("clip_grads", &clip_grads, py::arg("grads"), py::arg("max_norm"), py::arg("out"), py::arg("square_sum"));
  py::class_<AdamWState>(m, "AdamWState", "The tensors of a state that AdamW updates in place")
      .def(py::init<py::object, py::object, py::object, py::object, std::vector<std::string>, std::vector<int64_t>>(),
           py::arg("weight"), py::arg("exp_avg"), py::arg("exp_avg_sq"), py::arg("param"), py::arg("names"),
           py::arg("steps"))
      .def_property("steps", &AdamWState::steps, &AdamWState::set_steps)
      .def("step", &AdamWState::step, py::arg("grads"), py::arg("lr"), py::arg("beta1"),
           py::arg("beta2"), py::arg("eps"), py::arg("weight_decay"), py::arg("max_norm"), py::arg("square_sum"));
  m.def("vocab_embedding", &vocab_embedding, py::arg("tokens"), py::arg("weight"), py::arg("scale"),
        py::arg("vocab_start"), py::arg("out"));
  m.def("vocab_embedding_grad", &vocab_embedding_grad, py::arg("tokens"), py::arg("grad_output"), py::arg("rows"),
        py::arg("scale"), py::arg("vocab_start"), py::arg("dtype"), py::arg("out"), py::arg("accumulate"));
  m.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("targets"), py::arg("top"), py::arg("vocab"));
  m.def("token_logprobs_grad", &token_logprobs_grad, py::arg("logits"), py::arg("targets"), py::arg("lse"),
        py::arg("entropy"), py::arg("grad_logprob"), py::arg("grad_entropy"), py::arg("vocab"), py::arg("out"),
        py::arg("lse_low"));
  m.def("orthogonalize", &orthogonalize, py::arg("matrices"), py::arg("out"), py::arg("split"), py::arg("steps"),
        py::arg("coefficients"), py::arg("eps"), py::arg("all_reduce"));
  py::class_<MuonState>(m, "MuonState", "The matrices of a state that Muon updates in place")
      .def(py::init<py::object, py::object, py::object, std::vector<std::string>, std::vector<int32_t>, std::vector<double>>(),
           py::arg("weight"), py::arg("exp_avg"), py::arg("param"), py::arg("names"), py::arg("split"), py::arg("scale"))
      .def("step", &MuonState::step, py::arg("grads"), py::arg("lr"), py::arg("momentum"), py::arg("nesterov"),
           py::arg("weight_decay"), py::arg("steps"), py::arg("coefficients"), py::arg("eps"), py::arg("max_norm"),
           py::arg("square_sum"), py::arg("all_reduce"));
  m.def("gated_ffn", &gated_ffn, py::arg("x"), py::arg("gate"), py::arg("up"), py::arg("down"), py::arg("activation"),
        py::arg("keep"));
  m.def("gated_ffn_grad", &gated_ffn_grad, py::arg("x"), py::arg("gate"), py::arg("up"), py::arg("down"),
        py::arg("kept_gate"), py::arg("kept_up"), py::arg("grad_output"), py::arg("activation"), py::arg("wanted"));
}

}  // namespace suika_host
