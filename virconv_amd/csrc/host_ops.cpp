// The host side of the row operators: argument checks, allocation, autograd nodes and the launch in native code, on the C ABI of
// libvirconv_hip.so (its functions come in as addresses, so that whatever library the binding loaded is the one that runs).
//
// Why it is native: these operators run in 3 to 20 us on small inputs.  The same steps in Python took 9 us for a forward call, 125 us for a
// forward and backward pass through two Python autograd nodes, and 0.9 us a tensor for an optimizer step.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "../../include/virconv_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Abi {
  decltype(&vc_last_error) last_error = nullptr;
  decltype(&vc_layer_norm_forward) layer_norm_forward = nullptr;
  decltype(&vc_layer_norm_backward_workspace_bytes) layer_norm_backward_workspace_bytes = nullptr;
  decltype(&vc_layer_norm_backward) layer_norm_backward = nullptr;
  decltype(&vc_grouped_linear_workspace_bytes) grouped_linear_workspace_bytes = nullptr;
  decltype(&vc_grouped_linear_forward) grouped_linear_forward = nullptr;
  decltype(&vc_grouped_linear_backward_input) grouped_linear_backward_input = nullptr;
  decltype(&vc_grouped_linear_backward_weight) grouped_linear_backward_weight = nullptr;
  decltype(&vc_adamw) adamw = nullptr;
} abi;

struct VirConvError : std::runtime_error { using std::runtime_error::runtime_error; };
PyObject* error_class = nullptr;    // virconv_amd._lib.VirConvError

template <typename F> void set(F& f, uintptr_t address) { f = reinterpret_cast<F>(address); }

void bind(const std::unordered_map<std::string, uintptr_t>& fn, py::object error) {
  set(abi.last_error, fn.at("vc_last_error"));
  set(abi.layer_norm_forward, fn.at("vc_layer_norm_forward"));
  set(abi.layer_norm_backward_workspace_bytes, fn.at("vc_layer_norm_backward_workspace_bytes"));
  set(abi.layer_norm_backward, fn.at("vc_layer_norm_backward"));
  set(abi.grouped_linear_workspace_bytes, fn.at("vc_grouped_linear_workspace_bytes"));
  set(abi.grouped_linear_forward, fn.at("vc_grouped_linear_forward"));
  set(abi.grouped_linear_backward_input, fn.at("vc_grouped_linear_backward_input"));
  set(abi.grouped_linear_backward_weight, fn.at("vc_grouped_linear_backward_weight"));
  set(abi.adamw, fn.at("vc_adamw"));
  error_class = error.release().ptr();
}

void check(int status, const char* what) {
  if (status != VC_OK) throw VirConvError(std::string(what) + " failed with vc_status " + std::to_string(status) + ": " + abi.last_error());
}

int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return VC_F32;
    case at::kHalf: return VC_F16;
    case at::kBFloat16: return VC_BF16;
    default: throw VirConvError(std::string(name) + ": expected float32, float16 or bfloat16, got " + c10::toString(t.scalar_type()));
  }
}

void need_gpu(const Tensor& t, const char* name) {
  if (!t.is_cuda()) throw VirConvError(std::string(name) + ": expected a CUDA/HIP tensor; virconv_amd has no CPU path");
  if (t.layout() != at::kStrided) throw VirConvError(std::string(name) + ": expected a dense tensor");
}

void same_device(const Tensor& t, const Tensor& first, const char* name) {
  need_gpu(t, name);
  if (t.device() != first.device())
    throw VirConvError(std::string(name) + ": the tensors of a call lie on different devices: " + first.device().str() + " and " + t.device().str());
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// a matrix whose rows are dense (a column slice of a wider one passes as it is), and its row stride
Tensor rows_of(const Tensor& t, int64_t& stride) {
  const int64_t n = t.size(0), c = t.size(1);
  if ((t.stride(1) == 1 || c == 1) && (t.stride(0) >= c || n <= 1)) {
    stride = std::max<int64_t>(t.stride(0), c);
    return t;
  }
  stride = c;
  return t.contiguous();
}

Tensor workspace(size_t bytes, const Tensor& like) { return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor(); }

Tensor detached(const OptTensor& t) { return t.has_value() && t->defined() ? *t : Tensor(); }

OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// Forward-mode derivatives: there are none here, and the passes below would drop a tangent without a word.
void refuse_tangents(const char* who, std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), who, ": no forward-mode derivatives");
}

bool capturing(hipStream_t stream) {     // (the legacy stream never is, and must not be asked while another one is)
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return stream && hipStreamIsCapturing(stream, &status) == hipSuccess && status == hipStreamCaptureStatusActive;
}

// A backward pass under capture whose gradients go to nodes recorded before it on a stream that is not captured (a leaf's, while an eager graph of
// that leaf lives): the engine would make that stream wait for the captured one, which ends the process.  Said here instead, also where nodes of the
// capture lie in between (a view of the rows, a copy of a strided weight, layers in front of this one): all that this pass leads to is walked.
void refuse_uncaptured_consumers(const char* who, const Tensor& x) {
  const c10::hip::HIPStream here = c10::hip::getCurrentHIPStream(x.get_device());
  if (!capturing(here.stream())) return;
  const auto node = torch::autograd::get_current_node();
  const auto* tasks = torch::autograd::get_current_graph_task_exec_info();
  if (!node) return;
  std::vector<torch::autograd::Node*> stack{node.get()};
  std::unordered_set<torch::autograd::Node*> seen{node.get()};
  while (!stack.empty()) {
    torch::autograd::Node* const from = stack.back();
    stack.pop_back();
    for (const auto& edge : from->next_edges()) {
      torch::autograd::Node* const to = edge.function.get();
      if (!to || !seen.insert(to).second) continue;
      if (tasks && !tasks->empty()) {
        const auto it = tasks->find(to);
        if (it == tasks->end() || !it->second.should_execute()) continue;
      }
      stack.push_back(to);
      const auto there = to->stream();
      if (!there || there->id() == here.id() || there->device_index() != here.device_index()) continue;
      const c10::Stream plain(c10::Stream::UNSAFE, c10::Device(here.unwrap().device_type(), here.device_index()), there->id());
      if (!capturing(c10::hip::HIPStream(plain).stream()))
        throw VirConvError(std::string(who) + ": this backward pass is being captured, and a graph recorded before it, on a stream that is not, holds a node "
                           "its gradients go to (an eager result of the same leaf that is still alive): let go of that result before the capture");
    }
  }
}

// First-order gradients only: where a graph of the backward pass is asked for, its results hang on a node that says so when it is used.
struct OnceOnly : torch::autograd::Function<OnceOnly> {
  static Tensor forward(AutogradContext*, const Tensor& result, const OptTensor&, const OptTensor&, const OptTensor&) { return result.clone(); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "trying to differentiate twice a function of virconv_amd that has first-order gradients only");
  }
};

variable_list once(variable_list results, const Tensor& a, const Tensor& b, const Tensor& c) {
  if (!wants_grad({a, b, c})) return results;
  for (Tensor& t : results)
    if (t.defined()) t = OnceOnly::apply(t, given(a), given(b), given(c));
  return results;
}

// ---------------------------------------------------------------------------------------------------------------- layer norm
Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.size(0), c = x.size(1);
  int64_t ld;
  const Tensor xr = rows_of(x, ld);
  Tensor y = at::empty({n, c}, x.options());
  float *mean = nullptr, *rstd = nullptr;
  if (stats) {
    *stats = at::empty({2, n}, x.options().dtype(at::kFloat));
    mean = (float*)stats->data_ptr();
    rstd = mean + n;
  }
  check(abi.layer_norm_forward(xr.data_ptr(), ld, n, c, dtype_of(x, "layer_norm: x"), ptr(w), w.defined() ? dtype_of(w, "weight") : 0, ptr(b),
                               b.defined() ? dtype_of(b, "bias") : 0, (float)eps, y.data_ptr(), mean, rstd, stream_of(x)),
        "vc_layer_norm_forward");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    Tensor stats;
    const Tensor w = detached(weight), b = detached(bias);
    Tensor y = norm_forward(x, w, b, eps, &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["bias"] = b.defined() ? (int64_t)b.scalar_type() : (int64_t)-1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2], &dy = grads[0];
    refuse_uncaptured_consumers("layer_norm", x);
    // (edges are counted over the tensors that are there)
    const bool need_x = ctx->needs_input_grad(0), need_w = w.defined() && ctx->needs_input_grad(1);
    const int64_t bias_type = ctx->saved_data["bias"].toInt();
    const bool need_b = bias_type >= 0 && ctx->needs_input_grad(w.defined() ? 2 : 1);
    Tensor dx, dw, db;
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(x.device());
      const int64_t n = x.size(0), c = x.size(1);
      const int dt = dtype_of(x, "layer_norm: x");
      int64_t ld, dld;
      const Tensor xr = rows_of(x, ld), dyr = rows_of(dy, dld);
      if (need_x) dx = at::empty({n, c}, x.options());
      if (need_w) dw = at::empty({c}, w.options());
      if (need_b) db = at::empty({c}, x.options().dtype((at::ScalarType)bias_type));
      const size_t bytes = need_w || need_b ? abi.layer_norm_backward_workspace_bytes(n, c, dt) : 0;
      const Tensor ws = workspace(bytes, x);
      const float* mean = (const float*)stats.data_ptr();
      check(abi.layer_norm_backward(xr.data_ptr(), ld, dyr.data_ptr(), dld, n, c, dt, ptr(w), w.defined() ? dtype_of(w, "weight") : 0,
                                    need_b ? dtype_of(db, "bias") : 0, mean, mean + n, ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, stream_of(x)),
            "vc_layer_norm_backward");
    }
    variable_list out = once({dx, dw, db}, dy, x, w);
    out.push_back(Tensor());
    return out;
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: wants rows of at least one channel, got a tensor of shape ", x.sizes());
  const int64_t c = x.size(-1);
  Tensor w = detached(weight), b = detached(bias);
  for (const auto& [t, name] : {std::pair<Tensor&, const char*>{w, "weight"}, {b, "bias"}}) {
    if (!t.defined()) continue;
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == c, "layer_norm: ", name, " has shape ", t.sizes(), ", expected [", c, "]");
    TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, "layer_norm: ", name, " is ", t.scalar_type(), "; with ",
                      x.scalar_type(), " rows it has to be of that type or float32");
  }
  TORCH_CHECK_VALUE(eps >= 0.0, "layer_norm: eps = ", eps);
  refuse_tangents("layer_norm", {x, w, b});
  dtype_of(x, "layer_norm: x");
  need_gpu(x, "layer_norm: x");
  for (const auto& [t, name] : {std::pair<Tensor&, const char*>{w, "layer_norm: weight"}, {b, "layer_norm: bias"}})
    if (t.defined()) {
      same_device(t, x, name);
      if (!t.is_contiguous()) t = t.contiguous();
    }
  const Tensor rows = x.dim() == 2 ? x : x.reshape({-1, c});
  const Tensor y = wants_grad({x, w, b}) ? LayerNorm::apply(rows, given(w), given(b), eps) : norm_forward(rows, w, b, eps, nullptr);
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ---------------------------------------------------------------------------------------------------------------- grouped products
Tensor grouped_forward(const Tensor& x, const Tensor& w, const Tensor& offsets, const Tensor& b) {
  const c10::DeviceGuard guard(x.device());
  const int64_t n = x.size(0), groups = w.size(0), out = w.size(1), in = w.size(2);
  const int dt = dtype_of(x, "grouped_linear: x");
  int64_t ld;
  const Tensor xr = rows_of(x, ld);
  Tensor y = at::empty({n, out}, x.options());
  const size_t bytes = abi.grouped_linear_workspace_bytes(0, n, groups, in, out, dt);
  const Tensor ws = workspace(bytes, x);
  check(abi.grouped_linear_forward(xr.data_ptr(), ld, n, w.data_ptr(), ptr(b), offsets.data_ptr(), (int)(8 * offsets.element_size()), groups, in, out,
                                   dt, y.data_ptr(), ptr(ws), bytes, stream_of(x)),
        "vc_grouped_linear_forward");
  return y;
}

struct GroupedLinear : torch::autograd::Function<GroupedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& offsets, const OptTensor& bias) {
    const Tensor b = detached(bias);
    Tensor y = grouped_forward(x, w, offsets, b);
    ctx->save_for_backward({x, w, offsets});
    ctx->saved_data["bias"] = b.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &offsets = saved[2], &dy = grads[0];
    refuse_uncaptured_consumers("grouped_linear", x);
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
    Tensor dx, dw, db;
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(x.device());
      const int64_t n = x.size(0), groups = w.size(0), out = w.size(1), in = w.size(2);
      const int dt = dtype_of(x, "grouped_linear: x"), bits = (int)(8 * offsets.element_size());
      int64_t ld, dld;
      const Tensor xr = rows_of(x, ld), dyr = rows_of(dy, dld);
      if (need_x) {
        dx = at::empty({n, in}, x.options());
        const size_t bytes = abi.grouped_linear_workspace_bytes(1, n, groups, in, out, dt);
        const Tensor ws = workspace(bytes, x);
        check(abi.grouped_linear_backward_input(dyr.data_ptr(), dld, n, w.data_ptr(), offsets.data_ptr(), bits, groups, in, out, dt, dx.data_ptr(),
                                                ptr(ws), bytes, stream_of(x)),
              "vc_grouped_linear_backward_input");
      }
      if (need_w || need_b) {
        dw = at::empty({groups, out, in}, x.options());
        if (need_b) db = at::empty({groups, out}, x.options());
        const size_t bytes = abi.grouped_linear_workspace_bytes(2, n, groups, in, out, dt);
        const Tensor ws = workspace(bytes, x);
        check(abi.grouped_linear_backward_weight(xr.data_ptr(), ld, dyr.data_ptr(), dld, n, offsets.data_ptr(), bits, groups, in, out, dt,
                                                 dw.data_ptr(), ptr(db), ptr(ws), bytes, stream_of(x)),
              "vc_grouped_linear_backward_weight");
        if (!need_w) dw = Tensor();
      }
    }
    const variable_list d = once({dx, dw, db}, dy, x, w);
    return {d[0], d[1], Tensor(), d[2]};
  }
};

Tensor grouped_linear(const Tensor& x, const Tensor& weight, const Tensor& offsets, const OptTensor& bias) {
  const Tensor b0 = detached(bias);
  TORCH_CHECK_VALUE(x.dim() == 2 && weight.dim() == 3 && x.size(1) == weight.size(2) && weight.size(1) >= 1 && weight.size(2) >= 1,
                    "grouped_linear: wants x (N, in) and weight (G, out, in), got ", x.sizes(), " and ", weight.sizes());
  TORCH_CHECK_VALUE(weight.scalar_type() == x.scalar_type() && (!b0.defined() || b0.scalar_type() == x.scalar_type()),
                    "grouped_linear: x, weight and bias have to be of one type, got ", x.scalar_type(), ", ", weight.scalar_type(),
                    b0.defined() ? c10::str(", ", b0.scalar_type()) : std::string());
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.size(0) == weight.size(0) + 1 && (offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong),
                    "grouped_linear: offsets have to be ", weight.size(0) + 1, " int32 or int64 values, got ", offsets.sizes(), " ", offsets.scalar_type());
  TORCH_CHECK_VALUE(!b0.defined() || (b0.dim() == 2 && b0.size(0) == weight.size(0) && b0.size(1) == weight.size(1)), "grouped_linear: bias has shape ",
                    b0.defined() ? b0.sizes() : x.sizes(), ", expected [", weight.size(0), ", ", weight.size(1), "]");
  refuse_tangents("grouped_linear", {x, weight, b0});
  dtype_of(x, "grouped_linear: x");
  need_gpu(x, "grouped_linear: x");
  same_device(weight, x, "grouped_linear: weight");
  same_device(offsets, x, "grouped_linear: offsets");
  if (b0.defined()) same_device(b0, x, "grouped_linear: bias");
  const Tensor w = weight.is_contiguous() ? weight : weight.contiguous(), o = offsets.is_contiguous() ? offsets : offsets.contiguous();
  const Tensor b = !b0.defined() || b0.is_contiguous() ? b0 : b0.contiguous();
  return wants_grad({x, w, b}) ? GroupedLinear::apply(x, w, o, given(b)) : grouped_forward(x, w, o, b);
}

// ---------------------------------------------------------------------------------------------------------------- AdamW
bool plain(const Tensor& t, const Tensor& p, at::ScalarType type) {   // a tensor of p's shape, elements in p's (row-major) order, on p's device
  return t.layout() == at::kStrided && t.scalar_type() == type && t.device() == p.device() && t.sizes() == p.sizes() && t.is_contiguous();
}

// Memory that was written through a pointer: what keeps something by the tensor's version (autograd's saved tensors, packed weights) has to see it.
// (A tensor made in inference mode has no version.)
void written(c10::TensorImpl* t) {
  if (t && !t->is_inference()) t->bump_version();
}

constexpr const char* kCaptured = "AdamW: a step counts on the host (bias correction, random numbers): it cannot be captured into a graph";

// One step of `params` (those with gradients) with their state dicts (None: not there yet), all in the ordinary case: one device, row-major, one
// step count, moments as they are made; a call for each type.  -> the step taken, or -1 with nothing done: the caller sorts the case out.
int64_t adamw(const py::list& params, const py::list& states, int64_t first_place, int state_bits, double lr, double b1, double b2, double eps,
              double weight_decay, int64_t seed) {
  static PyObject* const kStep = PyUnicode_InternFromString("step");
  static PyObject* const kAvg = PyUnicode_InternFromString("exp_avg");
  static PyObject* const kSq = PyUnicode_InternFromString("exp_avg_sq");
  static PyObject* const kRms = PyUnicode_InternFromString("exp_avg_rms");
  static PyObject* const kExponents = PyUnicode_InternFromString("exponents");
  const size_t n = PyList_GET_SIZE(params.ptr());
  if ((size_t)PyList_GET_SIZE(states.ptr()) != n) return -1;
  const at::ScalarType moment = state_bits == 8 ? at::kFloat8_e4m3fn : at::kFloat;
  std::vector<vc_adamw_tensor> table[3];     // by vc_dtype
  bool any = false;
  struct Results { c10::TensorImpl* t[4]; PyObject* state; };     // what a tensor's step writes
  std::vector<Results> results[3];
  int64_t step = 0;
  Tensor first;
  for (size_t k = 0; k < n; ++k) {
    PyObject *po = PyList_GET_ITEM(params.ptr(), k), *st = PyList_GET_ITEM(states.ptr(), k);
    if (!THPVariable_Check(po)) return -1;
    const Tensor& p = THPVariable_Unpack(po);
    const Tensor& g = p.grad();
    if (!g.defined()) continue;
    if (!PyDict_Check(st)) return -1;
    if (!first.defined()) first = p;
    if (!p.is_cuda() || p.device() != first.device() || p.layout() != at::kStrided || !p.is_contiguous() || !plain(g, p, p.scalar_type())) return -1;
    int dt;
    switch (p.scalar_type()) {
      case at::kFloat: dt = VC_F32; break;
      case at::kHalf: dt = VC_F16; break;
      case at::kBFloat16: dt = VC_BF16; break;
      default: return -1;
    }
    PyObject *so = PyDict_GetItem(st, kStep), *mo = PyDict_GetItem(st, kAvg), *vo = PyDict_GetItem(st, state_bits == 8 ? kRms : kSq);
    if (!so || !PyLong_CheckExact(so) || !mo || !vo || !THPVariable_Check(mo) || !THPVariable_Check(vo)) return -1;
    const int64_t s = PyLong_AsLongLong(so);
    if (!any) step = s;
    if (s != step || s < 0) return -1;
    const Tensor &m = THPVariable_Unpack(mo), &v = THPVariable_Unpack(vo);
    if (!plain(m, p, moment) || !plain(v, p, moment)) return -1;
    vc_adamw_tensor t = {p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), nullptr, p.numel(), (uint32_t)(first_place + k), 0};
    Results r = {{p.unsafeGetTensorImpl(), m.unsafeGetTensorImpl(), v.unsafeGetTensorImpl(), nullptr}, st};
    if (state_bits == 8) {
      PyObject* eo = PyDict_GetItem(st, kExponents);
      if (!eo || !THPVariable_Check(eo)) return -1;
      const Tensor& e = THPVariable_Unpack(eo);
      if (e.scalar_type() != at::kChar || e.device() != p.device() || e.dim() != 2 || e.size(0) != (t.n + 127) / 128 || e.size(1) != 2 || !e.is_contiguous())
        return -1;
      t.exponents = (int8_t*)e.data_ptr();
      r.t[3] = e.unsafeGetTensorImpl();
    }
    if (table[dt].empty()) {
      table[dt].reserve(n - k);
      results[dt].reserve(n - k);
    }
    table[dt].push_back(t);
    results[dt].push_back(r);
    any = true;
  }
  if (!any) return 0;
  const py::object now = py::reinterpret_steal<py::object>(PyLong_FromLongLong(step + 1));
  const c10::DeviceGuard guard(first.device());
  if (capturing((hipStream_t)stream_of(first))) throw VirConvError(kCaptured);
  for (int dt = 0; dt < 3; ++dt) {
    if (table[dt].empty()) continue;
    check(abi.adamw(table[dt].data(), (int64_t)table[dt].size(), dt, state_bits, lr, b1, b2, eps, weight_decay, step + 1, (uint32_t)seed,
                    stream_of(first)),
          "vc_adamw");
    for (const Results& r : results[dt]) {     // (what the next type's call refuses does not take this step back)
      for (c10::TensorImpl* t : r.t) written(t);
      PyDict_SetItem(r.state, kStep, now.ptr());
    }
  }
  return step + 1;
}

// are the keys and values of `dict`, in order, the objects of `list`, a key and its value in turn?
bool same_items(const py::dict& dict, const py::list& list) {
  const Py_ssize_t n = PyList_GET_SIZE(list.ptr());
  if (2 * PyDict_Size(dict.ptr()) != n) return false;
  Py_ssize_t at = 0, k = 0;
  PyObject *key, *value;
  for (; PyDict_Next(dict.ptr(), &at, &key, &value); k += 2)
    if (k + 2 > n || PyList_GET_ITEM(list.ptr(), k) != key || PyList_GET_ITEM(list.ptr(), k + 1) != value) return false;
  return true;
}

bool same_objects(const py::list& a, const py::list& b) {
  const Py_ssize_t n = PyList_GET_SIZE(a.ptr());
  if (PyList_GET_SIZE(b.ptr()) != n) return false;
  for (Py_ssize_t k = 0; k < n; ++k)
    if (PyList_GET_ITEM(a.ptr(), k) != PyList_GET_ITEM(b.ptr(), k)) return false;
  return true;
}

}  // namespace

PYBIND11_MODULE(_host_ops, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const VirConvError& e) {
      PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
    }
  });
  m.attr("ABI_VERSION") = VC_ABI_VERSION;       // of the structs that are filled here
  m.attr("TORCH_VERSION") = VC_TORCH_VERSION;   // whose headers this was built against
  m.def("bind", &bind);
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  m.def("grouped_linear", &grouped_linear, py::call_guard<py::gil_scoped_release>());
  m.def("adamw", &adamw);
  m.attr("ADAMW_CAPTURED") = kCaptured;
  m.def("same_items", &same_items);
  m.def("same_objects", &same_objects);
}
