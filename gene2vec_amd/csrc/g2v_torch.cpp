// g2v_torch.cpp -- the tensor operators of libg2v as torch operators `g2v::...`
// and Python calls (gene2vec_amd/_g2v_torch.so; the public functions and their
// documentation are in gene2vec_amd/ops.py).
//
// A shell around the C ABI in three layers: the Python entry takes its arguments
// apart, the Autograd kernel records the lookup, the CUDA kernel checks the
// arguments, allocates results and workspaces on torch's allocator and enqueues
// the work on the current stream.  The layers call each other through torch's
// dispatcher, so that whatever sits in between (a tracer, a functional
// transform, a dispatch mode) sees one operator and not the empty tensors that
// it fills.  It is compiled because small calls are all host time: the same
// checks in Python cost a training step of 256 tokens 83 us, most of it in
// autograd's own thread, and a list of 600 tensors 310 us.
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>
#include <torch/version.h>

#include <cmath>
#include <cstdint>
#include <limits>
#include <stdexcept>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "g2v.h"

namespace py = pybind11;

namespace {

struct NativeError : std::runtime_error {
  int code;
  NativeError(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

[[noreturn]] void refuse(const std::string& m) { C10_THROW_ERROR(ValueError, m); }

void native(int rc) {
  if (rc == G2V_OK) return;
  const char* m = g2v_last_error();
  throw NativeError(rc, m ? m : "");
}

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return G2V_F32;
    case at::kHalf: return G2V_F16;
    case at::kBFloat16: return G2V_BF16;
    default: return -1;
  }
}

std::string name_of(at::ScalarType t) { return c10::toString(t); }

std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int device_index(const at::Tensor& t) { return t.device().index(); }

const at::Tensor& tensor(py::handle h, const char* name) {
  if (!THPVariable_Check(h.ptr()))
    refuse(std::string(name) + " must be a tensor, not " + Py_TYPE(h.ptr())->tp_name);
  return THPVariable_Unpack(h.ptr());
}

void on_gpu(const at::Tensor& t, const char* name) {
  if (!t.is_cuda() || t.layout() != at::kStrided)
    refuse(std::string(name) + " must be a dense tensor on the GPU (there is no CPU fallback)");
  if (t.is_neg()) refuse(std::string(name) + ": a lazily negated view; resolve_neg() it first");
}

void check_type(at::ScalarType t, const char* name) {
  if (type_code(t) < 0)
    refuse(std::string(name) + " must be float32, float16 or bfloat16, not " + name_of(t));
}

int id_bytes(const at::Tensor& ids) { return ids.scalar_type() == at::kInt ? 4 : 8; }

void check_ids(const at::Tensor& ids, const at::Tensor& rows) {
  on_gpu(ids, "ids");
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong)
    refuse("ids must be int32 or int64, not " + name_of(ids.scalar_type()));
  if (ids.device() != rows.device())
    refuse("ids are on " + ids.device().str() + ", the rows on " + rows.device().str());
}

at::ScalarType result_type(py::handle dtype, at::ScalarType otherwise) {
  if (dtype.is_none()) return otherwise;
  if (!THPDtype_Check(dtype.ptr())) refuse("dtype must be a torch.dtype");
  const at::ScalarType t = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
  check_type(t, "dtype");
  return t;
}

void check_scale(double scale) {
  if (!(std::fabs(scale) <= std::numeric_limits<float>::max()))
    refuse("scale must be finite in fp32, not " + std::to_string(scale));
}

// a whole number as Python gives it: int, numpy integer, 3.0
int64_t whole(py::handle h, const char* name) {
  const double d = PyFloat_AsDouble(h.ptr());  // a number: no text that holds one
  if (PyErr_Occurred()) throw py::error_already_set();
  if (d != std::floor(d) || std::fabs(d) > 9e15)
    refuse(std::string(name) + " must be a whole number, not " + std::string(py::str(h)));
  return (int64_t)d;
}

// -1, and only that, where there is none
int64_t padding_of(py::handle h) {
  if (h.is_none()) return -1;
  const int64_t pad = whole(h, "padding_idx");
  if (pad < 0) refuse("padding_idx " + std::to_string(pad) + " is negative");
  return pad;
}

void check_padding(int64_t pad, int64_t V) {
  if (pad < -1 || pad >= V)
    refuse("padding_idx " + std::to_string(pad) + " is not in [0, " + std::to_string(V) + ")");
}

// ---- the operators' handles: calls through the dispatcher ------------------------------
template <class F>
c10::TypedOperatorHandle<F> op(const char* name, const char* overload = "") {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, overload).typed<F>();
}

at::Tensor call_lookup(const at::Tensor& params, const at::Tensor& ids, double scale, int64_t pad,
                       at::ScalarType type) {
  static const auto h = op<at::Tensor(const at::Tensor&, const at::Tensor&, double, int64_t,
                                      at::ScalarType)>("g2v::embedding_lookup");
  return h.call(params, ids, scale, pad, type);
}

at::Tensor call_lookup_grad(const at::Tensor& dy, const at::Tensor& ids, int64_t V, double scale,
                            int64_t pad, at::ScalarType type) {
  static const auto h = op<at::Tensor(const at::Tensor&, const at::Tensor&, int64_t, double,
                                      int64_t, at::ScalarType)>("g2v::embedding_lookup_grad");
  return h.call(dy, ids, V, scale, pad, type);
}

at::Tensor call_norm(at::TensorList t_list) {
  static const auto h = op<at::Tensor(at::TensorList)>("g2v::global_norm");
  return h.call(t_list);
}

using Clipped = std::tuple<std::vector<at::Tensor>, at::Tensor>;

Clipped call_clip(at::TensorList t_list, double clip_norm) {
  static const auto h = op<Clipped(at::TensorList, double)>("g2v::clip_by_global_norm");
  return h.call(t_list, clip_norm);
}

at::Tensor call_clip_out(at::TensorList t_list, double clip_norm, at::TensorList out) {
  static const auto h =
      op<at::Tensor(at::TensorList, double, at::TensorList)>("g2v::clip_by_global_norm", "out");
  return h.call(t_list, clip_norm, out);
}

at::Tensor call_clip_(at::TensorList t_list, double clip_norm) {
  static const auto h = op<at::Tensor(at::TensorList, double)>("g2v::clip_by_global_norm_");
  return h.call(t_list, clip_norm);
}

// ---- the lookup --------------------------------------------------------------------------
at::Tensor lookup_cuda(const at::Tensor& params, const at::Tensor& given, double scale,
                       int64_t pad, at::ScalarType type) {
  on_gpu(params, "params");
  if (params.dim() != 2 || params.numel() == 0)
    refuse("params must be a matrix [V, D], not " + shape_of(params.sizes()));
  check_type(params.scalar_type(), "params");
  check_type(type, "dtype");
  const int64_t V = params.size(0), D = params.size(1);
  if (D > 1 && params.stride(1) != 1)
    refuse("the elements of a row of params must be contiguous");
  const int64_t ld = V > 1 ? params.stride(0) : D;
  if (ld < D) refuse("the rows of params overlap (strides " + shape_of(params.strides()) + ")");
  check_ids(given, params);
  check_scale(scale);
  check_padding(pad, V);
  const at::Tensor ids = given.contiguous();
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(D);
  at::Tensor out = at::empty(shape, params.options().dtype(type));
  native(g2v_embed_lookup(device_index(params), params.const_data_ptr(),
                          type_code(params.scalar_type()), V, D, ld, ids.const_data_ptr(),
                          id_bytes(ids), ids.numel(), (float)scale, out.mutable_data_ptr(),
                          type_code(type), stream_of(params)));
  return out;
}

at::Tensor lookup_grad_cuda(const at::Tensor& given, const at::Tensor& tokens, int64_t V,
                            double scale, int64_t pad, at::ScalarType type) {
  on_gpu(given, "dy");
  check_ids(tokens, given);
  check_type(given.scalar_type(), "dy");
  check_type(type, "dtype");
  if (given.dim() != tokens.dim() + 1 ||
      given.sizes().slice(0, tokens.dim()) != tokens.sizes() || given.size(-1) < 1)
    refuse("dy " + shape_of(given.sizes()) + " does not hold a row for each of ids " +
           shape_of(tokens.sizes()));
  if (V < 1) refuse("vocab_size must be positive, not " + std::to_string(V));
  check_scale(scale);
  check_padding(pad, V);
  const at::Tensor ids = tokens.contiguous();
  const int64_t n = ids.numel(), D = given.size(-1);
  at::Tensor dy = given.dim() == 2 ? given : given.reshape({n, D});
  int64_t ld = n > 1 ? dy.stride(0) : D;
  if ((D > 1 && dy.stride(1) != 1) || ld < D) {  // a transposed or broadcast gradient
    dy = dy.contiguous();
    ld = D;
  }
  int64_t bytes = 0;
  native(g2v_embed_grad_workspace(n, V, D, &bytes));
  at::Tensor grad = at::empty({V, D}, dy.options().dtype(type));
  at::Tensor ws = at::empty({bytes}, dy.options().dtype(at::kByte));
  native(g2v_embed_grad(device_index(dy), dy.const_data_ptr(), type_code(dy.scalar_type()), ld,
                        ids.const_data_ptr(), id_bytes(ids), n, V, D, (float)scale, pad,
                        grad.mutable_data_ptr(), type_code(type), ws.mutable_data_ptr(), bytes,
                        stream_of(dy)));
  return grad;
}

namespace ag = torch::autograd;

// A leaf's gradient is accumulated on the stream that its live graph was built
// on.  Where that is the default stream, which no capture can take in, a captured
// backward pass would end the capture, or the process: refused here, before
// anything is recorded.  The leaves are params itself or what it was computed from.
void check_capture(const at::Tensor& params) {
  const c10::DeviceGuard guard(params.device());  // the capture of its stream is asked for
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto check = [](ag::Node& leaf) {
    const auto stream = leaf.stream();
    if (stream &&
        stream->id() == c10::hip::getDefaultHIPStream(stream->device_index()).id())
      refuse("params: a graph of this leaf, or of one that it was computed from, is still alive "
             "from the default stream (a loss, say); drop it before capturing");
  };
  if (!params.grad_fn()) {
    if (const auto leaf = ag::impl::try_get_grad_accumulator(params)) check(*leaf);
    return;
  }
  std::vector<ag::Node*> todo{params.grad_fn().get()};
  std::unordered_set<ag::Node*> seen(todo.begin(), todo.end());
  while (!todo.empty()) {
    ag::Node* node = todo.back();
    todo.pop_back();
    if (dynamic_cast<ag::AccumulateGrad*>(node)) check(*node);
    for (const ag::Edge& e : node->next_edges())
      if (e.function && seen.insert(e.function.get()).second) todo.push_back(e.function.get());
  }
}

struct EmbeddingLookupBackward : public ag::Node {
  ag::SavedVariable ids;
  int64_t V = 0, D = 0, pad = -1;
  double scale = 1.0;
  at::TensorOptions table;  // type and device of the gradient

  std::string name() const override { return "EmbeddingLookupBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    ids.reset_data();
  }

  ag::variable_list apply(ag::variable_list&& dy) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const at::Tensor tokens = ids.unpack();
    if (!task_should_compute_output(0)) return {at::Tensor()};
    // in the grad mode of the pass (create_graph=True: recorded)
    const at::Tensor grad =
        dy[0].defined() ? call_lookup_grad(dy[0], tokens, V, scale, pad,
                                           c10::typeMetaToScalarType(table.dtype()))
                        : at::zeros({V, D}, table);
    return {grad};
  }
};

at::Tensor lookup_autograd(const at::Tensor& params, const at::Tensor& given, double scale,
                           int64_t pad, at::ScalarType type) {
  const at::Tensor ids = given.contiguous();
  std::shared_ptr<EmbeddingLookupBackward> node;
  if (ag::compute_requires_grad(params)) {
    check_capture(params);
    node = std::shared_ptr<EmbeddingLookupBackward>(new EmbeddingLookupBackward, ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(params));
  }
  at::Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = call_lookup(params, ids, scale, pad, type);
  }
  if (node) {
    node->ids = ag::SavedVariable(ids, false);
    node->V = params.size(0);
    node->D = params.size(1);
    node->pad = pad;
    node->scale = scale;
    node->table = params.options();
    ag::set_history(out, node);
  }
  const at::Tensor& tangent = params._fw_grad(0);  // linear in params
  if (tangent.defined())
    out._set_fw_grad(call_lookup(tangent, ids, scale, pad, type), 0, false);
  return out;
}

at::Tensor lookup_grad_autograd(const at::Tensor& dy, const at::Tensor& ids, int64_t V,
                                double scale, int64_t pad, at::ScalarType type) {
  at::Tensor grad;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    grad = call_lookup_grad(dy, ids, V, scale, pad, type);
  }
  if (ag::compute_requires_grad(dy))  // whoever differentiates the gradient is told
    ag::set_history(grad, std::make_shared<ag::Error>(
                              "embedding_lookup is differentiable once, not twice",
                              ag::collect_next_edges(dy)));
  const at::Tensor& tangent = dy._fw_grad(0);  // linear in dy
  if (tangent.defined())
    grad._set_fw_grad(call_lookup_grad(tangent, ids, V, scale, pad, type), 0, false);
  return grad;
}

at::Tensor embedding_lookup(py::handle params_, py::handle ids_, double scale,
                            py::handle padding_idx, py::handle dtype) {
  const at::Tensor& params = tensor(params_, "params");
  on_gpu(params, "params");
  const at::Tensor& ids = tensor(ids_, "ids");
  on_gpu(ids, "ids");
  const at::ScalarType type = result_type(dtype, params.scalar_type());
  const int64_t pad = padding_of(padding_idx);
  py::gil_scoped_release released;
  return call_lookup(params, ids, scale, pad, type);
}

at::Tensor embedding_lookup_grad(py::handle dy_, py::handle ids_, py::handle vocab_size,
                                 double scale, py::handle padding_idx, py::handle dtype) {
  const at::Tensor& dy = tensor(dy_, "dy");
  on_gpu(dy, "dy");
  if (ag::compute_requires_grad(dy))
    refuse("embedding_lookup_grad is not differentiable: pass a dy that requires no gradient, or "
           "call it under no_grad()");
  const at::Tensor& ids = tensor(ids_, "ids");
  on_gpu(ids, "ids");
  const at::ScalarType type = result_type(dtype, dy.scalar_type());
  const int64_t V = whole(vocab_size, "vocab_size"), pad = padding_of(padding_idx);
  py::gil_scoped_release released;
  return call_lookup_grad(dy, ids, V, scale, pad, type);
}

// ---- norm and clipping -------------------------------------------------------------------
// its elements fill one stretch of memory, each once, in whatever order
bool is_dense(const at::Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

// a list of tensors as the C entries take it
struct List {
  std::vector<const void*> src;
  std::vector<int64_t> numel;
  std::vector<int32_t> types;
  at::Tensor norm, ws;
  int device = 0;

  List(at::TensorList tensors, const char* what) {
    const size_t n = tensors.size();
    if (!n) refuse(std::string(what) + ": the list holds no tensor");
    src.reserve(n);
    numel.reserve(n);
    types.reserve(n);
    on_gpu(tensors[0], what);
    const c10::Device where = tensors[0].device();
    for (const at::Tensor& t : tensors) {  // other layouts have no kernel to come here by
      if (t.device() != where)
        refuse(std::string(what) + ": tensors on " + where.str() + " and " + t.device().str());
      const int type = type_code(t.scalar_type());
      if (type < 0)
        refuse(std::string(what) + ": tensors must be float32, float16 or bfloat16, not " +
               name_of(t.scalar_type()));
      if (!is_dense(t))
        refuse(std::string(what) + ": the elements of a tensor must be dense in memory (shape " +
               shape_of(t.sizes()) + ", strides " + shape_of(t.strides()) + ")");
      src.push_back(t.const_data_ptr());
      numel.push_back(t.numel());
      types.push_back(type);
    }
    int64_t bytes = 0;
    native(g2v_global_norm_workspace((int64_t)n, &bytes));
    norm = at::empty({}, tensors[0].options().dtype(at::kFloat));
    ws = at::empty({bytes}, tensors[0].options().dtype(at::kByte));
    device = device_index(norm);
  }
};

at::Tensor norm_cuda(at::TensorList t_list) {
  const List l(t_list, "global_norm");
  native(g2v_global_norm(l.device, l.src.data(), l.numel.data(), l.types.data(),
                         (int64_t)l.src.size(), l.norm.mutable_data_ptr<float>(),
                         l.ws.mutable_data_ptr(), l.ws.numel(), stream_of(l.norm)));
  return l.norm;
}

// t_list into outs, of the same shapes, types and strides; outs may be t_list
at::Tensor clip_into(at::TensorList t_list, at::TensorList outs, double clip_norm,
                     const char* what) {
  if (!(clip_norm > 0.0 && clip_norm < std::numeric_limits<double>::infinity()))
    refuse(std::string(what) + ": clip_norm must be positive and finite, not " +
           std::to_string(clip_norm));
  const List l(t_list, what);
  std::vector<void*> dst;
  dst.reserve(outs.size());
  for (const at::Tensor& o : outs) {
    if (o.is_inference() && !c10::InferenceMode::is_enabled())
      refuse(std::string(what) + ": an inference tensor is written in inference mode only");
    dst.push_back(o.mutable_data_ptr());
  }
  const int rc = g2v_clip_global_norm(
      l.device, l.src.data(), dst.data(), l.numel.data(), l.types.data(), (int64_t)l.src.size(),
      clip_norm, l.norm.mutable_data_ptr<float>(), l.ws.mutable_data_ptr(), l.ws.numel(),
      stream_of(l.norm));
  if (rc == G2V_EINVAL) refuse(g2v_last_error());  // tensors that overlap
  native(rc);
  for (const at::Tensor& o : outs)  // autograd learns that they changed
    if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  return l.norm;
}

Clipped clip_cuda(at::TensorList t_list, double clip_norm) {
  std::vector<at::Tensor> outs;
  outs.reserve(t_list.size());
  for (const at::Tensor& t : t_list) outs.push_back(at::empty_like(t));
  at::Tensor norm = clip_into(t_list, outs, clip_norm, "clip_by_global_norm");
  return {std::move(outs), std::move(norm)};
}

at::Tensor clip_out_cuda(at::TensorList t_list, double clip_norm, at::TensorList out) {
  const char* what = "clip_by_global_norm";
  if (out.size() != t_list.size())
    refuse(std::string(what) + ": " + std::to_string(out.size()) + " outputs for " +
           std::to_string(t_list.size()) + " tensors");
  for (size_t i = 0; i < out.size(); ++i) {
    const at::Tensor &o = out[i], &t = t_list[i];
    if (o.sizes() != t.sizes() || o.scalar_type() != t.scalar_type() ||
        o.device() != t.device() ||
        !((o.is_contiguous() && t.is_contiguous()) || o.strides() == t.strides()))
      refuse(std::string(what) +
             ": an output differs from its tensor in shape, type, strides or device");
  }
  return clip_into(t_list, out, clip_norm, what);
}

at::Tensor clip_inplace_cuda(at::TensorList t_list, double clip_norm) {
  return clip_into(t_list, t_list, clip_norm, "clip_by_global_norm_");
}

// none of these has a derivative, backward or forward
void no_derivative(at::TensorList tensors, const char* what) {
  const bool grad = at::GradMode::is_enabled();
  for (const at::Tensor& t : tensors) {
    if (!t.unsafeGetTensorImpl()->autograd_meta()) continue;  // plain data, as most are
    if (grad && t.requires_grad())
      refuse(std::string(what) +
             " is not differentiable: pass gradients, or call it under no_grad()");
    if (t._fw_grad(0).defined())
      refuse(std::string(what) + " is not differentiable: a tensor has a forward-mode tangent");
  }
}

at::Tensor norm_autograd(at::TensorList t_list) {
  no_derivative(t_list, "global_norm");
  at::AutoDispatchBelowADInplaceOrView below;
  return call_norm(t_list);
}

Clipped clip_autograd(at::TensorList t_list, double clip_norm) {
  no_derivative(t_list, "clip_by_global_norm");
  at::AutoDispatchBelowADInplaceOrView below;
  return call_clip(t_list, clip_norm);
}

at::Tensor clip_out_autograd(at::TensorList t_list, double clip_norm, at::TensorList out) {
  no_derivative(t_list, "clip_by_global_norm");
  no_derivative(out, "clip_by_global_norm: out");
  at::AutoDispatchBelowADInplaceOrView below;
  return call_clip_out(t_list, clip_norm, out);
}

at::Tensor clip_inplace_autograd(at::TensorList t_list, double clip_norm) {
  no_derivative(t_list, "clip_by_global_norm_");
  at::AutoDispatchBelowADInplaceOrView below;
  return call_clip_(t_list, clip_norm);
}

std::vector<py::object> items_of(py::handle seq, const char* what) {
  std::vector<py::object> v;
  if (THPVariable_Check(seq.ptr())) refuse(std::string(what) + ": a list of tensors is needed");
  for (py::handle h : py::iter(seq)) v.push_back(py::reinterpret_borrow<py::object>(h));
  return v;
}

// the tensors among them, without the None entries
std::vector<at::Tensor> tensors_of(const std::vector<py::object>& items, const char* what) {
  std::vector<at::Tensor> v;
  v.reserve(items.size());
  for (const py::object& o : items) {
    if (o.is_none()) continue;
    if (!THPVariable_Check(o.ptr()))
      refuse(std::string(what) + ": the list must hold tensors, not " + Py_TYPE(o.ptr())->tp_name);
    v.push_back(THPVariable_Unpack(o.ptr()));
    on_gpu(v.back(), what);
  }
  if (v.empty()) refuse(std::string(what) + ": the list holds no tensor");
  return v;
}

at::Tensor global_norm(py::handle t_list) {
  const std::vector<at::Tensor> tensors = tensors_of(items_of(t_list, "global_norm"),
                                                     "global_norm");
  py::gil_scoped_release released;
  return call_norm(tensors);
}

py::object wrap(at::Tensor t);

py::tuple clip_by_global_norm(py::handle t_list, double clip_norm, py::handle out) {
  const char* what = "clip_by_global_norm";
  const std::vector<py::object> items = items_of(t_list, what);
  const std::vector<at::Tensor> tensors = tensors_of(items, what);
  py::list result;
  at::Tensor norm;
  if (out.is_none()) {
    std::vector<at::Tensor> outs;
    {
      py::gil_scoped_release released;
      std::tie(outs, norm) = call_clip(tensors, clip_norm);
    }
    size_t k = 0;
    for (const py::object& o : items) result.append(o.is_none() ? py::none() : wrap(outs[k++]));
  } else {
    const std::vector<py::object> given = items_of(out, what);
    if (given.size() != items.size())
      refuse(std::string(what) + ": " + std::to_string(given.size()) + " outputs for " +
             std::to_string(items.size()) + " tensors");
    std::vector<at::Tensor> outs;
    outs.reserve(tensors.size());
    for (size_t i = 0; i < items.size(); ++i) {
      if (!items[i].is_none()) {
        outs.push_back(tensor(given[i], "clip_by_global_norm: out"));
        on_gpu(outs.back(), "clip_by_global_norm: out");
      }
      result.append(items[i].is_none() ? py::none() : given[i]);
    }
    py::gil_scoped_release released;
    norm = call_clip_out(tensors, clip_norm, outs);
  }
  return py::make_tuple(result, wrap(norm));
}

at::Tensor clip_by_global_norm_(py::handle t_list, double clip_norm) {
  const char* what = "clip_by_global_norm_";
  const std::vector<at::Tensor> tensors = tensors_of(items_of(t_list, what), what);
  py::gil_scoped_release released;
  return call_clip_(tensors, clip_norm);
}

py::object wrap(at::Tensor t) {
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t)));
}

}  // namespace

TORCH_LIBRARY(g2v, m) {
  m.def("embedding_lookup(Tensor params, Tensor ids, float scale, int padding_idx, "
        "ScalarType dtype) -> Tensor");
  m.def("embedding_lookup_grad(Tensor dy, Tensor ids, int vocab_size, float scale, "
        "int padding_idx, ScalarType dtype) -> Tensor");
  m.def("global_norm(Tensor[] t_list) -> Tensor");
  m.def("clip_by_global_norm(Tensor[] t_list, float clip_norm) -> (Tensor[], Tensor)");
  m.def("clip_by_global_norm.out(Tensor[] t_list, float clip_norm, *, Tensor(a!)[] out) -> Tensor");
  m.def("clip_by_global_norm_(Tensor(a!)[] t_list, float clip_norm) -> Tensor");
}

TORCH_LIBRARY_IMPL(g2v, CUDA, m) {
  m.impl("embedding_lookup", &lookup_cuda);
  m.impl("embedding_lookup_grad", &lookup_grad_cuda);
  m.impl("global_norm", &norm_cuda);
  m.impl("clip_by_global_norm", &clip_cuda);
  m.impl("clip_by_global_norm.out", &clip_out_cuda);
  m.impl("clip_by_global_norm_", &clip_inplace_cuda);
}

TORCH_LIBRARY_IMPL(g2v, Autograd, m) {
  m.impl("embedding_lookup", &lookup_autograd);
  m.impl("embedding_lookup_grad", &lookup_grad_autograd);
  m.impl("global_norm", &norm_autograd);
  m.impl("clip_by_global_norm", &clip_autograd);
  m.impl("clip_by_global_norm.out", &clip_out_autograd);
  m.impl("clip_by_global_norm_", &clip_inplace_autograd);
}

PYBIND11_MODULE(_g2v_torch, m) {
  // refusals as ValueError; the library's errors as the ctypes layer's
  // subclass of RuntimeError, with the code
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NativeError& e) {
      py::object type = py::module_::import("gene2vec_amd._native").attr("G2VError");
      PyErr_SetObject(type.ptr(), type(e.code, std::string(e.what())).ptr());
    } catch (const c10::ValueError& e) {
      PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
    }
  });
  // what this file was compiled against, not what libg2v answers at run time
  m.def("abi_version", [] { return G2V_ABI_VERSION; });
  m.def("torch_version", [] { return TORCH_VERSION; });
  m.def("embedding_lookup", [](py::handle p, py::handle i, double s, py::handle pad,
                               py::handle d) { return wrap(embedding_lookup(p, i, s, pad, d)); });
  m.def("embedding_lookup_grad",
        [](py::handle dy, py::handle i, py::handle v, double s, py::handle pad, py::handle d) {
          return wrap(embedding_lookup_grad(dy, i, v, s, pad, d));
        });
  m.def("global_norm", [](py::handle t) { return wrap(global_norm(t)); });
  m.def("clip_by_global_norm", &clip_by_global_norm);
  m.def("clip_by_global_norm_",
        [](py::handle t, double c) { return wrap(clip_by_global_norm_(t, c)); });
}
