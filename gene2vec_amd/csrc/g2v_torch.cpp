// g2v_torch.cpp -- the tensor operators of libg2v as Python calls on torch
// tensors (gene2vec_amd/_g2v_torch.so; the public functions and their
// documentation are in gene2vec_amd/ops.py).
//
// A shell around the C ABI: it checks the arguments, allocates results and
// workspaces on torch's allocator, finds the current stream and records the
// lookup for autograd.  It is compiled because small calls are all host time:
// the same checks in Python cost a training step of 256 tokens 83 us, most of
// it in autograd's own thread, and a list of 600 tensors 310 us.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <limits>
#include <stdexcept>
#include <string>
#include <vector>

#include "g2v.h"

namespace py = pybind11;

namespace {

struct NativeError : std::runtime_error {
  int code;
  NativeError(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

[[noreturn]] void refuse(const std::string& m) { throw py::value_error(m); }

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

double scale_of(double scale) {
  if (!(std::fabs(scale) <= std::numeric_limits<float>::max()))
    refuse("scale must be finite in fp32, not " + std::to_string(scale));
  return scale;
}

// a whole number as Python gives it: int, numpy integer, 3.0
int64_t whole(py::handle h, const char* name) {
  const double d = py::cast<double>(py::float_(py::reinterpret_borrow<py::object>(h)));
  if (d != std::floor(d) || std::fabs(d) > 9e15)
    refuse(std::string(name) + " must be a whole number, not " + std::string(py::str(h)));
  return (int64_t)d;
}

int64_t padding_of(py::handle h, int64_t V) {
  if (h.is_none()) return -1;
  const int64_t pad = whole(h, "padding_idx");
  if (pad < 0 || pad >= V)
    refuse("padding_idx " + std::to_string(pad) + " is not in [0, " + std::to_string(V) + ")");
  return pad;
}

at::Tensor lookup(const at::Tensor& params, const at::Tensor& ids, int64_t ld, double scale,
                  at::ScalarType type) {
  const int64_t V = params.size(0), D = params.size(1);
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(D);
  at::Tensor out = at::empty(shape, params.options().dtype(type));
  native(g2v_embed_lookup(device_index(params), params.const_data_ptr(),
                          type_code(params.scalar_type()), V, D, ld, ids.const_data_ptr(),
                          id_bytes(ids), ids.numel(), (float)scale, out.mutable_data_ptr(),
                          type_code(type), stream_of(params)));
  return out;
}

at::Tensor lookup_grad(at::Tensor dy, const at::Tensor& ids, int64_t V, int64_t D, double scale,
                       int64_t pad, at::ScalarType type) {
  const int64_t n = ids.numel();
  dy = dy.resolve_neg();
  if (dy.dim() != 2) dy = dy.reshape({n, D});
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
// anything is recorded.
void check_capture(const at::Tensor& params) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const std::shared_ptr<ag::Node> node = ag::impl::try_get_grad_accumulator(params);
  if (!node) return;
  const auto stream = node->stream();
  if (stream && stream->id() == c10::hip::getDefaultHIPStream(params.device().index()).id())
    refuse("params: a graph of this leaf from the default stream is still alive (its loss, "
           "say); drop it before capturing");
}

class EmbeddingLookup : public ag::Function<EmbeddingLookup> {
 public:
  static at::Tensor forward(ag::AutogradContext* ctx, const at::Tensor& params,
                            const at::Tensor& ids, int64_t ld, double scale, int64_t pad,
                            int64_t type) {
    ctx->save_for_backward({ids});
    ctx->saved_data["V"] = params.size(0);
    ctx->saved_data["D"] = params.size(1);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    ctx->saved_data["type"] = (int64_t)params.scalar_type();
    return lookup(params, ids, ld, scale, (at::ScalarType)type);
  }

  static ag::variable_list backward(ag::AutogradContext* ctx, ag::variable_list dy) {
    const bool again = at::GradMode::is_enabled();
    at::Tensor grad;
    {
      at::NoGradGuard no_grad;
      auto& d = ctx->saved_data;
      grad = lookup_grad(dy[0].detach(), ctx->get_saved_variables()[0], d["V"].toInt(),
                         d["D"].toInt(), d["scale"].toDouble(), d["pad"].toInt(),
                         (at::ScalarType)d["type"].toInt());
    }
    if (again) {  // create_graph=True: whoever differentiates the gradient is told
      auto error = std::make_shared<ag::DelayedError>(
          "embedding_lookup is differentiable once, not twice", 1);
      grad = (*error)({grad.set_requires_grad(true)})[0];
    }
    return {grad, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding_lookup(py::handle params_, py::handle ids_, double scale,
                            py::handle padding_idx, py::handle dtype) {
  const at::Tensor& params = tensor(params_, "params");
  on_gpu(params, "params");
  if (params.dim() != 2 || params.numel() == 0)
    refuse("params must be a matrix [V, D], not " + shape_of(params.sizes()));
  check_type(params.scalar_type(), "params");
  const int64_t V = params.size(0), D = params.size(1);
  if (D > 1 && params.stride(1) != 1)
    refuse("the elements of a row of params must be contiguous");
  const int64_t ld = V > 1 ? params.stride(0) : D;
  if (ld < D) refuse("the rows of params overlap (strides " + shape_of(params.strides()) + ")");
  const at::Tensor& given = tensor(ids_, "ids");
  check_ids(given, params);
  const at::ScalarType type = result_type(dtype, params.scalar_type());
  scale_of(scale);
  const int64_t pad = padding_of(padding_idx, V);
  py::gil_scoped_release released;
  const at::Tensor ids = given.contiguous();
  if (params.requires_grad() && at::GradMode::is_enabled()) {
    check_capture(params);
    return EmbeddingLookup::apply(params, ids, ld, scale, pad, (int64_t)type);
  }
  return lookup(params, ids, ld, scale, type);
}

at::Tensor embedding_lookup_grad(py::handle dy_, py::handle ids_, py::handle vocab_size,
                                 double scale, py::handle padding_idx, py::handle dtype) {
  const at::Tensor& dy = tensor(dy_, "dy");
  on_gpu(dy, "dy");
  const at::Tensor& ids = tensor(ids_, "ids");
  check_ids(ids, dy);
  check_type(dy.scalar_type(), "dy");
  if (dy.dim() != ids.dim() + 1 || dy.sizes().slice(0, ids.dim()) != ids.sizes() ||
      dy.size(-1) < 1)
    refuse("dy " + shape_of(dy.sizes()) + " does not hold a row for each of ids " +
           shape_of(ids.sizes()));
  const int64_t V = whole(vocab_size, "vocab_size");
  if (V < 1) refuse("vocab_size must be positive, not " + std::to_string(V));
  const at::ScalarType type = result_type(dtype, dy.scalar_type());
  scale_of(scale);
  const int64_t pad = padding_of(padding_idx, V);
  py::gil_scoped_release released;
  at::NoGradGuard no_grad;
  return lookup_grad(dy.detach(), ids.contiguous(), V, dy.size(-1), scale, pad, type);
}

// its elements fill one stretch of memory, each once, in whatever order
bool is_dense(const at::Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

// a list of tensors as the C entries take it, without its None entries
struct List {
  std::vector<at::Tensor> tensors;
  std::vector<const void*> src;
  std::vector<int64_t> numel;
  std::vector<int32_t> types;
  size_t size() const { return tensors.size(); }
};

std::vector<py::object> items_of(py::handle seq, const char* what) {
  std::vector<py::object> v;
  if (THPVariable_Check(seq.ptr())) refuse(std::string(what) + ": a list of tensors is needed");
  for (py::handle h : py::iter(seq)) v.push_back(py::reinterpret_borrow<py::object>(h));
  return v;
}

List list_of(const std::vector<py::object>& items, const char* what) {
  List l;
  const size_t n = items.size();
  l.tensors.reserve(n);
  l.src.reserve(n);
  l.numel.reserve(n);
  l.types.reserve(n);
  const bool grad = at::GradMode::is_enabled();
  for (const py::object& o : items) {
    if (o.is_none()) continue;
    if (!THPVariable_Check(o.ptr()))
      refuse(std::string(what) + ": the list must hold tensors, not " + Py_TYPE(o.ptr())->tp_name);
    const at::Tensor& t = THPVariable_Unpack(o.ptr());
    on_gpu(t, what);
    if (l.size() && t.device() != l.tensors[0].device())
      refuse(std::string(what) + ": tensors on " + l.tensors[0].device().str() + " and " +
             t.device().str());
    const int type = type_code(t.scalar_type());
    if (type < 0)
      refuse(std::string(what) + ": tensors must be float32, float16 or bfloat16, not " +
             name_of(t.scalar_type()));
    if (grad && t.requires_grad())
      refuse(std::string(what) +
             " is not differentiable: pass gradients, or call it under no_grad()");
    if (!is_dense(t))
      refuse(std::string(what) + ": the elements of a tensor must be dense in memory (shape " +
             shape_of(t.sizes()) + ", strides " + shape_of(t.strides()) + ")");
    l.tensors.push_back(t);
    l.src.push_back(t.const_data_ptr());
    l.numel.push_back(t.numel());
    l.types.push_back(type);
  }
  if (!l.size()) refuse(std::string(what) + ": the list holds no tensor");
  return l;
}

at::Tensor norm_workspace(const List& l) {
  int64_t bytes = 0;
  native(g2v_global_norm_workspace((int64_t)l.size(), &bytes));
  return at::empty({bytes}, l.tensors[0].options().dtype(at::kByte));
}

at::Tensor global_norm(py::handle t_list) {
  const std::vector<py::object> items = items_of(t_list, "global_norm");
  const List l = list_of(items, "global_norm");
  py::gil_scoped_release released;
  at::Tensor norm = at::empty({}, l.tensors[0].options().dtype(at::kFloat));
  at::Tensor ws = norm_workspace(l);
  native(g2v_global_norm(device_index(norm), l.src.data(), l.numel.data(), l.types.data(),
                         (int64_t)l.size(), norm.mutable_data_ptr<float>(), ws.mutable_data_ptr(),
                         ws.numel(), stream_of(norm)));
  return norm;
}

at::Tensor clip(const List& l, const std::vector<at::Tensor>& outs, double clip_norm,
                const char* what) {
  if (!(clip_norm > 0.0 && clip_norm < std::numeric_limits<double>::infinity()))
    refuse(std::string(what) + ": clip_norm must be positive and finite, not " +
           std::to_string(clip_norm));
  std::vector<void*> dst;
  dst.reserve(outs.size());
  for (const at::Tensor& o : outs) {
    if (o.is_inference() && !c10::InferenceMode::is_enabled())
      refuse(std::string(what) + ": an inference tensor is written in inference mode only");
    dst.push_back(o.mutable_data_ptr());
  }
  at::Tensor norm = at::empty({}, l.tensors[0].options().dtype(at::kFloat));
  at::Tensor ws = norm_workspace(l);
  const int rc = g2v_clip_global_norm(
      device_index(norm), l.src.data(), dst.data(), l.numel.data(), l.types.data(),
      (int64_t)l.size(), clip_norm, norm.mutable_data_ptr<float>(), ws.mutable_data_ptr(),
      ws.numel(), stream_of(norm));
  if (rc == G2V_EINVAL) refuse(g2v_last_error());  // tensors that overlap
  native(rc);
  for (const at::Tensor& o : outs)  // autograd learns that they changed
    if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
  return norm;
}

py::tuple clip_by_global_norm(py::handle t_list, double clip_norm, py::handle out) {
  const char* what = "clip_by_global_norm";
  const std::vector<py::object> items = items_of(t_list, what);
  const List l = list_of(items, what);
  std::vector<at::Tensor> outs;
  outs.reserve(l.size());
  py::list result;
  if (out.is_none()) {
    for (const at::Tensor& t : l.tensors) outs.push_back(at::empty_like(t));
    size_t k = 0;
    for (const py::object& o : items) {
      if (o.is_none()) result.append(py::none());
      else result.append(py::reinterpret_steal<py::object>(THPVariable_Wrap(outs[k++])));
    }
  } else {
    const std::vector<py::object> given = items_of(out, what);
    if (given.size() != items.size())
      refuse(std::string(what) + ": " + std::to_string(given.size()) + " outputs for " +
             std::to_string(items.size()) + " tensors");
    const bool grad = at::GradMode::is_enabled();
    for (size_t i = 0; i < items.size(); ++i) {
      if (items[i].is_none()) {
        result.append(py::none());
        continue;
      }
      const at::Tensor& t = l.tensors[outs.size()];
      const at::Tensor& o = tensor(given[i], "clip_by_global_norm: out");
      on_gpu(o, "clip_by_global_norm: out");
      if (o.sizes() != t.sizes() || o.scalar_type() != t.scalar_type() ||
          o.device() != t.device() ||
          !((o.is_contiguous() && t.is_contiguous()) || o.strides() == t.strides()))
        refuse(std::string(what) +
               ": an output differs from its tensor in shape, type, strides or device");
      if (grad && o.requires_grad())
        refuse(std::string(what) + ": an output requires a gradient");
      outs.push_back(o);
      result.append(given[i]);
    }
  }
  at::Tensor norm;
  {
    py::gil_scoped_release released;
    norm = clip(l, outs, clip_norm, what);
  }
  return py::make_tuple(result, py::reinterpret_steal<py::object>(THPVariable_Wrap(norm)));
}

at::Tensor clip_by_global_norm_(py::handle t_list, double clip_norm) {
  const std::vector<py::object> items = items_of(t_list, "clip_by_global_norm_");
  const List l = list_of(items, "clip_by_global_norm_");
  py::gil_scoped_release released;
  return clip(l, l.tensors, clip_norm, "clip_by_global_norm_");
}

py::object wrap(at::Tensor t) {
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t)));
}

}  // namespace

PYBIND11_MODULE(_g2v_torch, m) {
  // RuntimeError's subclass of the ctypes layer, with the code
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NativeError& e) {
      py::object type = py::module_::import("gene2vec_amd._native").attr("G2VError");
      PyErr_SetObject(type.ptr(), type(e.code, std::string(e.what())).ptr());
    }
  });
  m.def("abi_version", &g2v_abi_version);
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
