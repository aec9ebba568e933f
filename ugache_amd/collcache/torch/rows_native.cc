// The calls of collcache.torch.rows: checks of the tensors, memory for the outputs, and the launch through the C-ABI of
// include/ugache_hip.h, compiled because a call in Python costs more than the kernels of a decoding step take (one launch, us per
// call in Python / here: sort of one token's assignments 11 / 5, dispatch 9 / 4, combine with its gradients 29 / 11).
//
// Tensors are torch's own (ATen); the raw stream comes from torch through its Python function, so that no HIP header is
// needed.  Built by python -m ugache_amd.build; collcache.torch.rows is the public face and documents the calls.
#include <ATen/ATen.h>
#include <ATen/core/DimVector.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <iterator>
#include <string>
#include <vector>

#include "ugache_hip.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using c10::ScalarType;

PyObject *g_raw_stream = nullptr;  // torch._C._cuda_getCurrentRawStream, for the life of the process
PyObject *g_launch_error = nullptr;

int ElemOf(const Tensor &t) {  // 0: none of the three
  switch (t.scalar_type()) {
    case ScalarType::Float: return 4;
    case ScalarType::Half: return 2;
    case ScalarType::BFloat16: return UGK_ELEM_BF16;
    default: return 0;
  }
}
bool IsInt(const Tensor &t) { return t.scalar_type() == ScalarType::Int || t.scalar_type() == ScalarType::Long; }

// The operators have no forward-mode derivative: a tangent is refused instead of left out of the result, which would make the
// derivative zero without a word.  (Not where torch has forward mode switched off: inside a Function that brings its own.)
void NoTangent(const char *what, const Tensor &t) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined()) return;
  PyErr_SetString(PyExc_NotImplementedError,
                  (std::string(what) + " has a tangent: the operators on rows have no forward-mode derivative").c_str());
  throw py::error_already_set();
}

enum Kind { kRowsKind, kIntKind, kInt32Kind };
Tensor Unpack(const char *what, py::handle h, Kind kind, int dev = -1) {
  const char *types = kind == kRowsKind ? "float32, float16, bfloat16" : kind == kIntKind ? "int32, int64" : "int32";
  if (!THPVariable_Check(h.ptr())) throw py::type_error(std::string(what) + " must be a GPU tensor of " + types);
  const Tensor &t = THPVariable_Unpack(h.ptr());
  NoTangent(what, t);
  const bool right = kind == kRowsKind ? ElemOf(t) != 0 : kind == kIntKind ? IsInt(t) : t.scalar_type() == ScalarType::Int;
  if (!t.is_cuda() || t.layout() != c10::kStrided || !right) throw py::type_error(std::string(what) + " must be a GPU tensor of " + types);
  if (dev >= 0 && t.get_device() != dev) throw py::value_error(std::string(what) + " must be on the GPU of the other tensors");
  return t.is_neg() ? t.resolve_neg() : t;  // memory that torch holds negated until it is read
}

// enqueues on torch's current stream of GPU `dev`, which is the current device while the call runs
class On {
 public:
  explicit On(const Tensor &t) : _guard(t.device()) {
    py::object dev = py::reinterpret_steal<py::object>(PyLong_FromLong(t.get_device()));
    py::object raw = py::reinterpret_steal<py::object>(PyObject_CallOneArg(g_raw_stream, dev.ptr()));
    if (!raw) throw py::error_already_set();
    stream = PyLong_AsVoidPtr(raw.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
  }
  void *stream;

 private:
  c10::DeviceGuard _guard;
};
void Launched(int rc) {
  if (rc == 0) return;
  PyErr_SetString(g_launch_error, ugk_last_error());
  throw py::error_already_set();
}

// rows of at least one element: a run of elements each, in ascending order of memory; a copy where they are not
struct Rows {
  Tensor t;
  int64_t n, dim, stride;
  int elem;
};
Rows RowsOf(const char *what, py::handle h, int dev = -1) {
  Tensor t = Unpack(what, h, kRowsKind, dev);
  if (t.dim() < 1 || t.size(-1) < 1) throw py::value_error(std::string(what) + " must be rows of at least one element");
  if (t.dim() != 2) t = t.reshape({-1, t.size(-1)});
  int64_t n = t.size(0);
  const int64_t dim = t.size(1);
  if ((dim > 1 && t.stride(1) != 1) || (n > 1 && t.stride(0) < dim)) t = t.contiguous();
  const int64_t stride = n > 1 ? t.stride(0) : dim;
  const int elem = ElemOf(t);
  return Rows{std::move(t), n, dim, stride, elem};
}

struct Order {
  Tensor slot, offsets;
  int64_t tokens, top, n;
  const int32_t *live;
};
Order OrderOf(py::handle slot_h, py::handle offsets_h, int dev) {
  Order o;
  o.slot = Unpack("order.slot", slot_h, kInt32Kind, dev).contiguous();
  o.offsets = Unpack("order.offsets", offsets_h, kInt32Kind, dev).contiguous();
  if (o.slot.dim() < 1 || o.slot.dim() > 2 || (o.slot.dim() == 2 && o.slot.size(1) < 1) || o.offsets.dim() != 1 || o.offsets.numel() < 2)
    throw py::value_error("order must be what coll_torch_expert_sort returned");
  o.tokens = o.slot.size(0);
  o.top = o.slot.dim() == 2 ? o.slot.size(1) : 1;
  o.n = o.slot.numel();
  o.live = o.offsets.data_ptr<int32_t>() + (o.offsets.numel() - 1);
  return o;
}

// sizes without those of one, which say nothing of the order
at::DimVector Wide(at::IntArrayRef sizes) {
  at::DimVector out;
  std::copy_if(sizes.begin(), sizes.end(), std::back_inserter(out), [](int64_t n) { return n != 1; });
  return out;
}

struct Weights {
  Tensor t;
  const void *data = nullptr;
  int elem = 4;
};
Weights WeightsOf(py::handle h, const Order &o, int dev) {
  Weights w;
  if (h.is_none()) return w;
  w.t = Unpack("weights", h, kRowsKind, dev).contiguous();
  if (w.t.numel() != o.n)
    throw py::value_error(std::to_string(w.t.numel()) + " weights for " + std::to_string(o.n) + " assignments");
  // one after the other, or those of a token beside one another; any other shape has them in another order
  const at::DimVector wide = Wide(w.t.sizes());
  if (o.n && wide.size() > 1 && o.top > 1 && wide.back() != o.top)
    throw py::value_error("weights must be shaped [tokens, top_k] or [tokens * top_k]: the last size is " + std::to_string(wide.back()) +
                          ", top_k " + std::to_string(o.top));
  w.data = w.t.data_ptr();
  w.elem = ElemOf(w.t);
  return w;
}

Tensor NewRows(int64_t n, const Rows &like) { return at::empty({n, like.dim}, like.t.options()); }
Tensor NewInts(at::IntArrayRef sizes, const Tensor &like) { return at::empty(sizes, like.options().dtype(at::kInt)); }
// bytes of scratch memory, none where none are needed
Tensor Scratch(size_t nbytes, const Tensor &like) {
  return nbytes ? at::empty({(int64_t)nbytes}, like.options().dtype(at::kByte)) : Tensor();
}
void *Data(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
py::object Wrap(Tensor t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t))); }

py::tuple ExpertSort(py::handle ids_h, int64_t num_experts) {
  Tensor ids = Unpack("expert_ids", ids_h, kIntKind);
  if (num_experts < 1 || num_experts > 1024)
    throw py::value_error("num_experts must be 1 to 1024, got " + std::to_string(num_experts));
  if (ids.dim() < 1 || ids.dim() > 2 || (ids.dim() == 2 && ids.size(1) < 1))
    throw py::value_error("expert_ids must be [tokens, top_k] or [tokens]");
  ids = ids.contiguous();
  const int64_t n = ids.numel();
  if (n >= (int64_t)1 << 31) throw py::value_error(std::to_string(n) + " assignments are more than positions of 31 bits name");
  const On on(ids);
  Tensor slot = NewInts(ids.sizes(), ids), src = NewInts({n}, ids), offsets = NewInts({num_experts + 1}, ids);
  const size_t nbytes = ugk_expert_sort_workspace_bytes((size_t)n, (uint32_t)num_experts);
  const Tensor scratch = Scratch(nbytes, ids);
  int32_t *s = slot.data_ptr<int32_t>(), *p = src.data_ptr<int32_t>(), *o = offsets.data_ptr<int32_t>();
  if (ids.scalar_type() == ScalarType::Long)
    Launched(ugk_expert_sort_i64(ids.data_ptr<int64_t>(), (size_t)n, (uint32_t)num_experts, s, p, o, Data(scratch), nbytes, on.stream));
  else
    Launched(ugk_expert_sort_i32(ids.data_ptr<int32_t>(), (size_t)n, (uint32_t)num_experts, s, p, o, Data(scratch), nbytes, on.stream));
  return py::make_tuple(Wrap(std::move(slot)), Wrap(std::move(src)), Wrap(std::move(offsets)));
}

py::object Dispatch(py::handle x_h, py::handle slot_h, py::handle offsets_h) {
  const Rows x = RowsOf("x", x_h);
  const Order o = OrderOf(slot_h, offsets_h, x.t.get_device());
  if (x.n != o.tokens)
    throw py::value_error(std::to_string(x.n) + " rows, but the order is of " + std::to_string(o.tokens) + " tokens");
  const On on(x.t);
  Tensor rows = NewRows(o.n, x);
  Launched(ugk_expert_dispatch(x.t.data_ptr(), (size_t)x.stride, o.slot.data_ptr<int32_t>(), o.live, (size_t)o.tokens, (uint32_t)o.top,
                               (size_t)x.dim, x.elem, rows.data_ptr(), on.stream));
  return Wrap(std::move(rows));
}

py::object Combine(const char *what, py::handle rows_h, py::handle slot_h, py::handle offsets_h, py::handle weights_h) {
  const Rows rows = RowsOf(what, rows_h);
  const int dev = rows.t.get_device();
  const Order o = OrderOf(slot_h, offsets_h, dev);
  if (rows.n != o.n)
    throw py::value_error(std::to_string(rows.n) + " rows, but the order is of " + std::to_string(o.n) + " assignments");
  const Weights w = WeightsOf(weights_h, o, dev);
  const On on(rows.t);
  Tensor out = NewRows(o.tokens, rows);
  Launched(ugk_expert_combine(rows.t.data_ptr(), (size_t)rows.n, (size_t)rows.stride, o.slot.data_ptr<int32_t>(), (size_t)o.tokens,
                              (uint32_t)o.top, w.data, w.elem, (size_t)rows.dim, rows.elem, out.data_ptr(), on.stream));
  return Wrap(std::move(out));
}

// rows_h None: only where the gradient of the weights is not wanted (weights_too false), which alone reads the rows
py::tuple CombineGrad(py::handle grad_h, py::handle rows_h, py::handle slot_h, py::handle offsets_h, py::handle weights_h,
                      bool weights_too) {
  const Rows grad = RowsOf("grad_out", grad_h);
  const int dev = grad.t.get_device();
  Rows rows{Tensor(), 0, grad.dim, grad.dim, grad.elem};
  const bool read = weights_too || !rows_h.is_none();
  if (read) rows = RowsOf("rows", rows_h, dev);
  const Order o = OrderOf(slot_h, offsets_h, dev);
  if (grad.n != o.tokens || (read && rows.n != o.n) || grad.dim != rows.dim || grad.elem != rows.elem)
    throw py::value_error("grad_out and rows are not rows of one type and length of " + std::to_string(o.tokens) + " tokens and " +
                          std::to_string(o.n) + " assignments");
  const Weights w = WeightsOf(weights_h, o, dev);
  const On on(grad.t);
  Tensor grad_rows = NewRows(o.n, grad);
  Tensor grad_w;
  if (w.data && weights_too) grad_w = at::empty(w.t.sizes(), w.t.options());
  else if (w.t.defined() && weights_too) grad_w = at::empty_like(w.t);  // no assignments
  Launched(ugk_expert_combine_grad(grad.t.data_ptr(), (size_t)grad.stride, Data(rows.t), (size_t)rows.stride, o.slot.data_ptr<int32_t>(),
                                   o.live, (size_t)o.tokens, (uint32_t)o.top, w.data, w.elem, (size_t)grad.dim, grad.elem,
                                   grad_rows.data_ptr(), Data(grad_w), on.stream));
  return py::make_tuple(Wrap(std::move(grad_rows)), grad_w.defined() ? Wrap(std::move(grad_w)) : py::none());
}

py::object TakeRows(py::handle table_h, py::handle index_h) {
  const Tensor &whole = Unpack("table", table_h, kRowsKind);
  if (whole.dim() != 2) throw py::value_error("table must be [rows, dim]");
  const Rows table = RowsOf("table", table_h);
  const Tensor index = Unpack("index", index_h, kIntKind, table.t.get_device()).contiguous();
  const On on(table.t);
  std::vector<int64_t> sizes(index.sizes().begin(), index.sizes().end());
  sizes.push_back(table.dim);
  Tensor out = at::empty(sizes, table.t.options());
  if (index.scalar_type() == ScalarType::Long)
    Launched(ugk_take_rows_i64(table.t.data_ptr(), (uint64_t)table.n, (size_t)table.stride, index.data_ptr<int64_t>(), (size_t)index.numel(),
                               (size_t)table.dim, table.elem, out.data_ptr(), on.stream));
  else
    Launched(ugk_take_rows_i32(table.t.data_ptr(), (uint64_t)table.n, (size_t)table.stride, index.data_ptr<int32_t>(), (size_t)index.numel(),
                               (size_t)table.dim, table.elem, out.data_ptr(), on.stream));
  return Wrap(std::move(out));
}

py::object TakeRowsGrad(py::handle grad_h, py::handle index_h, int64_t num_rows) {
  const Rows grad = RowsOf("grad", grad_h);
  const Tensor index = Unpack("index", index_h, kIntKind, grad.t.get_device()).contiguous();
  const int64_t n = index.numel();
  if (grad.n != n) throw py::value_error(std::to_string(grad.n) + " rows for " + std::to_string(n) + " indices");
  // of the index's shape, or one of the two is a list
  const at::IntArrayRef of = THPVariable_Unpack(grad_h.ptr()).sizes();
  const at::DimVector wide = Wide(of.slice(0, of.size() - 1)), index_wide = Wide(index.sizes());
  if (n && wide.size() > 1 && index_wide.size() > 1 && wide != index_wide)
    throw py::value_error("grad must be shaped [*index.shape, dim] or [indices, dim]");
  if (num_rows < 0 || num_rows >= (int64_t)1 << 31 || n >= (int64_t)1 << 31)
    throw py::value_error(std::to_string(n) + " indices into " + std::to_string(num_rows) + " rows: both must be below 2^31");
  const On on(grad.t);
  Tensor out = NewRows(num_rows, grad);
  const size_t nbytes = ugk_take_rows_grad_workspace_bytes((size_t)n, (uint64_t)num_rows, (size_t)grad.dim);
  const Tensor scratch = Scratch(nbytes, grad.t);
  if (index.scalar_type() == ScalarType::Long)
    Launched(ugk_take_rows_grad_i64(grad.t.data_ptr(), (size_t)grad.stride, index.data_ptr<int64_t>(), (size_t)n, (uint64_t)num_rows,
                                    (size_t)grad.dim, grad.elem, out.data_ptr(), Data(scratch), nbytes, on.stream));
  else
    Launched(ugk_take_rows_grad_i32(grad.t.data_ptr(), (size_t)grad.stride, index.data_ptr<int32_t>(), (size_t)n, (uint64_t)num_rows,
                                    (size_t)grad.dim, grad.elem, out.data_ptr(), Data(scratch), nbytes, on.stream));
  return Wrap(std::move(out));
}

// the tensors of a sequence or an iterator, or one tensor, or none of them, held while the call runs
class Items {
 public:
  explicit Items(py::handle h) {
    if (h.is_none()) return;
    if (THPVariable_Check(h.ptr())) {
      _one = h.ptr();
      return;
    }
    _seq = py::reinterpret_steal<py::object>(PySequence_Fast(h.ptr(), "gradients must be a tensor or a sequence of tensors"));
    if (!_seq) throw py::error_already_set();
  }
  size_t size() const { return _one ? 1 : !_seq ? 0 : (size_t)PySequence_Fast_GET_SIZE(_seq.ptr()); }
  PyObject *operator[](size_t i) const { return _one ? _one : PySequence_Fast_GET_ITEM(_seq.ptr(), (Py_ssize_t)i); }

 private:
  PyObject *_one = nullptr;
  py::object _seq;
};

const Tensor &ListedTensor(const char *what, PyObject *o, int dev) {
  const Tensor *t = THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
  if (t) NoTangent(what, *t);
  if (!t || !t->is_cuda() || t->layout() != c10::kStrided || ElemOf(*t) == 0)
    throw py::type_error(std::string(what) + " must be a GPU tensor of float32, float16, bfloat16");
  if (dev >= 0 && t->get_device() != dev) throw py::value_error(std::string(what) + " must be on the GPU of the other tensors");
  return *t;
}

struct Span {
  uintptr_t from, to;
  Span(const void *at, size_t nbytes) : from((uintptr_t)at), to((uintptr_t)at + nbytes) {}
};
// what is written is written once, and is nothing that the call reads but its own gradient; read[i] goes with written[i],
// or is left out where it is that place
void CheckPlaces(const std::vector<Span> &read, std::vector<Span> written) {
  std::vector<Span> elsewhere;
  for (size_t i = 0; i < read.size(); ++i)
    if (read[i].from != written[i].from) elsewhere.push_back(read[i]);
  std::sort(written.begin(), written.end(), [](const Span &a, const Span &b) { return a.from < b.from; });
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].from < written[i - 1].to) throw py::value_error("two gradients are written to the same place");
  for (const Span &r : elsewhere) {
    // the first that ends behind the start of r
    const auto w = std::upper_bound(written.begin(), written.end(), r.from, [](uintptr_t at, const Span &s) { return at < s.to; });
    if (w != written.end() && w->from < r.to)
      throw py::value_error("an output is in the same place as another gradient, or as a part of its own");
  }
}

// max_norm None: the norm alone; out None: in place
py::object GradNorm(py::handle grads_h, py::handle max_norm_h, py::handle out_h) {
  const bool clip = !max_norm_h.is_none(), elsewhere = !out_h.is_none();
  double max_norm = 0;
  if (clip) {
    max_norm = max_norm_h.cast<double>();
    if (!(max_norm >= 0)) throw py::value_error("max_norm must be at least 0, got " + std::to_string(max_norm));
  }
  const Items grads(grads_h);  // once: it may be an iterator
  const Items outs(elsewhere ? out_h : py::handle(Py_None));
  const size_t n = grads.size();
  if (elsewhere && outs.size() != n)
    throw py::value_error(std::to_string(outs.size()) + " outputs for " + std::to_string(n) + " gradients");
  std::vector<ugk_tensor_t> listed;
  std::vector<Tensor> copies;
  std::vector<Span> read, written;
  std::vector<c10::TensorImpl *> changed;
  listed.reserve(n);
  if (clip) written.reserve(n);
  if (clip && elsewhere) read.reserve(n);
  changed.reserve(n);
  const Tensor *first = nullptr;
  int dev = -1;
  for (size_t i = 0; i < n; ++i) {
    if (grads[i] == Py_None) continue;
    const Tensor *g = &ListedTensor("a gradient", grads[i], dev);
    if (!first) first = g, dev = (int)g->get_device();
    // in place and for the norm alone the order of the elements is nobody's matter, so long as they are one run of memory
    if (g->is_neg() || (!g->is_contiguous() && (elsewhere || !g->is_non_overlapping_and_dense()))) {
      if (clip && !elsewhere && g->numel())
        throw py::value_error("a gradient whose elements are no run of memory cannot be scaled in place");
      copies.push_back(g->resolve_neg().contiguous());
      g = nullptr;
    }
    const Tensor &from = g ? *g : copies.back();
    void *at = from.data_ptr(), *to = at;
    if (elsewhere) {
      const Tensor &o = ListedTensor("an output", outs[i], dev);
      if (o.scalar_type() != from.scalar_type() || o.sizes() != from.sizes() || !o.is_contiguous() || o.is_neg())
        throw py::value_error("an output must be contiguous and of its gradient's shape, type and GPU");
      to = o.data_ptr();
      changed.push_back(o.unsafeGetTensorImpl());
    } else if (clip) {
      changed.push_back(from.unsafeGetTensorImpl());
    }
    listed.push_back(ugk_tensor_t{at, to, (uint64_t)from.numel(), ElemOf(from), 0});
    if (clip && from.numel()) written.push_back(Span(to, from.nbytes()));
    if (clip && elsewhere && from.numel()) read.push_back(Span(at, from.nbytes()));
  }
  if (!first) throw py::value_error("no gradients");
  CheckPlaces(read, written);
  const On on(*first);
  for (c10::TensorImpl *t : changed) t->bump_version();  // what autograd has saved of them is stale
  const size_t nbytes = ugk_grad_norm_workspace_bytes(listed.data(), listed.size());
  Tensor norm = at::empty({}, first->options().dtype(at::kFloat));
  const Tensor scratch = Scratch(nbytes, *first);
  Launched(clip ? ugk_grad_clip(listed.data(), listed.size(), max_norm, Data(scratch), nbytes, norm.data_ptr<float>(), on.stream)
                : ugk_grad_norm(listed.data(), listed.size(), Data(scratch), nbytes, norm.data_ptr<float>(), on.stream));
  return Wrap(std::move(norm));
}

// torch's exceptions reach Python as torch's own (out of memory among them)
template <typename R, typename... A>
auto Guarded(R (*f)(A...)) {
  return [f](A... args) -> R {
    HANDLE_TH_ERRORS
    return f(args...);
    END_HANDLE_TH_ERRORS_PYBIND
  };
}

py::object CombineRows(py::handle rows, py::handle slot, py::handle offsets, py::handle weights) {
  return Combine("rows", rows, slot, offsets, weights);
}
py::object DispatchGrad(py::handle rows, py::handle slot, py::handle offsets) { return Combine("grad_rows", rows, slot, offsets, py::none()); }

}  // namespace

PYBIND11_MODULE(rows_native, m) {
  m.doc() = "the calls of collcache.torch.rows, compiled";
  if (ugk_abi_version() != UGK_ABI_VERSION) throw py::import_error("libugache_hip.so and rows_native come from different builds");
  g_raw_stream = py::object(py::module_::import("torch._C").attr("_cuda_getCurrentRawStream")).release().ptr();
  g_launch_error = py::object(py::module_::import("builtins").attr("RuntimeError")).release().ptr();
  m.def("expert_sort", Guarded(&ExpertSort));
  m.def("dispatch", Guarded(&Dispatch));
  m.def("dispatch_grad", Guarded(&DispatchGrad));
  m.def("combine", Guarded(&CombineRows));
  m.def("combine_grad", Guarded(&CombineGrad));
  m.def("take_rows", Guarded(&TakeRows));
  m.def("take_rows_grad", Guarded(&TakeRowsGrad));
  m.def("grad_norm", Guarded(&GradNorm));
}
