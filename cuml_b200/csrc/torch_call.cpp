// Native call path for device tensors: `DeviceCall(X, preds, kind, chunk_size, threshold)`.
//
// A prediction of a small batch takes a few microseconds on the GPU, so what its caller waits for
// is host work: attribute look-ups, shape checks, `torch.empty`, the current stream and a ctypes
// call cost about 8 us from Python, as much as all kernel launches together.  This object does the
// same with torch's C++ interface in under 2 us.  It handles the common call only - a CUDA tensor
// of the forest's own dtype on the forest's device with unit column stride, results to a new
// tensor or to a fitting `preds` - and returns None for everything else, which the Python code
// then converts or rejects with its usual messages.
#include <Python.h>

#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/autocast_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>

#include "../../include/b2fil.h"

namespace {

using PredictFn = int (*)(const b2fil_forest*, int, const void*, int64_t, int64_t, void*, int,
                          double, void*);

struct DeviceCall {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  PredictFn predict;            // b2fil_predict of the library that owns the forest
  const b2fil_forest* forest;
  int64_t n_features, n_trees, n_outputs;
  int device;
  bool f64, vector_leaves;
};

// Shape and element type of an output kind.
struct OutSpec {
  int ndim;
  int64_t dims[3];
  at::ScalarType dtype;
};

bool out_spec(const DeviceCall* c, int64_t kind, int64_t n, OutSpec& s)
{
  s.dtype = c->f64 ? at::kDouble : at::kFloat;
  s.ndim  = 2;
  s.dims[0] = n;
  switch (kind) {
    case B2FIL_INFER_DEFAULT: s.dims[1] = c->n_outputs; return true;
    case B2FIL_INFER_PROBA2: s.dims[1] = 2; return true;
    case B2FIL_INFER_CLASS:
      s.ndim  = 1;
      s.dtype = at::kInt;
      return true;
    case B2FIL_INFER_LEAF_ID:
      s.dims[1] = c->n_trees;
      s.dtype   = at::kInt;
      return true;
    case B2FIL_INFER_PER_TREE:
      s.dims[1] = c->n_trees;
      if (c->vector_leaves) {
        s.ndim    = 3;
        s.dims[2] = c->n_outputs;
      }
      return true;
    default: return false;
  }
}

// X, preds (tensor or None), kind, chunk_size, threshold.  Returns the output tensor, None when
// the call is not one of the common ones, or the library's error code as an int.  Any of torch's
// functions may throw (a tensor subclass answers even size() in Python): the macros turn what they
// throw into the Python exception.
PyObject* device_call(PyObject* self, PyObject* const* args, size_t nargsf, PyObject*)
{
  HANDLE_TH_ERRORS
  const DeviceCall* c = reinterpret_cast<const DeviceCall*>(self);
  if (PyVectorcall_NARGS(nargsf) != 5) {
    PyErr_SetString(PyExc_TypeError, "DeviceCall takes X, preds, kind, chunk_size, threshold");
    return nullptr;
  }
  if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
  const at::Tensor& X = THPVariable_Unpack(args[0]);
  const auto want     = c->f64 ? at::kDouble : at::kFloat;
  if (!X.is_cuda() || X.layout() != at::kStrided || X.dim() != 2 || X.scalar_type() != want ||
      X.get_device() != c->device || X.size(1) != c->n_features || X.stride(1) != 1)
    Py_RETURN_NONE;
  const int64_t kind  = PyLong_AsLongLong(args[2]);
  const int64_t chunk = PyLong_AsLongLong(args[3]);
  const double thr    = PyFloat_AsDouble(args[4]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t n = X.size(0);
  OutSpec s;
  if (!out_spec(c, kind, n, s)) Py_RETURN_NONE;
  const at::IntArrayRef dims(s.dims, s.ndim);
  const void* from      = X.const_data_ptr();
  const int64_t stride  = X.stride(0);
  at::TensorBase made;
  const bool given = args[1] != Py_None;
  if (given) {
    if (!THPVariable_Check(args[1])) Py_RETURN_NONE;
    const at::Tensor& out = THPVariable_Unpack(args[1]);
    if (out.sizes() != dims || out.scalar_type() != s.dtype || !out.is_cuda() ||
        !out.is_contiguous())
      Py_RETURN_NONE;
    made = out;
  } else {
    made = at::detail::empty_cuda(dims, s.dtype, X.device(), std::nullopt);
  }
  void* to     = made.mutable_data_ptr();
  void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(c->device)).stream();
  int rc;
  // (nothing in here throws: the lock has to come back)
  Py_BEGIN_ALLOW_THREADS;
  rc = c->predict(c->forest, static_cast<int>(kind), from, n, stride, to, static_cast<int>(chunk), thr,
                  stream);
  Py_END_ALLOW_THREADS;
  if (rc != B2FIL_OK) return PyLong_FromLong(rc);
  if (given) return Py_NewRef(args[1]);
  return THPVariable_Wrap(std::move(made));
  END_HANDLE_TH_ERRORS
}

// DeviceCall(predict_address, forest_address, n_features, n_trees, n_outputs, device, f64, vector)
PyObject* device_call_new(PyTypeObject* type, PyObject* args, PyObject*)
{
  unsigned long long predict = 0, forest = 0;
  long long nf = 0, nt = 0, no = 0;
  int device = 0, f64 = 0, vec = 0;
  if (!PyArg_ParseTuple(args, "KKLLLipp", &predict, &forest, &nf, &nt, &no, &device, &f64, &vec))
    return nullptr;
  DeviceCall* c = reinterpret_cast<DeviceCall*>(type->tp_alloc(type, 0));
  if (!c) return nullptr;
  c->vectorcall    = device_call;
  c->predict       = reinterpret_cast<PredictFn>(static_cast<uintptr_t>(predict));
  c->forest        = reinterpret_cast<const b2fil_forest*>(static_cast<uintptr_t>(forest));
  c->n_features    = nf;
  c->n_trees       = nt;
  c->n_outputs     = no;
  c->device        = device;
  c->f64           = f64 != 0;
  c->vector_leaves = vec != 0;
  return reinterpret_cast<PyObject*>(c);
}

PyTypeObject device_call_type = [] {
  PyTypeObject t         = {PyVarObject_HEAD_INIT(nullptr, 0)};
  t.tp_name              = "b2fil_torch.DeviceCall";
  t.tp_basicsize         = sizeof(DeviceCall);
  t.tp_flags             = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  t.tp_vectorcall_offset = offsetof(DeviceCall, vectorcall);
  t.tp_call              = PyVectorcall_Call;
  t.tp_new               = device_call_new;
  t.tp_doc               = "Predict call of one forest on CUDA tensors.";
  return t;
}();

// ---- distillation ----------------------------------------------------------------------------
using at::Tensor;
namespace ag = torch::autograd;

// The library's entry points (`bind`).
struct Library {
  decltype(&b2fil_last_error) last_error;
  decltype(&b2fil_top_scores_workspace) top_workspace;
  decltype(&b2fil_top_scores) top;
  decltype(&b2fil_distill_loss_workspace) loss_workspace;
  decltype(&b2fil_distill_loss) loss;
  decltype(&b2fil_distill_loss_grad) loss_grad;
  decltype(&b2fil_linear_loss_workspace) linear_workspace;
  decltype(&b2fil_linear_loss) linear;
  decltype(&b2fil_linear_loss_grad_workspace) linear_grad_workspace;
  decltype(&b2fil_linear_loss_grad) linear_grad;
  decltype(&b2fil_log_probs_workspace) score_workspace;
  decltype(&b2fil_log_probs) score;
  decltype(&b2fil_log_probs_grad) score_grad;
  decltype(&b2fil_linear_log_probs_workspace) linear_score_workspace;
  decltype(&b2fil_linear_log_probs) linear_score;
  decltype(&b2fil_linear_log_probs_grad_workspace) linear_score_grad_workspace;
  decltype(&b2fil_linear_log_probs_grad) linear_score_grad;
  decltype(&b2fil_clip_gradients_workspace) clip_workspace;
  decltype(&b2fil_clip_gradients) clip;
} library;

struct LibraryError {
  int code;
};
int64_t ok(int64_t rc)
{
  if (rc < 0) throw LibraryError{static_cast<int>(rc)};
  return rc;
}

int type_of(const Tensor& t)
{
  switch (t.scalar_type()) {
    case at::kFloat: return B2FIL_TYPE_F32;
    case at::kDouble: return B2FIL_TYPE_F64;
    case at::kBFloat16: return B2FIL_TYPE_BF16;
    case at::kHalf: return B2FIL_TYPE_F16;
    default: return -1;
  }
}
void* stream_of(int device)
{
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}
Tensor make(at::IntArrayRef size, at::ScalarType type, const Tensor& like)
{
  return Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}

// An ordinary CUDA tensor of two dimensions whose rows lie one after the other.
bool plain_rows(PyObject* o)
{
  if (!THPVariable_Check(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && t.dim() == 2 && !at::isTensorSubclassLike(t) && !t.is_neg() &&
         !t.is_conj() && (t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= t.size(1) || t.size(0) == 1) &&
         t.size(0) > 0 && t.size(1) > 0;
}
// Whether a student's tensor carries a forward-mode tangent: the ctypes path's autograd function refuses that, a
// node of this file would leave it out.
bool has_tangent(PyObject* o) { return THPVariable_Unpack(o)._fw_grad(/*level=*/0).defined(); }
bool on(const Tensor& t, const Tensor& like) { return t.device() == like.device(); }

// A teacher's numbers in 32 bits (scores of 16 or 64 bits are converted), constants to autograd.
Tensor as_floats(const Tensor& x)
{
  if (x.scalar_type() == at::kFloat) return x;
  at::AutoDispatchBelowADInplaceOrView below;
  return x.to(at::kFloat);
}

// The teacher of one call.  values and logsumexp may be undefined.
struct TeacherOf {
  Tensor values, index, logsumexp;
  int64_t ignore;
  b2fil_teacher c() const
  {
    b2fil_teacher t{};
    if (values.defined()) {
      t.values        = values.const_data_ptr<float>();
      t.values_stride = values.stride(0);
    }
    t.index        = index.const_data_ptr();
    t.index_stride = index.stride(0);
    t.index64      = index.scalar_type() == at::kLong;
    if (logsumexp.defined()) t.logsumexp = logsumexp.const_data_ptr<float>();
    t.ignore = ignore;
    t.k      = static_cast<int32_t>(index.size(1));
    return t;
  }
};
// False: not what the library takes as it is.
bool teacher_of(PyObject* values, PyObject* index, PyObject* lse, const Tensor& like, TeacherOf& t)
{
  const int64_t n = like.size(0);
  if (values == Py_None) {  // one class per row
    if (!THPVariable_Check(index)) return false;
    t.index = THPVariable_Unpack(index);
    if (t.index.dim() != 1 || !t.index.is_cuda() || t.index.layout() != at::kStrided || at::isTensorSubclassLike(t.index) ||
        t.index.is_neg())
      return false;
    t.index = t.index.unsqueeze(1);
  } else {
    if (!plain_rows(index)) return false;
    t.index = THPVariable_Unpack(index);
  }
  if ((t.index.scalar_type() != at::kInt && t.index.scalar_type() != at::kLong) || t.index.size(0) != n ||
      t.index.size(1) > B2FIL_MOST_TOP || !on(t.index, like))
    return false;
  if (values != Py_None) {
    if (!plain_rows(values)) return false;
    t.values = THPVariable_Unpack(values);
    if (type_of(t.values) < 0 || t.values.sizes() != t.index.sizes() || !on(t.values, like)) return false;
    t.values = as_floats(t.values);
  }
  if (lse != Py_None) {
    if (!THPVariable_Check(lse)) return false;
    t.logsumexp = THPVariable_Unpack(lse);
    if (!t.logsumexp.is_cuda() || t.logsumexp.layout() != at::kStrided || type_of(t.logsumexp) < 0 ||
        t.logsumexp.dim() != 1 || t.logsumexp.size(0) != n || (n > 1 && t.logsumexp.stride(0) != 1) ||
        at::isTensorSubclassLike(t.logsumexp) || t.logsumexp.is_neg() || !on(t.logsumexp, like))
      return false;
    t.logsumexp = as_floats(t.logsumexp);
  }
  return true;
}

// Options of a loss: temperature, ignored class, reduction.
struct Options {
  double temperature;
  int64_t ignore;
  int reduction;
};
bool options_of(PyObject* const* args, Options& o)
{
  o.temperature = PyFloat_AsDouble(args[0]);
  o.ignore      = PyLong_AsLongLong(args[1]);
  o.reduction   = static_cast<int>(PyLong_AsLong(args[2]));
  return !PyErr_Occurred();
}

// What a node keeps of its inputs.
struct Saved {
  ag::SavedVariable variable;
  at::ScalarType type;
  int64_t rows, cols;
  at::Device device = at::kCPU;
  void set(const Tensor& x)
  {
    variable = ag::SavedVariable(x, false);
    type     = x.scalar_type();
    rows     = x.size(0);
    cols     = x.size(1);
    device   = x.device();
  }
  // Called outside of dispatch guards: hooks may compute it again, through autograd.
  Tensor unpack()
  {
    Tensor x = variable.unpack();
    TORCH_CHECK(x.layout() == at::kStrided && x.dim() == 2 && x.size(0) == rows && x.size(1) == cols &&
                  x.scalar_type() == type && x.device() == device,
                "a hook gave back another tensor than the distillation loss had saved");
    return x;
  }
};
// Rows one after the other: what hooks return may lie in another order.
Tensor in_rows(const Tensor& given)
{
  const Tensor x = given.is_neg() ? given.resolve_neg() : given;  // (the call by itself would cost 0.5 us of a step)
  const bool as_saved = (x.stride(1) == 1 || x.size(1) == 1) && (x.stride(0) >= x.size(1) || x.size(0) == 1);
  return as_saved ? x : x.contiguous();
}

// What a node's gradient is by the loss: 32-bit values, and elements from one row's to the next.  (The gradient of a part of a
// conjugate may be a view whose numbers are the negatives of those in memory.)
Tensor upstream_of(const Tensor& g, int64_t& stride)
{
  const Tensor x = g.scalar_type() != at::kFloat ? g.to(at::kFloat) : g.is_neg() ? g.resolve_neg() : g;
  stride         = x.dim() ? x.stride(0) : 0;
  return x;
}
[[noreturn]] void raise_library_error(const LibraryError& e)
{
  TORCH_CHECK(false, "b2fil error ", e.code, ": ", library.last_error());
}
// A second derivative is an error where it is taken, not a silent zero.
void no_second_derivative(Tensor& grad, const ag::variable_list& of)
{
  if (!grad.defined() || !at::GradMode::is_enabled()) return;
  auto node = std::shared_ptr<ag::Error>(new ag::Error("the distillation losses have first derivatives only",
                                                       ag::collect_next_edges(of)), ag::deleteNode);
  ag::set_history(grad, node);
}

struct LossNode : ag::Node {
  Saved logits;
  Tensor kept;
  Options o;
  int k;
  bool gone = false;

  ag::variable_list apply(ag::variable_list&& grads) override
  {
    TORCH_CHECK(!gone, "the distillation loss's graph has been freed: retain_graph=True keeps it");
    if (!grads[0].defined()) return {Tensor()};
    const Tensor saved = logits.unpack();
    Tensor grad;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      at::NoGradGuard no_grad;
      const Tensor x  = in_rows(saved);
      const int64_t n = x.size(0), c = x.size(1);
      grad = make({n, c}, x.scalar_type(), x);
      int64_t stride;
      const Tensor g     = upstream_of(grads[0], stride);
      const float* at    = kept.const_data_ptr<float>();
      const float* named = at + 4 * n + 4;
      const int device   = x.get_device();
      try {
        ok(library.loss_grad(type_of(x), x.const_data_ptr(), n, c, x.stride(0), k, o.temperature, at, named,
                             reinterpret_cast<const int32_t*>(named + n * k), g.const_data_ptr<float>(), stride,
                             o.reduction ? at + 4 * n : nullptr, grad.mutable_data_ptr(), c, device, stream_of(device)));
      } catch (const LibraryError& e) {
        raise_library_error(e);
      }
    }
    no_second_derivative(grad, {grads[0], saved});
    return {grad};
  }
  void release_variables() override
  {
    logits.variable.reset_data();
    kept = Tensor();
    gone = true;
  }
  std::string name() const override { return "DistillLossBackward"; }
};

// logits, values, index, logsumexp or None, temperature, ignored class, reduction
PyObject* distill_loss(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
  HANDLE_TH_ERRORS
  if (nargs != 7) return PyErr_Format(PyExc_TypeError, "distill_loss takes 7 arguments");
  Options o;
  if (!options_of(args + 4, o)) return nullptr;
  if (!library.loss || !plain_rows(args[0]) || has_tangent(args[0])) Py_RETURN_NONE;
  const Tensor& x = THPVariable_Unpack(args[0]);
  const int type  = type_of(x);
  TeacherOf t;
  if (type < 0 || type == B2FIL_TYPE_F64 || !teacher_of(args[1], args[2], args[3], x, t)) Py_RETURN_NONE;
  t.ignore        = o.ignore;
  const int64_t n = x.size(0), c = x.size(1);
  const int k     = static_cast<int>(t.index.size(1));
  Tensor kept, loss;
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    const int device   = x.get_device();
    const int64_t room = ok(library.loss_workspace(type, n, c, k, device));
    // statistics, factor, the named classes' arrays, losses of the rows where they are not what is
    // returned, workspace
    const int64_t named_at = 4 * n + 4, rows_at = named_at + 2 * n * k,
                  work_at = (rows_at + (o.reduction ? n : 0) + 63) / 64 * 64;
    kept          = make({work_at + room / 4}, at::kFloat, x);
    loss          = o.reduction ? make({}, at::kFloat, x) : make({n}, at::kFloat, x);
    float* at     = kept.mutable_data_ptr<float>();
    float* to     = loss.mutable_data_ptr<float>();
    const auto tc = t.c();
    ok(library.loss(type, x.const_data_ptr(), n, c, x.stride(0), &tc, o.temperature, o.reduction,
                    o.reduction ? at + rows_at : to, at, at + named_at, reinterpret_cast<int32_t*>(at + named_at + n * k), to,
                    at + 4 * n, at + work_at, room, device, stream_of(device)));
  } catch (const LibraryError& e) {
    return PyLong_FromLong(e.code);
  }
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    auto node = std::shared_ptr<LossNode>(new LossNode(), ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(x));
    node->logits.set(x);
    node->kept = std::move(kept);
    node->o    = o;
    node->k    = k;
    ag::set_history(loss, node);
  }
  return THPVariable_Wrap(std::move(loss));
  END_HANDLE_TH_ERRORS
}

struct LinearNode : ag::Node {
  Saved hidden, weight;
  Tensor kept;
  Options o;
  int k;
  bool gone = false;

  ag::variable_list apply(ag::variable_list&& grads) override
  {
    TORCH_CHECK(!gone, "the distillation loss's graph has been freed: retain_graph=True keeps it");
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const Tensor saved_h = hidden.unpack(), saved_w = weight.unpack();
    Tensor dh, dw;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      at::NoGradGuard no_grad;
      const Tensor h = in_rows(saved_h), w = in_rows(saved_w);
      const int64_t n = h.size(0), width = h.size(1), c = w.size(0);
      auto step = [&](const Tensor& x) { return x.size(0) == 1 ? width : x.stride(0); };
      const bool wants_h = task_should_compute_output(0), wants_w = task_should_compute_output(1);
      if (wants_h) dh = make({n, width}, h.scalar_type(), h);
      if (wants_w) dw = make({c, width}, h.scalar_type(), h);
      int64_t stride;
      const Tensor g   = upstream_of(grads[0], stride);
      const float* at  = kept.const_data_ptr<float>();
      const float* named = at + 4 * n + 4;
      const int device = h.get_device(), type = type_of(h);
      try {
        const int64_t room = ok(library.linear_grad_workspace(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w),
                                                               n, c, width, k, wants_h, wants_w, device));
        const Tensor work  = make({room}, at::kByte, h);
        ok(library.linear_grad(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w), n, c, width, k,
                               o.temperature, at, named, named + n * k, reinterpret_cast<const int32_t*>(named + 2 * n * k),
                               g.const_data_ptr<float>(), stride, o.reduction ? at + 4 * n : nullptr,
                               wants_h ? dh.mutable_data_ptr() : nullptr, wants_w ? dw.mutable_data_ptr() : nullptr,
                               work.mutable_data_ptr(), room, device, stream_of(device)));
      } catch (const LibraryError& e) {
        raise_library_error(e);
      }
    }
    no_second_derivative(dh, {grads[0], saved_h, saved_w});
    no_second_derivative(dw, {grads[0], saved_h, saved_w});
    return {dh, dw};
  }
  void release_variables() override
  {
    hidden.variable.reset_data();
    weight.variable.reset_data();
    kept = Tensor();
    gone = true;
  }
  std::string name() const override { return "LinearDistillLossBackward"; }
};

// hidden, weight, values or None, index, temperature, ignored class, reduction, whether autocast has been heeded
PyObject* linear_loss(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
  HANDLE_TH_ERRORS
  if (nargs != 8) return PyErr_Format(PyExc_TypeError, "linear_loss takes 8 arguments");
  Options o;
  const int cast = PyObject_IsTrue(args[7]);
  if (cast < 0 || !options_of(args + 4, o)) return nullptr;
  if (!library.linear || (!cast && at::autocast::is_autocast_enabled(at::kCUDA)) || !plain_rows(args[0]) || !plain_rows(args[1]) ||
      has_tangent(args[0]) || has_tangent(args[1]))
    Py_RETURN_NONE;
  const Tensor& h = THPVariable_Unpack(args[0]);
  const Tensor& w = THPVariable_Unpack(args[1]);
  const int type  = type_of(h);
  const int64_t n = h.size(0), width = h.size(1), c = w.size(0);
  // (a single row's stride says nothing)
  auto step = [&](const Tensor& x) { return x.size(0) == 1 ? width : x.stride(0); };
  TeacherOf t;
  if ((type != B2FIL_TYPE_BF16 && type != B2FIL_TYPE_F16) || w.scalar_type() != h.scalar_type() || !on(w, h) ||
      w.size(1) != width || !teacher_of(args[2], args[3], Py_None, h, t))
    Py_RETURN_NONE;
  t.ignore    = o.ignore;
  const int k = static_cast<int>(t.index.size(1));
  Tensor kept, loss;
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    const int device   = h.get_device();
    const int64_t room = ok(library.linear_workspace(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w), n, c, width,
                                                      k, device));
    const Tensor work  = make({room}, at::kByte, h);
    // statistics, factor, the named classes' arrays, losses of the rows where they are not what is returned
    kept          = make({4 * n + 4 + 3 * n * k + (o.reduction ? n : 0)}, at::kFloat, h);
    loss          = o.reduction ? make({}, at::kFloat, h) : make({n}, at::kFloat, h);
    float* at     = kept.mutable_data_ptr<float>();
    float* named  = at + 4 * n + 4;
    float* to     = loss.mutable_data_ptr<float>();
    const auto tc = t.c();
    ok(library.linear(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w), n, c, width, &tc,
                      o.temperature, o.reduction, o.reduction ? named + 3 * n * k : to, at, named, named + n * k,
                      reinterpret_cast<int32_t*>(named + 2 * n * k), to, at + 4 * n, work.mutable_data_ptr(), room, device,
                      stream_of(device)));
  } catch (const LibraryError& e) {
    return PyLong_FromLong(e.code);
  }
  if (at::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad())) {
    auto node = std::shared_ptr<LinearNode>(new LinearNode(), ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(h, w));
    node->hidden.set(h);
    node->weight.set(w);
    node->kept = std::move(kept);
    node->o    = o;
    node->k    = k;
    ag::set_history(loss, node);
  }
  return THPVariable_Wrap(std::move(loss));
  END_HANDLE_TH_ERRORS
}

// scores, k, temperature, probabilities -> (values, index, logsumexp)
PyObject* top_scores(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
  HANDLE_TH_ERRORS
  if (nargs != 4) return PyErr_Format(PyExc_TypeError, "top_scores takes 4 arguments");
  const int64_t k  = PyLong_AsLongLong(args[1]);
  const double tau = PyFloat_AsDouble(args[2]);
  const int prob   = PyObject_IsTrue(args[3]);
  if (PyErr_Occurred()) return nullptr;
  if (!library.top || !plain_rows(args[0])) Py_RETURN_NONE;
  const Tensor& x = THPVariable_Unpack(args[0]);
  const int type  = type_of(x);
  if (type < 0 || k < 1 || k > x.size(1) || k > B2FIL_MOST_TOP) Py_RETURN_NONE;
  Tensor values, index, lse;
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t n = x.size(0), c = x.size(1);
    const int device   = x.get_device();
    const int64_t room = ok(library.top_workspace(type, n, c, static_cast<int>(k), device));
    Tensor work;
    if (room) work = make({room}, at::kByte, x);
    values = make({n, k}, x.scalar_type(), x);
    index  = make({n, k}, at::kInt, x);
    lse    = make({n}, type == B2FIL_TYPE_F64 ? at::kDouble : at::kFloat, x);
    ok(library.top(type, x.const_data_ptr(), n, c, x.stride(0), static_cast<int>(k), prob, tau, values.mutable_data_ptr(),
                   index.mutable_data_ptr<int>(), lse.mutable_data_ptr(), room ? work.mutable_data_ptr() : nullptr, room,
                   device, stream_of(device)));
  } catch (const LibraryError& e) {
    return PyLong_FromLong(e.code);
  }
  PyObject* out[3] = {THPVariable_Wrap(std::move(values)), THPVariable_Wrap(std::move(index)), THPVariable_Wrap(std::move(lse))};
  PyObject* r      = out[0] && out[1] && out[2] ? PyTuple_Pack(3, out[0], out[1], out[2]) : nullptr;
  for (PyObject* x : out) Py_XDECREF(x);
  return r;
  END_HANDLE_TH_ERRORS
}

// ---- scores ----------------------------------------------------------------------------------
// One class per row, or none.  False: not what the library takes as it is.
bool target_of(PyObject* o, const Tensor& like, int64_t ignore, Tensor& index, b2fil_target& t)
{
  t        = b2fil_target{};
  t.ignore = ignore;
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  index = THPVariable_Unpack(o);
  if (index.dim() != 1 || !index.is_cuda() || index.layout() != at::kStrided || at::isTensorSubclassLike(index) || index.is_neg() ||
      (index.scalar_type() != at::kInt && index.scalar_type() != at::kLong) || index.size(0) != like.size(0) || !on(index, like))
    return false;
  t.index   = index.const_data_ptr();
  t.stride  = index.stride(0);
  t.index64 = index.scalar_type() == at::kLong;
  return true;
}

// A node's gradients by the rows' log probabilities and entropies, which may not be there.
struct Upstreams {
  Tensor log_prob, entropy;
  int64_t log_prob_stride = 0, entropy_stride = 0;
  Upstreams(const Tensor& g, const Tensor& h)
  {
    if (g.defined()) log_prob = upstream_of(g, log_prob_stride);
    if (h.defined()) entropy = upstream_of(h, entropy_stride);
  }
  static const float* at(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
};
constexpr const char* kFreed = "the scores' graph has been freed: retain_graph=True keeps it";

// Outputs: log probability (where a target is given), entropy.
struct ScoreNode : ag::Node {
  Saved logits;
  Tensor kept;
  double temperature;
  bool has_target, gone = false;

  ag::variable_list apply(ag::variable_list&& grads) override
  {
    TORCH_CHECK(!gone, kFreed);
    const Tensor g = has_target ? grads[0] : Tensor(), h = grads[has_target];
    if (!g.defined() && !h.defined()) return {Tensor()};
    const Tensor saved = logits.unpack();
    Tensor grad;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      at::NoGradGuard no_grad;
      const Tensor x  = in_rows(saved);
      const int64_t n = x.size(0), c = x.size(1);
      grad = make({n, c}, x.scalar_type(), x);
      const Upstreams up(g, h);
      const int device = x.get_device();
      try {
        ok(library.score_grad(type_of(x), x.const_data_ptr(), n, c, x.stride(0), temperature, kept.const_data_ptr<float>(),
                              Upstreams::at(up.log_prob), up.log_prob_stride, Upstreams::at(up.entropy), up.entropy_stride,
                              grad.mutable_data_ptr(), c, device, stream_of(device)));
      } catch (const LibraryError& e) {
        raise_library_error(e);
      }
    }
    no_second_derivative(grad, {g, h, saved});
    return {grad};
  }
  void release_variables() override
  {
    logits.variable.reset_data();
    kept = Tensor();
    gone = true;
  }
  std::string name() const override { return "LogProbsBackward"; }
};

struct LinearScoreNode : ag::Node {
  Saved hidden, weight;
  Tensor kept;
  double temperature;
  bool has_target, gone = false;

  ag::variable_list apply(ag::variable_list&& grads) override
  {
    TORCH_CHECK(!gone, kFreed);
    const Tensor g = has_target ? grads[0] : Tensor(), h_up = grads[has_target];
    if (!g.defined() && !h_up.defined()) return {Tensor(), Tensor()};
    const Tensor saved_h = hidden.unpack(), saved_w = weight.unpack();
    Tensor dh, dw;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      at::NoGradGuard no_grad;
      const Tensor h = in_rows(saved_h), w = in_rows(saved_w);
      const int64_t n = h.size(0), width = h.size(1), c = w.size(0);
      auto step = [&](const Tensor& x) { return x.size(0) == 1 ? width : x.stride(0); };
      const bool wants_h = task_should_compute_output(0), wants_w = task_should_compute_output(1);
      if (wants_h) dh = make({n, width}, h.scalar_type(), h);
      if (wants_w) dw = make({c, width}, h.scalar_type(), h);
      const Upstreams up(g, h_up);
      const int device = h.get_device(), type = type_of(h);
      try {
        const int64_t room = ok(library.linear_score_grad_workspace(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w),
                                                                     n, c, width, wants_h, wants_w, device));
        const Tensor work  = make({room}, at::kByte, h);
        ok(library.linear_score_grad(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w), n, c, width, temperature,
                                     kept.const_data_ptr<float>(), Upstreams::at(up.log_prob), up.log_prob_stride,
                                     Upstreams::at(up.entropy), up.entropy_stride, wants_h ? dh.mutable_data_ptr() : nullptr,
                                     wants_w ? dw.mutable_data_ptr() : nullptr, work.mutable_data_ptr(), room, device,
                                     stream_of(device)));
      } catch (const LibraryError& e) {
        raise_library_error(e);
      }
    }
    no_second_derivative(dh, {g, h_up, saved_h, saved_w});
    no_second_derivative(dw, {g, h_up, saved_h, saved_w});
    return {dh, dw};
  }
  void release_variables() override
  {
    hidden.variable.reset_data();
    weight.variable.reset_data();
    kept = Tensor();
    gone = true;
  }
  std::string name() const override { return "LinearLogProbsBackward"; }
};

// The log probabilities (None without a target), the entropies and two more, as a tuple of `n`.
PyObject* pack_scores(Tensor log_prob, Tensor entropy, Tensor top, Tensor index, int n)
{
  PyObject* out[4] = {THPVariable_Wrap(std::move(log_prob)), THPVariable_Wrap(std::move(entropy)), nullptr, nullptr};
  for (int i = 2; i < n; ++i) out[i] = THPVariable_Wrap(i == 2 ? std::move(top) : std::move(index));  // (undefined: None)
  PyObject* r = nullptr;
  if (out[0] && out[1] && (n < 3 || (out[2] && out[3])))
    r = n == 2 ? PyTuple_Pack(2, out[0], out[1]) : PyTuple_Pack(4, out[0], out[1], out[2], out[3]);
  for (PyObject* x : out) Py_XDECREF(x);
  return r;
}
// Room for a row's scores in `kept`: what the gradient needs comes first.
Tensor score_room(int64_t n, int64_t more, const Tensor& like) { return make({4 * n + more}, at::kFloat, like); }

// logits, target or None, temperature, k, ignored class -> (log_prob or None, entropy, best log probabilities, their classes)
PyObject* log_probs(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
  HANDLE_TH_ERRORS
  if (nargs != 5) return PyErr_Format(PyExc_TypeError, "log_probs takes 5 arguments");
  const double temperature = PyFloat_AsDouble(args[2]);
  const int64_t k = PyLong_AsLongLong(args[3]), ignore = PyLong_AsLongLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  if (!library.score || !plain_rows(args[0]) || has_tangent(args[0])) Py_RETURN_NONE;
  const Tensor& x = THPVariable_Unpack(args[0]);
  const int type  = type_of(x);
  Tensor index;
  b2fil_target t;
  if (type < 0 || type == B2FIL_TYPE_F64 || k < 0 || k > x.size(1) || k > B2FIL_MOST_TOP || !target_of(args[1], x, ignore, index, t))
    Py_RETURN_NONE;
  const bool has_target = t.index != nullptr;
  const int64_t n = x.size(0), c = x.size(1);
  Tensor kept, log_prob, entropy, top, classes;
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    const int device   = x.get_device();
    const int64_t room = ok(library.score_workspace(type, n, c, static_cast<int>(k), device));
    const int64_t work_at = (4 * n + 63) / 64 * 64;
    kept    = score_room(n, work_at - 4 * n + room / 4, x);
    entropy = make({n}, at::kFloat, x);
    if (has_target) log_prob = make({n}, at::kFloat, x);
    if (k) {
      top     = make({n, k}, at::kFloat, x);
      classes = make({n, k}, at::kInt, x);
    }
    float* at = kept.mutable_data_ptr<float>();
    ok(library.score(type, x.const_data_ptr(), n, c, x.stride(0), &t, temperature, static_cast<int>(k),
                     has_target ? log_prob.mutable_data_ptr<float>() : nullptr, entropy.mutable_data_ptr<float>(), at,
                     k ? top.mutable_data_ptr<float>() : nullptr, k ? classes.mutable_data_ptr<int>() : nullptr, at + work_at, room,
                     device, stream_of(device)));
  } catch (const LibraryError& e) {
    return PyLong_FromLong(e.code);
  }
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    auto node = std::shared_ptr<ScoreNode>(new ScoreNode(), ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(x));
    node->logits.set(x);
    node->kept        = std::move(kept);
    node->temperature = temperature;
    node->has_target  = has_target;
    if (has_target) ag::set_history(log_prob, node);
    ag::set_history(entropy, node);
  }
  return pack_scores(std::move(log_prob), std::move(entropy), std::move(top), std::move(classes), 4);
  END_HANDLE_TH_ERRORS
}

// hidden, weight, target or None, temperature, ignored class, whether autocast has been heeded -> (log_prob or None, entropy)
PyObject* linear_log_probs(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
  HANDLE_TH_ERRORS
  if (nargs != 6) return PyErr_Format(PyExc_TypeError, "linear_log_probs takes 6 arguments");
  const double temperature = PyFloat_AsDouble(args[3]);
  const int64_t ignore     = PyLong_AsLongLong(args[4]);
  const int cast           = PyObject_IsTrue(args[5]);
  if (PyErr_Occurred()) return nullptr;
  if (!library.linear_score || (!cast && at::autocast::is_autocast_enabled(at::kCUDA)) || !plain_rows(args[0]) ||
      !plain_rows(args[1]) || has_tangent(args[0]) || has_tangent(args[1]))
    Py_RETURN_NONE;
  const Tensor& h = THPVariable_Unpack(args[0]);
  const Tensor& w = THPVariable_Unpack(args[1]);
  const int type  = type_of(h);
  const int64_t n = h.size(0), width = h.size(1), c = w.size(0);
  auto step = [&](const Tensor& x) { return x.size(0) == 1 ? width : x.stride(0); };
  Tensor index;
  b2fil_target t;
  if ((type != B2FIL_TYPE_BF16 && type != B2FIL_TYPE_F16) || w.scalar_type() != h.scalar_type() || !on(w, h) ||
      w.size(1) != width || !target_of(args[2], h, ignore, index, t))
    Py_RETURN_NONE;
  const bool has_target = t.index != nullptr;
  Tensor kept, log_prob, entropy;
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    const int device   = h.get_device();
    const int64_t room = ok(library.linear_score_workspace(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w), n, c,
                                                            width, device));
    const Tensor work  = make({room}, at::kByte, h);
    kept    = score_room(n, 0, h);
    entropy = make({n}, at::kFloat, h);
    if (has_target) log_prob = make({n}, at::kFloat, h);
    ok(library.linear_score(type, h.const_data_ptr(), step(h), w.const_data_ptr(), step(w), n, c, width, &t, temperature,
                            has_target ? log_prob.mutable_data_ptr<float>() : nullptr, entropy.mutable_data_ptr<float>(),
                            kept.mutable_data_ptr<float>(), work.mutable_data_ptr(), room, device, stream_of(device)));
  } catch (const LibraryError& e) {
    return PyLong_FromLong(e.code);
  }
  if (at::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad())) {
    auto node = std::shared_ptr<LinearScoreNode>(new LinearScoreNode(), ag::deleteNode);
    node->set_next_edges(ag::collect_next_edges(h, w));
    node->hidden.set(h);
    node->weight.set(w);
    node->kept        = std::move(kept);
    node->temperature = temperature;
    node->has_target  = has_target;
    if (has_target) ag::set_history(log_prob, node);
    ag::set_history(entropy, node);
  }
  return pack_scores(std::move(log_prob), std::move(entropy), Tensor(), Tensor(), 2);
  END_HANDLE_TH_ERRORS
}

// ---- gradients -------------------------------------------------------------------------------
// A gradient (or what takes it) whose elements lie one after the other in some order.
bool dense(const Tensor& t, const Tensor& like)
{
  const int type = type_of(t);
  return t.is_cuda() && t.layout() == at::kStrided && !at::isTensorSubclassLike(t) && !t.is_neg() && !t.is_conj() &&
         (type == B2FIL_TYPE_F32 || type == B2FIL_TYPE_BF16 || type == B2FIL_TYPE_F16) && on(t, like) &&
         t.is_non_overlapping_and_dense();
}

// gradients, out (lists; out may be None), largest norm, kind of norm, whether to scale -> norm
PyObject* clip_gradients(PyObject*, PyObject* const* args, Py_ssize_t nargs)
{
  HANDLE_TH_ERRORS
  if (nargs != 5) return PyErr_Format(PyExc_TypeError, "clip_gradients takes 5 arguments");
  const double most = PyFloat_AsDouble(args[2]);
  const int kind    = static_cast<int>(PyLong_AsLong(args[3]));
  const int scales  = PyObject_IsTrue(args[4]);
  if (PyErr_Occurred()) return nullptr;
  const bool apart = args[1] != Py_None;
  if (!library.clip || !PyList_Check(args[0]) || (apart && (!PyList_Check(args[1]) || PyList_GET_SIZE(args[0]) != PyList_GET_SIZE(args[1]))))
    Py_RETURN_NONE;
  std::vector<b2fil_gradient> entries;
  std::vector<Tensor> written;
  Tensor first;
  const Py_ssize_t size = PyList_GET_SIZE(args[0]);
  entries.reserve(size);
  written.reserve(size);
  for (Py_ssize_t i = 0; i < size; ++i) {
    PyObject* o = PyList_GET_ITEM(args[0], i);
    if (o == Py_None) continue;
    if (!THPVariable_Check(o)) Py_RETURN_NONE;
    Tensor x = THPVariable_Unpack(o);
    if (at::isTensorSubclassLike(x)) Py_RETURN_NONE;
    if (x.requires_grad() && x.is_leaf()) x = x.grad();
    if (!x.defined()) continue;
    if (!first.defined()) first = x;
    if (!dense(x, first)) Py_RETURN_NONE;
    Tensor to = x;
    if (apart) {
      PyObject* p = PyList_GET_ITEM(args[1], i);
      if (!THPVariable_Check(p)) Py_RETURN_NONE;
      to = THPVariable_Unpack(p);
      if (!dense(to, first) || to.sizes() != x.sizes() || to.strides() != x.strides() || to.requires_grad()) Py_RETURN_NONE;
    }
    b2fil_gradient g{};
    // (a tensor that is written first gets memory of its own where it shares some)
    g.to        = scales ? to.mutable_data_ptr() : const_cast<void*>(to.const_data_ptr());
    g.from      = x.const_data_ptr();
    g.rows      = 1;
    g.cols      = x.numel();
    g.from_col  = g.to_col = 1;
    g.from_type = type_of(x);
    g.to_type   = type_of(to);
    g.tensor    = static_cast<int32_t>(i);
    entries.push_back(g);
    if (scales) written.push_back(std::move(to));
  }
  if (!first.defined()) Py_RETURN_NONE;
  Tensor norm;
  try {
    at::AutoDispatchBelowADInplaceOrView below;
    const int device   = first.get_device();
    const int64_t n    = static_cast<int64_t>(entries.size());
    const int64_t room = ok(library.clip_workspace(entries.data(), n, device));
    const Tensor work  = make({room}, at::kByte, first);
    norm               = make({}, at::kFloat, first);
    ok(library.clip(entries.data(), n, kind, scales, most, norm.mutable_data_ptr<float>(), work.mutable_data_ptr(), room, device,
                    stream_of(device)));
  } catch (const LibraryError& e) {
    return PyLong_FromLong(e.code);
  }
  for (const Tensor& x : written)
    if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(std::move(norm));
  END_HANDLE_TH_ERRORS
}

// Addresses of the library's entry points, in the order of `Library`.
PyObject* bind(PyObject*, PyObject* args)
{
  constexpr int N = 19;
  static_assert(sizeof(Library) == N * sizeof(void*), "one address each");
  unsigned long long a[N];
  if (PyTuple_GET_SIZE(args) != N) return PyErr_Format(PyExc_TypeError, "bind takes %d addresses", N);
  for (int i = 0; i < N; ++i) {
    a[i] = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(args, i));
    if (PyErr_Occurred()) return nullptr;
  }
  Library l;
  auto put = [](auto& f, unsigned long long at) { f = reinterpret_cast<std::decay_t<decltype(f)>>(static_cast<uintptr_t>(at)); };
  put(l.last_error, a[0]);
  put(l.top_workspace, a[1]);
  put(l.top, a[2]);
  put(l.loss_workspace, a[3]);
  put(l.loss, a[4]);
  put(l.loss_grad, a[5]);
  put(l.linear_workspace, a[6]);
  put(l.linear, a[7]);
  put(l.linear_grad_workspace, a[8]);
  put(l.linear_grad, a[9]);
  put(l.score_workspace, a[10]);
  put(l.score, a[11]);
  put(l.score_grad, a[12]);
  put(l.linear_score_workspace, a[13]);
  put(l.linear_score, a[14]);
  put(l.linear_score_grad_workspace, a[15]);
  put(l.linear_score_grad, a[16]);
  put(l.clip_workspace, a[17]);
  put(l.clip, a[18]);
  library = l;
  Py_RETURN_NONE;
}

PyMethodDef module_methods[] = {
  {"bind", bind, METH_VARARGS, "Entry points of libb2fil that the distillation calls use."},
  {"top_scores", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(top_scores)), METH_FASTCALL, nullptr},
  {"distill_loss", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(distill_loss)), METH_FASTCALL, nullptr},
  {"linear_loss", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_loss)), METH_FASTCALL, nullptr},
  {"log_probs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(log_probs)), METH_FASTCALL, nullptr},
  {"linear_log_probs", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_log_probs)), METH_FASTCALL, nullptr},
  {"clip_gradients", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(clip_gradients)), METH_FASTCALL, nullptr},
  {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "b2fil_torch",
                          "Native call path of libb2fil for torch tensors.", -1, module_methods};

}  // namespace

PyMODINIT_FUNC PyInit_b2fil_torch()
{
  if (PyType_Ready(&device_call_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (!m) return nullptr;
  if (PyModule_AddObjectRef(m, "DeviceCall", reinterpret_cast<PyObject*>(&device_call_type)) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
