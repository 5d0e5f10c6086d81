// xgboost._encoder: the leaf encoder's C entries called with torch tensors.
// The small calls are a few microseconds of kernel, less than argument checks,
// allocations and a foreign-function call cost in Python (a lookup of 16 rows:
// 12.3 us of host time that way), so those are here.
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <string>

#include "mgb_kernels.h"

namespace {

using at::Tensor;

PyObject* g_error = nullptr;  // xgboost.XGBoostError

[[noreturn]] void type_error(const std::string& message) {
  PyErr_SetString(PyExc_TypeError, message.c_str());
  throw python_error();
}

[[noreturn]] void value_error(const std::string& message) {
  PyErr_SetString(PyExc_ValueError, message.c_str());
  throw python_error();
}

void check(int status) {
  if (status == 0) return;
  PyErr_SetString(g_error, mgb_last_error());
  throw python_error();
}

std::string text(at::IntArrayRef shape) {
  std::string s = "(";
  for (size_t k = 0; k < shape.size(); ++k) s += (k ? ", " : "") + std::to_string(shape[k]);
  return s + ")";
}

[[noreturn]] void not_implemented(const std::string& message) {
  PyErr_SetString(PyExc_NotImplementedError, message.c_str());
  throw python_error();
}

// The calls are no operators of torch's, so what records operators does not see
// them: a trace would hold their results as constants.
bool recording() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  if (c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer)) return true;
  return c10::impl::dispatch_mode_enabled() &&
         (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL));
}

// What a view that torch negates on reading stands for is a copy.
Tensor tensor(const char* name, PyObject* object) {
  if (!THPVariable_Check(object))
    type_error(std::string(name) + " must be a torch.Tensor, got " + Py_TYPE(object)->tp_name);
  if (recording()) not_implemented("the encoder's operators cannot be traced");
  const Tensor& t = THPVariable_Unpack(object);
  // The tangent would be lost, and a tensor without one counts as constant.
  if (t._fw_grad(0).defined())
    not_implemented(std::string(name) + " has a forward-mode tangent, which the encoder's operators do not carry");
  return t.is_neg() ? t.resolve_neg() : t;
}

// A tensor of one of the three types on a GPU.
int dtype(const char* name, const Tensor& t) {
  int code;
  switch (t.scalar_type()) {
    case at::kFloat: code = MGB_F32; break;
    case at::kHalf: code = MGB_F16; break;
    case at::kBFloat16: code = MGB_BF16; break;
    default: type_error(std::string(name) + " must be float32, float16 or bfloat16, is " + toString(t.scalar_type()));
  }
  if (!t.is_cuda()) value_error(std::string(name) + " must be on a GPU, is on " + t.device().str());
  return code;
}

void same_device(const Tensor& t, const char* name, const Tensor& other) {
  if (other.device() != t.device())
    value_error(std::string(name) + " must be on " + t.device().str() + ", is on " + other.device().str());
}

// t, or a copy of it, as rows of its last axis at one distance.
struct Rows {
  Tensor t;
  int64_t stride;
};

Rows rows_of(const Tensor& t) {
  const int64_t dim = t.size(-1);
  if (t.is_contiguous()) return {t, dim};
  if (t.dim() == 2 && (t.stride(1) == 1 || dim == 1)) return {t, t.stride(0)};
  return {t.contiguous(), dim};
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}

Tensor workspace(size_t bytes, const Tensor& like) { return empty({(int64_t)bytes}, at::kByte, like); }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int64_t count(at::IntArrayRef shape) {
  int64_t n = 1;
  for (int64_t s : shape) n *= s;
  return n;
}

double real(PyObject* object) {
  const double v = PyFloat_AsDouble(object);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

int64_t integer(PyObject* object) {
  const int64_t v = PyLong_AsLongLong(object);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

bool truth(PyObject* object) {
  const int v = PyObject_IsTrue(object);
  if (v < 0) throw python_error();
  return v != 0;
}

void arguments(const char* name, Py_ssize_t got, Py_ssize_t want) {
  if (got != want)
    type_error(std::string(name) + " takes " + std::to_string(want) + " arguments, got " + std::to_string(got));
}

// Tokens without gaps, their rows' count and length.
struct Tokens {
  Tensor t;
  int bytes;
  at::IntArrayRef rows;
  int64_t bag;
};

Tokens tokens_of(PyObject* object, bool pool) {
  const Tensor t = tensor("tokens", object);
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong)
    type_error(std::string("tokens must be int32 or int64, are ") + toString(t.scalar_type()));
  if (pool && t.dim() == 0) value_error("pool needs tokens with an axis to sum over");
  Tokens out{t.is_contiguous() ? t : t.contiguous(), t.scalar_type() == at::kInt ? 4 : 8, {}, 1};
  out.rows = out.t.sizes();
  if (pool) {
    out.bag = out.rows.back();
    out.rows = out.rows.slice(0, out.rows.size() - 1);
  }
  return out;
}

at::DimVector with_dim(at::IntArrayRef rows, int64_t dim) {
  at::DimVector shape(rows.begin(), rows.end());
  shape.push_back(dim);
  return shape;
}

// (weight, tokens, scale, pool)
PyObject* lookup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("lookup", n, 4);
  const Tensor table = tensor("weight", args[0]);
  const int type = dtype("weight", table);
  if (table.dim() != 2) value_error("weight must be a table of rows, has shape " + text(table.sizes()));
  const Tokens tokens = tokens_of(args[1], truth(args[3]));
  same_device(table, "tokens", tokens.t);
  const Rows weight = rows_of(table);
  const int64_t dim = table.size(1);
  const c10::DeviceGuard guard(table.device());
  Tensor out = empty(with_dim(tokens.rows, dim), table.scalar_type(), table);
  check(mgb_embedding_lookup(out.data_ptr(), weight.t.data_ptr(), tokens.t.data_ptr(), count(tokens.rows), tokens.bag,
                             table.size(0), dim, weight.stride, (float)real(args[2]), type, tokens.bytes,
                             stream_of(table)));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (grad, tokens, num_embeddings, scale, pool)
PyObject* lookup_gradient(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("lookup_gradient", n, 5);
  const Tensor given = tensor("grad", args[0]);
  const int type = dtype("grad", given);
  const Tokens tokens = tokens_of(args[1], truth(args[4]));
  same_device(given, "tokens", tokens.t);
  if (given.dim() < 1 || given.sizes().slice(0, given.dim() - 1) != tokens.rows)
    value_error("grad must have shape " + text(tokens.rows) + " and a last axis for these tokens, has " +
                text(given.sizes()));
  const int64_t table = integer(args[2]);
  if (table < 1) value_error("num_embeddings must be at least 1, is " + std::to_string(table));
  const Rows grad = rows_of(given);
  const int64_t dim = given.size(-1);
  const c10::DeviceGuard guard(given.device());
  const size_t need = mgb_embedding_gradient_workspace_bytes(count(tokens.rows), tokens.bag, table, dim, type);
  Tensor out = empty({table, dim}, given.scalar_type(), given), space = workspace(need, given);
  check(mgb_embedding_gradient(out.data_ptr(), grad.t.data_ptr(), tokens.t.data_ptr(), count(tokens.rows), tokens.bag,
                               table, dim, grad.stride, (float)real(args[3]), type, tokens.bytes, space.data_ptr(),
                               need, stream_of(given)));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

void check_normalised(const Tensor& x) {
  if (x.dim() == 0 || x.size(-1) == 0)
    value_error("x must have a last axis to normalise, has shape " + text(x.sizes()));
}

// A parameter row of layer norm without gaps, or none.
Tensor parameter(const char* name, PyObject* object, const Tensor& x) {
  if (object == Py_None) return {};
  const Tensor t = tensor(name, object);
  dtype(name, t);
  if (t.dim() != 1 || t.size(0) != x.size(-1))
    value_error(std::string(name) + " must have shape (" + std::to_string(x.size(-1)) + "), has " + text(t.sizes()));
  same_device(x, name, t);
  return t.is_contiguous() ? t : t.contiguous();
}

int weight_type(const Tensor& x, const Tensor& weight) {
  const int type = dtype("weight", weight);
  if (type != MGB_F32 && weight.scalar_type() != x.scalar_type())
    type_error(std::string("weight must be ") + toString(x.scalar_type()) + " or Float, is " +
               toString(weight.scalar_type()));
  return type;
}

void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// (x, weight or None, bias or None, eps)
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("norm", n, 4);
  const Tensor given = tensor("x", args[0]);
  const int type = dtype("x", given);
  check_normalised(given);
  const Tensor weight = parameter("weight", args[1], given), bias = parameter("bias", args[2], given);
  int wtype = type;
  if (weight.defined()) wtype = weight_type(given, weight);
  if (bias.defined()) {
    if (!weight.defined()) value_error("a bias needs a weight");
    if (bias.scalar_type() != weight.scalar_type())
      type_error(std::string("bias must be ") + toString(weight.scalar_type()) + " as the weight, is " +
                 toString(bias.scalar_type()));
  }
  const Rows x = rows_of(given);
  const at::IntArrayRef shape = given.sizes(), rows = shape.slice(0, shape.size() - 1);
  const c10::DeviceGuard guard(given.device());
  Tensor y = empty(shape, given.scalar_type(), given);
  Tensor mean = empty(rows, at::kFloat, given), rstd = empty(rows, at::kFloat, given);
  check(mgb_layer_norm(y.data_ptr(), (float*)mean.data_ptr(), (float*)rstd.data_ptr(), x.t.data_ptr(), pointer(weight),
                       pointer(bias), count(rows), given.size(-1), x.stride, (float)real(args[3]), type, wtype,
                       stream_of(given)));
  return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(mean)),
                       THPVariable_Wrap(std::move(rstd)));
  END_HANDLE_TH_ERRORS
}

// (grad, x, mean, rstd, weight or None)
PyObject* norm_gradient(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("norm_gradient", n, 5);
  const Tensor g = tensor("grad", args[0]), given = tensor("x", args[1]);
  const int type = dtype("x", given);
  if (dtype("grad", g) != type || g.sizes() != given.sizes())
    value_error(std::string("grad must be like x, ") + toString(given.scalar_type()) + " " + text(given.sizes()) +
                ", is " + toString(g.scalar_type()) + " " + text(g.sizes()));
  check_normalised(given);
  same_device(given, "grad", g);
  const at::IntArrayRef shape = given.sizes(), rows = shape.slice(0, shape.size() - 1);
  const char* names[2] = {"mean", "rstd"};
  Tensor statistics[2];
  for (int k = 0; k < 2; ++k) {
    const Tensor t = tensor(names[k], args[2 + k]);
    if (t.scalar_type() != at::kFloat || t.sizes() != rows)
      value_error(std::string(names[k]) + " must be Float " + text(rows) + ", is " + toString(t.scalar_type()) + " " +
                  text(t.sizes()));
    same_device(given, names[k], t);
    statistics[k] = t.is_contiguous() ? t : t.contiguous();
  }
  const Tensor weight = parameter("weight", args[4], given);
  const int wtype = weight.defined() ? weight_type(given, weight) : type;
  const Rows x = rows_of(given), grad = rows_of(g);
  const int64_t dim = given.size(-1);
  const c10::DeviceGuard guard(given.device());
  Tensor dx = empty(shape, given.scalar_type(), given), dweight, dbias, space;
  size_t need = 0;
  if (weight.defined()) {
    dweight = empty({dim}, weight.scalar_type(), given);
    dbias = empty({dim}, weight.scalar_type(), given);
    need = mgb_layer_norm_gradient_workspace_bytes(count(rows), dim, type);
    space = workspace(need, given);
  }
  check(mgb_layer_norm_gradient(dx.data_ptr(), pointer(dweight), pointer(dbias), grad.t.data_ptr(), x.t.data_ptr(),
                                (const float*)statistics[0].data_ptr(), (const float*)statistics[1].data_ptr(),
                                pointer(weight), count(rows), dim, grad.stride, x.stride, type, wtype, pointer(space),
                                need, stream_of(given)));
  if (!weight.defined()) return Py_BuildValue("(NOO)", THPVariable_Wrap(std::move(dx)), Py_None, Py_None);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(dx)), THPVariable_Wrap(std::move(dweight)),
                       THPVariable_Wrap(std::move(dbias)));
  END_HANDLE_TH_ERRORS
}

// (update, steps, coefficients, eps)
PyObject* orthogonalize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("orthogonalize", n, 4);
  const Tensor given = tensor("update", args[0]);
  const int type = dtype("update", given);
  if (given.dim() < 2) value_error("update must be a matrix, has shape " + text(given.sizes()));
  float coefficients[3];
  THPObjectPtr sequence(PySequence_Fast(args[2], "coefficients must be three numbers"));
  if (!sequence) throw python_error();
  if (PySequence_Fast_GET_SIZE(sequence.get()) != 3) value_error("coefficients must be three numbers");
  for (int k = 0; k < 3; ++k) coefficients[k] = (float)real(PySequence_Fast_GET_ITEM(sequence.get(), k));
  const int64_t steps = integer(args[1]);
  if (steps < 1 || steps > 100) value_error("steps must be 1 to 100, is " + std::to_string(steps));
  const int64_t rows = given.size(-2), columns = given.size(-1);
  const int64_t batch = count(given.sizes().slice(0, given.dim() - 2));
  Rows update = {given, columns};
  int64_t batch_stride = rows * columns;
  if (given.dim() == 2) {
    update = rows_of(given);
  } else if (!given.is_contiguous()) {
    update.t = given.contiguous();
  }
  const c10::DeviceGuard guard(given.device());
  const size_t need = mgb_orthogonalize_workspace_bytes(batch, rows, columns);
  Tensor out = empty(given.sizes(), given.scalar_type(), given), space = workspace(need, given);
  check(mgb_orthogonalize(out.data_ptr(), update.t.data_ptr(), batch, rows, columns, update.stride, batch_stride,
                          (int)steps, coefficients, (float)real(args[3]), type, space.data_ptr(), need,
                          stream_of(given)));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

#define ENTRY(fn) {#fn, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {ENTRY(lookup), ENTRY(lookup_gradient), ENTRY(norm), ENTRY(norm_gradient),
                           ENTRY(orthogonalize), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_encoder", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__encoder(void) {
  THPObjectPtr core(PyImport_ImportModule("xgboost.core"));
  if (!core) return nullptr;
  g_error = PyObject_GetAttrString(core.get(), "XGBoostError");
  if (!g_error) return nullptr;
  return PyModule_Create(&g_module);
}
