// xgboost._encoder: the leaf encoder's C entries called with torch tensors.
// The small calls are a few microseconds of kernel, less than argument checks,
// allocations and a foreign-function call cost in Python (a lookup of 16 rows:
// 12.3 us of host time that way), so those are here.
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cstring>
#include <string>
#include <utility>
#include <vector>

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

int activation_of(PyObject* object) {
  const char* name = PyUnicode_Check(object) ? PyUnicode_AsUTF8(object) : nullptr;
  if (PyErr_Occurred()) throw python_error();
  if (name && !strcmp(name, "silu")) return MGB_SILU;
  if (name && !strcmp(name, "gelu")) return MGB_GELU;
  value_error("activation must be \"silu\" or \"gelu\"");
}

// The block's matrices, in x's type and on its device.
struct Matrices {
  Rows gate, up, down;
  int64_t dim, hidden;
};

Matrices matrices_of(const Tensor& x, PyObject* const* args) {
  if (x.dim() == 0 || x.size(-1) == 0) value_error("x must have a last axis, has shape " + text(x.sizes()));
  const char* names[3] = {"gate", "up", "down"};
  Tensor t[3];
  for (int k = 0; k < 3; ++k) {
    t[k] = tensor(names[k], args[k]);
    dtype(names[k], t[k]);
    if (t[k].scalar_type() != x.scalar_type())
      type_error(std::string(names[k]) + " must be " + toString(x.scalar_type()) + " as x, is " +
                 toString(t[k].scalar_type()));
    same_device(x, names[k], t[k]);
  }
  const int64_t dim = x.size(-1), hidden = t[0].dim() == 2 ? t[0].size(0) : 0;
  if (t[0].dim() != 2 || t[0].size(1) != dim || hidden == 0)
    value_error("gate must have shape (hidden, " + std::to_string(dim) + "), has " + text(t[0].sizes()));
  if (t[1].sizes() != t[0].sizes()) value_error("up must have shape " + text(t[0].sizes()) + ", has " + text(t[1].sizes()));
  if (t[2].dim() != 2 || t[2].size(0) != dim || t[2].size(1) != hidden)
    value_error("down must have shape (" + std::to_string(dim) + ", " + std::to_string(hidden) + "), has " +
                text(t[2].sizes()));
  return {rows_of(t[0]), rows_of(t[1]), rows_of(t[2]), dim, hidden};
}

at::IntArrayRef rows_shape(const Tensor& x) { return x.sizes().slice(0, x.dim() - 1); }

// (x, gate, up, down, activation, keep)
PyObject* feed_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("feed_forward", n, 6);
  const Tensor given = tensor("x", args[0]);
  const int type = dtype("x", given);
  const Matrices m = matrices_of(given, args + 1);
  const int activation = activation_of(args[4]);
  const bool keep = truth(args[5]);
  const Rows x = rows_of(given);
  const c10::DeviceGuard guard(given.device());
  Tensor y = empty(given.sizes(), given.scalar_type(), given), kept;
  if (keep) {
    at::DimVector shape = with_dim(rows_shape(given), 2);
    shape.push_back(m.hidden);
    kept = empty(shape, at::kFloat, given);
  }
  const MgbFeedForward p = {y.data_ptr(), (float*)pointer(kept), x.t.data_ptr(), m.gate.t.data_ptr(), m.up.t.data_ptr(),
                            m.down.t.data_ptr(), count(rows_shape(given)), m.dim, m.hidden, x.stride, m.gate.stride,
                            m.up.stride, m.down.stride, activation, type};
  const size_t need = mgb_feed_forward_workspace_bytes(&p);
  const Tensor space = workspace(need, given);
  check(mgb_feed_forward(&p, space.data_ptr(), need, stream_of(given)));
  if (!keep) return THPVariable_Wrap(std::move(y));
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(kept)));
  END_HANDLE_TH_ERRORS
}

// (grad, x, kept, gate, up, down, activation, which of the four are wanted)
PyObject* feed_forward_gradient(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("feed_forward_gradient", n, 8);
  const Tensor g = tensor("grad", args[0]), given = tensor("x", args[1]);
  const int type = dtype("x", given);
  if (dtype("grad", g) != type || g.sizes() != given.sizes())
    value_error(std::string("grad must be like x, ") + toString(given.scalar_type()) + " " + text(given.sizes()) +
                ", is " + toString(g.scalar_type()) + " " + text(g.sizes()));
  same_device(given, "grad", g);
  const Matrices m = matrices_of(given, args + 3);
  at::DimVector kept_shape = with_dim(rows_shape(given), 2);
  kept_shape.push_back(m.hidden);
  Tensor kept = tensor("kept", args[2]);
  if (kept.scalar_type() != at::kFloat || kept.sizes() != at::IntArrayRef(kept_shape))
    value_error("kept must be Float " + text(kept_shape) + ", is " + toString(kept.scalar_type()) + " " +
                text(kept.sizes()));
  same_device(given, "kept", kept);
  if (!kept.is_contiguous()) kept = kept.contiguous();
  const int activation = activation_of(args[6]);
  const int64_t wanted = integer(args[7]);
  const Rows x = rows_of(given), grad = rows_of(g);
  const c10::DeviceGuard guard(given.device());
  Tensor out[4];
  if (wanted & 1) out[0] = empty(given.sizes(), given.scalar_type(), given);
  if (wanted & 2) out[1] = empty({m.hidden, m.dim}, given.scalar_type(), given);
  if (wanted & 4) out[2] = empty({m.hidden, m.dim}, given.scalar_type(), given);
  if (wanted & 8) out[3] = empty({m.dim, m.hidden}, given.scalar_type(), given);
  const MgbFeedForwardGradient p = {pointer(out[0]), pointer(out[1]), pointer(out[2]), pointer(out[3]),
                                    grad.t.data_ptr(), x.t.data_ptr(), (const float*)kept.data_ptr(),
                                    m.gate.t.data_ptr(), m.up.t.data_ptr(), m.down.t.data_ptr(),
                                    count(rows_shape(given)), m.dim, m.hidden, grad.stride, x.stride, m.gate.stride,
                                    m.up.stride, m.down.stride, activation, type};
  const size_t need = mgb_feed_forward_gradient_workspace_bytes(&p);
  const Tensor space = workspace(need, given);
  check(mgb_feed_forward_gradient(&p, space.data_ptr(), need, stream_of(given)));
  PyObject* result = PyTuple_New(4);
  if (!result) throw python_error();
  for (int k = 0; k < 4; ++k) {
    PyObject* item = Py_None;
    if (out[k].defined()) item = THPVariable_Wrap(std::move(out[k]));
    else Py_INCREF(item);
    PyTuple_SET_ITEM(result, k, item);
  }
  return result;
  END_HANDLE_TH_ERRORS
}

constexpr int64_t kBlock = 128;

// (values, scales) as quantize_blocks gives them: whole blocks in 8 bits, their
// scales in rows of whole words.  Others are laid out anew.
struct Blocks {
  Tensor values, scales;
  MgbBlocks blocks;
};

Blocks blocks_of(const char* name, PyObject* values_object, PyObject* scales_object) {
  Tensor values = tensor(name, values_object), scales = tensor(name, scales_object);
  if (values.scalar_type() != at::kFloat8_e4m3fn)
    type_error(std::string(name) + "'s values must be float8_e4m3fn, are " + toString(values.scalar_type()));
  if (scales.scalar_type() != at::kFloat8_e8m0fnu)
    type_error(std::string(name) + "'s scales must be float8_e8m0fnu, are " + toString(scales.scalar_type()));
  if (!values.is_cuda()) value_error(std::string(name) + " must be on a GPU, is on " + values.device().str());
  same_device(values, "its scales", scales);
  if (values.dim() == 0 || values.size(-1) == 0 || values.size(-1) % kBlock)
    value_error(std::string(name) + "'s values must be rows of whole blocks of 128, have shape " + text(values.sizes()));
  const int64_t blocks = values.size(-1) / kBlock;
  at::DimVector want(values.sizes().begin(), values.sizes().end());
  want.back() = blocks;
  if (scales.sizes() != at::IntArrayRef(want))
    value_error(std::string(name) + "'s scales must have shape " + text(want) + ", have " + text(scales.sizes()));
  Rows v = rows_of(values);
  if (v.stride % 16 || v.stride < values.size(-1) || v.stride > (int64_t(1) << 20) || (uintptr_t)v.t.data_ptr() % 16)
    v = {values.clone(at::MemoryFormat::Contiguous), values.size(-1)};
  const int64_t rows = count(values.sizes().slice(0, values.dim() - 1)), words = (blocks + 3) / 4 * 4;
  // Rows of scales: the view that quantize_blocks gives has whole words behind it.
  bool well = scales.stride(-1) == 1 && (uintptr_t)scales.data_ptr() % 4 == 0;
  int64_t step = words;
  for (int64_t axis = scales.dim() - 2; axis >= 0 && well; --axis) {
    well = scales.size(axis) <= 1 || scales.stride(axis) == step;
    step *= scales.size(axis);
  }
  well = well && (scales.storage_offset() + rows * words) * (int64_t)scales.element_size() <= (int64_t)scales.storage().nbytes();
  if (!well) {
    at::DimVector wide(want);
    wide.back() = words;
    const c10::DeviceGuard guard(values.device());
    Tensor copy = empty(wide, at::kFloat8_e8m0fnu, scales);
    copy.narrow(-1, 0, blocks).copy_(scales);
    scales = copy;
  }
  return {v.t, scales, {v.t.data_ptr(), scales.data_ptr(), rows, blocks, v.stride, words}};
}

// (x) -> values (..., whole blocks), scales (..., blocks)
PyObject* quantize_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("quantize_blocks", n, 1);
  const Tensor given = tensor("x", args[0]);
  const int type = dtype("x", given);
  if (given.dim() == 0 || given.size(-1) == 0) value_error("x must have a last axis, has shape " + text(given.sizes()));
  const Rows x = rows_of(given);
  const int64_t dim = given.size(-1), blocks = (dim + kBlock - 1) / kBlock, words = (blocks + 3) / 4 * 4;
  const c10::DeviceGuard guard(given.device());
  Tensor values = empty(with_dim(rows_shape(given), blocks * kBlock), at::kFloat8_e4m3fn, given);
  Tensor scales = empty(with_dim(rows_shape(given), words), at::kFloat8_e8m0fnu, given);
  const MgbBlocks out = {values.data_ptr(), scales.data_ptr(), count(rows_shape(given)), blocks, blocks * kBlock, words};
  check(mgb_quantize_blocks(&out, x.t.data_ptr(), dim, x.stride, type, stream_of(given)));
  if (words != blocks) scales = scales.narrow(-1, 0, blocks);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(values)), THPVariable_Wrap(std::move(scales)));
  END_HANDLE_TH_ERRORS
}

at::ScalarType result_type(PyObject* object, int* code) {
  if (!THPDtype_Check(object)) type_error(std::string("dtype must be a torch.dtype, got ") + Py_TYPE(object)->tp_name);
  const at::ScalarType type = reinterpret_cast<THPDtype*>(object)->scalar_type;
  switch (type) {
    case at::kFloat: *code = MGB_F32; break;
    case at::kHalf: *code = MGB_F16; break;
    case at::kBFloat16: *code = MGB_BF16; break;
    default: type_error(std::string("dtype must be float32, float16 or bfloat16, is ") + toString(type));
  }
  return type;
}

// (x values, x scales, weight values, weight scales, dtype)
PyObject* block_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("block_matmul", n, 5);
  int type = 0;
  const at::ScalarType result = result_type(args[4], &type);
  const Blocks x = blocks_of("x", args[0], args[1]), weight = blocks_of("weight", args[2], args[3]);
  same_device(x.values, "weight", weight.values);
  if (weight.values.dim() != 2) value_error("weight must be a matrix, has shape " + text(weight.values.sizes()));
  if (x.blocks.blocks != weight.blocks.blocks)
    value_error("x and weight must have rows of as many blocks, have " + std::to_string(x.blocks.blocks) + " and " +
                std::to_string(weight.blocks.blocks));
  const c10::DeviceGuard guard(x.values.device());
  Tensor out = empty(with_dim(rows_shape(x.values), weight.blocks.rows), result, x.values);
  const MgbBlockMatmul p = {out.data_ptr(), x.blocks, weight.blocks, type};
  const size_t need = mgb_block_matmul_workspace_bytes(&p);
  const Tensor space = workspace(need, x.values);
  check(mgb_block_matmul(&p, space.data_ptr(), need, stream_of(x.values)));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (x, gate values, scales, up values, scales, down values, scales, activation)
PyObject* block_feed_forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("block_feed_forward", n, 8);
  const Tensor given = tensor("x", args[0]);
  const int type = dtype("x", given);
  if (given.dim() == 0 || given.size(-1) == 0) value_error("x must have a last axis, has shape " + text(given.sizes()));
  const char* names[3] = {"gate", "up", "down"};
  std::vector<Blocks> m;
  for (int k = 0; k < 3; ++k) {
    m.push_back(blocks_of(names[k], args[1 + 2 * k], args[2 + 2 * k]));
    same_device(given, names[k], m[k].values);
    if (m[k].values.dim() != 2)
      value_error(std::string(names[k]) + " must be a matrix, has shape " + text(m[k].values.sizes()));
  }
  const int64_t dim = given.size(-1), hidden = m[0].blocks.rows;
  const int64_t blocks = (dim + kBlock - 1) / kBlock, hidden_blocks = (hidden + kBlock - 1) / kBlock;
  if (hidden == 0 || m[0].blocks.blocks != blocks)
    value_error("gate must have rows of " + std::to_string(blocks) + " blocks, has shape " + text(m[0].values.sizes()));
  if (m[1].values.sizes() != m[0].values.sizes())
    value_error("up must have shape " + text(m[0].values.sizes()) + ", has " + text(m[1].values.sizes()));
  if (m[2].blocks.rows != dim || m[2].blocks.blocks != hidden_blocks)
    value_error("down must have " + std::to_string(dim) + " rows of " + std::to_string(hidden_blocks) +
                " blocks, has shape " + text(m[2].values.sizes()));
  if (m[0].blocks.stride != m[1].blocks.stride)
    for (int k = 0; k < 2; ++k)
      if (m[k].blocks.stride != m[k].values.size(-1)) {
        m[k].values = m[k].values.clone(at::MemoryFormat::Contiguous);
        m[k].blocks.values = m[k].values.data_ptr();
        m[k].blocks.stride = m[k].values.size(-1);
      }
  const int activation = activation_of(args[7]);
  const Rows x = rows_of(given);
  const c10::DeviceGuard guard(given.device());
  Tensor y = empty(given.sizes(), given.scalar_type(), given);
  const MgbBlockFeedForward p = {y.data_ptr(), x.t.data_ptr(), m[0].blocks, m[1].blocks, m[2].blocks,
                                 count(rows_shape(given)), dim, hidden, x.stride, activation, type};
  const size_t need = mgb_block_feed_forward_workspace_bytes(&p);
  const Tensor space = workspace(need, given);
  check(mgb_block_feed_forward(&p, space.data_ptr(), need, stream_of(given)));
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// Rows of logits and a teacher's entries for each.
struct Distillation {
  Rows logits, values, indices;
  at::IntArrayRef rows;
  MgbDistillation p;
};

Distillation distillation_of(const Tensor& logits, PyObject* values_object, PyObject* indices_object, PyObject* temperature) {
  Distillation d = {};
  const int type = dtype("logits", logits);
  if (logits.dim() == 0 || logits.size(-1) == 0)
    value_error("logits must have a last axis, have shape " + text(logits.sizes()));
  const Tensor values = tensor("values", values_object), indices = tensor("indices", indices_object);
  const int value_type = dtype("values", values);
  if (indices.scalar_type() != at::kInt && indices.scalar_type() != at::kLong)
    type_error(std::string("indices must be int32 or int64, are ") + toString(indices.scalar_type()));
  same_device(logits, "values", values);
  same_device(logits, "indices", indices);
  d.rows = rows_shape(logits);
  if (values.dim() != logits.dim() || rows_shape(values) != d.rows)
    value_error("values must have shape " + text(d.rows) + " and a last axis for these logits, have " + text(values.sizes()));
  if (indices.sizes() != values.sizes())
    value_error("indices must have shape " + text(values.sizes()) + " as values, have " + text(indices.sizes()));
  if (values.size(-1) > 1024)
    value_error("a teacher's row must have at most 1,024 entries, has " + std::to_string(values.size(-1)));
  const double t = real(temperature);
  if (!((float)t > 0.0f && (float)t <= 3.4e38f)) value_error("temperature must be positive, is " + std::to_string(t));
  d.logits = rows_of(logits);
  d.values = rows_of(values);
  d.indices = rows_of(indices);
  d.p.logits = d.logits.t.data_ptr();
  d.p.values = d.values.t.data_ptr();
  d.p.indices = d.indices.t.data_ptr();
  d.p.rows = count(d.rows);
  d.p.classes = logits.size(-1);
  d.p.top = values.size(-1);
  d.p.stride = d.logits.stride;
  d.p.value_stride = d.values.stride;
  d.p.index_stride = d.indices.stride;
  d.p.temperature = (float)t;
  d.p.dtype = type;
  d.p.value_dtype = value_type;
  d.p.index_bytes = indices.scalar_type() == at::kInt ? 4 : 8;
  return d;
}

// (logits, values, indices, temperature) -> loss, lse
PyObject* distillation_loss(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("distillation_loss", n, 4);
  const Tensor given = tensor("logits", args[0]);
  Distillation d = distillation_of(given, args[1], args[2], args[3]);
  const c10::DeviceGuard guard(given.device());
  Tensor loss = empty(d.rows, at::kFloat, given), lse = empty(d.rows, at::kFloat, given);
  d.p.loss = (float*)loss.data_ptr();
  d.p.lse = (float*)lse.data_ptr();
  const size_t need = mgb_distillation_loss_workspace_bytes(&d.p);
  const Tensor space = workspace(need, given);
  check(mgb_distillation_loss(&d.p, space.data_ptr(), need, stream_of(given)));
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(loss)), THPVariable_Wrap(std::move(lse)));
  END_HANDLE_TH_ERRORS
}

// (grad, logits, lse, values, indices, temperature)
PyObject* distillation_gradient(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("distillation_gradient", n, 6);
  Tensor grad = tensor("grad", args[0]);
  const Tensor given = tensor("logits", args[1]);
  Tensor lse = tensor("lse", args[2]);
  Distillation d = distillation_of(given, args[3], args[4], args[5]);
  for (const auto& [name, t] : {std::pair<const char*, Tensor*>{"grad", &grad}, {"lse", &lse}}) {
    if (t->scalar_type() != at::kFloat || t->sizes() != d.rows)
      value_error(std::string(name) + " must be Float " + text(d.rows) + ", is " + toString(t->scalar_type()) + " " +
                  text(t->sizes()));
    same_device(given, name, *t);
  }
  if (!lse.is_contiguous()) lse = lse.contiguous();
  // The gradient of a sum is one value for all rows.
  d.p.grad_stride = grad.dim() == 1 ? grad.stride(0) : 1;
  if (grad.dim() != 1 && !grad.is_contiguous()) grad = grad.contiguous();
  const c10::DeviceGuard guard(given.device());
  Tensor out = empty(given.sizes(), given.scalar_type(), given);
  d.p.dlogits = out.data_ptr();
  d.p.grad = (const float*)grad.data_ptr();
  d.p.lse = (float*)lse.data_ptr();
  check(mgb_distillation_gradient(&d.p, stream_of(given)));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (result of a pass that has a backward pass)
// What adds up a leaf's gradient runs on the stream of the first graph that holds the
// leaf, for as long as a graph does, be it of torch's operators.  If that is the default
// stream, a backward pass that is captured would have it wait for the capture, which ends
// the process.
PyObject* check_capture(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments("check_capture", n, 1);
  const Tensor& result = THPVariable_Unpack(args[0]);
  const c10::DeviceGuard guard(result.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None && result.grad_fn())
    for (const torch::autograd::Edge& edge : result.grad_fn()->next_edges()) {
      const auto* leaf = dynamic_cast<const torch::autograd::AccumulateGrad*>(edge.function.get());
      if (leaf && leaf->input_metadata(0).stream().id() == 0) {
        PyErr_SetString(PyExc_RuntimeError,
                        "a graph made on the default stream still holds a leaf of this capture: its backward pass cannot "
                        "be captured; drop the eager pass's results first, or run it on another stream");
        throw python_error();
      }
    }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define ENTRY(fn) {#fn, (PyCFunction)(void (*)(void))fn, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {ENTRY(lookup), ENTRY(lookup_gradient), ENTRY(norm), ENTRY(norm_gradient),
                           ENTRY(orthogonalize), ENTRY(feed_forward), ENTRY(feed_forward_gradient),
                           ENTRY(quantize_blocks), ENTRY(block_matmul), ENTRY(block_feed_forward), ENTRY(distillation_loss),
                           ENTRY(distillation_gradient), ENTRY(check_capture), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_encoder", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__encoder(void) {
  THPObjectPtr core(PyImport_ImportModule("xgboost.core"));
  if (!core) return nullptr;
  g_error = PyObject_GetAttrString(core.get(), "XGBoostError");
  if (!g_error) return nullptr;
  return PyModule_Create(&g_module);
}
