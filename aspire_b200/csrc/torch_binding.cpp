// The feed-forward operators' Python calls: argument checks, outputs and the
// call of the C ABI (include/aspire_b200.h) on torch's current stream.
//
// A decode step's calls are a few microseconds on the device, less than the
// same checks take attribute by attribute in Python, so they are made here on
// the tensors themselves.  Host time of one call, Python -> here: product 10.2
// -> 5.1 us, routing 15.1 -> 7.1, combine 10.4 -> 3.8 (an output's allocation
// alone is 2.4).  Everything a kernel needs still crosses the C ABI, through
// the entry points of the library that the package has loaded (bind()); this
// file launches nothing.
#include <Python.h>

#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <utility>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "aspire_b200.h"

namespace {

using at::Tensor;

// The C ABI's entry points, set by bind().
struct {
  decltype(&aspire_last_error) last_error;
  decltype(&aspire_w4_linear) w4_linear;
  decltype(&aspire_moe_route) moe_route;
  decltype(&aspire_moe_route_workspace) moe_route_workspace;
  decltype(&aspire_moe_route_grad) moe_route_grad;
  decltype(&aspire_moe_dispatch) moe_dispatch;
  decltype(&aspire_moe_combine) moe_combine;
  decltype(&aspire_moe_combine_grad) moe_combine_grad;
} abi = {};

// A refused argument; becomes ValueError.
struct Invalid : std::invalid_argument {
  using std::invalid_argument::invalid_argument;
};

void require(bool ok, const char* what) {
  if (!ok) throw Invalid(what);
}

void check(int rc, const char* what) {
  if (rc == ASPIRE_OK) return;
  const std::string msg = abi.last_error();
  if (rc == ASPIRE_ERR_INVALID) throw Invalid(what + (": " + msg));
  throw std::runtime_error(what + (" failed (" + std::to_string(rc) + "): " + msg));
}

// Runs `f(stream)` with the tensor's device current.
template <typename F>
void on_device(const Tensor& t, F&& f) {
  const c10::cuda::CUDAGuard guard(t.device());
  f(static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()));
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return ASPIRE_T_F32;
    case at::kBFloat16: return ASPIRE_T_BF16;
    case at::kHalf: return ASPIRE_T_F16;
    default: return -1;
  }
}

const Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw Invalid("a tensor is required");
  const Tensor& t = THPVariable_Unpack(o);
  // A tangent would be dropped, not carried through.
  require(!t._fw_grad(0).defined(), "the feed-forward operators have no forward-mode derivative");
  return t;
}
// NULL for None.
const Tensor* optional(PyObject* o) { return o == Py_None ? nullptr : &tensor(o); }
long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Invalid("an integer is required");
  }
  return v;
}

uint32_t* status_word(const Tensor* s, const Tensor& like) {
  if (!s) return nullptr;
  require(s->device() == like.device() && s->numel() >= 1 && s->element_size() == 4,
          "status must be a 32-bit tensor on the operands' device");
  return static_cast<uint32_t*>(s->data_ptr());
}

// ------------------------------------------------------------------- outputs
// Rows of `bytes` bytes each, `pitch` (at least as many) bytes apart.
struct Block {
  uintptr_t at;
  int64_t rows, bytes, pitch;
};

Block block_of(const Tensor& t, int64_t stride) {
  const int64_t size = t.element_size();
  return {reinterpret_cast<uintptr_t>(t.data_ptr()), t.size(0), t.size(1) * size, stride * size};
}

// Whether two blocks have a byte in common.  Blocks whose address ranges cross
// may lie between one another's rows (columns of one buffer): their rows are
// then compared in order of address.
bool share(const Block& a, const Block& b) {
  if (a.rows == 0 || b.rows == 0 || a.bytes == 0 || b.bytes == 0) return false;
  const auto end = [](const Block& v) { return v.at + uintptr_t((v.rows - 1) * v.pitch + v.bytes); };
  if (end(a) <= b.at || end(b) <= a.at) return false;
  if (a.pitch < a.bytes || b.pitch < b.bytes) return true;
  for (int64_t i = 0, j = 0; i < a.rows && j < b.rows;) {
    const uintptr_t pa = a.at + uintptr_t(i * a.pitch), pb = b.at + uintptr_t(j * b.pitch);
    if (pa + uintptr_t(a.bytes) <= pb)
      ++i;
    else if (pb + uintptr_t(b.bytes) <= pa)
      ++j;
    else
      return true;
  }
  return false;
}

// A given output: apart from what is read, except the residual as a whole
// (each of its elements is read before it is written, by the same thread or
// warp).  Autograd learns of the write by the tensor's version.
void check_out(const Tensor& out, int64_t stride, const Tensor& in, int64_t in_stride, const Tensor* residual,
               int64_t res_stride) {
  require(!(at::GradMode::is_enabled() && out.requires_grad()), "out requires a gradient: give another, or use torch.no_grad()");
  const Block o = block_of(out, stride);
  require(!share(o, block_of(in, in_stride)), "out must not overlap the operator's input");
  if (residual) {
    const Block r = block_of(*residual, res_stride);
    require((r.at == o.at && (r.pitch == o.pitch || o.rows <= 1)) || !share(o, r),
            "out may be the residual itself, but must not overlap it otherwise");
  }
  out.unsafeGetTensorImpl()->bump_version();
}

// ------------------------------------------------------------ 4-bit products
// Row stride of an output or residual.
int64_t output_stride(const Tensor& t, const Tensor& x, int64_t rows, int64_t n) {
  require(t.scalar_type() == x.scalar_type() && t.dim() == 2 && t.size(0) == rows && t.size(1) == n &&
              t.device() == x.device() && (n <= 1 || rows == 0 || t.stride(1) == 1),
          "out and residual must be [rows, n] of x's type with contiguous rows on x's device");
  return rows > 1 ? t.stride(0) : n;
}

Tensor w4(const Tensor& x, const Tensor& codes, const Tensor& scales, const Tensor* zeros, const Tensor* residual,
          const Tensor* out_given, bool swiglu, const Tensor* offsets, const Tensor* status) {
  const int lead = offsets ? 1 : 0;
  // The result has no history, so a gradient would stop here without a word.
  require(!at::GradMode::is_enabled() ||
              !(x.requires_grad() || scales.requires_grad() || (residual && residual->requires_grad())),
          "the 4-bit products have no gradient: detach the operands or call them under torch.no_grad()");
  require(x.dim() == 2 && codes.dim() == 2 + lead && scales.dim() == 2 + lead,
          "x must be [rows, k] and codes / scales [n, ...], with a leading expert dimension for experts");
  const int type = type_of(x);
  require((type == ASPIRE_T_BF16 || type == ASPIRE_T_F16) && scales.scalar_type() == x.scalar_type(),
          "x and scales must both be bfloat16 or both float16");
  require(codes.scalar_type() == at::kInt, "codes must be int32");
  require(x.is_cuda() && codes.device() == x.device() && scales.device() == x.device(),
          "x, codes and scales must be on one CUDA device");
  const int64_t rows = x.size(0), k = x.size(1), r = codes.size(lead), groups = scales.size(-1);
  require(codes.size(-1) * 8 == k, "codes and x disagree on k");
  require(scales.size(lead) == r && (!lead || scales.size(0) == codes.size(0)) && groups > 0 && k % groups == 0,
          "scales must be [..., n, k / group]");
  const int64_t group = k / groups;
  require(group == 32 || group == 64 || (group > 0 && group % 128 == 0), "group must be 32, 64 or a multiple of 128");
  require(!swiglu || r % 2 == 0, "the gated form needs as many gate as up rows");
  const int64_t n = swiglu ? r / 2 : r;
  require((rows == 0 || x.stride(1) == 1) && codes.stride(-1) == 1 && (groups == 1 || scales.stride(-1) == 1),
          "x, codes and scales need contiguous rows");
  if (zeros) {
    require(zeros->scalar_type() == at::kByte && zeros->sizes() == scales.sizes() && zeros->device() == x.device(),
            "zeros must be uint8 of the scales' shape on their device");
    require(groups == 1 || zeros->stride(-1) == 1, "zeros need contiguous rows");
  }
  require(!offsets || (offsets->scalar_type() == at::kInt && offsets->device() == x.device() &&
                       offsets->is_contiguous() && offsets->dim() == 1 && offsets->size(0) == codes.size(0) + 1),
          "offsets must be contiguous int32 [experts + 1] on x's device");
  const int64_t res_stride = residual ? output_stride(*residual, x, rows, n) : 0;
  int64_t out_stride = n;
  Tensor out;
  if (out_given) {
    out = *out_given;
    out_stride = output_stride(out, x, rows, n);
    check_out(out, out_stride, x, rows > 1 ? x.stride(0) : k, residual, res_stride);
  } else {
    out = at::empty({rows, n}, x.options());
  }
  if (rows == 0 || n == 0) return out;
  require(k <= INT32_MAX && n <= INT32_MAX && (!lead || codes.size(0) <= INT32_MAX), "sizes past 32 bits");
  AspireW4Args a = {};
  a.x = x.data_ptr();
  a.x_stride = rows > 1 ? x.stride(0) : k;
  a.rows = rows;
  a.codes = static_cast<const uint32_t*>(codes.data_ptr());
  // (The stride of a dimension of size one says nothing.)
  a.codes_stride = r > 1 ? codes.stride(lead) : k / 8;
  a.scales = scales.data_ptr();
  a.scales_stride = r > 1 ? scales.stride(lead) : groups;
  if (zeros) {
    a.zeros = static_cast<const uint8_t*>(zeros->data_ptr());
    a.zeros_stride = r > 1 ? zeros->stride(lead) : groups;
  }
  if (residual) {
    a.residual = residual->data_ptr();
    a.residual_stride = res_stride;
  }
  a.out = out.data_ptr();
  a.out_stride = out_stride;
  a.n = int32_t(n);
  a.k = int32_t(k);
  a.group = int32_t(group);
  a.type = type;
  a.swiglu = swiglu ? 1 : 0;
  if (lead) {
    a.offsets = static_cast<const int32_t*>(offsets->data_ptr());
    a.experts = int32_t(codes.size(0));
    if (a.experts > 1) {
      a.codes_stride_e = codes.stride(0);
      a.scales_stride_e = scales.stride(0);
      if (zeros) a.zeros_stride_e = zeros->stride(0);
    }
  }
  a.status = status_word(status, x);
  on_device(x, [&](void* stream) { check(abi.w4_linear(&a, stream), "aspire_w4_linear"); });
  return out;
}

// ------------------------------------------------------------------- routing
struct Routed {
  Tensor weights, experts, position, source, offsets;
};

// Of logits [tokens, experts], or of given choices (experts_in) the sort alone.
Routed route(const Tensor* logits, const Tensor* experts_in, int64_t num_experts, int64_t top_k, bool renormalize) {
  const Tensor& given = logits ? *logits : *experts_in;
  const int64_t tokens = given.size(0);
  Routed r;
  const auto i32 = given.options().dtype(at::kInt).requires_grad(false);
  if (logits) {
    r.weights = at::empty({tokens, top_k}, given.options().dtype(at::kFloat).requires_grad(false));
    r.experts = at::empty({tokens, top_k}, i32);
  } else {
    r.experts = *experts_in;
  }
  r.position = at::empty({tokens, top_k}, i32);
  r.source = at::empty({tokens * top_k}, i32);
  r.offsets = at::empty({num_experts + 1}, i32);
  AspireMoeRouteArgs a = {};
  if (logits) {
    a.logits = given.data_ptr();
    a.logits_type = type_of(given);
    a.logits_stride = given.stride(0);
    a.weights = static_cast<float*>(r.weights.data_ptr());
  }
  a.tokens = tokens;
  a.num_experts = int32_t(num_experts);
  a.top_k = int32_t(top_k);
  a.renormalize = renormalize ? 1 : 0;
  a.experts = static_cast<int32_t*>(r.experts.data_ptr());
  a.position = static_cast<int32_t*>(r.position.data_ptr());
  a.source = static_cast<int32_t*>(r.source.data_ptr());
  a.offsets = static_cast<int32_t*>(r.offsets.data_ptr());
  Tensor workspace;
  a.workspace_bytes = abi.moe_route_workspace(tokens, a.num_experts, a.top_k);
  if (a.workspace_bytes) {
    workspace = at::empty({int64_t(a.workspace_bytes / 4)}, i32);
    a.workspace = static_cast<int32_t*>(workspace.data_ptr());
  }
  on_device(given, [&](void* stream) { check(abi.moe_route(&a, stream), "aspire_moe_route"); });
  return r;
}

Tensor route_grad(const Tensor& grad_in, const Tensor& weights, const Tensor& experts, const Tensor* logits,
                  int64_t num_experts, int type, bool renormalize) {
  const Tensor grad = grad_in.to(at::kFloat).contiguous();
  const auto as = type == ASPIRE_T_F32 ? at::kFloat : type == ASPIRE_T_BF16 ? at::kBFloat16 : at::kHalf;
  Tensor out = at::empty({weights.size(0), num_experts}, weights.options().dtype(as).requires_grad(false));
  if (out.numel() == 0) return out;
  AspireMoeRouteGradArgs a = {};
  a.logits_type = type_of(out);
  if (logits) {
    a.logits = logits->data_ptr();
    a.logits_stride = logits->stride(0);
  }
  a.weights = static_cast<const float*>(weights.data_ptr());
  a.experts = static_cast<const int32_t*>(experts.data_ptr());
  a.grad_weights = static_cast<const float*>(grad.data_ptr());
  a.tokens = weights.size(0);
  a.num_experts = int32_t(num_experts);
  a.top_k = int32_t(weights.size(1));
  a.renormalize = renormalize ? 1 : 0;
  a.grad_logits = out.data_ptr();
  on_device(weights, [&](void* stream) { check(abi.moe_route_grad(&a, stream), "aspire_moe_route_grad"); });
  return out;
}

// ---------------------------------------------------------- dispatch, combine
// Pointer and row stride of a [rows, width] operand.
struct Rows {
  void* ptr;
  int64_t stride;
};

Rows rows_of(const char* name, const Tensor& t, int64_t rows, const Tensor* like) {
  const std::string who(name);
  if (type_of(t) < 0 || t.dim() != 2 || !t.is_cuda())
    throw Invalid(who + " must be a 2-D CUDA tensor of float32, bfloat16 or float16");
  if (t.size(0) != rows) throw Invalid(who + " has the wrong shape");
  if (like && (t.size(1) != like->size(1) || t.scalar_type() != like->scalar_type() || t.device() != like->device()))
    throw Invalid(who + " must have the rows' width, type and device");
  const int64_t vec = 16 / t.element_size(), width = t.size(1);
  if (width == 0 || width % vec || width > INT32_MAX)
    throw Invalid(who + ": rows must be a positive multiple of 16 bytes");
  if (rows && (t.stride(1) != 1 || (rows > 1 && (t.stride(0) % vec || t.stride(0) < width))))
    throw Invalid(who + ": rows must be contiguous and a multiple of 16 bytes apart");
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) throw Invalid(who + " must be 16-byte aligned");
  return {t.data_ptr(), rows > 1 ? t.stride(0) : width};
}

// What autograd hands over may have any strides.
Tensor grad_rows(const Tensor& g) {
  const int64_t vec = 16 / g.element_size();
  const bool ok = g.stride(1) == 1 && (g.size(0) <= 1 || (g.stride(0) % vec == 0 && g.stride(0) >= g.size(1))) &&
                  (reinterpret_cast<uintptr_t>(g.data_ptr()) & 15) == 0;
  return ok ? g : g.clone(at::MemoryFormat::Contiguous);
}

struct Order {
  const Tensor& position;
  const Tensor& source;
  const Tensor& offsets;
  int64_t tokens, top_k;

  Order(const Tensor& p, const Tensor& s, const Tensor& o, const Tensor& like)
      : position(p), source(s), offsets(o), tokens(0), top_k(0) {
    for (const Tensor* t : {&p, &s, &o})
      require(t->scalar_type() == at::kInt && t->device() == like.device() && t->is_contiguous(),
              "the order's tensors must be contiguous int32 on the rows' device");
    require(p.dim() == 2 && s.dim() == 1 && s.size(0) == p.numel() && o.dim() == 1 && o.size(0) >= 1,
            "order must be what moe_route or moe_sort returned");
    tokens = p.size(0);
    top_k = p.size(1);
    require(top_k >= 1 && top_k <= 32, "between 1 and 32 choices are supported");
  }
  AspireMoePermuteArgs args(const Tensor& like, const Tensor* status) const {
    AspireMoePermuteArgs a = {};
    a.type = type_of(like);
    a.position = static_cast<const int32_t*>(position.data_ptr());
    a.offsets = static_cast<const int32_t*>(offsets.data_ptr());
    a.num_experts = int32_t(offsets.size(0) - 1);
    a.top_k = int32_t(top_k);
    a.tokens = tokens;
    a.width = int32_t(like.size(1));
    a.status = status_word(status, like);
    return a;
  }
};

Tensor empty_rows(const Tensor& like, int64_t rows) {
  return at::empty({rows, like.size(1)}, like.options().requires_grad(false));
}

Tensor dispatch(const Tensor& x, const Order& o, const Tensor* status) {
  const Rows in = rows_of("x", x, o.tokens, nullptr);
  Tensor out = empty_rows(x, o.tokens * o.top_k);
  if (o.tokens == 0) return out;
  AspireMoePermuteArgs a = o.args(x, status);
  a.in = in.ptr;
  a.in_stride = in.stride;
  a.out = out.data_ptr();
  a.out_stride = x.size(1);
  on_device(x, [&](void* stream) { check(abi.moe_dispatch(&a, stream), "aspire_moe_dispatch"); });
  return out;
}

void check_weights(const Tensor& w, const Order& o, const Tensor& like) {
  require(w.scalar_type() == at::kFloat && w.sizes() == o.position.sizes() && w.device() == like.device() &&
              w.is_contiguous(),
          "weights must be contiguous float32 [tokens, top_k] on the rows' device");
}

Tensor combine(const Tensor& rows, const Tensor* weights, const Order& o, const Tensor* residual,
               const Tensor* out_given, const Tensor* status) {
  const Rows in = rows_of("rows", rows, o.tokens * o.top_k, nullptr);
  if (weights) check_weights(*weights, o, rows);
  Rows res = {nullptr, 0};
  if (residual) res = rows_of("residual", *residual, o.tokens, &rows);
  Tensor out = out_given ? *out_given : empty_rows(rows, o.tokens);
  const Rows to = out_given ? rows_of("out", out, o.tokens, &rows) : Rows{out.data_ptr(), rows.size(1)};
  if (out_given) check_out(out, to.stride, rows, in.stride, residual, res.stride);
  if (o.tokens == 0) return out;
  AspireMoePermuteArgs a = o.args(rows, status);
  a.in = in.ptr;
  a.in_stride = in.stride;
  a.residual = res.ptr;
  a.residual_stride = res.stride;
  if (weights) a.weights = static_cast<const float*>(weights->data_ptr());
  a.out = to.ptr;
  a.out_stride = to.stride;
  on_device(rows, [&](void* stream) { check(abi.moe_combine(&a, stream), "aspire_moe_combine"); });
  return out;
}

// Gradients of combine; an undefined tensor where none is wanted.
std::pair<Tensor, Tensor> combine_grad(const Tensor& grad_in, const Tensor& rows, const Tensor& weights, const Order& o,
                                       bool need_rows, bool need_weights, const Tensor* status) {
  Tensor d_rows, d_weights;
  if (need_rows) d_rows = empty_rows(rows, rows.size(0));
  if (need_weights) d_weights = at::empty(weights.sizes(), weights.options().requires_grad(false));
  if (o.tokens == 0) return {d_rows, d_weights};
  const Tensor grad = grad_rows(grad_in);
  const Rows in = rows_of("rows", rows, o.tokens * o.top_k, nullptr);
  const Rows g = rows_of("the gradient", grad, o.tokens, &rows);
  check_weights(weights, o, rows);
  AspireMoePermuteArgs a = o.args(rows, status);
  a.in = in.ptr;
  a.in_stride = in.stride;
  a.weights = static_cast<const float*>(weights.data_ptr());
  a.grad = g.ptr;
  a.grad_stride = g.stride;
  if (need_rows) {
    a.out = d_rows.data_ptr();
    a.out_stride = rows.size(1);
  }
  if (need_weights) a.grad_weights = static_cast<float*>(d_weights.data_ptr());
  on_device(rows, [&](void* stream) { check(abi.moe_combine_grad(&a, stream), "aspire_moe_combine_grad"); });
  return {d_rows, d_weights};
}

// -------------------------------------------------------------------- Python
PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <typename... T>
PyObject* wrap_all(const T&... t) {
  PyObject* tuple = PyTuple_New(sizeof...(t));
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  bool ok = true;
  const auto put = [&](const Tensor& v) {
    PyObject* o = ok ? wrap(v) : nullptr;
    if (o)
      PyTuple_SET_ITEM(tuple, i++, o);
    else
      ok = false;
  };
  (put(t), ...);
  if (!ok) {
    Py_DECREF(tuple);
    return nullptr;
  }
  return tuple;
}

template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& f) {
  if (given != wanted) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return f();
  } catch (const Invalid& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// (x, codes, scales, zeros, residual, out, swiglu, offsets, status)
PyObject* py_w4(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    return wrap(w4(tensor(v[0]), tensor(v[1]), tensor(v[2]), optional(v[3]),
                   optional(v[4]), optional(v[5]), v[6] == Py_True, optional(v[7]),
                   optional(v[8])));
  });
}
// (logits, top_k, renormalize) -> weights, experts, position, source, offsets
PyObject* py_route(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 3, [&] {
    const Tensor& l = tensor(v[0]);
    const long top_k = integer(v[1]);
    require(l.dim() == 2 && type_of(l) >= 0 && l.is_cuda(),
            "logits must be a [tokens, experts] CUDA tensor of float32, bfloat16 or float16");
    require(l.size(1) >= 1 && l.size(1) <= 512, "between 1 and 512 experts are supported");
    require(top_k >= 1 && top_k <= 32 && top_k <= l.size(1), "top_k must be between 1 and min(32, experts)");
    require(l.stride(1) == 1 || l.size(1) == 1 || l.size(0) == 0, "logits need contiguous rows");
    const Routed r = route(&l, nullptr, l.size(1), top_k, v[2] == Py_True);
    return wrap_all(r.weights, r.experts, r.position, r.source, r.offsets);
  });
}
// (experts, num_experts) -> position, source, offsets
PyObject* py_sort(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 2, [&] {
    const Tensor& e = tensor(v[0]);
    const long num = integer(v[1]);
    require(e.dim() == 2 && e.scalar_type() == at::kInt && e.is_cuda() && e.is_contiguous(),
            "experts must be a contiguous int32 [tokens, top_k] CUDA tensor");
    require(num >= 1 && num <= 512 && e.size(1) >= 1 && e.size(1) <= 32,
            "between 1 and 512 experts and 1 and 32 choices are supported");
    const Routed r = route(nullptr, &e, num, e.size(1), false);
    return wrap_all(r.position, r.source, r.offsets);
  });
}
// (gradient, weights, experts, logits or None, num_experts, the logits' type, renormalize)
PyObject* py_route_grad(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 7, [&] {
    return wrap(route_grad(tensor(v[0]), tensor(v[1]), tensor(v[2]),
                           optional(v[3]), integer(v[4]), int(integer(v[5])), v[6] == Py_True));
  });
}
// (x, position, source, offsets, status)
PyObject* py_dispatch(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    const Tensor& x = tensor(v[0]);
    const Order o(tensor(v[1]), tensor(v[2]), tensor(v[3]), x);
    return wrap(dispatch(x, o, optional(v[4])));
  });
}
// (gradient of the rows, position, source, offsets, status)
PyObject* py_dispatch_grad(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    const Tensor& g = tensor(v[0]);
    const Order o(tensor(v[1]), tensor(v[2]), tensor(v[3]), g);
    return wrap(combine(grad_rows(g), nullptr, o, nullptr, nullptr, optional(v[4])));
  });
}
// (rows, weights, position, source, offsets, residual, out, status)
PyObject* py_combine(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 8, [&] {
    const Tensor& rows = tensor(v[0]);
    const Order o(tensor(v[2]), tensor(v[3]), tensor(v[4]), rows);
    return wrap(combine(rows, &tensor(v[1]), o, optional(v[5]), optional(v[6]),
                        optional(v[7])));
  });
}
// (gradient, rows, weights, position, source, offsets, need_rows, need_weights, status)
PyObject* py_combine_grad(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    const Tensor& rows = tensor(v[1]);
    const Order o(tensor(v[3]), tensor(v[4]), tensor(v[5]), rows);
    const auto d = combine_grad(tensor(v[0]), rows, tensor(v[2]), o, v[6] == Py_True,
                                v[7] == Py_True, optional(v[8]));
    return wrap_all(d.first, d.second);
  });
}

// (addresses of the entry points, in the order of `abi`)
PyObject* py_bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const auto at = [&](int i, auto& fn) {
      fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(PyLong_AsVoidPtr(v[i]));
      if (!fn) throw Invalid("an address is required");
    };
    at(0, abi.last_error);
    at(1, abi.w4_linear);
    at(2, abi.moe_route);
    at(3, abi.moe_route_workspace);
    at(4, abi.moe_route_grad);
    at(5, abi.moe_dispatch);
    at(6, abi.moe_combine);
    at(7, abi.moe_combine_grad);
    Py_RETURN_NONE;
  });
}

#define ASPIRE_METHOD(name, fn) \
  { name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr }
PyMethodDef kMethods[] = {
    ASPIRE_METHOD("bind", py_bind),
    ASPIRE_METHOD("w4", py_w4),
    ASPIRE_METHOD("route", py_route),
    ASPIRE_METHOD("sort", py_sort),
    ASPIRE_METHOD("route_grad", py_route_grad),
    ASPIRE_METHOD("dispatch", py_dispatch),
    ASPIRE_METHOD("dispatch_grad", py_dispatch_grad),
    ASPIRE_METHOD("combine", py_combine),
    ASPIRE_METHOD("combine_grad", py_combine_grad),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding(void) {
  PyObject* m = PyModule_Create(&kModule);
  // The torch and the Python it was built for, as build.py finds them in the file.
  if (m && PyModule_AddStringConstant(m, "built_for", "aspire binding for [" ASPIRE_BUILT_FOR "]") < 0) Py_CLEAR(m);
  return m;
}
