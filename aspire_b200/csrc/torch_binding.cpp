// The feed-forward and tree-step operators' Python calls: argument checks,
// outputs and the call of the C ABI (include/aspire_b200.h) on torch's current
// stream.
//
// A decode step's calls are a few microseconds on the device, less than the
// same checks take attribute by attribute in Python, so they are made here on
// the tensors themselves.  Host time of one call, Python -> here: product 10.2
// -> 5.1 us, routing 15.1 -> 7.1, combine 10.4 -> 3.8 (an output's allocation
// alone is 2.4).  Everything a kernel needs still crosses the C ABI, through
// the entry points of the library that the package has loaded (bind()); this
// file launches nothing.
#include <Python.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

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
  decltype(&aspire_step_tables) step_tables;
  decltype(&aspire_logits_workspace) logits_workspace;
  decltype(&aspire_adjust_logits) adjust_logits;
  decltype(&aspire_tree_accept) tree_accept;
  decltype(&aspire_tree_attention) tree_attention;
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
  require(!t._fw_grad(0).defined(), "the feed-forward and tree-step operators have no forward-mode derivative");
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

// ----------------------------------------------------------------- tree step
// A contiguous int32 vector of `n` entries (any number for n < 0) on `like`'s device.
int32_t* ints(const Tensor* t, int64_t n, const Tensor& like, const char* name) {
  if (!t) return nullptr;
  if (t->scalar_type() != at::kInt || t->dim() != 1 || !t->is_contiguous() || t->device() != like.device() ||
      (n >= 0 && t->size(0) != n))
    throw Invalid(std::string(name) + " must be a contiguous int32 vector of the right length on the operands' device");
  return static_cast<int32_t*>(t->data_ptr());
}

// A 2-D int32 tensor with contiguous rows.
int32_t* int_rows(const Tensor& t, int64_t rows, const Tensor& like, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != rows || t.device() != like.device() ||
      (t.size(1) > 1 && rows > 0 && t.stride(1) != 1) || t.size(1) > INT32_MAX)
    throw Invalid(std::string(name) + " must be a 2-D int32 tensor with contiguous rows on the operands' device");
  return static_cast<int32_t*>(t.data_ptr());
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// A tensor's memory, first to last element.
std::pair<uintptr_t, uintptr_t> span_of(const Tensor& t) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {at, at};
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {at, at + uintptr_t((last + 1) * t.element_size())};
}

// Whether two tensors' memory has a byte in common.
bool in_common(const Tensor& a, const Tensor& b) {
  const auto x = span_of(a), y = span_of(b);
  return x.first < y.second && y.first < x.second;
}

// Whether two [tokens, heads, dim] tensors with contiguous dims have a byte in
// common.  Vectors of one buffer may lie between one another's (the parts of a
// fused projection): by rows first, vector by vector only where rows cross.
bool share_vectors(const Tensor& a, const Tensor& b) {
  if (!in_common(a, b)) return false;
  const auto rows_of = [](const Tensor& t) {
    const int64_t size = t.element_size();
    return Block{reinterpret_cast<uintptr_t>(t.data_ptr()), t.size(0), ((t.size(1) - 1) * t.stride(1) + t.size(2)) * size,
                 t.stride(0) * size};
  };
  if (!share(rows_of(a), rows_of(b))) return false;
  const auto vectors_of = [](const Tensor& t) {
    std::vector<uintptr_t> at;
    at.reserve(size_t(t.size(0) * t.size(1)));
    for (int64_t n = 0; n < t.size(0); ++n)
      for (int64_t h = 0; h < t.size(1); ++h)
        at.push_back(reinterpret_cast<uintptr_t>(t.data_ptr()) + uintptr_t((n * t.stride(0) + h * t.stride(1)) * t.element_size()));
    std::sort(at.begin(), at.end());
    return at;
  };
  const std::vector<uintptr_t> x = vectors_of(a), y = vectors_of(b);
  const uintptr_t xb = uintptr_t(a.size(2) * a.element_size()), yb = uintptr_t(b.size(2) * b.element_size());
  for (size_t i = 0, j = 0; i < x.size() && j < y.size();) {
    if (x[i] + xb <= y[j])
      ++i;
    else if (y[j] + yb <= x[i])
      ++j;
    else
      return true;
  }
  return false;
}

// Tensors of one type in one allocation, each 16-byte aligned: a step has many
// small tables, and an allocation is most of what a small tensor costs.
class Pieces {
 public:
  Pieces(std::initializer_list<int64_t> counts, const at::TensorOptions& options, int64_t size) : step_(16 / size) {
    int64_t total = 0;
    for (const int64_t c : counts) total += (c + step_ - 1) / step_ * step_;
    all_ = at::empty({total}, options);
  }
  // The next piece, of these sizes.
  Tensor take(at::IntArrayRef sizes) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all_.storage()), all_.key_set(), all_.dtype());
    c10::TensorImpl* impl = t.unsafeGetTensorImpl();
    impl->set_storage_offset(at_);
    impl->set_sizes_contiguous(sizes);
    at_ += (t.numel() + step_ - 1) / step_ * step_;
    return t;
  }

 private:
  Tensor all_;
  int64_t step_, at_ = 0;
};

struct Tables {
  Tensor qo_indptr, kv_indptr, kv_len, last_page_len, positions, slots, tree_mask;
};

Tables step_tables(const Tensor& lengths, const Tensor* new_tokens, const Tensor& table, const Tensor& held,
                   const Tensor& free_pages, const Tensor& free_count, int64_t tokens, const Tensor* parents,
                   int64_t max_nodes, int64_t page_size, const Tensor* status) {
  require(lengths.is_cuda() && lengths.dim() == 1, "lengths must be a 1-D CUDA tensor");
  const int64_t rows = lengths.size(0);
  require(rows <= INT32_MAX && tokens >= 0 && tokens <= INT32_MAX, "sizes past 32 bits");
  require(page_size >= 1 && page_size <= INT32_MAX, "page_size must be positive");
  require(!parents || (max_nodes >= 1 && max_nodes <= INT32_MAX - 31), "parents need max_nodes, the nodes of the largest tree");
  AspireStepTablesArgs a = {};
  a.lengths = ints(&lengths, rows, lengths, "lengths");
  a.new_tokens = ints(new_tokens, rows, lengths, "new_tokens");
  a.rows = int32_t(rows);
  a.page_size = int32_t(page_size);
  a.block_table = int_rows(table, rows, lengths, "block_table");
  a.block_table_stride = row_stride(table);
  a.block_table_cols = int32_t(table.size(1));
  require(rows <= 1 || table.stride(0) >= table.size(1), "block_table's rows must not overlap");
  a.held = ints(&held, rows, lengths, "held");
  a.free_pages = ints(&free_pages, -1, lengths, "free_pages");
  a.free_capacity = free_pages.size(0);
  require(a.free_capacity <= INT32_MAX, "sizes past 32 bits");
  a.free_count = ints(&free_count, 1, lengths, "free_count");
  a.parents = ints(parents, tokens, lengths, "parents");
  const Tensor* written[] = {&table, &held, &free_pages, &free_count};
  const Tensor* read[] = {&lengths, new_tokens, parents};
  for (int i = 0; i < 4; ++i) {
    for (int j = i + 1; j < 4; ++j)
      require(!in_common(*written[i], *written[j]), "block_table, held, free_pages and free_count must not overlap");
    for (const Tensor* r : read)
      require(!r || !in_common(*written[i], *r), "what the call changes must not overlap what it reads");
  }
  for (const Tensor* w : written) w->unsafeGetTensorImpl()->bump_version();
  const auto i32 = lengths.options();
  Tables t;
  const int64_t words = parents ? (max_nodes + 31) / 32 : 0;
  Pieces pieces({rows + 1, rows + 1, rows, rows, tokens, tokens * words}, i32, 4);
  t.qo_indptr = pieces.take({rows + 1});
  t.kv_indptr = pieces.take({rows + 1});
  t.kv_len = pieces.take({rows});
  t.last_page_len = pieces.take({rows});
  t.positions = pieces.take({tokens});
  t.slots = at::empty({tokens}, i32.dtype(at::kLong));
  a.qo_indptr = static_cast<int32_t*>(t.qo_indptr.data_ptr());
  a.kv_indptr = static_cast<int32_t*>(t.kv_indptr.data_ptr());
  a.kv_len = static_cast<int32_t*>(t.kv_len.data_ptr());
  a.last_page_len = static_cast<int32_t*>(t.last_page_len.data_ptr());
  a.positions = static_cast<int32_t*>(t.positions.data_ptr());
  a.slots = static_cast<int64_t*>(t.slots.data_ptr());
  a.tokens = tokens;
  if (parents) {
    a.tree_mask_words = int32_t(words);
    t.tree_mask = pieces.take({tokens, words});
    a.tree_mask = static_cast<int32_t*>(t.tree_mask.data_ptr());
    if (!a.parents) a.parents = a.qo_indptr;  // (no tokens, no address: nothing is read through it)
  }
  if (rows == 0) {  // (no kernel writes the tokens' tables)
    t.positions.zero_();
    t.slots.fill_(-1);
    if (parents) t.tree_mask.zero_();
  }
  a.status = status_word(status, lengths);
  on_device(lengths, [&](void* stream) { check(abi.step_tables(&a, stream), "aspire_step_tables"); });
  return t;
}

const float* row_terms(const Tensor* t, int64_t rows, const Tensor& like, const char* name) {
  if (!t) return nullptr;
  if (t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != rows || !t->is_contiguous() ||
      t->device() != like.device())
    throw Invalid(std::string(name) + " must be contiguous float32 [rows] on the logits' device");
  return static_cast<const float*>(t->data_ptr());
}

struct LogitsCall {
  const Tensor &logits;
  const Tensor *history, *history_len, *prompt_len, *indptr, *tokens, *tree_mask, *repetition, *frequency, *presence,
      *bias_indptr, *bias_ids, *bias_values, *allowed, *out;
  bool want_out, want_ids;
  const Tensor* status;
};

std::pair<Tensor, Tensor> adjust_logits(const LogitsCall& c) {
  const Tensor& x = c.logits;
  require(x.dim() == 2 && type_of(x) >= 0 && x.is_cuda(),
          "logits must be a [tokens, vocab] CUDA tensor of float32, bfloat16 or float16");
  for (const Tensor* t : {&x, c.repetition, c.frequency, c.presence, c.bias_values})
    require(!t || !at::GradMode::is_enabled() || !t->requires_grad(),
            "adjusted logits have no gradient: detach the operands or call under torch.no_grad()");
  const int64_t tokens = x.size(0), vocab = x.size(1);
  require(vocab >= 1 && vocab <= INT32_MAX && tokens <= INT32_MAX, "tokens or vocab out of range");
  require(tokens == 0 || vocab == 1 || x.stride(1) == 1, "logits need contiguous rows");
  const int64_t rows = c.indptr ? c.indptr->numel() - 1 : tokens;
  require(!c.indptr || rows >= 0, "indptr must be [rows + 1]");
  require(rows <= 65534, "at most 65534 rows are supported");
  AspireLogitsArgs a = {};
  a.logits = x.data_ptr();
  a.logits_stride = tokens > 1 ? x.stride(0) : vocab;
  require(a.logits_stride >= vocab, "logits' rows must not overlap");
  a.type = type_of(x);
  a.tokens = tokens;
  a.vocab = int32_t(vocab);
  a.rows = int32_t(rows);
  a.indptr = ints(c.indptr, rows + 1, x, "indptr");
  require(!c.history == !c.history_len, "history and history_len go together");
  require(!c.prompt_len || c.history, "prompt_len needs a history");
  if (c.history) {
    a.history = int_rows(*c.history, rows, x, "history");
    a.history_stride = row_stride(*c.history);
    a.history_cols = int32_t(c.history->size(1));
    a.history_len = ints(c.history_len, rows, x, "history_len");
    a.prompt_len = ints(c.prompt_len, rows, x, "prompt_len");
    if (a.history_cols == 0) a.history = nullptr;
  }
  a.step_tokens = ints(c.tokens, tokens, x, "tokens");
  if (c.tree_mask) {
    require(c.tokens, "tree_mask needs tokens");
    a.tree_mask = int_rows(*c.tree_mask, tokens, x, "tree_mask");
    require(c.tree_mask->is_contiguous() && c.tree_mask->size(1) >= 1, "tree_mask must be contiguous [tokens, words]");
    a.tree_mask_words = int32_t(c.tree_mask->size(1));
  }
  a.repetition = row_terms(c.repetition, rows, x, "repetition");
  a.frequency = row_terms(c.frequency, rows, x, "frequency");
  a.presence = row_terms(c.presence, rows, x, "presence");
  require(!c.bias_indptr == !c.bias_ids && !c.bias_ids == !c.bias_values, "bias must be (indptr, ids, values)");
  if (c.bias_indptr && c.bias_ids->numel() > 0) {
    a.bias_indptr = ints(c.bias_indptr, rows + 1, x, "bias indptr");
    a.bias_ids = ints(c.bias_ids, -1, x, "bias ids");
    a.bias_values = row_terms(c.bias_values, c.bias_ids->numel(), x, "bias values");
    a.bias_entries = c.bias_ids->numel();
    require(a.bias_entries < INT32_MAX, "sizes past 32 bits");
  }
  if (c.allowed) {
    a.allowed = int_rows(*c.allowed, tokens, x, "allowed");
    a.allowed_stride = row_stride(*c.allowed);
    require(c.allowed->size(1) >= (vocab + 31) / 32, "allowed must be [tokens, vocab / 32 rounded up]");
  }
  Tensor out, ids, workspace;
  if (c.want_out) {
    if (c.out) {
      out = *c.out;
      require(out.scalar_type() == x.scalar_type() && out.sizes() == x.sizes() && out.device() == x.device() &&
                  (tokens == 0 || vocab == 1 || out.stride(1) == 1),
              "out must be [tokens, vocab] of the logits' type with contiguous rows on their device");
      a.out_stride = tokens > 1 ? out.stride(0) : vocab;
      require(a.out_stride >= vocab, "out's rows must not overlap");
      require(!(at::GradMode::is_enabled() && out.requires_grad()),
              "out requires a gradient: give another, or use torch.no_grad()");
      const Block o = block_of(out, a.out_stride), l = block_of(x, a.logits_stride);
      require((o.at == l.at && (o.pitch == l.pitch || o.rows <= 1)) || !share(o, l),
              "out may be the logits themselves, but must not overlap them otherwise");
      for (const Tensor* t : {c.history, c.history_len, c.prompt_len, c.indptr, c.tokens, c.tree_mask, c.repetition,
                              c.frequency, c.presence, c.bias_indptr, c.bias_ids, c.bias_values, c.allowed})
        require(!t || !in_common(out, *t), "out must not overlap what the call reads");
      out.unsafeGetTensorImpl()->bump_version();
    } else {
      out = at::empty({tokens, vocab}, x.options().requires_grad(false));
      a.out_stride = vocab;
    }
    a.out = out.data_ptr();
  }
  a.status = status_word(c.status, x);
  on_device(x, [&](void* stream) {
    const auto i32 = x.options().dtype(at::kInt).requires_grad(false);
    if (c.want_ids) {
      ids = at::empty({tokens}, i32);
      a.ids = static_cast<int32_t*>(ids.data_ptr());
    }
    if (tokens == 0) return;
    a.workspace_bytes = abi.logits_workspace(&a);
    if (a.workspace_bytes) {
      workspace = at::empty({int64_t(a.workspace_bytes / 4)}, i32);
      a.workspace = workspace.data_ptr();
    }
    check(abi.adjust_logits(&a, stream), "aspire_adjust_logits");
  });
  return {out, ids};
}

struct Walked {
  Tensor count, path, tokens, lengths;
};

Walked tree_accept(const Tensor& tokens, const Tensor& parents, const Tensor& targets, const Tensor& indptr,
                   const Tensor& lengths, int64_t max_path, const std::vector<const Tensor*>& caches,
                   const Tensor* table, const Tensor* status, const Tensor* kv_len) {
  require(tokens.is_cuda() && tokens.dim() == 1, "tokens must be a 1-D CUDA tensor");
  require(max_path >= 1 && max_path <= ASPIRE_MAX_PATH, "max_path must be between 1 and 64");
  const int64_t total = tokens.size(0), rows = lengths.numel();
  require(total <= INT32_MAX && rows <= INT32_MAX, "sizes past 32 bits");
  AspireTreeAcceptArgs a = {};
  a.tokens = ints(&tokens, total, tokens, "tokens");
  a.parents = ints(&parents, total, tokens, "parents");
  a.targets = ints(&targets, total, tokens, "targets");
  a.lengths = ints(&lengths, rows, tokens, "lengths");
  a.indptr = ints(&indptr, rows + 1, tokens, "indptr");
  a.kv_len = ints(kv_len, rows, tokens, "kv_len");
  a.total = total;
  a.rows = int32_t(rows);
  a.max_path = int32_t(max_path);
  std::vector<void*> at;
  if (!caches.empty()) {
    require(table, "caches need a block table");
    a.block_table = int_rows(*table, rows, tokens, "block_table");
    a.block_table_stride = row_stride(*table);
    a.block_table_cols = int32_t(table->size(1));
    const Tensor& first = *caches[0];
    require(first.dim() == 5 && first.size(1) == 2, "a cache must be [pages, 2, page_size, heads, head_dim]");
    const bool grads = at::GradMode::is_enabled();
    const size_t bytes = first.nbytes();
    std::vector<uintptr_t> starts;
    at.reserve(caches.size());
    starts.reserve(caches.size());
    for (const Tensor* c : caches) {
      require(c->sizes() == first.sizes() && c->scalar_type() == first.scalar_type() && c->is_contiguous() &&
                  c->device() == tokens.device() && !(grads && c->requires_grad()),
              "caches must be contiguous tensors of one shape and type on the tokens' device, without gradients");
      at.push_back(c->data_ptr());
      starts.push_back(reinterpret_cast<uintptr_t>(at.back()));
    }
    std::sort(starts.begin(), starts.end());
    for (size_t i = 1; i < starts.size(); ++i)
      require(bytes == 0 || starts[i] - starts[i - 1] >= bytes, "a cache is given twice, or two of them overlap");
    for (const Tensor* t : {&tokens, &parents, &targets, &indptr, &lengths, table, kv_len}) {
      if (!t) continue;
      const auto s = span_of(*t);
      const auto next = std::upper_bound(starts.begin(), starts.end(), s.first);
      require(s.first == s.second || bytes == 0 ||
                  ((next == starts.end() || s.second <= *next) && (next == starts.begin() || *(next - 1) + bytes <= s.first)),
              "a cache overlaps what the call reads");
    }
    a.pages = first.size(0);
    a.token_bytes = first.size(3) * first.size(4) * first.element_size();
    require(first.size(2) >= 1 && first.size(2) <= INT32_MAX, "bad page size");
    a.page_size = int32_t(first.size(2));
    require(a.token_bytes >= 16 && a.token_bytes % 16 == 0, "a token's keys must be a positive multiple of 16 bytes");
    for (const Tensor* c : caches) c->unsafeGetTensorImpl()->bump_version();
  }
  const auto i32 = tokens.options();
  Walked w;
  Pieces pieces({rows, rows * max_path, rows * max_path, rows}, i32, 4);
  w.count = pieces.take({rows});
  w.path = pieces.take({rows, max_path});
  w.tokens = pieces.take({rows, max_path});
  w.lengths = pieces.take({rows});
  a.count = static_cast<int32_t*>(w.count.data_ptr());
  a.path = static_cast<int32_t*>(w.path.data_ptr());
  a.out_tokens = static_cast<int32_t*>(w.tokens.data_ptr());
  a.new_lengths = static_cast<int32_t*>(w.lengths.data_ptr());
  a.status = status_word(status, tokens);
  if (rows == 0) return w;
  on_device(tokens, [&](void* stream) {
    size_t done = 0;
    do {  // (more layers than a call takes: the walk is the same each time)
      a.num_caches = int32_t(std::min(at.size() - done, size_t(ASPIRE_MAX_CACHES)));
      a.caches = at.data() + done;
      check(abi.tree_accept(&a, stream), "aspire_tree_accept");
      done += size_t(a.num_caches);
    } while (done < at.size());
  });
  return w;
}

// `fixed` holds what a plan's calls share (heads, pages, workspaces, scale); q_total the query rows it addresses.
std::pair<Tensor, Tensor> tree_attention(const Tensor& q, const Tensor& cache, const Tensor& mask,
                                         const Tensor* out_given, const Tensor* lse_given, bool want_lse,
                                         const AspireAttnArgs& fixed, const AspirePlanInfo& plan, int64_t q_total,
                                         const Tensor* k_new, const Tensor* v_new) {
  require(q.scalar_type() == at::kBFloat16 && cache.scalar_type() == at::kBFloat16, "q and paged_kv_cache must be bfloat16");
  require(cache.dim() == 5 && cache.size(1) == 2 && cache.is_contiguous() && cache.device() == q.device(),
          "paged_kv_cache must be a contiguous [pages, 2, page_size, num_kv_heads, head_dim] tensor on q's device");
  require(q.is_cuda() && q.dim() == 3 && q.size(1) == fixed.num_qo_heads && q.size(2) == cache.size(4),
          "q's shape does not match the plan");
  require(q.stride(2) == 1, "q head_dim must be contiguous");
  require(cache.size(2) == fixed.page_size && cache.size(3) == fixed.num_kv_heads,
          "paged_kv_cache geometry does not match the plan");
  require(q.size(0) >= q_total, "q has fewer rows than the plan addresses");
  require(!at::GradMode::is_enabled() || !(q.requires_grad() || cache.requires_grad()),
          "the attention has no gradient: detach the operands or call under torch.no_grad()");
  require(mask.scalar_type() == at::kInt && mask.dim() == 2 && mask.is_contiguous() && mask.device() == q.device() &&
              mask.size(0) >= q.size(0) && mask.size(1) >= 1 && mask.size(1) <= INT32_MAX,
          "tree_mask must be a contiguous int32 [tokens, words] tensor on q's device");
  require(!k_new == !v_new, "append needs both the new keys and the new values");
  for (const Tensor* t : {k_new, v_new}) {
    if (!t) continue;
    const std::string name = t == k_new ? "k_new" : "v_new";
    if (t->scalar_type() != at::kBFloat16 || t->dim() != 3 || t->stride(2) != 1 || t->device() != q.device())
      throw Invalid(name + " must be a bf16 [tokens, num_kv_heads, 128] tensor on q's device");
    if (t->size(1) != cache.size(3) || t->size(2) != q.size(2) || t->size(0) < q.size(0))
      throw Invalid(name + "'s shape does not match the plan");
    require(!at::GradMode::is_enabled() || !t->requires_grad(),
            "the attention has no gradient: detach the operands or call under torch.no_grad()");
    // (The append writes the cache.)
    require(!in_common(*t, cache) && !in_common(q, cache) && !in_common(mask, cache),
            "the cache must not overlap what the call reads");
  }
  Tensor out, lse;
  if (out_given) {
    out = *out_given;
    require(out.scalar_type() == q.scalar_type() && out.sizes() == q.sizes() && out.stride(2) == 1 &&
                out.device() == q.device(),
            "out must match q's shape and type with a contiguous head_dim on its device");
    require(!(at::GradMode::is_enabled() && out.requires_grad()),
            "out requires a gradient: give another, or use torch.no_grad()");
  } else {
    out = at::empty(q.sizes(), q.options().requires_grad(false));
  }
  if (lse_given) {
    lse = *lse_given;
    require(lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.dim() == 2 && lse.size(0) == q.size(0) &&
                lse.size(1) == q.size(1) && lse.device() == q.device(),
            "lse must be a contiguous fp32 [tokens, num_qo_heads] tensor");
    require(!(at::GradMode::is_enabled() && lse.requires_grad()),
            "lse requires a gradient: give another, or use torch.no_grad()");
  } else if (want_lse) {
    lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat).requires_grad(false));
  }
  if (out_given) {
    require(!in_common(out, cache) && !in_common(out, mask), "out must not overlap the cache or the mask");
    // (An item reads its queries before it writes their rows, and no other item reads them.)
    const bool same = out.data_ptr() == q.data_ptr() && (q.size(0) <= 1 || out.stride(0) == q.stride(0)) &&
                      (q.size(1) <= 1 || out.stride(1) == q.stride(1));
    require(same || !share_vectors(out, q), "out may be q itself, but must not overlap it otherwise");
    for (const Tensor* t : {k_new, v_new})
      require(!t || !share_vectors(out, *t), "out must not overlap the new keys and values");
  }
  if (lse_given) {
    require(!in_common(lse, cache) && !in_common(lse, mask) && !in_common(lse, q) && !in_common(lse, out),
            "lse must not overlap the other operands");
    for (const Tensor* t : {k_new, v_new}) require(!t || !in_common(lse, *t), "lse must not overlap the other operands");
  }
  if (k_new) cache.unsafeGetTensorImpl()->bump_version();
  if (out_given) out.unsafeGetTensorImpl()->bump_version();
  if (lse_given) lse.unsafeGetTensorImpl()->bump_version();
  AspireAttnArgs a = fixed;
  a.q = q.data_ptr();
  a.q_stride_n = q.stride(0);
  a.q_stride_h = q.stride(1);
  a.q_rows = q.size(0);
  a.head_dim = int32_t(q.size(2));
  a.kv_cache = cache.data_ptr();
  a.num_pages_total = cache.size(0);
  a.out = out.data_ptr();
  a.o_stride_n = out.stride(0);
  a.o_stride_h = out.stride(1);
  a.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
  if (k_new) {
    a.k_new = k_new->data_ptr();
    a.k_new_stride_n = k_new->stride(0);
    a.k_new_stride_h = k_new->stride(1);
    a.v_new = v_new->data_ptr();
    a.v_new_stride_n = v_new->stride(0);
    a.v_new_stride_h = v_new->stride(1);
  }
  on_device(q, [&](void* stream) {
    check(abi.tree_attention(&a, static_cast<const int32_t*>(mask.data_ptr()), int32_t(mask.size(1)), &plan, stream),
          "aspire_tree_attention");
  });
  return {out, lse};
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

// (lengths, new_tokens, block_table, held, free_pages, free_count, tokens, parents, max_nodes, page_size, status)
PyObject* py_step_tables(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 11, [&] {
    const Tables t = step_tables(tensor(v[0]), optional(v[1]), tensor(v[2]), tensor(v[3]), tensor(v[4]), tensor(v[5]),
                                 integer(v[6]), optional(v[7]), integer(v[8]), integer(v[9]), optional(v[10]));
    return wrap_all(t.qo_indptr, t.kv_indptr, t.kv_len, t.last_page_len, t.positions, t.slots, t.tree_mask);
  });
}
// (logits, history, history_len, prompt_len, indptr, tokens, tree_mask, repetition, frequency, presence, bias indptr,
// ids, values, allowed, out, want_out, want_ids, status) -> out, ids
PyObject* py_adjust_logits(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 18, [&] {
    const LogitsCall c = {tensor(v[0]),    optional(v[1]),  optional(v[2]),  optional(v[3]),  optional(v[4]),
                          optional(v[5]),  optional(v[6]),  optional(v[7]),  optional(v[8]),  optional(v[9]),
                          optional(v[10]), optional(v[11]), optional(v[12]), optional(v[13]), optional(v[14]),
                          v[15] == Py_True, v[16] == Py_True, optional(v[17])};
    const auto r = adjust_logits(c);
    return wrap_all(r.first, r.second);
  });
}
// (tokens, parents, targets, indptr, lengths, max_path, caches, block_table, status, kv_len) -> count, path, tokens,
// lengths
PyObject* py_tree_accept(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    require(PyList_Check(v[6]) || PyTuple_Check(v[6]), "caches must be a list or tuple of tensors");
    std::vector<const Tensor*> caches;
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(v[6]); ++i)
      caches.push_back(&tensor(PySequence_Fast_GET_ITEM(v[6], i)));
    const Walked w = tree_accept(tensor(v[0]), tensor(v[1]), tensor(v[2]), tensor(v[3]), tensor(v[4]), integer(v[5]),
                                 caches, optional(v[7]), optional(v[8]), optional(v[9]));
    return wrap_all(w.count, w.path, w.tokens, w.lengths);
  });
}

// (q, cache, mask, out, lse, want_lse, address of the plan's AspireAttnArgs, of its AspirePlanInfo, q_total, k_new,
// v_new) -> out, lse
PyObject* py_tree_attention(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const void* fixed = PyLong_AsVoidPtr(v[6]);
    const void* plan = PyLong_AsVoidPtr(v[7]);
    if (!fixed || !plan) throw Invalid("an address is required");
    const auto r = tree_attention(tensor(v[0]), tensor(v[1]), tensor(v[2]), optional(v[3]), optional(v[4]),
                                  v[5] == Py_True, *static_cast<const AspireAttnArgs*>(fixed),
                                  *static_cast<const AspirePlanInfo*>(plan), integer(v[8]), optional(v[9]),
                                  optional(v[10]));
    return wrap_all(r.first, r.second);
  });
}

// (addresses of the entry points, in the order of `abi`)
PyObject* py_bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
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
    at(8, abi.step_tables);
    at(9, abi.logits_workspace);
    at(10, abi.adjust_logits);
    at(11, abi.tree_accept);
    at(12, abi.tree_attention);
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
    ASPIRE_METHOD("step_tables", py_step_tables),
    ASPIRE_METHOD("adjust_logits", py_adjust_logits),
    ASPIRE_METHOD("tree_accept", py_tree_accept),
    ASPIRE_METHOD("tree_attention", py_tree_attention),
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
