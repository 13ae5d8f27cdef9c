// Native host path of fhob.rotary and fhob.layer_norm: checks, strides, allocation and the autograd functions.
//
// All arguments are checked here (the calls are bound by the host at small sizes), and an argument that is
// refused raises ValueError or TypeError.  Views that the kernels cannot read in place are copied first.
// Nothing is kept between calls: what a call needs besides its results is allocated on its stream.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include "../../include/fhob.h"
#include "host_layer.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// An argument of an autograd function that may be missing: these take no undefined tensors.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor given(const Maybe& t) { return t ? *t : Tensor(); }

int type_of(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kBFloat16 ? FHOB_BF16 : s == at::kHalf ? FHOB_F16 : s == at::kFloat ? FHOB_F32 : -1;
}

Tensor new_like(const Tensor& t) { return at::detail::empty_cuda(t.sizes(), t.scalar_type(), t.device(), std::nullopt); }

// Runs `call` on the current stream of the tensor's device, with that device current.
template <class F>
void launch(const Tensor& t, const char* what, F&& call) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != t.get_device()) guard.set_index(static_cast<c10::DeviceIndex>(t.get_device()));
  const int status = call(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
  TORCH_CHECK(status == FHOB_OK, what, " failed with status ", status, ": ", fhob_strerror(status), status == FHOB_ERR_CUDA ? ": " : "",
              status == FHOB_ERR_CUDA ? fhob_last_cuda_error() : "");
}

// ------------------------------------------------------------------ rotary positions

using Axes = std::vector<int64_t>;

// Turns one or two tensors (the second may be undefined).  Everything but their strides has been checked.
std::array<Tensor, 2> rotate(const Tensor& x0, const Tensor& x1, const Tensor& positions, const Tensor& frequencies, const Axes& axis_of_pair,
                             bool interleaved, bool inverse) {
  FhobRotary r;
  memset(&r, 0, sizeof(r));
  std::array<Tensor, 2> out;
  Tensor keep[2];
  const Tensor* inputs[2] = {&x0, &x1};
  const Tensor* some = nullptr;
  uint8_t axes[FHOB_ROTARY_MAX_PAIRS];
  for (int t = 0; t < 2; ++t) {
    if (!inputs[t]->defined()) continue;
    out[t] = new_like(*inputs[t]);
    if (out[t].numel() == 0) continue;
    const int dim = static_cast<int>(inputs[t]->dim());
    keep[t] = inputs[t]->stride(dim - 1) == 1 || inputs[t]->size(dim - 1) == 1 ? *inputs[t] : inputs[t]->contiguous();
    const Tensor& x = keep[t];
    some = &x;
    // the stride of a dim with one element says nothing
    auto stride = [&](int i) -> int64_t { return x.size(i) > 1 ? x.stride(i) : 0; };
    FhobRotaryTensor& d = r.tensor[r.tensors++];
    d.in = x.const_data_ptr();
    d.out = out[t].mutable_data_ptr();
    TORCH_CHECK_VALUE(x.size(dim - 3) <= (1 << 20), "at most 2^20 heads are turned in one call, got ", x.size(dim - 3));
    d.heads = static_cast<int32_t>(x.size(dim - 3));
    d.row = stride(dim - 2);
    d.head = stride(dim - 3);
    d.batch = dim == 4 ? stride(0) : 0;
    r.batch = dim == 4 ? x.size(0) : 1;
    r.n = x.size(dim - 2);
    r.d = static_cast<int32_t>(x.size(dim - 1));
    r.dtype = type_of(x);
  }
  if (!some) return out;
  r.pairs = static_cast<int32_t>(frequencies.size(0));
  r.axes = static_cast<int32_t>(positions.size(0));
  for (int i = 0; i < r.pairs; ++i) axes[i] = static_cast<uint8_t>(axis_of_pair.empty() ? 0 : axis_of_pair[i]);
  r.axis_of_pair = axes;
  r.interleaved = interleaved;
  r.inverse = inverse;
  r.positions = positions.const_data_ptr();
  r.positions_are_64_bit = positions.scalar_type() == at::kLong;
  r.pos_axis = positions.stride(0);
  r.pos_batch = positions.dim() == 3 && positions.size(1) > 1 ? positions.stride(1) : 0;
  r.pos_n = positions.stride(positions.dim() - 1);
  const Tensor f = frequencies.contiguous();
  r.frequencies = f.const_data_ptr();
  r.frequencies_are_64_bit = f.scalar_type() == at::kDouble;
  launch(*some, "fhob_rotary", [&](cudaStream_t s) { return fhob_rotary(&r, s); });
  return out;
}

// The rotation is linear and its transpose is the rotation by the negative angles, so the backward pass is the
// function itself and can be differentiated as often as one likes.
struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, Tensor x0, Maybe second, Tensor positions, Tensor frequencies, Axes axes, bool interleaved,
                               bool inverse) {
    const Tensor x1 = given(second);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["axes"] = axes;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["both"] = x1.defined();
    const auto out = rotate(x0, x1, positions, frequencies, axes, interleaved, inverse);
    if (!x1.defined()) return {out[0]};
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const Axes axes = ctx->saved_data["axes"].toIntVector();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = !ctx->saved_data["inverse"].toBool();
    Tensor d[2];
    const bool has0 = g[0].defined(), has1 = ctx->saved_data["both"].toBool() && g[1].defined();
    if (!has0 && !has1) return variable_list(7);
    if (!at::GradMode::is_enabled() && !has_tangent({&g[0], has1 ? &g[1] : &g[0]})) {   // no derivative of this is asked for
      const auto r = rotate(has0 ? g[0] : g[1], has0 && has1 ? g[1] : Tensor(), s[0], s[1], axes, interleaved, inverse);
      d[has0 ? 0 : 1] = r[0];
      if (has0 && has1) d[1] = r[1];
    } else {
      const auto r = Rotary::apply(has0 ? g[0] : g[1], has0 && has1 ? Maybe(g[1]) : Maybe(), s[0], s[1], axes, interleaved, inverse);
      d[has0 ? 0 : 1] = r[0];
      if (has0 && has1) d[1] = r[1];
    }
    return {d[0], d[1], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

void check_rotary(const Tensor* const* x, int count, const Tensor& positions, const Tensor& frequencies, const Axes& axes) {
  const Tensor& q = *x[0];
  TORCH_CHECK_TYPE(type_of(q) >= 0, "dtype ", q.scalar_type(), " not supported: bfloat16, float16 or float32");
  for (int i = 0; i < count; ++i) {
    const Tensor& t = *x[i];
    TORCH_CHECK_VALUE(t.dim() == 3 || t.dim() == 4, "expected (H, N, D) or (B, H, N, D), got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == q.device(), "tensor ", i, " is on ", t.device(), ", the first one on ", q.device());
    TORCH_CHECK_TYPE(t.scalar_type() == q.scalar_type(), "tensor ", i, " has dtype ", t.scalar_type(), ", the first one ", q.scalar_type());
    TORCH_CHECK_VALUE(t.dim() == q.dim() && t.size(-1) == q.size(-1) && t.size(-2) == q.size(-2) && (t.dim() == 3 || t.size(0) == q.size(0)),
                      "tensors may differ in their heads only, got ", q.sizes(), " and ", t.sizes());
  }
  TORCH_CHECK_TYPE(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "positions must be int32 or int64, got ",
                   positions.scalar_type());
  TORCH_CHECK_VALUE(positions.device() == q.device(), "positions are on ", positions.device(), ", the tensors on ", q.device());
  const int64_t batch = q.dim() == 4 ? q.size(0) : 1, n = q.size(-2);
  TORCH_CHECK_VALUE((positions.dim() == 2 && positions.size(1) == n) ||
                        (positions.dim() == 3 && (positions.size(1) == batch || positions.size(1) == 1) && positions.size(2) == n),
                    "positions: expected (axes, N) or (axes, B, N) with B = ", batch, ", N = ", n, ", got ", positions.sizes());
  TORCH_CHECK_VALUE(positions.size(0) >= 1 && positions.size(0) <= 255, "positions: between 1 and 255 axes, got ", positions.size(0));
  TORCH_CHECK_TYPE(frequencies.scalar_type() == at::kFloat || frequencies.scalar_type() == at::kDouble, "frequencies must be float32 or float64, got ",
                   frequencies.scalar_type());
  TORCH_CHECK_VALUE(frequencies.device() == q.device(), "frequencies are on ", frequencies.device(), ", the tensors on ", q.device());
  TORCH_CHECK_VALUE(!frequencies.requires_grad() && !has_tangent({&frequencies}), "frequencies are constants: no gradient flows into them (pass frequencies.detach())");
  TORCH_CHECK_VALUE(frequencies.dim() == 1 && frequencies.size(0) >= 1 && 2 * frequencies.size(0) <= q.size(-1),
                    "frequencies: expected one for each of at most D / 2 = ", q.size(-1) / 2, " pairs, got ", frequencies.sizes());
  TORCH_CHECK_VALUE(q.size(-1) <= FHOB_ROTARY_MAX_DIM, "rows of at most ", FHOB_ROTARY_MAX_DIM, " elements, got ", q.size(-1));
  TORCH_CHECK_VALUE(!axes.empty() || positions.size(0) == 1, "axis_of_pair is needed with positions of ", positions.size(0), " axes");
  TORCH_CHECK_VALUE(axes.empty() || static_cast<int64_t>(axes.size()) == frequencies.size(0), "axis_of_pair: expected ", frequencies.size(0),
                    " entries, got ", axes.size());
  for (const int64_t a : axes) TORCH_CHECK_VALUE(a >= 0 && a < positions.size(0), "axis_of_pair: ", a, " is not an axis of positions (", positions.size(0), ")");
  TORCH_CHECK_VALUE(q.is_cuda(), "rotary needs CUDA tensors, got one on ", q.device());
}

// ------------------------------------------------------------------ layer norm

// Rows of a tensor (..., cols) at one stride, or a contiguous copy's.
struct Rows {
  Tensor t;
  int64_t stride = 0;
  const void* ptr() const { return t.const_data_ptr(); }
};
Rows rows_of(const Tensor& x) {
  Rows r;
  const int64_t cols = x.size(-1);
  // the dims in front of the last, from the inside: one stride for all their rows?
  bool one = x.stride(-1) == 1 || cols == 1;
  int64_t inside = 0;   // rows of the dims seen so far
  for (int64_t i = x.dim() - 2; i >= 0 && one; --i) {
    if (x.size(i) == 1) continue;
    if (!inside) r.stride = x.stride(i);
    else one = x.stride(i) == r.stride * inside;
    inside = (inside ? inside : 1) * x.size(i);
  }
  r.t = one ? x : x.contiguous();
  if (!one || !inside) r.stride = cols;
  return r;
}

FhobLayerNorm describe(const Rows& x, const Tensor& w, const Tensor& mean, const Tensor& rstd) {
  FhobLayerNorm n;
  memset(&n, 0, sizeof(n));
  n.cols = static_cast<int32_t>(x.t.size(-1));
  n.rows = x.t.numel() / n.cols;
  n.dtype = n.w_dtype = type_of(x.t);
  n.x = x.ptr();
  n.x_row = x.stride;
  if (w.defined()) {
    n.w = w.const_data_ptr();
    n.w_dtype = type_of(w);
  }
  n.mean = static_cast<float*>(mean.data_ptr());
  n.rstd = static_cast<float*>(rstd.data_ptr());
  return n;
}

Tensor column_workspace(FhobLayerNorm& n, const Tensor& x) {
  const size_t bytes = fhob_layer_norm_workspace_bytes(n.cols);
  Tensor ws = at::detail::empty_cuda({static_cast<int64_t>(bytes)}, at::kByte, x.device(), std::nullopt);
  n.workspace = ws.data_ptr();
  n.workspace_bytes = bytes;
  return ws;
}

void norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor& y, Tensor& mean, Tensor& rstd) {
  y = new_like(x);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  mean = at::detail::empty_cuda(lead, at::kFloat, x.device(), std::nullopt);
  rstd = at::detail::empty_cuda(lead, at::kFloat, x.device(), std::nullopt);
  if (x.numel() == 0) return;
  const Rows r = rows_of(x);
  const Tensor wc = w.defined() ? w.contiguous() : w, bc = b.defined() ? b.contiguous() : b;
  FhobLayerNorm n = describe(r, wc, mean, rstd);
  if (bc.defined()) {
    n.b = bc.const_data_ptr();
    n.w_dtype = type_of(bc);
  }
  n.eps = static_cast<float>(eps);
  launch(x, "fhob_layer_norm", [&](cudaStream_t s) { return fhob_layer_norm(&n, y.data_ptr(), s); });
}

// dx, and where wanted dw and db of type `wt`
void norm_backward(const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& mean, const Tensor& rstd, bool want_dw, bool want_db,
                   at::ScalarType wt, Tensor& dx, Tensor& dw, Tensor& db) {
  dx = new_like(x);
  const int64_t cols = x.size(-1);
  if (x.numel() == 0) {
    const auto options = x.options().dtype(wt);
    if (want_dw) dw = at::zeros({cols}, options);
    if (want_db) db = at::zeros({cols}, options);
    return;
  }
  if (want_dw) dw = at::detail::empty_cuda({cols}, wt, x.device(), std::nullopt);
  if (want_db) db = at::detail::empty_cuda({cols}, wt, x.device(), std::nullopt);
  const Rows r = rows_of(x), g = rows_of(dy);
  const Tensor wc = w.defined() ? w.contiguous() : w;
  FhobLayerNorm n = describe(r, wc, mean, rstd);
  n.w_dtype = wt == at::kFloat ? FHOB_F32 : type_of(x);
  Tensor ws;
  if (want_dw || want_db) ws = column_workspace(n, x);
  launch(x, "fhob_layer_norm_backward", [&](cudaStream_t s) {
    return fhob_layer_norm_backward(&n, g.ptr(), g.stride, dx.data_ptr(), want_dw ? dw.data_ptr() : nullptr, want_db ? db.data_ptr() : nullptr, s);
  });
}

// ddy, dx2, and dw2 if there is a weight; any of the cotangents may be undefined
void norm_bwdbwd(const Tensor& ddx, const Tensor& ddw, const Tensor& ddb, const Tensor& dy, const Tensor& x, const Tensor& w, const Tensor& mean,
                 const Tensor& rstd, Tensor& ddy, Tensor& dx2, Tensor& dw2) {
  ddy = new_like(x);
  dx2 = new_like(x);
  if (x.numel() == 0) {
    if (w.defined()) dw2 = at::zeros_like(w);
    return;
  }
  const Rows r = rows_of(x), g = rows_of(dy), v = ddx.defined() ? rows_of(ddx) : Rows();
  const Tensor wc = w.defined() ? w.contiguous() : w;
  const Tensor vw = ddw.defined() ? ddw.contiguous() : ddw, vb = ddb.defined() ? ddb.contiguous() : ddb;
  FhobLayerNorm n = describe(r, wc, mean, rstd);
  if (vw.defined() || vb.defined()) n.w_dtype = type_of(vw.defined() ? vw : vb);
  Tensor ws;
  if (w.defined()) {
    dw2 = new_like(w);
    ws = column_workspace(n, x);
  }
  launch(x, "fhob_layer_norm_bwdbwd", [&](cudaStream_t s) {
    return fhob_layer_norm_bwdbwd(&n, g.ptr(), g.stride, ddx.defined() ? v.ptr() : nullptr, v.stride, vw.defined() ? vw.const_data_ptr() : nullptr,
                                  vb.defined() ? vb.const_data_ptr() : nullptr, ddy.data_ptr(), dx2.data_ptr(), dw2.defined() ? dw2.data_ptr() : nullptr, s);
  });
}

// Stands behind the results of the double backward when a graph of them is asked for: they have no derivative of
// their own here, which must not pass for zero.
struct NoThirdDerivative : torch::autograd::Function<NoThirdDerivative> {
  static variable_list forward(AutogradContext*, Tensor ddy, Tensor dx2, Maybe dw2, Tensor, Tensor, Maybe, Maybe, Maybe, Maybe) {
    variable_list out = {ddy, dx2};
    if (dw2) out.push_back(*dw2);
    return out;
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "fhob.layer_norm is differentiable twice: its third derivative is not implemented");
  }
};

struct LayerNormBackward : torch::autograd::Function<LayerNormBackward> {
  // results: dx, then dw and db where wanted
  static variable_list forward(AutogradContext* ctx, Tensor dy, Tensor x, Maybe weight, Tensor mean, Tensor rstd, bool want_dw, bool want_db, int64_t wt) {
    const Tensor w = given(weight);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({dy, x, w, mean, rstd});
    ctx->saved_data["want_dw"] = want_dw;
    ctx->saved_data["want_db"] = want_db;
    Tensor dx, dw, db;
    norm_backward(dy, x, w, mean, rstd, want_dw, want_db, static_cast<at::ScalarType>(wt), dx, dw, db);
    variable_list out = {dx};
    if (want_dw) out.push_back(dw);
    if (want_db) out.push_back(db);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const bool has_dw = ctx->saved_data["want_dw"].toBool(), has_db = ctx->saved_data["want_db"].toBool();
    const Tensor ddw = has_dw ? g[1] : Tensor(), ddb = has_db ? g[1 + has_dw] : Tensor();
    Tensor ddy, dx2, dw2;
    norm_bwdbwd(g[0], ddw, ddb, s[0], s[1], s[2], s[3], s[4], ddy, dx2, dw2);
    if (at::GradMode::is_enabled() || has_tangent({&g[0], &ddw, &ddb})) {
      const auto r = NoThirdDerivative::apply(ddy, dx2, maybe(dw2), s[0], s[1], maybe(s[2]), maybe(g[0]), maybe(ddw), maybe(ddb));
      ddy = r[0];
      dx2 = r[1];
      if (dw2.defined()) dw2 = r[2];
    }
    return {ddy, dx2, dw2, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Maybe weight, Maybe bias, double eps) {
    const Tensor w = given(weight), b = given(bias);
    Tensor y, mean, rstd;
    norm_forward(x, w, b, eps, y, mean, rstd);
    ctx->save_for_backward({x, w, mean, rstd});
    ctx->saved_data["bias"] = b.defined();
    ctx->saved_data["type"] = static_cast<int64_t>(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const bool has_w = s[1].defined();   // (inputs are counted without those that are missing)
    const bool want_dw = has_w && ctx->needs_input_grad(1), want_db = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(1 + has_w);
    if (!at::GradMode::is_enabled() && !has_tangent({&g[0]})) {   // no derivative of this is asked for
      Tensor dx, dw, db;
      norm_backward(g[0], s[0], s[1], s[2], s[3], want_dw, want_db, static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()), dx, dw, db);
      return {dx, dw, db, Tensor()};
    }
    const auto r = LayerNormBackward::apply(g[0], s[0], maybe(s[1]), s[2], s[3], want_dw, want_db, ctx->saved_data["type"].toInt());
    return {r[0], want_dw ? r[1] : Tensor(), want_db ? r[1 + want_dw] : Tensor(), Tensor()};
  }
};

void check_norm_input(const Tensor& x) {
  TORCH_CHECK_TYPE(type_of(x) >= 0, "dtype ", x.scalar_type(), " not supported: bfloat16, float16 or float32");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= FHOB_LAYER_NORM_MAX_COLS, "x: rows of 1 to ", FHOB_LAYER_NORM_MAX_COLS,
                    " elements, got ", x.sizes());
}
void check_device(const Tensor& x) { TORCH_CHECK_VALUE(x.is_cuda(), "layer_norm needs CUDA tensors, got one on ", x.device()); }
// a vector over the columns of x (or undefined)
void check_vector(const Tensor& v, const char* name, const Tensor& x, const Tensor& like) {
  if (!v.defined()) return;
  TORCH_CHECK_VALUE(v.device() == x.device(), name, " is on ", v.device(), ", x on ", x.device());
  TORCH_CHECK_VALUE(v.dim() == 1 && v.size(0) == x.size(-1), name, ": expected (", x.size(-1), "), got ", v.sizes());
  TORCH_CHECK_TYPE(v.scalar_type() == at::kFloat || v.scalar_type() == x.scalar_type(), name, " must be float32 or ", x.scalar_type(), ", got ",
                   v.scalar_type());
  TORCH_CHECK_TYPE(!like.defined() || like.scalar_type() == v.scalar_type(), name, " has dtype ", v.scalar_type(), ", the weight ", like.defined() ? like.scalar_type() : v.scalar_type());
}
void check_matrix(const Tensor& m, const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(m.device() == x.device(), name, " is on ", m.device(), ", x on ", x.device());
  TORCH_CHECK_TYPE(m.scalar_type() == x.scalar_type(), name, " has dtype ", m.scalar_type(), ", x ", x.scalar_type());
  TORCH_CHECK_VALUE(m.sizes() == x.sizes(), name, ": expected ", x.sizes(), ", got ", m.sizes());
}
Tensor check_statistic(const Tensor& m, const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(m.device() == x.device(), name, " is on ", m.device(), ", x on ", x.device());
  TORCH_CHECK_TYPE(m.scalar_type() == at::kFloat, name, " must be float32, got ", m.scalar_type());
  TORCH_CHECK_VALUE(m.sizes() == x.sizes().slice(0, x.dim() - 1), name, ": expected ", x.sizes().slice(0, x.dim() - 1), ", got ", m.sizes());
  return m.contiguous();
}

// ------------------------------------------------------------------ module functions

const Tensor& tensor_arg(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}
Tensor optional_arg(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor_arg(o, name); }

// Does the call go through its autograd function?
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (has_tangent(ts)) return true;
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

PyObject* to_tuple(const Tensor* t, int n) {   // None for undefined
  PyObject* r = PyTuple_New(n);
  for (int i = 0; r && i < n; ++i) {
    if (!t[i].defined()) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(r, i, t[i].defined() ? THPVariable_Wrap(t[i]) : Py_None);
  }
  return r;
}

double eps_arg(PyObject* o) {
  const double eps = PyFloat_AsDouble(o);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "eps must not be negative, got ", eps);
  return eps;
}

}  // namespace

// rotary(tensors (a tuple of one or two), positions, frequencies, axis_of_pair (None or a sequence), interleaved, inverse) -> tuple
PyObject* fhob_py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6 && PyTuple_Check(a[0]), "rotary takes 6 arguments");
  const Py_ssize_t count = PyTuple_GET_SIZE(a[0]);
  TORCH_CHECK_VALUE(count == 1 || count == 2, "rotary takes one or two tensors, got ", count);
  const Tensor* x[2] = {nullptr, nullptr};
  for (Py_ssize_t i = 0; i < count; ++i) x[i] = &tensor_arg(PyTuple_GET_ITEM(a[0], i), "x");
  const Tensor &positions = tensor_arg(a[1], "positions"), &frequencies = tensor_arg(a[2], "frequencies");
  Axes axes;
  if (a[3] != Py_None) {
    PyObject* list = PySequence_Fast(a[3], "axis_of_pair must be a sequence of integers");
    if (!list) throw python_error();
    const py::object own = py::reinterpret_steal<py::object>(list);
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(list); ++i) {
      const long long axis = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(list, i));
      if (axis == -1 && PyErr_Occurred()) throw python_error();
      axes.push_back(axis);
    }
    TORCH_CHECK_VALUE(!axes.empty(), "axis_of_pair is empty");
  }
  const int interleaved = PyObject_IsTrue(a[4]), inverse = PyObject_IsTrue(a[5]);
  if (interleaved < 0 || inverse < 0) throw python_error();
  check_rotary(x, static_cast<int>(count), positions, frequencies, axes);
  const Tensor second = count == 2 ? *x[1] : Tensor();
  Tensor r[2];
  {
    pybind11::gil_scoped_release nogil;
    if (wants_grad({x[0], &second})) {
      const auto out = Rotary::apply(*x[0], maybe(second), positions, frequencies, axes, interleaved == 1, inverse == 1);
      for (size_t i = 0; i < out.size(); ++i) r[i] = out[i];
    } else {
      const auto out = rotate(*x[0], second, positions, frequencies, axes, interleaved == 1, inverse == 1);
      r[0] = out[0];
      r[1] = out[1];
    }
  }
  return to_tuple(r, static_cast<int>(count));
  END_HANDLE_TH_ERRORS
}

// layer_norm(x, weight, bias, eps) -> y, differentiable twice
PyObject* fhob_py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4, "layer_norm takes 4 arguments");
  const Tensor& x = tensor_arg(a[0], "x");
  const Tensor w = optional_arg(a[1], "weight"), b = optional_arg(a[2], "bias");
  const double eps = eps_arg(a[3]);
  check_norm_input(x);
  check_vector(w, "weight", x, Tensor());
  check_vector(b, "bias", x, w);
  check_device(x);
  Tensor y;
  {
    pybind11::gil_scoped_release nogil;
    if (wants_grad({&x, &w, &b})) {
      y = LayerNorm::apply(x, maybe(w), maybe(b), eps);
    } else {
      Tensor mean, rstd;
      norm_forward(x, w, b, eps, y, mean, rstd);
    }
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// layer_norm_forward(x, weight, bias, eps) -> (y, mean, rstd)
PyObject* fhob_py_layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4, "layer_norm_forward takes 4 arguments");
  const Tensor& x = tensor_arg(a[0], "x");
  const Tensor w = optional_arg(a[1], "weight"), b = optional_arg(a[2], "bias");
  const double eps = eps_arg(a[3]);
  check_norm_input(x);
  check_vector(w, "weight", x, Tensor());
  check_vector(b, "bias", x, w);
  check_device(x);
  Tensor r[3];
  {
    pybind11::gil_scoped_release nogil;
    norm_forward(x, w, b, eps, r[0], r[1], r[2]);
  }
  return to_tuple(r, 3);
  END_HANDLE_TH_ERRORS
}

// layer_norm_backward(dy, x, weight, mean, rstd, want_db) -> (dx, dw or None, db or None)
PyObject* fhob_py_layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "layer_norm_backward takes 6 arguments");
  const Tensor &dy = tensor_arg(a[0], "dy"), &x = tensor_arg(a[1], "x");
  const Tensor w = optional_arg(a[2], "weight");
  check_norm_input(x);
  check_matrix(dy, "dy", x);
  check_vector(w, "weight", x, Tensor());
  const Tensor mean = check_statistic(tensor_arg(a[3], "mean"), "mean", x), rstd = check_statistic(tensor_arg(a[4], "rstd"), "rstd", x);
  check_device(x);
  const int want_db = PyObject_IsTrue(a[5]);
  if (want_db < 0) throw python_error();
  Tensor r[3];
  {
    pybind11::gil_scoped_release nogil;
    norm_backward(dy, x, w, mean, rstd, w.defined(), want_db == 1, w.defined() ? w.scalar_type() : x.scalar_type(), r[0], r[1], r[2]);
  }
  return to_tuple(r, 3);
  END_HANDLE_TH_ERRORS
}

// layer_norm_bwdbwd(ddx, ddw, ddb, dy, x, weight, mean, rstd) -> (ddy, dx2, dw2 or None)
PyObject* fhob_py_layer_norm_bwdbwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "layer_norm_bwdbwd takes 8 arguments");
  const Tensor ddx = optional_arg(a[0], "ddx"), ddw = optional_arg(a[1], "ddw"), ddb = optional_arg(a[2], "ddb");
  const Tensor &dy = tensor_arg(a[3], "dy"), &x = tensor_arg(a[4], "x");
  const Tensor w = optional_arg(a[5], "weight");
  check_norm_input(x);
  check_matrix(dy, "dy", x);
  if (ddx.defined()) check_matrix(ddx, "ddx", x);
  check_vector(w, "weight", x, Tensor());
  TORCH_CHECK_VALUE(w.defined() || !ddw.defined(), "ddw needs a weight");
  check_vector(ddw, "ddw", x, w);
  check_vector(ddb, "ddb", x, w);
  const Tensor mean = check_statistic(tensor_arg(a[6], "mean"), "mean", x), rstd = check_statistic(tensor_arg(a[7], "rstd"), "rstd", x);
  check_device(x);
  Tensor r[3];
  {
    pybind11::gil_scoped_release nogil;
    norm_bwdbwd(ddx, ddw, ddb, dy, x, w, mean, rstd, r[0], r[1], r[2]);
  }
  return to_tuple(r, 3);
  END_HANDLE_TH_ERRORS
}
