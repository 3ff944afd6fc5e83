// The ranking-head operators as differentiable functions of torch tensors (the extension module behind
// collie_amd/functional.py, which documents them): checks, outputs, workspaces and the autograd nodes
// around the C entry points.  Unlike the other operators these are not called through ctypes: a
// training step of a small batch is host time here, and nodes in Python, which autograd runs on its
// own thread, took several times as long as the launches.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>

#include "../../include/collie_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

namespace {

// becomes collie_amd._lib.CollieHipError
struct HipError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
#define REFUSE_VALUE(cond, ...) \
  if (cond) throw py::value_error(c10::str(__VA_ARGS__))
#define REFUSE(cond, ...) \
  if (cond) throw HipError(c10::str(__VA_ARGS__))

void check(int rc, const char* what) {
  REFUSE(rc != 0, what, " failed (", rc, "): ", collie_last_error());
}

collie_stream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void require_hip(const Tensor& t, const char* what) {
  REFUSE(!t.is_cuda(), what, ": tensor is on ", t.device(),
         "; collie_amd computes on a HIP device only (no CPU fallback). Move the model and data with "
         "``.to(\"cuda\")``.");
}

// The kernels see memory.  A tensor that stands for something else (a batch of vmap, a subclass such as a
// fake tensor), one with a tangent of forward-mode differentiation, and any tensor while a graph is
// being recorded from torch's own calls, would lose that silently.
bool plain(const Tensor& t) {
  using c10::DispatchKey;
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  static const c10::DispatchKeySet wrapped({DispatchKey::Python, DispatchKey::FuncTorchBatched,
                                            DispatchKey::FuncTorchGradWrapper,
                                            DispatchKey::Functionalize});
  if (t.key_set().has_any(wrapped) || !t.has_storage() || t._fw_grad(0).defined()) return false;
  return !torch::jit::tracer::isTracing() && !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) &&
         !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) &&
         !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL);
}

void require_plain(const MaybeTensor& t) {
  REFUSE(t && t->defined() && !plain(*t),
         "collie_amd computes on memory: tensors under vmap, torch.func or torch.jit.trace, fake tensors and "
         "tensors with a forward-mode tangent are not supported");
}
template <typename... Rest>
void require_plain(const MaybeTensor& t, const Rest&... rest) {
  require_plain(t);
  require_plain(rest...);
}

std::string dtype(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kDouble: return "torch.float64";
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    default: return c10::toString(t.scalar_type());
  }
}

int32_t element_type(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return COLLIE_F32;
    case at::kBFloat16: return COLLIE_BF16;
    case at::kHalf: return COLLIE_F16;
    default:
      throw HipError(c10::str(what, " must be float32, bfloat16 or float16, not ", dtype(t)));
  }
}

int32_t id_type(const Tensor& ids) {
  REFUSE(ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong,
         "index tensors must be int32 or int64, not ", dtype(ids));
  return ids.scalar_type() == at::kLong ? COLLIE_I64 : COLLIE_I32;
}

// widths are 32-bit numbers at the C entry points
void check_width(int64_t n) {
  REFUSE_VALUE(n > INT32_MAX, "rows of ", n, " elements are too wide");
}

void* at_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// a tensor as [rows, width] with contiguous rows that do not overlap (a copy only if it must be)
struct Rows {
  Tensor t;
  int64_t ld;
};
Rows rows_view(const Tensor& t, int64_t width) {
  if (t.is_contiguous()) return {t.dim() == 2 ? t : t.reshape({-1, width}), width};
  if (t.dim() != 2 || t.stride(1) != 1 || (t.size(0) > 1 && t.stride(0) < width))
    return {t.contiguous().reshape({-1, width}), width};
  return {t, t.size(0) > 1 ? t.stride(0) : width};
}

// a parameter of a layer: on x's device, of its type (or float32 where `f32`), contiguous
Tensor param(const MaybeTensor& p, const Tensor& x, at::IntArrayRef shape, const char* what,
             bool f32 = false) {
  if (!p || !p->defined()) return Tensor();
  REFUSE_VALUE(p->sizes() != shape, what, " must have shape ", shape, ", not ", p->sizes());
  REFUSE(p->device() != x.device(), what, " is on ", p->device(), ", x is on ", x.device());
  REFUSE(p->scalar_type() != x.scalar_type() && !(f32 && p->scalar_type() == at::kFloat), what, " is ",
         dtype(*p), ", x is ", dtype(x));
  return p->contiguous();
}

Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// an argument that may be absent, for a node: absent ones have no edge in the graph
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }
Tensor given(const MaybeTensor& t) { return t.value_or(Tensor()); }

// which of a node's tensors are there, a bit each
int64_t present(std::initializer_list<const Tensor*> tensors) {
  int64_t bits = 0, i = 0;
  for (const Tensor* t : tensors) bits |= static_cast<int64_t>(t->defined()) << i++;
  return bits;
}

// which of them take a gradient in this backward pass (edges count the present ones)
int64_t wanted(AutogradContext* ctx, int64_t there) {
  int64_t want = 0, edge = 0;
  for (int i = 0; there >> i; ++i)
    if (there >> i & 1) want |= static_cast<int64_t>(ctx->needs_input_grad(edge++)) << i;
  return want;
}

bool takes_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  return at::GradMode::is_enabled() &&
         std::any_of(tensors.begin(), tensors.end(), [](const Tensor* t) { return takes_grad(*t); });
}

// Gradients that cannot be differentiated again, with respect to any of the tensors they come from, say
// so when that is tried; without create_graph (grad mode off) nobody can.
variable_list once(variable_list grads, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::Error>(
      "collie_amd: this layer can be differentiated once", torch::autograd::collect_next_edges(from));
  for (Tensor& g : grads)
    if (g.defined()) torch::autograd::set_history(g, error);
  return grads;
}

// ---- embedding rows --------------------------------------------------------------------------------
Tensor lookup(const Tensor& table, const Tensor& ids, double scale, const Tensor& status) {
  const int32_t tag = element_type(table, "table");
  const Tensor w = table.contiguous(), i = ids.contiguous();
  auto shape = ids.sizes().vec();
  shape.push_back(w.size(1));
  Tensor out = at::empty(shape, w.options());
  c10::DeviceGuard guard(w.device());
  check(collie_embedding_rows(w.data_ptr(), tag, w.size(0), w.size(1), i.data_ptr(), id_type(i),
                              i.numel(), scale, out.data_ptr(),
                              static_cast<int32_t*>(at_or_null(status)), stream_of(w)),
        "collie_embedding_rows");
  return out;
}

Tensor lookup_grad(const Tensor& ids, const Tensor& dy, int64_t num_rows, double scale,
                   int64_t padding, const Tensor& status) {
  const int64_t dim = dy.size(-1), n = ids.numel();
  const Tensor i = ids.contiguous();
  const Rows g = rows_view(dy, dim);
  Tensor grad = at::empty({num_rows, dim}, dy.options());
  const Tensor ws = scratch(collie_embedding_rows_grad_workspace_bytes(n, dim), dy);
  c10::DeviceGuard guard(dy.device());
  check(collie_embedding_rows_grad(i.data_ptr(), id_type(i), n, g.t.data_ptr(), g.ld,
                                   element_type(dy, "dy"), num_rows, dim, scale, padding,
                                   grad.data_ptr(), ws.data_ptr(), ws.numel(),
                                   static_cast<int32_t*>(at_or_null(status)), stream_of(dy)),
        "collie_embedding_rows_grad");
  return grad;
}

// The same for tensors that are not plain (a gradient under vmap or with a forward-mode tangent), in
// torch's operations: ids outside the table go to a row of zeros behind it.
Tensor inside(const Tensor& ids, int64_t num_rows) {
  return ids.reshape({-1}).to(at::kLong).clamp(-1, num_rows).remainder(num_rows + 1);
}

Tensor plain_lookup(const Tensor& table, const Tensor& ids, double scale) {
  auto shape = ids.sizes().vec();
  shape.push_back(table.size(1));
  const Tensor rows = at::cat({table, at::zeros({1, table.size(1)}, table.options())});
  return (rows.index_select(0, inside(ids, table.size(0))).to(at::kFloat) * scale)
      .to(table.scalar_type())
      .reshape(shape);
}

Tensor plain_lookup_grad(const Tensor& ids, const Tensor& dy, int64_t num_rows, double scale,
                         int64_t padding) {
  Tensor to = inside(ids, num_rows);
  if (padding >= 0) to = to.masked_fill(to == padding, num_rows);
  const Tensor vals = dy.reshape({-1, dy.size(-1)}).to(at::kFloat) * scale;
  return at::zeros({num_rows + 1, vals.size(1)}, vals.options())
      .index_add(0, to, vals)
      .narrow(0, 0, num_rows)
      .to(dy.scalar_type());
}

struct LookupGrad;

struct Lookup : torch::autograd::Function<Lookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids,
                        const MaybeTensor& status, double scale, int64_t padding, bool sparse) {
    ctx->save_for_backward({ids});
    ctx->saved_data["status"] = status;   // a flag that others set in place: no saved variable
    ctx->saved_data["rest"] = c10::IValue(std::vector<int64_t>{table.size(0), padding, sparse});
    ctx->saved_data["scale"] = scale;
    return lookup(table, ids, scale, given(status));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

// the gradient is linear in dy: its own gradient is the lookup again
struct LookupGrad : torch::autograd::Function<LookupGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dy, const Tensor& ids,
                        const MaybeTensor& status, int64_t num_rows, double scale,
                        int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["status"] = status;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["scale"] = scale;
    return lookup_grad(ids, dy, num_rows, scale, padding, given(status));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor out = plain(grads[0])
                     ? Lookup::apply(grads[0], ids, ctx->saved_data["status"].toOptional<Tensor>(), scale,
                                     padding, false)
                     : plain_lookup(grads[0], ids, scale);
    if (padding >= 0) out = out.masked_fill((ids == padding).unsqueeze(-1), 0.0);
    return {out, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

variable_list Lookup::backward(AutogradContext* ctx, variable_list grads) {
  const Tensor ids = ctx->get_saved_variables()[0];
  const MaybeTensor status = ctx->saved_data["status"].toOptional<Tensor>();
  const auto rest = ctx->saved_data["rest"].toIntVector();
  const double scale = ctx->saved_data["scale"].toDouble();
  const int64_t rows = rest[0], padding = rest[1];
  Tensor dw;
  if (rest[2]) {
    // the uncoalesced COO gradient of nn.Embedding(sparse=True), without entries that take no gradient: an
    // index outside the table would be an address outside of it for whoever uses the tensor
    Tensor flat = ids.reshape({-1}).to(at::kLong), vals = grads[0].reshape({-1, grads[0].size(-1)});
    Tensor live = flat.ge(0).logical_and(flat.lt(rows));
    if (padding >= 0) live = live.logical_and(flat.ne(padding));
    const Tensor which = live.nonzero().reshape({-1});
    flat = flat.index_select(0, which);
    vals = vals.index_select(0, which);
    if (scale != 1.0) vals = vals * scale;
    dw = at::sparse_coo_tensor(flat.unsqueeze(0), vals, {rows, vals.size(1)});
  } else if (!plain(grads[0])) {
    dw = plain_lookup_grad(ids, grads[0], rows, scale, padding);
  } else if (at::GradMode::is_enabled()) {
    dw = LookupGrad::apply(grads[0], ids, status, rows, scale, padding);
  } else {
    dw = lookup_grad(ids, grads[0], rows, scale, padding, given(status));
  }
  return {dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
}

Tensor flag_of(const MaybeTensor& status, const Tensor& like) {
  if (!status || !status->defined()) return Tensor();
  REFUSE(status->scalar_type() != at::kInt || status->device() != like.device() || status->numel() < 1,
         "status must be an int32 tensor on the device of the table");
  return *status;
}

Tensor embedding_rows_grad(const Tensor& ids, const Tensor& dy, int64_t num_rows, double scale,
                           std::optional<int64_t> padding, const MaybeTensor& status) {
  require_plain(dy, ids, status);
  REFUSE_VALUE(dy.dim() < 1 || dy.sizes().slice(0, dy.dim() - 1) != ids.sizes(), "dy ", dy.sizes(),
               " does not belong to ids ", ids.sizes());
  REFUSE_VALUE(padding && (*padding < 0 || *padding >= num_rows), "padding_idx ", *padding,
               " is no row of the table");
  check_width(dy.size(-1));
  const Tensor flag = flag_of(status, dy);
  element_type(dy, "dy");
  id_type(ids);
  require_hip(dy, "dy");
  REFUSE(ids.device() != dy.device(), "ids are on ", ids.device(), ", dy is on ", dy.device());
  return lookup_grad(ids, dy, num_rows, scale, padding.value_or(-1), flag);
}

Tensor embedding_rows(const Tensor& weight, const Tensor& ids, double scale,
                      std::optional<int64_t> padding, bool sparse, const MaybeTensor& status) {
  require_plain(weight, ids, status);
  REFUSE_VALUE(weight.dim() != 2, "table must be [rows, dim], not ", weight.sizes());
  REFUSE_VALUE(padding && (*padding < 0 || *padding >= weight.size(0)), "padding_idx ", *padding,
               " is no row of the table");
  check_width(weight.size(1));
  const Tensor flag = flag_of(status, weight);
  element_type(weight, "table");
  id_type(ids);
  require_hip(weight, "table");
  REFUSE(ids.device() != weight.device(), "ids are on ", ids.device(), ", the table is on ",
         weight.device());
  if (!wants_grad({&weight})) return lookup(weight, ids, scale, flag);
  return Lookup::apply(weight, ids, maybe(flag), scale, padding.value_or(-1), sparse);
}

// ---- layer norm ------------------------------------------------------------------------------------
int32_t norm_param_type(const Tensor& w, const Tensor& b, const Tensor& x) {
  return element_type(w.defined() ? w : b.defined() ? b : x, "weight");
}

// y, and mean (two parts) and rstd [3, rows] with `keep`
std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps,
                                       bool keep) {
  const int64_t dim = x.size(-1);
  const Rows r = rows_view(x, dim);
  const int64_t m = r.t.size(0);
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor stats = keep ? at::empty({3, m}, x.options().dtype(at::kFloat)) : Tensor();
  float* mean = static_cast<float*>(at_or_null(stats));
  c10::DeviceGuard guard(x.device());
  check(collie_layer_norm_forward(r.t.data_ptr(), r.ld, element_type(x, "x"), m, dim, at_or_null(w),
                                  at_or_null(b), norm_param_type(w, b, x), eps, y.data_ptr(), mean,
                                  mean ? mean + 2 * m : nullptr, stream_of(x)),
        "collie_layer_norm_forward");
  return {y, stats};
}

struct Norm : torch::autograd::Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight,
                        const MaybeTensor& bias, double eps) {
    const Tensor w = given(weight), b = given(bias);
    auto [y, stats] = norm_forward(x, w, b, eps, true);
    ctx->save_for_backward({x, w, b, stats});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &b = s[2], &stats = s[3];
    require_plain(grads[0]);
    const int64_t dim = x.size(-1);
    const Rows r = rows_view(x, dim), g = rows_view(grads[0], dim);
    const int64_t m = r.t.size(0);
    const int64_t want = wanted(ctx, present({&x, &w, &b}));
    Tensor dx = want & 1 ? at::empty(x.sizes(), x.options()) : Tensor();
    Tensor dw = want & 2 ? at::empty({dim}, w.options()) : Tensor();
    Tensor db = want & 4 ? at::empty({dim}, b.options()) : Tensor();
    const Tensor ws = scratch(collie_layer_norm_backward_workspace_bytes(m, dim), x);
    const float* mean = stats.data_ptr<float>();
    c10::DeviceGuard guard(x.device());
    check(collie_layer_norm_backward(g.t.data_ptr(), g.ld, r.t.data_ptr(), r.ld, element_type(x, "x"),
                                     m, dim, at_or_null(w), norm_param_type(w, b, x), mean, mean + 2 * m,
                                     at_or_null(dx), at_or_null(dw), at_or_null(db), ws.data_ptr(),
                                     ws.numel(), stream_of(x)),
          "collie_layer_norm_backward");
    return once({dx, dw, db, Tensor()}, {grads[0], x, w});
  }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
  require_plain(x, weight, bias);
  REFUSE_VALUE(!(eps >= 0), "eps must not be negative, not ", eps);
  element_type(x, "x");
  REFUSE_VALUE(x.dim() < 1 || x.size(-1) < 1, "x must have a last dimension to normalise, not ",
               x.sizes());
  check_width(x.size(-1));
  const Tensor w = param(weight, x, {x.size(-1)}, "weight", true);
  const Tensor b = param(bias, x, {x.size(-1)}, "bias", true);
  REFUSE(w.defined() && b.defined() && w.scalar_type() != b.scalar_type(), "weight is ",
         dtype(w), ", bias is ", dtype(b));
  require_hip(x, "x");
  if (!wants_grad({&x, &w, &b})) return norm_forward(x, w, b, eps, false).first;
  return Norm::apply(x, maybe(w), maybe(b), eps);
}

// ---- linear and gated layers -----------------------------------------------------------------------
void check_layer(const Tensor& x, const Tensor& weight) {
  element_type(x, "x");
  REFUSE_VALUE(weight.dim() != 2 || x.dim() < 1 || x.size(-1) != weight.size(1), "x ", x.sizes(),
               " and weight ", weight.sizes(),
               " do not fit: expected x [..., n_in] and weight [n_out, n_in]");
  REFUSE_VALUE(weight.numel() == 0, "weight ", weight.sizes(), " is empty");
  check_width(weight.size(0));
  check_width(weight.size(1));
}

struct Forward {
  Tensor y, keep, keep2;
};

// (w2 undefined: the linear layer)
Forward layer_forward(const Tensor& x, const Tensor& w, const Tensor& w2, const Tensor& b,
                      const Tensor& b2, const Tensor& residual, int32_t act, bool keep) {
  const int64_t n_out = w.size(0), n_in = w.size(1);
  const int32_t tag = element_type(x, "x");
  const Rows r = rows_view(x, n_in);
  const int64_t m = r.t.size(0);
  auto shape = x.sizes().vec();
  shape.back() = n_out;
  Rows res{Tensor(), 0};
  if (residual.defined()) res = rows_view(residual, n_out);
  Forward f;
  f.y = at::empty(shape, x.options());
  if (keep && w2.defined()) {
    f.keep = at::empty({m, n_out}, x.options().dtype(at::kFloat));
    f.keep2 = at::empty({m, n_out}, x.options().dtype(at::kFloat));
  } else if (keep && act != COLLIE_ACT_IDENTITY) {
    const bool sign_only = act == COLLIE_ACT_RELU || act == COLLIE_ACT_LEAKY_RELU;
    f.keep = at::empty({m, n_out}, sign_only ? x.options() : x.options().dtype(at::kFloat));
  }
  const Tensor ws = scratch(collie_layer_forward_workspace_bytes(r.t.data_ptr(), r.ld, tag, m, n_in,
                                                                 w.data_ptr(), at_or_null(w2), n_out),
                            x);
  c10::DeviceGuard guard(x.device());
  if (w2.defined())
    check(collie_gated_forward(r.t.data_ptr(), r.ld, tag, m, n_in, w.data_ptr(), w2.data_ptr(),
                               at_or_null(b), at_or_null(b2), n_out, act, at_or_null(f.keep),
                               at_or_null(f.keep2), f.y.data_ptr(), ws.data_ptr(), ws.numel(),
                               stream_of(x)),
          "collie_gated_forward");
  else
    check(collie_linear_forward(r.t.data_ptr(), r.ld, tag, m, n_in, w.data_ptr(), at_or_null(b),
                                n_out, act, at_or_null(res.t), res.ld, at_or_null(f.keep),
                                f.y.data_ptr(), ws.data_ptr(), ws.numel(), stream_of(x)),
          "collie_linear_forward");
  return f;
}

// dx, dw, dw2, db, db2 as far as `want` (a bit each) says so
std::array<Tensor, 5> layer_backward(const Tensor& dy, const Tensor& x, const Tensor& w,
                                     const Tensor& w2, const Tensor& keep, const Tensor& keep2,
                                     int32_t act, int64_t want) {
  const int64_t n_out = w.size(0), n_in = w.size(1);
  const int32_t tag = element_type(x, "x");
  const Rows r = rows_view(x, n_in), g = rows_view(dy, n_out);
  const int64_t m = r.t.size(0);
  std::array<Tensor, 5> d;
  const at::IntArrayRef weights = w.sizes(), bias = weights.slice(0, 1);
  for (int i = 0; i < 5; ++i)
    if (want >> i & 1) {
      const at::IntArrayRef shape = i == 0 ? x.sizes() : i < 3 ? weights : bias;
      d[i] = m ? at::empty(shape, x.options()) : at::zeros(shape, x.options());
    }
  if (m == 0) return d;
  const Tensor ws = scratch(
      collie_layer_backward_workspace_bytes(g.t.data_ptr(), g.ld, r.t.data_ptr(), r.ld, tag, m, n_in,
                                            w.data_ptr(), at_or_null(w2), n_out, act),
      x);
  c10::DeviceGuard guard(x.device());
  if (w2.defined())
    check(collie_gated_backward(g.t.data_ptr(), g.ld, r.t.data_ptr(), r.ld, tag, m, n_in,
                                w.data_ptr(), w2.data_ptr(), n_out, act, keep.data_ptr(),
                                keep2.data_ptr(), at_or_null(d[0]), at_or_null(d[1]),
                                at_or_null(d[2]), at_or_null(d[3]), at_or_null(d[4]), ws.data_ptr(),
                                ws.numel(), stream_of(x)),
          "collie_gated_backward");
  else
    check(collie_linear_backward(g.t.data_ptr(), g.ld, r.t.data_ptr(), r.ld, tag, m, n_in,
                                 w.data_ptr(), n_out, act, at_or_null(keep), at_or_null(d[0]),
                                 at_or_null(d[1]), at_or_null(d[3]), ws.data_ptr(), ws.numel(),
                                 stream_of(x)),
          "collie_linear_backward");
  return d;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                        const MaybeTensor& bias, const MaybeTensor& residual, int64_t act) {
    const Tensor b = given(bias), r = given(residual);
    const bool keep = takes_grad(x) || takes_grad(w) || takes_grad(b);
    const Forward f = layer_forward(x, w, Tensor(), b, Tensor(), r, act, keep);
    ctx->save_for_backward({x, w, f.keep});
    ctx->saved_data["act"] = act;
    ctx->saved_data["there"] = present({&x, &w, &b, &r});
    return f.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const int64_t want = wanted(ctx, ctx->saved_data["there"].toInt());
    std::array<Tensor, 5> d;
    require_plain(grads[0]);
    if (want & 7)
      d = layer_backward(grads[0], s[0], s[1], Tensor(), s[2], Tensor(),
                         ctx->saved_data["act"].toInt(), (want & 3) | (want & 4) << 1);
    variable_list out = once({d[0], d[1], d[3]}, {grads[0], s[0], s[1]});
    // the residual's gradient is dy itself, and as differentiable
    return {out[0], out[1], out[2], want & 8 ? grads[0] : Tensor(), Tensor()};
  }
};

struct Gated : torch::autograd::Function<Gated> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& w2,
                        const MaybeTensor& bias, const MaybeTensor& bias2, int64_t act) {
    const Tensor b = given(bias), b2 = given(bias2);
    const Forward f = layer_forward(x, w, w2, b, b2, Tensor(), act, true);
    ctx->save_for_backward({x, w, w2, f.keep, f.keep2});
    ctx->saved_data["act"] = act;
    ctx->saved_data["there"] = present({&x, &w, &w2, &b, &b2});
    return f.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    require_plain(grads[0]);
    const auto d = layer_backward(grads[0], s[0], s[1], s[2], s[3], s[4],
                                  ctx->saved_data["act"].toInt(),
                                  wanted(ctx, ctx->saved_data["there"].toInt()));
    return once({d[0], d[1], d[2], d[3], d[4], Tensor()}, {grads[0], s[0], s[1], s[2]});
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const MaybeTensor& bias,
              int64_t act, const MaybeTensor& residual) {
  require_plain(x, weight, bias, residual);
  check_layer(x, weight);
  const Tensor w = param(weight, x, weight.sizes(), "weight");
  const Tensor b = param(bias, x, {weight.size(0)}, "bias"), r = given(residual);
  if (r.defined()) {
    auto shape = x.sizes().vec();
    shape.back() = w.size(0);
    REFUSE_VALUE(r.sizes() != at::IntArrayRef(shape), "residual must have shape ",
                 at::IntArrayRef(shape), ", not ", r.sizes());
    REFUSE(r.device() != x.device() || r.scalar_type() != x.scalar_type(), "residual is ", dtype(r),
           " on ", r.device(), ", x is ", dtype(x), " on ", x.device());
  }
  require_hip(x, "x");
  if (!wants_grad({&x, &w, &b, &r}))
    return layer_forward(x, w, Tensor(), b, Tensor(), r, act, false).y;
  return Linear::apply(x, w, maybe(b), maybe(r), act);
}

Tensor gated_linear(const Tensor& x, const Tensor& gate_weight, const Tensor& up_weight,
                    const MaybeTensor& gate_bias, const MaybeTensor& up_bias,
                    int64_t act) {
  require_plain(x, gate_weight, up_weight, gate_bias, up_bias);
  REFUSE_VALUE(gate_bias.has_value() != up_bias.has_value(), "gate_bias and up_bias: both or none");
  check_layer(x, gate_weight);
  const Tensor w = param(gate_weight, x, gate_weight.sizes(), "gate_weight");
  const Tensor w2 = param(up_weight, x, gate_weight.sizes(), "up_weight");
  const Tensor b = param(gate_bias, x, {w.size(0)}, "gate_bias");
  const Tensor b2 = param(up_bias, x, {w.size(0)}, "up_bias");
  require_hip(x, "x");
  if (!wants_grad({&x, &w, &w2, &b, &b2}))
    return layer_forward(x, w, w2, b, b2, Tensor(), act, false).y;
  return Gated::apply(x, w, w2, maybe(b), maybe(b2), act);
}

}  // namespace

PYBIND11_MODULE(_head_autograd, m) {
  static PyObject* error =
      py::object(py::module_::import("collie_amd._lib").attr("CollieHipError")).release().ptr();
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const HipError& e) {
      PyErr_SetString(error, e.what());
    }
  });
  // launches need no interpreter
  using Unlocked = py::call_guard<py::gil_scoped_release>;
  m.def("embedding_rows", &embedding_rows, Unlocked());
  m.def("embedding_rows_grad", &embedding_rows_grad, Unlocked());
  m.def("layer_norm", &layer_norm, Unlocked());
  m.def("linear", &linear, Unlocked());
  m.def("gated_linear", &gated_linear, Unlocked());
  m.def("plain", &plain);
  m.def("rows_view", [](const Tensor& t, int64_t width) {
    const Rows r = rows_view(t, width);
    return std::make_pair(r.t, r.ld);
  });
}
