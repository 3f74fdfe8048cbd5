// Host path of layer norm and the feed-forward block in native code: checks,
// allocations, the C ABI call and the autograd node, on operands in the form
// nearly every call gives them (norm.py and feed_forward.py decide the same in
// Python; there a forward of 187 rows took 35 us of host time, its kernel 4).
//
// Both functions return None for anything but that form (tensors of several
// devices or dtypes, subclasses, lengths that are not integers on the device,
// calls that torch records, forward-mode derivatives, calls the library
// refuses): the caller then takes the Python path, which handles or rejects it.
// The library refuses before it launches a kernel. A launch error raises.
// Nothing is kept between calls but the library's entry points.
#include "fst_block_host.h"

#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>
#include <stdexcept>
#include <string>

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct Library {
  decltype(&fst_layer_norm_forward) norm_forward = nullptr;
  decltype(&fst_layer_norm_backward_workspace_bytes) norm_workspace = nullptr;
  decltype(&fst_layer_norm_backward) norm_backward = nullptr;
  decltype(&fst_ffn_forward) ffn_forward = nullptr;
  decltype(&fst_ffn_backward_workspace_bytes) ffn_workspace = nullptr;
  decltype(&fst_ffn_backward) ffn_backward = nullptr;
  decltype(&fst_last_error) last_error = nullptr;
} lib;

// The library's refusal of a call (before any launch): the Python path reports it.
struct Refused {};

void check(int rc, const char* what, bool may_refuse) {
  if (rc == FST_OK) return;
  if (may_refuse && (rc == FST_EINVAL || rc == FST_EUNSUPPORTED)) throw Refused();
  throw std::runtime_error(std::string(what) + ": " + lib.last_error());
}

// Whether torch's tracer or make_fx is recording: they would take this path's
// outputs for what at::empty gives, as they do not see the launch that fills them.
// The tracer records the Python path as a call; make_fx it refuses.
bool recorded_by_fx() {
  return c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
}
bool recorded() { return torch::jit::tracer::isTracing() || recorded_by_fx(); }

// A tensor with a forward-mode derivative is not plain: without a node here its
// derivative would be lost, and the Python path refuses it.
bool plain(const Tensor& t, const at::Device& dev) {
  return t.defined() && t.layout() == at::kStrided && t.device() == dev && !at::isTensorSubclassLike(t) &&
         !t.is_neg() && !t.is_conj() && !t._fw_grad(/*level=*/0).defined();
}
bool plain(const Maybe& t, const at::Device& dev) { return !t.has_value() || plain(*t, dev); }

int dtype_of(at::ScalarType t) {
  return t == at::kBFloat16 ? FST_BF16 : t == at::kHalf ? FST_F16 : t == at::kFloat ? FST_F32 : -1;
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const int32_t* ints(const Tensor& t) { return static_cast<const int32_t*>(data(t)); }

// The current stream of the tensor's device, made current.
struct OnDevice {
  c10::DeviceGuard guard;
  void* stream;
  explicit OnDevice(const Tensor& t) : guard(t.device()) {
    stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
  }
};

// t [.., n] as rows a fixed stride apart (norm.token_rows): t itself, or a copy.
Tensor token_rows(const Tensor& t, int64_t& stride, size_t align) {
  const int64_t n = t.size(-1);
  const auto sizes = t.sizes(), strides = t.strides();
  bool ok = n == 1 || strides.back() == 1;
  int64_t step = -1, span = 1;  // stride of a row; rows of the dimensions seen
  for (int64_t d = t.dim() - 2; d >= 0 && ok; --d) {
    if (sizes[d] == 1) continue;
    if (step < 0)
      step = strides[d];
    else
      ok = strides[d] == step * span;
    span *= sizes[d];
  }
  stride = step < 0 ? n : step;
  if (!ok || stride < n) {
    stride = n;
    return t.contiguous();
  }
  if (align > 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) % align || stride * t.element_size() % align)) {
    stride = n;
    return t.clone(at::MemoryFormat::Contiguous);
  }
  return t;
}

Tensor dense16(const Maybe& t) {
  if (!t.has_value()) return Tensor();
  const Tensor c = t->contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

// Events of padded x [B, L, n] with lengths, one of rows [L, n] with one length, or
// one of all rows.
struct Batch {
  int64_t B = 1, L = 0;
  Tensor lens;
};
bool batch_of(const Tensor& x, const Maybe& seqlens, Batch& b) {
  if (!seqlens.has_value()) {
    b.L = x.numel() / x.size(-1);
    return b.L <= INT32_MAX;
  }
  const auto t = seqlens->scalar_type();
  if ((x.dim() != 3 && x.dim() != 2) || seqlens->dim() != 1 || (t != at::kInt && t != at::kLong)) return false;
  b.B = x.dim() == 2 ? 1 : x.size(0);
  b.L = x.size(x.dim() - 2);
  if (seqlens->size(0) != b.B) return false;
  b.lens = seqlens->to(at::kInt).contiguous();
  return b.B <= INT32_MAX && b.L <= INT32_MAX;
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const Maybe& t) { return t.has_value() && t->requires_grad(); }

// Gradients of gradients are not offered: where a graph of the backward is
// asked for, differentiating it raises.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list vars;
  for (Tensor& g : grads)
    if (g.defined()) {
      g = g.detach();
      g.set_requires_grad(true);
      vars.push_back(g);
    }
  auto fail = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice ") + what + ", which offers first derivatives only", (int64_t)vars.size());
  vars = (*fail)(std::move(vars));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = vars[i++];
  return grads;
}

// --- layer norm -------------------------------------------------------------

struct NormCall {
  int dtype, param_dtype;
  Batch batch;
  double eps;
};

void norm_forward(const NormCall& c, const Tensor& x, const Maybe& residual, const Tensor& w, const Tensor& b,
                  bool keep, Tensor& xr, int64_t& xs, Tensor& y, Tensor& s, Tensor& stats) {
  const int64_t n = x.size(-1);
  OnDevice on(x);
  xr = token_rows(x, xs, 1);
  int64_t rs = 0;
  Tensor rr;
  if (residual.has_value()) rr = token_rows(*residual, rs, 1);
  const auto opt = x.options().requires_grad(false);
  y = at::empty(x.sizes(), opt);
  if (rr.defined()) s = at::empty(x.sizes(), opt);
  if (keep) stats = at::empty({c.batch.B * c.batch.L, 2}, opt.dtype(at::kFloat));
  check(lib.norm_forward(c.dtype, c.param_dtype, (int)c.batch.B, (int)c.batch.L, (int)n, data(xr), xs, data(rr), rs,
                         data(w), data(b), ints(c.batch.lens), (float)c.eps, data(y), data(s),
                         static_cast<float*>(data(stats)), on.stream),
        "flash_layer_norm", true);
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, const Maybe& weight,
                               const Maybe& bias, const NormCall& c) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor w = weight.has_value() ? weight->contiguous() : Tensor();
    const Tensor b = bias.has_value() ? bias->contiguous() : Tensor();
    Tensor xr, y, s, stats;
    int64_t xs;
    norm_forward(c, x, residual, w, b, true, xr, xs, y, s, stats);
    ctx->save_for_backward({s.defined() ? s : xr, w, c.batch.lens, stats});
    ctx->set_materialize_grads(false);
    ctx->saved_data["call"] = c10::List<int64_t>(
        {c.dtype, c.param_dtype, c.batch.B, c.batch.L, s.defined() ? x.size(-1) : xs, wants_grad(x),
         wants_grad(residual), wants_grad(weight), wants_grad(bias), s.defined()});
    return s.defined() ? variable_list{y, s} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!recorded_by_fx(), "flash_layer_norm backward: make_fx cannot record it");
    const variable_list saved = ctx->get_saved_variables();
    const auto call = ctx->saved_data["call"].toIntVector();
    variable_list out(5);
    const bool residual = call[9];
    const Tensor& s = saved[0];
    const Tensor ds_in = residual ? grads[1] : Tensor();
    if (!grads[0].defined() && !ds_in.defined()) return out;
    {
      at::AutoGradMode no_graph(false);
      OnDevice on(s);
      const auto opt = s.options().requires_grad(false);
      const int64_t n = s.size(-1), B = call[2], L = call[3];
      int64_t dys, dss = 0;
      const Tensor dy = token_rows(grads[0].defined() ? grads[0].to(s.scalar_type()) : at::zeros(s.sizes(), opt), dys, 1);
      const Tensor ds = ds_in.defined() ? token_rows(ds_in.to(s.scalar_type()), dss, 1) : Tensor();
      TORCH_CHECK(dy.sizes() == s.sizes() && dy.device() == s.device() && (!ds.defined() || (ds.sizes() == s.sizes() && ds.device() == s.device())),
                  "flash_layer_norm backward: gradients must have the outputs' shape and device");
      const auto param = opt.dtype(call[1] == FST_F32 ? at::kFloat : s.scalar_type());
      Tensor dx, dw, db, ws;
      if (call[5] || call[6]) dx = at::empty(s.sizes(), opt);
      if (call[7]) dw = at::empty({n}, param);
      if (call[8]) db = at::empty({n}, param);
      size_t bytes = 0;
      if (call[7] || call[8]) {
        bytes = lib.norm_workspace((int)call[0], (int)B, (int)L, (int)n);
        ws = at::empty({(int64_t)std::max<size_t>(bytes, 1)}, opt.dtype(at::kByte));
      }
      check(lib.norm_backward((int)call[0], (int)call[1], (int)B, (int)L, (int)n, data(s), call[4], data(saved[1]),
                              ints(saved[2]), static_cast<const float*>(data(saved[3])), data(dy), dys, data(ds), dss,
                              data(dx), data(dw), data(db), data(ws), bytes, on.stream),
            "flash_layer_norm backward", false);
      if (call[5]) out[0] = dx;
      if (call[6]) out[1] = dx;
      out[2] = dw;
      out[3] = db;
    }
    return once(std::move(out), "flash_layer_norm");
  }
};

py::object norm_call(const Tensor& x, const Maybe& residual, const Maybe& weight, const Maybe& bias, double eps,
                     const Maybe& seqlens) {
  const at::Device dev = x.device();
  if (!lib.norm_forward || !dev.is_cuda() || recorded() || !plain(x, dev) || !plain(residual, dev) || !plain(weight, dev) ||
      !plain(bias, dev) || !plain(seqlens, dev))
    return py::none();
  NormCall c;
  c.dtype = c.param_dtype = dtype_of(x.scalar_type());
  c.eps = eps;
  if (c.dtype < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > INT32_MAX || !(eps >= 0)) return py::none();
  if (residual.has_value() && (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type()))
    return py::none();
  for (const Maybe* t : {&weight, &bias}) {
    if (!t->has_value()) continue;
    if ((*t)->dim() != 1 || (*t)->size(0) != x.size(-1)) return py::none();
    if ((*t)->scalar_type() != x.scalar_type() && (*t)->scalar_type() != at::kFloat) return py::none();
    c.param_dtype = dtype_of((*t)->scalar_type());
  }
  if (weight.has_value() && bias.has_value() && weight->scalar_type() != bias->scalar_type()) return py::none();
  if (!batch_of(x, seqlens, c.batch)) return py::none();
  variable_list out;
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(residual) || wants_grad(weight) || wants_grad(bias))) {
    out = NormFunction::apply(x, residual, weight, bias, c);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor w = weight.has_value() ? weight->contiguous() : Tensor();
    const Tensor b = bias.has_value() ? bias->contiguous() : Tensor();
    Tensor xr, y, s, stats;
    int64_t xs;
    norm_forward(c, x, residual, w, b, false, xr, xs, y, s, stats);
    out = s.defined() ? variable_list{y, s} : variable_list{y};
  }
  if (residual.has_value()) return py::make_tuple(out[0], out[1]);
  return py::cast(out[0]);
}

// --- feed-forward block -----------------------------------------------------

struct FfnCall {
  int dtype, act;
  Batch batch;
  int64_t D, F;
};

struct FfnKept {
  Tensor x, wg, wu, wd, bg, bu, hidden, gate, up, rowmap, y;
  int64_t xs;
};

FfnKept ffn_forward(const FfnCall& c, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                    const Maybe& bg, const Maybe& bu, const Maybe& bd, bool keep) {
  OnDevice on(x);
  FfnKept k;
  k.x = token_rows(x, k.xs, 16);
  k.wg = dense16(wg), k.wu = dense16(wu), k.wd = dense16(wd), k.bg = dense16(bg), k.bu = dense16(bu);
  const Tensor down = dense16(bd);
  const auto opt = x.options().requires_grad(false);
  const int64_t rows = c.batch.B * c.batch.L;
  k.y = at::empty(x.sizes(), opt);
  k.hidden = at::empty({rows, c.F}, opt);
  if (keep && c.dtype == FST_F32) k.gate = at::empty({rows, c.F}, opt), k.up = at::empty({rows, c.F}, opt);
  if (c.batch.lens.defined()) k.rowmap = at::empty({rows + 1}, opt.dtype(at::kInt));
  check(lib.ffn_forward(c.dtype, c.act, (int)c.batch.B, (int)c.batch.L, (int)c.D, (int)c.F, data(k.x), k.xs, data(k.wg),
                        data(k.wu), data(k.wd), data(k.bg), data(k.bu), data(down), ints(c.batch.lens),
                        data(k.hidden), data(k.gate), data(k.up), static_cast<int32_t*>(data(k.rowmap)), data(k.y),
                        on.stream),
        "flash_gated_feed_forward", true);
  return k;
}

struct FfnFunction : torch::autograd::Function<FfnFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                        const Maybe& bg, const Maybe& bu, const Maybe& bd, const FfnCall& c) {
    at::AutoDispatchBelowADInplaceOrView below;
    const FfnKept k = ffn_forward(c, x, wg, wu, wd, bg, bu, bd, true);
    ctx->save_for_backward({k.x, k.wg, k.wu, k.wd, k.bg, k.bu, c.batch.lens, k.hidden, k.gate, k.up, k.rowmap});
    ctx->saved_data["call"] = c10::List<int64_t>({c.dtype, c.act, c.batch.B, c.batch.L, c.D, c.F, k.xs, wants_grad(x),
                                                  wants_grad(wg), wants_grad(wu), wants_grad(wd), wants_grad(bg),
                                                  wants_grad(bu), wants_grad(bd)});
    return k.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!recorded_by_fx(), "flash_gated_feed_forward backward: make_fx cannot record it");
    const variable_list v = ctx->get_saved_variables();
    const auto call = ctx->saved_data["call"].toIntVector();
    variable_list out(8);
    {
      at::AutoGradMode no_graph(false);
      const Tensor& x = v[0];
      OnDevice on(x);
      const auto opt = x.options().requires_grad(false);
      const int64_t B = call[2], L = call[3], D = call[4], F = call[5];
      int64_t dys;
      const Tensor dy = token_rows(grads[0].to(x.scalar_type()), dys, 16);
      TORCH_CHECK(dy.numel() == x.numel() && dy.size(-1) == D && dy.device() == x.device(),
                  "flash_gated_feed_forward backward: the gradient must have the output's shape and device");
      const std::vector<int64_t> shapes[7] = {x.sizes().vec(), {F, D}, {F, D}, {D, F}, {F}, {F}, {D}};
      for (int i = 0; i < 7; ++i)
        if (call[7 + i]) out[i] = at::empty(shapes[i], opt);
      const size_t bytes = lib.ffn_workspace((int)call[0], (int)B, (int)L, (int)D, (int)F);
      const Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 1)}, opt.dtype(at::kByte));
      check(lib.ffn_backward((int)call[0], (int)call[1], (int)B, (int)L, (int)D, (int)F, data(x), call[6], data(v[1]),
                             data(v[2]), data(v[3]), data(v[4]), data(v[5]), ints(v[6]), data(v[7]), data(v[8]),
                             data(v[9]), ints(v[10]), data(dy), dys, data(out[0]), data(out[1]), data(out[2]),
                             data(out[3]), data(out[4]), data(out[5]), data(out[6]), data(ws), bytes, on.stream),
            "flash_gated_feed_forward backward", false);
    }
    return once(std::move(out), "flash_gated_feed_forward");
  }
};

py::object ffn_call(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const Maybe& bg,
                    const Maybe& bu, const Maybe& bd, int act, const Maybe& seqlens) {
  const at::Device dev = x.device();
  if (!lib.ffn_forward || !dev.is_cuda() || recorded()) return py::none();
  for (const Tensor* t : {&x, &wg, &wu, &wd})
    if (!plain(*t, dev) || t->scalar_type() != x.scalar_type()) return py::none();
  for (const Maybe* t : {&bg, &bu, &bd})
    if (!plain(*t, dev) || (t->has_value() && (*t)->scalar_type() != x.scalar_type())) return py::none();
  if (!plain(seqlens, dev)) return py::none();
  FfnCall c;
  c.dtype = dtype_of(x.scalar_type());
  c.act = act;
  if (c.dtype < 0 || x.dim() < 1 || x.size(-1) < 1 || wg.dim() != 2) return py::none();
  c.D = x.size(-1), c.F = wg.size(0);
  if (c.D > INT32_MAX || c.F > INT32_MAX || wg.size(1) != c.D || wu.sizes() != wg.sizes() ||
      wd.sizes() != at::IntArrayRef({c.D, c.F}))
    return py::none();
  for (const auto& [t, n] : {std::pair<const Maybe*, int64_t>{&bg, c.F}, {&bu, c.F}, {&bd, c.D}})
    if (t->has_value() && ((*t)->dim() != 1 || (*t)->size(0) != n)) return py::none();
  if (!batch_of(x, seqlens, c.batch)) return py::none();
  bool graph = false;
  for (const Tensor* t : {&x, &wg, &wu, &wd}) graph |= wants_grad(*t);
  for (const Maybe* t : {&bg, &bu, &bd}) graph |= wants_grad(*t);
  if (at::GradMode::is_enabled() && graph) return py::cast(FfnFunction::apply(x, wg, wu, wd, bg, bu, bd, c));
  at::AutoDispatchBelowADInplaceOrView below;
  return py::cast(ffn_forward(c, x, wg, wu, wd, bg, bu, bd, false).y);
}

// A refused call and a failed allocation are the Python path's to report.
template <typename F, typename... A>
py::object or_none(F f, const A&... args) {
  try {
    return f(args...);
  } catch (const Refused&) {
  } catch (const c10::OutOfMemoryError&) {
  }
  return py::none();
}

}  // namespace

void bind_block_library(size_t norm_fwd, size_t norm_ws, size_t norm_bwd, size_t ffn_fwd, size_t ffn_ws,
                        size_t ffn_bwd, size_t last_error) {
  lib.norm_forward = reinterpret_cast<decltype(lib.norm_forward)>(norm_fwd);
  lib.norm_workspace = reinterpret_cast<decltype(lib.norm_workspace)>(norm_ws);
  lib.norm_backward = reinterpret_cast<decltype(lib.norm_backward)>(norm_bwd);
  lib.ffn_forward = reinterpret_cast<decltype(lib.ffn_forward)>(ffn_fwd);
  lib.ffn_workspace = reinterpret_cast<decltype(lib.ffn_workspace)>(ffn_ws);
  lib.ffn_backward = reinterpret_cast<decltype(lib.ffn_backward)>(ffn_bwd);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(last_error);
}

void define_block_operators(py::module_& m) {
  m.def("layer_norm", [](const Tensor& x, const Maybe& residual, const Maybe& weight, const Maybe& bias, double eps,
                         const Maybe& seqlens) { return or_none(norm_call, x, residual, weight, bias, eps, seqlens); });
  m.def("feed_forward", [](const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const Maybe& bg,
                           const Maybe& bu, const Maybe& bd, int act, const Maybe& seqlens) {
    return or_none(ffn_call, x, wg, wu, wd, bg, bu, bd, act, seqlens);
  });
}
