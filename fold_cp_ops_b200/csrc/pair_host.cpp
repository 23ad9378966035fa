// Host side of the pair-stream operators: argument checks, allocation and gradients over the C ABI of
// include/pair_stream_sm100.h, as the Python module `_pair_host`.
//
// A step of a small pair tensor is host time (the kernels take 2 to 10 us), so what runs between the caller and
// the launch is native: a forward call takes about 6 us and the gradient of one runs in the autograd engine's own thread
// without the interpreter.  A training step takes 54 to 70 us, where one of torch's addition takes 53: the engine's own.  (The
// same in Python: 14 us, and 90 to 130.)  The library's functions come as addresses from the loader, which has checked them against
// the sources; nothing here links to it.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <torch/version.h>

#include <cmath>
#include <cstring>
#include <limits>
#include <string>

#include "../../include/pair_stream_sm100.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---------------------------------------------------------------------------------------------
// the library
// ---------------------------------------------------------------------------------------------
struct Api {
  decltype(&pair_sm100_add_norm) add_norm;
  decltype(&pair_sm100_add_norm_grad_workspace) add_norm_grad_workspace;
  decltype(&pair_sm100_add_norm_grad) add_norm_grad;
  decltype(&pair_sm100_embed) embed;
  decltype(&pair_sm100_embed_grad_workspace) embed_grad_workspace;
  decltype(&pair_sm100_embed_grad) embed_grad;
  decltype(&trimul_sm100_last_error) last_error;
} api = {};

PyObject* library_error = nullptr;  // the loader's exception type

struct LibraryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <typename F>
void take(F& f, const py::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

void bind(const py::dict& addresses, const py::object& error) {
  take(api.add_norm, addresses, "pair_sm100_add_norm");
  take(api.add_norm_grad_workspace, addresses, "pair_sm100_add_norm_grad_workspace");
  take(api.add_norm_grad, addresses, "pair_sm100_add_norm_grad");
  take(api.embed, addresses, "pair_sm100_embed");
  take(api.embed_grad_workspace, addresses, "pair_sm100_embed_grad_workspace");
  take(api.embed_grad, addresses, "pair_sm100_embed_grad");
  take(api.last_error, addresses, "trimul_sm100_last_error");
  library_error = error.inc_ref().ptr();
}

void ok(int rc, const char* what) {
  if (rc == TRIMUL_OK) return;
  const std::string msg = c10::str(what, ": ", api.last_error());
  if (rc == TRIMUL_ERR_INVALID_ARGUMENT || rc == TRIMUL_ERR_UNSUPPORTED_SHAPE) throw py::value_error(msg);
  throw LibraryError(c10::str(what, " failed (code ", rc, "): ", api.last_error()));
}

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  throw py::value_error(c10::str(parts...));
}

// ---------------------------------------------------------------------------------------------
// tensors
// ---------------------------------------------------------------------------------------------
int kind_of(at::ScalarType t) {
  return t == at::kBFloat16 ? PAIR_BF16 : t == at::kHalf ? PAIR_FP16 : t == at::kFloat ? PAIR_FP32 : -1;
}

bool same(const Tensor& a, const Tensor& b) {
  return a.sizes() == b.sizes() && a.scalar_type() == b.scalar_type() && a.device() == b.device();
}

std::string describe(const Tensor& t) { return c10::str(t.sizes(), " ", t.scalar_type(), " on ", t.device()); }

// What the memory holds is what the tensor says (no lazy negation).
Tensor unlazy(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

// Contiguous channels (a copy where they are not).
Tensor channels(const Tensor& t) {
  return !t.defined() || t.size(-1) == 1 || t.stride(-1) == 1 ? unlazy(t) : unlazy(t).contiguous();
}

Tensor packed(const Tensor& t) { return t.defined() ? unlazy(t).contiguous() : t; }

// The last one to four axes are (b, i, j, d).
pair_tensor_t view(const Tensor& t) {
  pair_tensor_t v = {nullptr, 0, 0, 0};
  if (!t.defined()) return v;
  const auto s = t.strides();
  const int64_t n = t.dim();
  v.data = t.data_ptr();
  if (n >= 2) v.stride_j = s[n - 2];
  if (n >= 3) v.stride_i = s[n - 3];
  if (n >= 4) v.stride_b = s[n - 4];
  return v;
}

void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor fresh(const Tensor& like) { return at::empty(like.sizes(), like.options()); }

trimul_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<trimul_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

Tensor or_none(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// A dropout comes as the bytes of its pair_dropout_t and, where the seed lives on the device, its tensor.
struct Dropping {
  pair_dropout_t record;
  Tensor seed;
  bool on() const { return record.keep < 65536u; }
};

const pair_dropout_t kNoDropout = {0, 0, 65536u, nullptr, PAIR_SHARED_NONE, 0, 0, 0};

Dropping dropping(const std::string& bytes, const Tensor& seed, const Tensor& like) {
  Dropping d{kNoDropout, seed};
  if (seed.defined() && seed.device() != like.device())
    refuse("the dropout's seed must be on ", like.device(), " like the tensors; it is on ", seed.device());
  if (!bytes.empty()) {
    TORCH_CHECK(bytes.size() == sizeof(pair_dropout_t), "a dropout record has ", sizeof(pair_dropout_t), " bytes");
    std::memcpy(&d.record, bytes.data(), sizeof(pair_dropout_t));
  }
  if (seed.defined()) d.record.device_seed = static_cast<const uint64_t*>(seed.data_ptr());
  return d;
}

pair_norm_desc_t norm_desc(const Tensor& x, const Tensor& weight, double eps, int group, const Dropping& drop) {
  const int64_t n = x.dim();
  pair_norm_desc_t d;
  const bool empty = x.numel() == 0;  // its other axes may be of any length
  d.b = empty ? 0 : n >= 4 ? static_cast<int32_t>(x.size(n - 4)) : 1;
  d.i = empty ? 0 : n >= 3 ? static_cast<int32_t>(x.size(n - 3)) : 1;
  d.j = empty ? 0 : n >= 2 ? static_cast<int32_t>(x.size(n - 2)) : 1;
  d.d = static_cast<int32_t>(x.size(n - 1));
  d.dtype = kind_of(x.scalar_type());
  d.weight_dtype = weight.defined() ? kind_of(weight.scalar_type()) : d.dtype;
  d.group = group;
  d.eps = static_cast<float>(eps);
  d.dropout = drop.record;
  return d;
}

// ---------------------------------------------------------------------------------------------
// checks
// ---------------------------------------------------------------------------------------------
// The kernels run on memory and show themselves to no dispatcher: a wrapper's memory is not found, a tangent would be lost without a word, which reads as zero, and a trace would
// keep the empty outputs and not what fills them.
void check_visible(std::initializer_list<const Tensor*> tensors) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  if (torch::jit::tracer::isTracing() || (TorchDispatchModeTLS::any_modes_set() && TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value()))
    refuse("the pair-stream operators cannot be traced");
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    if (t->_fw_grad(0).defined()) refuse("the pair-stream operators have no forward-mode derivative; an input has a tangent");
    // subclasses that only wrap another tensor; to the library a null pointer is an absent tensor
    if (t->numel() > 0 && t->const_data_ptr() == nullptr) refuse("the pair-stream operators need tensors with memory of their own; got one without");
  }
}

const Tensor kAbsent;
const Tensor* seed_of(const std::optional<Tensor>& seed) { return seed.has_value() ? &*seed : &kAbsent; }

void check_pair(const Tensor& update, const Tensor& residual) {
  if (!update.is_cuda()) refuse("update must be a CUDA tensor; the pair-stream kernels have no CPU path");
  if (kind_of(update.scalar_type()) < 0) refuse("update must be bfloat16, float16 or float32; got ", update.scalar_type());
  if (update.dim() < 1 || update.dim() > 4)
    refuse("update must have one to four dims, (B, N_i, N_j, D) or its last ones; got ", update.sizes());
  const int64_t d = update.size(-1);
  if (d < 1 || d > PAIR_MAX_WIDTH) refuse("the width D must be in [1, ", PAIR_MAX_WIDTH, "]; got ", d);
  if (update.numel() / d >= int64_t{1} << 31) refuse("at most 2^31 - 1 rows in one call; got ", update.sizes());
  if (residual.defined() && !same(residual, update))
    refuse("residual must be ", describe(update), " like update; got ", describe(residual));
}

void check_weight(const Tensor& weight, const Tensor& update, double eps) {
  if (weight.dim() != 1 || weight.size(0) != update.size(-1) || kind_of(weight.scalar_type()) < 0 ||
      weight.device() != update.device())
    refuse("weight must be a (", update.size(-1), ",) bfloat16, float16 or float32 tensor on ", update.device(), "; got ",
           describe(weight));
  if (!(eps >= 1.1754944e-38 && eps < 3.4e38)) refuse("eps must be a normal float32 number > 0; got ", eps);
}

// First byte and end of the memory that a tensor reaches.
std::pair<uintptr_t, uintptr_t> span(const Tensor& t) {
  int64_t last = 0;
  for (int64_t k = 0; k < t.dim(); ++k) last += (t.size(k) - 1) * t.stride(k);
  const auto at = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {at, at + (1 + last) * t.element_size()};
}

void check_overlap(const Tensor& out, const Tensor& t, const char* name) {
  if (!t.defined() || out.numel() == 0) return;
  const auto a = span(out), b = span(t);
  if (a.first < b.second && b.first < a.second && !(a.first == b.first && t.is_contiguous()))
    refuse("out overlaps ", name, " without being it");
}

// A captured backward pass may only touch the capturing stream, but the engine also waits for the streams that the leaves'
// accumulators belong to.  An accumulator lives as long as any graph that uses the leaf: one that an eager graph on another
// stream still holds would break the capture from inside the engine, so the call is refused while nothing is lost.
void check_capture(std::initializer_list<const Tensor*> tensors) {
  const c10::cuda::OptionalCUDAGuard guard((*tensors.begin())->device());  // all are on one device, which need not be the current one
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  for (const Tensor* t : tensors) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (accumulator == nullptr) continue;
    const auto stream = accumulator->stream();
    if (stream.has_value() && *stream != c10::cuda::getCurrentCUDAStream(t->get_device()).unwrap())
      throw std::runtime_error(
          "cannot capture a gradient: an eager graph of the same leaf, made on another stream, is still alive. Drop its outputs "
          "(and run warm-up passes on the capturing stream) before the capture");
  }
}

// ---------------------------------------------------------------------------------------------
// the calls: checked tensors in, new tensors out, on the current stream of the tensors' device
// ---------------------------------------------------------------------------------------------
Tensor run_add(const Tensor& update, const Tensor& residual, const Dropping& drop, const Tensor& out) {
  const c10::cuda::OptionalCUDAGuard guard(update.device());
  const Tensor u = channels(update), r = channels(residual), z = out.defined() ? out : fresh(update);
  const pair_norm_desc_t d = norm_desc(u, Tensor(), 1.0, 0, drop);
  const pair_tensor_t uv = view(u), rv = view(r);
  ok(api.add_norm(&d, &uv, &rv, nullptr, z.data_ptr(), nullptr, nullptr, stream_of(u)), "pair_sm100_add_norm");
  return z;
}

// (y, z): z is undefined where the stream is the update itself.
std::tuple<Tensor, Tensor> run_norm(const Tensor& update, const Tensor& residual, const Tensor& weight, double eps,
                                    const Dropping& drop, int group, const Tensor& scales) {
  const c10::cuda::OptionalCUDAGuard guard(update.device());
  const Tensor u = channels(update), r = channels(residual), w = packed(weight);
  const Tensor z = residual.defined() || drop.on() ? fresh(update) : Tensor();
  const Tensor y = group != 0 ? at::empty(update.sizes(), update.options().dtype(at::kFloat8_e4m3fn)) : fresh(update);
  const pair_norm_desc_t d = norm_desc(u, w, eps, group, drop);
  const pair_tensor_t uv = view(u), rv = view(r);
  ok(api.add_norm(&d, &uv, &rv, w.data_ptr(), at_of(z), y.data_ptr(), static_cast<float*>(at_of(scales)), stream_of(u)),
     "pair_sm100_add_norm");
  return {y, z};
}

// (d_update, d_residual, d_weight); without a dropout the first two are one tensor.
std::tuple<Tensor, Tensor, Tensor> run_norm_grad(const Tensor& stream, const Tensor& dy, const Tensor& dz, const Tensor& weight,
                                                 double eps, const Dropping& drop, bool need_u, bool need_r, bool need_w) {
  const c10::cuda::OptionalCUDAGuard guard(stream.device());
  const Tensor z = channels(stream), y = channels(dy), g = channels(dz), w = packed(weight);
  const bool own_u = need_u && (drop.on() || !need_r);
  const Tensor du = own_u ? fresh(stream) : Tensor(), dr = need_r ? fresh(stream) : Tensor();
  const pair_norm_desc_t d = norm_desc(z, w, eps, 0, drop);
  Tensor dw, workspace;
  if (need_w) {
    uint64_t bytes = 0;
    ok(api.add_norm_grad_workspace(&d, &bytes), "pair_sm100_add_norm_grad_workspace");
    dw = fresh(w);
    workspace = at::empty({static_cast<int64_t>(bytes)}, z.options().dtype(at::kByte));
  }
  const pair_tensor_t zv = view(z), yv = view(y), gv = view(g);
  ok(api.add_norm_grad(&d, &zv, &yv, &gv, w.data_ptr(), at_of(dr), at_of(du), at_of(dw), at_of(workspace), stream_of(z)),
     "pair_sm100_add_norm_grad");
  return {own_u ? du : need_u ? dr : Tensor(), dr, dw};
}

pair_embed_desc_t embed_desc(const Tensor& index, int64_t rows, int64_t d, at::ScalarType dtype, at::ScalarType table_dtype,
                             double scale) {
  pair_embed_desc_t e;
  e.tokens = index.numel();
  e.d = static_cast<int32_t>(d);
  e.rows = static_cast<int32_t>(rows);
  e.index_bits = index.scalar_type() == at::kInt ? 32 : 64;
  e.dtype = kind_of(dtype);
  e.table_dtype = kind_of(table_dtype);
  e.scale = static_cast<float>(scale);
  return e;
}

Tensor run_embed(const Tensor& index, const Tensor& table, const Tensor& base, double scale, at::ScalarType dtype) {
  const c10::cuda::OptionalCUDAGuard guard(index.device());
  const Tensor x = index.contiguous(), t = packed(table), b = packed(base);
  std::vector<int64_t> shape(index.sizes().begin(), index.sizes().end());
  shape.push_back(table.size(1));
  const Tensor out = at::empty(shape, table.options().dtype(dtype));
  const pair_embed_desc_t d = embed_desc(x, table.size(0), table.size(1), dtype, table.scalar_type(), scale);
  ok(api.embed(&d, x.data_ptr(), t.data_ptr(), at_of(b), out.data_ptr(), stream_of(x)), "pair_sm100_embed");
  return out;
}

Tensor run_embed_grad(const Tensor& index, const Tensor& d_out, int64_t rows, at::ScalarType table_dtype, double scale) {
  const c10::cuda::OptionalCUDAGuard guard(index.device());
  const Tensor x = index.contiguous(), g = packed(d_out);
  const Tensor d_table = at::empty({rows, g.size(-1)}, g.options().dtype(table_dtype));
  const pair_embed_desc_t d = embed_desc(x, rows, g.size(-1), g.scalar_type(), table_dtype, scale);
  uint64_t bytes = 0;
  ok(api.embed_grad_workspace(&d, &bytes), "pair_sm100_embed_grad_workspace");
  const Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, g.options().dtype(at::kByte));
  ok(api.embed_grad(&d, x.data_ptr(), g.data_ptr(), d_table.data_ptr(), workspace.data_ptr(), stream_of(x)), "pair_sm100_embed_grad");
  return d_table;
}

// ---------------------------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------------------------
// The gradients are kernels' results without a graph of their own: where one is being made of them, using it is an error.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      "the pair-stream operators are differentiable once: their gradients have no gradient", static_cast<int64_t>(grads.size()));
  for (Tensor& g : grads)
    if (g.defined()) {
      g = g.detach();
      g.set_requires_grad(true);
    }
  return (*error)(std::move(grads));
}

// The engine numbers a function's edges over the tensors that were given: an absent residual or base has none.
struct DropoutAdd : torch::autograd::Function<DropoutAdd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& update, const std::optional<Tensor>& residual,
                        const std::optional<Tensor>& seed, const std::string& drop) {
    ctx->set_materialize_grads(false);
    ctx->saved_data["drop"] = drop;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->save_for_backward({or_none(seed)});
    return run_add(update, or_none(residual), dropping(drop, or_none(seed), update), Tensor());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor du, dz = grads[0];
    const variable_list saved = ctx->get_saved_variables();  // raises where the seed's values were changed
    if (dz.defined() && ctx->needs_input_grad(0)) {
      const Dropping drop = dropping(ctx->saved_data["drop"].toStringRef(), saved[0], dz);
      du = drop.on() ? run_add(dz, Tensor(), drop, Tensor()) : dz;
    }
    const bool need_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1);
    variable_list out = once({du, need_r ? dz : Tensor()});
    out.resize(4);
    return out;
  }
};

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& update, const std::optional<Tensor>& residual, const Tensor& weight,
                               const std::optional<Tensor>& seed, double eps, const std::string& drop) {
    ctx->set_materialize_grads(false);
    auto [y, z] = run_norm(update, or_none(residual), weight, eps, dropping(drop, or_none(seed), update), 0, Tensor());
    if (!z.defined()) z = update.view_as(update);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["drop"] = drop;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->save_for_backward({z, weight, or_none(seed)});
    return {y, z};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(3);
    if (grads[0].defined() || grads[1].defined()) {
      const variable_list saved = ctx->get_saved_variables();
      const bool residual = ctx->saved_data["residual"].toBool();
      std::tie(out[0], out[1], out[2]) =
          run_norm_grad(saved[0], grads[0], grads[1], saved[1], ctx->saved_data["eps"].toDouble(),
                        dropping(ctx->saved_data["drop"].toStringRef(), saved[2], saved[0]), ctx->needs_input_grad(0),
                        residual && ctx->needs_input_grad(1), ctx->needs_input_grad(residual ? 2 : 1));
    }
    out = once(std::move(out));
    out.resize(6);
    return out;
  }
};

struct PairEmbedding : torch::autograd::Function<PairEmbedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& index, const Tensor& table, const std::optional<Tensor>& base, double scale,
                        int64_t dtype) {
    ctx->set_materialize_grads(false);
    ctx->saved_data["base"] = base.has_value();
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["type"] = static_cast<int64_t>(table.scalar_type());
    ctx->saved_data["scale"] = scale;
    ctx->save_for_backward({index});
    return run_embed(index, table, or_none(base), scale, static_cast<at::ScalarType>(dtype));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(3);
    if (grads[0].defined()) {
      if (ctx->needs_input_grad(1))
        out[1] = run_embed_grad(ctx->get_saved_variables()[0], grads[0], ctx->saved_data["rows"].toInt(),
                                static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()), ctx->saved_data["scale"].toDouble());
      if (ctx->saved_data["base"].toBool() && ctx->needs_input_grad(2)) out[2] = grads[0];
    }
    out = once(std::move(out));
    out.resize(5);
    return out;
  }
};

// ---------------------------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------------------------
Tensor dropout_add(const Tensor& update, const std::optional<Tensor>& residual_, const std::string& drop,
                   const std::optional<Tensor>& seed, const std::optional<Tensor>& out_) {
  const Tensor residual = or_none(residual_), out = or_none(out_);
  check_visible({&update, &residual, &out, seed_of(seed)});
  check_pair(update, residual);
  if (out.defined()) {
    if (wants_grad({&update, &residual, &out})) refuse("out= has no gradient: leave it out, or run under torch.no_grad()");
    if (!same(out, update) || !out.is_contiguous() || out.is_neg()) refuse("out must be a contiguous ", describe(update), " tensor; got ", describe(out));
    check_overlap(out, update, "update");
    check_overlap(out, residual, "residual");
  } else if (wants_grad({&update, &residual})) {
    check_capture({&update, &residual});
    return DropoutAdd::apply(update, residual_, seed, drop);
  }
  const Tensor z = run_add(update, residual, dropping(drop, or_none(seed), update), out);
  if (out.defined() && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();  // graphs that saved out's old values notice
  return z;
}

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& update, const std::optional<Tensor>& residual_, const Tensor& weight, double eps,
                                        const std::string& drop, const std::optional<Tensor>& seed) {
  const Tensor residual = or_none(residual_);
  check_visible({&update, &residual, &weight, seed_of(seed)});
  check_pair(update, residual);
  check_weight(weight, update, eps);
  if (wants_grad({&update, &residual, &weight})) {
    check_capture({&update, &residual, &weight});
    variable_list out = AddRmsNorm::apply(update, residual_, weight, seed, eps, drop);
    return {out[0], out[1]};
  }
  auto [y, z] = run_norm(update, residual, weight, eps, dropping(drop, or_none(seed), update), 0, Tensor());
  return {y, z.defined() ? z : update};
}

// Lanes reduce a group's octs: rows have to start on 16-byte boundaries (a copy where they do not).
Tensor aligned(const Tensor& given) {
  const Tensor t = unlazy(given);
  if (!t.defined() || t.numel() == 0) return t;
  const int64_t unit = 16 / t.element_size();
  bool fits = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.size(-1) == 1 || t.stride(-1) == 1);
  for (int64_t k = 0; k + 1 < t.dim(); ++k) fits = fits && (t.size(k) == 1 || t.stride(k) % unit == 0);
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_fp8(const Tensor& update_, const std::optional<Tensor>& residual_, const Tensor& weight,
                                                    double eps, const std::optional<int64_t>& group, const std::string& drop,
                                                    const std::optional<Tensor>& seed) {
  Tensor update = update_, residual = or_none(residual_);
  check_visible({&update, &residual, &weight, seed_of(seed)});
  check_pair(update, residual);
  check_weight(weight, update, eps);
  const int64_t width = update.size(-1);
  if (group.has_value() && ((*group != 32 && *group != 64 && *group != 128) || width % *group != 0))
    refuse("group must be 32, 64 or 128 and divide D=", width, ", or None for one scale per row; got ", *group);
  if (wants_grad({&update, &residual, &weight})) refuse("the e4m3 form has no gradient: run it under torch.no_grad()");
  if (group.has_value()) update = aligned(update), residual = aligned(residual);
  const int64_t g = group.value_or(width);
  std::vector<int64_t> shape(update.sizes().begin(), update.sizes().end());
  shape.back() = width / g;
  const Tensor scales = at::empty(shape, update.options().dtype(at::kFloat));
  auto [q, z] = run_norm(update, residual, weight, eps, dropping(drop, or_none(seed), update), static_cast<int>(g), scales);
  return {q, scales, z.defined() ? z : update_};
}

Tensor pair_embedding(const Tensor& index, const Tensor& table, double scale, const std::optional<Tensor>& base_,
                      const std::optional<at::ScalarType>& dtype_) {
  const Tensor base = or_none(base_);
  check_visible({&index, &table, &base});
  if (index.scalar_type() != at::kInt && index.scalar_type() != at::kLong)
    refuse("index must be an int32 or int64 tensor; got ", index.scalar_type());
  if (!index.is_cuda()) refuse("index must be a CUDA tensor; the pair-stream kernels have no CPU path");
  if (table.dim() != 2 || table.size(0) < 1 || kind_of(table.scalar_type()) < 0 || table.device() != index.device())
    refuse("table must be a (V, D) bfloat16, float16 or float32 tensor on ", index.device(), "; got ", describe(table));
  if (table.size(0) > std::numeric_limits<int32_t>::max()) refuse("table has at most 2^31 - 1 rows; got ", table.size(0));
  const int64_t d = table.size(1);
  if (d < 1 || d > PAIR_MAX_WIDTH) refuse("the width D must be in [1, ", PAIR_MAX_WIDTH, "]; got ", d);
  if (index.numel() >= int64_t{1} << 31) refuse("at most 2^31 - 1 tokens in one call; got ", index.numel());
  if (base.defined()) {
    const auto s = base.sizes();
    if (base.dim() != index.dim() + 1 || s.slice(0, s.size() - 1) != index.sizes() || s.back() != d || base.device() != index.device())
      refuse("base must have index's shape ", index.sizes(), " and D=", d, " channels on ", index.device(), "; got ", describe(base));
    if (dtype_.has_value() && *dtype_ != base.scalar_type())
      refuse("the result has base's type ", base.scalar_type(), "; got dtype=", *dtype_);
  }
  const at::ScalarType dtype = base.defined() ? base.scalar_type() : dtype_.value_or(table.scalar_type());
  if (kind_of(dtype) < 0) refuse("the embedding's type must be bfloat16, float16 or float32; got ", dtype);
  if (!std::isfinite(static_cast<float>(scale))) refuse("scale must be finite in float32; got ", scale);
  if (wants_grad({&table, &base})) {
    check_capture({&table, &base});
    return PairEmbedding::apply(index, table, base_, scale, static_cast<int64_t>(dtype));
  }
  return run_embed(index, table, base, scale, dtype);
}

const char* build_id() {
#ifdef TRIMUL_BUILD_ID
  return TRIMUL_BUILD_ID;
#else
  return "unknown";
#endif
}

}  // namespace

PYBIND11_MODULE(_pair_host, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const LibraryError& e) {
      PyErr_SetString(library_error, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("build_id", &build_id);
  m.attr("torch_version") = TORCH_VERSION;  // the headers that this was compiled against
  m.def("dropout_add", &dropout_add);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("add_rms_norm_fp8", &add_rms_norm_fp8);
  m.def("pair_embedding", &pair_embedding);
}
