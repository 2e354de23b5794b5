// Thin torch binding over the C ABI (include/fpscan_b200.h): the fast path of
// fpscan_b200.ops for the reference's own entry points, and of the calls of
// delta.py and checkpoint8.py, where a serving step's kernel takes less time
// than a Python + ctypes call.  It plays the role of
// the reference's pybind module (csrc/main.cpp:10, fullscan_forward) -- tensor
// checks, output allocation, the caller's current stream -- in C++, so a
// call costs what the reference's does instead of a Python + ctypes round
// trip.  All work is done by libfpscan_b200.so; this file has no kernels.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <map>
#include <mutex>
#include <tuple>

#include "../../include/fpscan_b200.h"

namespace {

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return FPSCAN_F32;
    case at::kHalf:
      return FPSCAN_F16;
    case at::kBFloat16:
      return FPSCAN_BF16;
    default:
      TORCH_CHECK(false, "tokens must be float16 or bfloat16 or float32");
  }
  return -1;
}

// Same conditions and order as ops.validate (CHECK_INPUT of
// csrc/full_scan/full_scan.h:7-15, then shapes); the C ABI re-checks sizes,
// alignment and overlap.
void check_pair(const at::Tensor& gates, const at::Tensor& tokens, const char* gname) {
  TORCH_CHECK(gates.is_cuda(), gname, " must be a CUDA tensor");
  TORCH_CHECK(tokens.is_cuda(), "tokens must be a CUDA tensor");
  TORCH_CHECK(gates.is_contiguous(), gname, " must be contiguous");
  TORCH_CHECK(tokens.is_contiguous(), "tokens must be contiguous");
  TORCH_CHECK(tokens.dim() == 3, "tokens must be 3-D (batch, dim, seqlen)");
  TORCH_CHECK(gates.sizes() == tokens.sizes(), gname, " and tokens must have the same shape");
  TORCH_CHECK(gates.scalar_type() == tokens.scalar_type(), gname,
              " dtype must equal tokens dtype");
  TORCH_CHECK(gates.device() == tokens.device(), gname, " and tokens must be on the same device");
}

// Workspaces of the split-row paths, one per (device, stream, kind), zeroed
// once when (re)allocated; calls on one stream are ordered, so they may
// share it.  Kept for the life of the process (a few KB each).
at::Tensor workspace(const at::Tensor& like, int64_t bytes, int kind) {
  static std::mutex mu;
  static std::map<std::tuple<int, void*, int>, at::Tensor> cache;
  const auto key = std::make_tuple((int)like.get_device(),
                                   (void*)at::cuda::getCurrentCUDAStream().stream(), kind);
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(key);
  if (it != cache.end() && it->second.numel() >= bytes) return it->second;
  at::Tensor w = at::zeros({std::max<int64_t>(bytes, 1 << 16)}, like.options().dtype(at::kByte));
  cache[key] = w;
  return w;
}

void raise_on(int rc, const char* what) {
  if (rc != FPSCAN_OK) TORCH_CHECK(false, what, ": ", fpscan_last_error());
}

at::Tensor fullscan_forward(const at::Tensor& gates, const at::Tensor& tokens, at::Tensor out,
                            bool reverse) {
  check_pair(gates, tokens, "gates");
  TORCH_CHECK(out.sizes() == tokens.sizes() && out.scalar_type() == tokens.scalar_type() &&
                  out.device() == tokens.device(),
              "out must match tokens in shape, dtype and device");
  TORCH_CHECK(out.is_contiguous(), "out must be contiguous");
  const int code = dtype_code(tokens);
  const int64_t b = tokens.size(0), d = tokens.size(1), l = tokens.size(2);
  const c10::cuda::CUDAGuard guard(tokens.device());
  void* stream = at::cuda::getCurrentCUDAStream().stream();
  const int64_t ws = fpscan_scan_fwd_workspace_bytes(b, d, l, code);
  if (ws > 0) {
    // few, long rows: the split-row kernel and its workspace
    at::Tensor w = workspace(tokens, ws, 0);
    raise_on(fpscan_scan_fwd_ws(gates.data_ptr(), tokens.data_ptr(), out.data_ptr(), b, d, l, code,
                                reverse ? 1 : 0, w.data_ptr(), w.numel(), stream),
             "fpscan_scan_fwd_ws");
  } else {
    raise_on(fpscan_scan_fwd(gates.data_ptr(), tokens.data_ptr(), out.data_ptr(), b, d, l, code,
                             reverse ? 1 : 0, stream),
             "fpscan_scan_fwd");
  }
  return out;
}

at::Tensor scan_forward(const at::Tensor& gates, const at::Tensor& tokens, bool reverse) {
  return fullscan_forward(gates, tokens, at::empty_like(tokens), reverse);
}

std::tuple<at::Tensor, at::Tensor> scan_backward(const at::Tensor& gates, const at::Tensor& y,
                                                 const at::Tensor& grad_out) {
  check_pair(gates, grad_out, "gates");
  check_pair(y, grad_out, "y");
  const int code = dtype_code(grad_out);
  const int64_t b = grad_out.size(0), d = grad_out.size(1), l = grad_out.size(2);
  const c10::cuda::CUDAGuard guard(grad_out.device());
  at::Tensor dgates = at::empty_like(grad_out), dtokens = at::empty_like(grad_out);
  void* stream = at::cuda::getCurrentCUDAStream().stream();
  const int64_t ws = fpscan_scan_bwd_workspace_bytes(b, d, l, code);
  if (ws > 0) {
    // few, long rows: the split-row backward and its workspace
    at::Tensor w = workspace(grad_out, ws, 1);
    raise_on(fpscan_scan_bwd_ws(gates.data_ptr(), y.data_ptr(), grad_out.data_ptr(),
                                dgates.data_ptr(), dtokens.data_ptr(), b, d, l, code,
                                w.data_ptr(), w.numel(), stream),
             "fpscan_scan_bwd_ws");
  } else {
    raise_on(fpscan_scan_bwd(gates.data_ptr(), y.data_ptr(), grad_out.data_ptr(),
                             dgates.data_ptr(), dtokens.data_ptr(), b, d, l, code, stream),
             "fpscan_scan_bwd");
  }
  return {dgates, dtokens};
}

// ---------------------------------------------------------------- gated delta rule
// Same conditions and wording as delta.validate_delta.
struct DeltaSizes {
  int64_t b, l, hk, h, dk, dv;
  int code;
};

DeltaSizes check_delta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                       const at::Tensor& log_decay, const at::Tensor& beta,
                       const c10::optional<at::Tensor>& state,
                       const c10::optional<at::Tensor>& out) {
  const at::Tensor* all[5] = {&q, &k, &v, &log_decay, &beta};
  static const char* const names[5] = {"q", "k", "v", "log_decay", "beta"};
  for (int i = 0; i < 5; ++i) {
    TORCH_CHECK(all[i]->is_cuda(), names[i], " must be a CUDA tensor");
    TORCH_CHECK(all[i]->is_contiguous(), names[i], " must be contiguous");
    TORCH_CHECK(all[i]->scalar_type() == at::kFloat || all[i]->scalar_type() == at::kHalf ||
                    all[i]->scalar_type() == at::kBFloat16,
                names[i], " must be float16 or bfloat16 or float32");
  }
  for (int i = 0; i < 3; ++i)
    TORCH_CHECK(all[i]->dim() == 4, names[i], " must be 4-D (batch, seqlen, heads, channels), got ",
                all[i]->sizes());
  DeltaSizes s{v.size(0), v.size(1), q.size(2), v.size(2), q.size(3), v.size(3), dtype_code(v)};
  TORCH_CHECK(q.sizes() == k.sizes(), "q ", q.sizes(), " and k ", k.sizes(),
              " must have the same shape");
  TORCH_CHECK(q.size(0) == s.b && q.size(1) == s.l, "q ", q.sizes(), " and v ", v.sizes(),
              " must agree in batch and seqlen");
  TORCH_CHECK(s.hk >= 1 && s.h >= 1 && s.h % s.hk == 0, "heads of v (", s.h,
              ") must be a positive multiple of the heads of q and k (", s.hk, ")");
  TORCH_CHECK(s.l >= 1, "seqlen must be >= 1 (got ", s.l, ")");
  TORCH_CHECK(s.dk % 8 == 0 && s.dk >= 8 && s.dk <= 128,
              "dk must be a multiple of 8 in [8, 128] (got ", s.dk, ")");
  TORCH_CHECK(s.dv % 8 == 0 && s.dv >= 8 && s.dv <= 65536,
              "dv must be a multiple of 8 in [8, 65536] (got ", s.dv, ")");
  for (int i = 3; i < 5; ++i)
    TORCH_CHECK(all[i]->dim() == 3 && all[i]->size(0) == s.b && all[i]->size(1) == s.l &&
                    all[i]->size(2) == s.h,
                names[i], " must have shape (", s.b, ", ", s.l, ", ", s.h,
                ") (batch, seqlen, heads), got ", all[i]->sizes());
  for (int i = 0; i < 5; ++i) {
    TORCH_CHECK(all[i]->scalar_type() == v.scalar_type(), names[i], " dtype ",
                all[i]->scalar_type(), " must equal v dtype ", v.scalar_type());
    TORCH_CHECK(all[i]->device() == v.device(), names[i], " and v must be on the same device");
  }
  if (state) {
    TORCH_CHECK(state->dim() == 4 && state->size(0) == s.b && state->size(1) == s.h &&
                    state->size(2) == s.dv && state->size(3) == s.dk,
                "the state must have shape (", s.b, ", ", s.h, ", ", s.dv, ", ", s.dk,
                ") (batch, heads, dv, dk), got ", state->sizes());
    TORCH_CHECK(state->device() == v.device(), "the state must be on the device of v");
    TORCH_CHECK(state->scalar_type() == at::kFloat && state->is_contiguous(),
                "the state must be float32 and contiguous");
  }
  if (out) {
    TORCH_CHECK(out->sizes() == v.sizes() && out->scalar_type() == v.scalar_type() &&
                    out->device() == v.device(),
                "out must match v in shape, dtype and device");
    TORCH_CHECK(out->is_contiguous(), "out must be contiguous");
  }
  return s;
}

at::Tensor delta_workspace(const at::Tensor& v, const DeltaSizes& s, bool wide, bool backward) {
  const int64_t n = fpscan_delta_workspace_bytes(s.b, s.l, s.hk, s.h, s.dk, s.dv, s.code, wide, backward);
  return at::empty({std::max<int64_t>(n, 16)}, v.options().dtype(at::kByte));
}

// One token of `heads` values, or one sequence of a batch, starts anywhere: a
// contiguous tensor that does not start on 16 bytes, as the sequence kernels'
// operands must, is copied.
at::Tensor aligned(const at::Tensor& t) {
  return t.numel() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t;
}

// A backward pass that has saved a tensor must notice that it is overwritten.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_written(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), name,
              " requires a gradient, which writing it here would lose: detach it");
}

float* state_ptr(const c10::optional<at::Tensor>& t) {
  return t && t->numel() ? t->data_ptr<float>() : nullptr;
}

at::Tensor delta_step(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                      const at::Tensor& log_decay, const at::Tensor& beta, at::Tensor state,
                      double scale, const c10::optional<at::Tensor>& out_) {
  const DeltaSizes s = check_delta(q, k, v, log_decay, beta, state, out_);
  check_written(state, "state");
  if (out_) check_written(*out_, "out");
  const c10::cuda::CUDAGuard guard(v.device());
  at::Tensor out = out_ ? *out_ : at::empty_like(v);
  raise_on(fpscan_delta_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
                             beta.data_ptr(), state_ptr(state), out.data_ptr(), state_ptr(state),
                             s.b, s.l, s.hk, s.h, s.dk, s.dv, (float)scale, s.code,
                             at::cuda::getCurrentCUDAStream().stream()),
           "fpscan_delta_step");
  written(state);
  if (out_) written(out);
  return out;
}

std::tuple<at::Tensor, c10::optional<at::Tensor>> delta_forward(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay_,
    const at::Tensor& beta_, const c10::optional<at::Tensor>& initial, double scale,
    bool return_state, const c10::optional<at::Tensor>& out_) {
  const DeltaSizes s = check_delta(q, k, v, log_decay_, beta_, initial, out_);
  if (out_) check_written(*out_, "out");
  const c10::cuda::CUDAGuard guard(v.device());
  const at::Tensor log_decay = aligned(log_decay_), beta = aligned(beta_);
  const bool wide = initial || return_state;
  at::Tensor out = out_ ? *out_ : at::empty_like(v);
  c10::optional<at::Tensor> last;
  if (return_state) last = at::empty({s.b, s.h, s.dv, s.dk}, v.options().dtype(at::kFloat));
  const at::Tensor ws = delta_workspace(v, s, wide, false);
  raise_on(fpscan_delta_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
                            beta.data_ptr(), state_ptr(initial), out.data_ptr(), state_ptr(last),
                            s.b, s.l, s.hk, s.h, s.dk, s.dv, (float)scale, s.code, wide,
                            ws.data_ptr(), ws.numel(), at::cuda::getCurrentCUDAStream().stream()),
           "fpscan_delta_fwd");
  if (out_) written(out);
  return {out, last};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, c10::optional<at::Tensor>>
delta_backward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
               const at::Tensor& log_decay_, const at::Tensor& beta_, const at::Tensor& grad_out_,
               const c10::optional<at::Tensor>& initial,
               const c10::optional<at::Tensor>& grad_final_, double scale, bool need_initial) {
  const DeltaSizes s = check_delta(q, k, v, log_decay_, beta_, initial, grad_out_);
  if (grad_final_) check_delta(q, k, v, log_decay_, beta_, grad_final_, c10::nullopt);
  const c10::cuda::CUDAGuard guard(v.device());
  const at::Tensor log_decay = aligned(log_decay_), beta = aligned(beta_), grad_out = aligned(grad_out_);
  c10::optional<at::Tensor> grad_final;
  if (grad_final_) grad_final = aligned(*grad_final_);
  const bool wide = initial || grad_final || need_initial;
  at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v),
             dg = at::empty_like(log_decay), db = at::empty_like(beta);
  c10::optional<at::Tensor> di;
  if (need_initial) di = at::empty({s.b, s.h, s.dv, s.dk}, v.options().dtype(at::kFloat));
  const at::Tensor ws = delta_workspace(v, s, wide, true);
  raise_on(fpscan_delta_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
                            beta.data_ptr(), state_ptr(initial), grad_out.data_ptr(),
                            state_ptr(grad_final), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                            dg.data_ptr(), db.data_ptr(), state_ptr(di), s.b, s.l, s.hk, s.h, s.dk,
                            s.dv, (float)scale, s.code, wide, ws.data_ptr(), ws.numel(),
                            at::cuda::getCurrentCUDAStream().stream()),
           "fpscan_delta_bwd");
  return {dq, dk, dv, dg, db, di};
}

// delta.GatedDelta, in C++: a training step's layer is half a dozen kernels,
// and a Python autograd function costs as much as some of them.
std::tuple<at::Tensor, at::Tensor> quantize8(const at::Tensor& x);
at::Tensor dequantize8(const at::Tensor& codes, const at::Tensor& steps, at::ScalarType dtype);

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// Gradients of a backward pass that is not differentiable itself: taken with
// create_graph, they raise when they are differentiated instead of counting
// as constants.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const at::Tensor& g : grads)
    if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " is differentiable once", (int64_t)in.size());
  const variable_list out = (*error)(std::move(in));
  size_t i = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

struct GatedDelta : public torch::autograd::Function<GatedDelta> {
  static variable_list forward(AutogradContext* ctx, const Variable& q, const Variable& k,
                               const Variable& v, const Variable& log_decay, const Variable& beta,
                               const c10::optional<Variable>& state, double scale,
                               bool return_state, bool checkpoint8) {
    c10::optional<at::Tensor> held;
    if (state) held = state->to(at::kFloat).contiguous();
    auto [out, last] = delta_forward(q, k, v, log_decay, beta, held, scale, return_state, c10::nullopt);
    variable_list kept;
    if (checkpoint8) {
      for (const Variable* x : {&q, &k, &v}) {
        auto [codes, steps] = quantize8(*x);
        kept.push_back(codes);
        kept.push_back(steps);
      }
    } else {
      kept = {q, k, v};
    }
    kept.push_back(log_decay);
    kept.push_back(beta);
    kept.push_back(held ? *held : at::Tensor());
    ctx->save_for_backward(kept);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["checkpoint8"] = checkpoint8;
    ctx->saved_data["dtype"] = (int64_t)v.scalar_type();
    ctx->saved_data["state_dtype"] = state ? (int64_t)state->scalar_type() : (int64_t)-1;
    ctx->set_materialize_grads(false);
    if (return_state) return {out, *last};
    return {out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor none;
    const at::Tensor grad_final = grads.size() > 1 ? grads[1] : none;
    if (!grads[0].defined() && !grad_final.defined()) return variable_list(9);
    variable_list kept = ctx->get_saved_variables();
    const size_t n = kept.size();
    at::Tensor q, k, v;
    if (ctx->saved_data["checkpoint8"].toBool()) {
      const auto dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
      q = dequantize8(kept[0], kept[1], dtype);
      k = dequantize8(kept[2], kept[3], dtype);
      v = dequantize8(kept[4], kept[5], dtype);
    } else {
      q = kept[0];
      k = kept[1];
      v = kept[2];
    }
    const at::Tensor grad_out = grads[0].defined() ? grads[0].contiguous() : at::zeros_like(v);
    c10::optional<at::Tensor> initial, gf;
    if (kept[n - 1].defined()) initial = kept[n - 1];
    if (grad_final.defined()) gf = grad_final.to(at::kFloat).contiguous();
    const int64_t state_dtype = ctx->saved_data["state_dtype"].toInt();
    const bool need = state_dtype >= 0 && ctx->needs_input_grad(5);
    auto [dq, dk, dv, dg, db, di] =
        delta_backward(q, k, v, kept[n - 3], kept[n - 2], grad_out, initial, gf,
                       ctx->saved_data["scale"].toDouble(), need);
    at::Tensor dstate;
    if (di) dstate = di->to((at::ScalarType)state_dtype);
    return once({dq, dk, dv, dg, db, dstate, none, none, none}, "gated_delta");
  }
};

// Whether a backward pass can follow: without one no checkpoint is made.
bool wanted(std::initializer_list<const at::Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : inputs)
    if (t->requires_grad()) return true;
  return false;
}

std::tuple<at::Tensor, c10::optional<at::Tensor>> gated_delta(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
    const at::Tensor& beta, const c10::optional<at::Tensor>& state, double scale,
    bool return_state, bool checkpoint8) {
  const at::Tensor none;
  checkpoint8 = checkpoint8 && wanted({&q, &k, &v, &log_decay, &beta, state ? &*state : &none});
  const variable_list r =
      GatedDelta::apply(q, k, v, log_decay, beta, state, scale, return_state, checkpoint8);
  if (return_state) return {r[0], r[1]};
  return {r[0], c10::nullopt};
}

// ---------------------------------------------------------------- 8-bit checkpoints
std::tuple<at::Tensor, at::Tensor> quantize8(const at::Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK(x.is_contiguous(), "x must be contiguous");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kHalf ||
                  x.scalar_type() == at::kBFloat16,
              "x must be float16 or bfloat16 or float32");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t n = x.numel();
  at::Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar).requires_grad(false));
  at::Tensor steps = at::empty({(n + 63) / 64}, x.options().dtype(at::kFloat).requires_grad(false));
  if (n)
    raise_on(fpscan_quantize8(x.data_ptr(), codes.data_ptr(), steps.data_ptr<float>(), n,
                              dtype_code(x), at::cuda::getCurrentCUDAStream().stream()),
             "fpscan_quantize8");
  return {codes, steps};
}

// Called with checked codes and steps (checkpoint8.dequantize8).
at::Tensor dequantize8(const at::Tensor& codes, const at::Tensor& steps, at::ScalarType dtype) {
  const c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype));
  if (codes.numel())
    raise_on(fpscan_dequantize8(codes.data_ptr(), steps.data_ptr<float>(), out.data_ptr(),
                                codes.numel(), dtype_code(out),
                                at::cuda::getCurrentCUDAStream().stream()),
             "fpscan_dequantize8");
  return out;
}

// ops.PScanChannelsLast8, in C++ for the same reason.
struct Scan8 : public torch::autograd::Function<Scan8> {
  // Same conditions as ops.validate_channels_last.
  static void check(const at::Tensor& gates, const at::Tensor& tokens) {
    const at::Tensor* all[2] = {&gates, &tokens};
    static const char* const names[2] = {"gates", "tokens"};
    for (int i = 0; i < 2; ++i) {
      TORCH_CHECK(all[i]->is_cuda(), names[i], " must be a CUDA tensor");
      TORCH_CHECK(all[i]->is_contiguous(), names[i], " must be contiguous");
      TORCH_CHECK(all[i]->scalar_type() == at::kFloat || all[i]->scalar_type() == at::kHalf ||
                      all[i]->scalar_type() == at::kBFloat16,
                  names[i], " must be float16 or bfloat16 or float32");
    }
    TORCH_CHECK(tokens.dim() == 3, "tokens must be 3-D (batch, seqlen, dim), got ", tokens.sizes());
    TORCH_CHECK(gates.sizes() == tokens.sizes() && gates.scalar_type() == tokens.scalar_type() &&
                    gates.device() == tokens.device(),
                "gates and tokens must have the same shape, dtype and device");
    TORCH_CHECK(tokens.size(1) >= 1, "seqlen must be >= 1 (got ", tokens.size(1), ")");
    const int64_t vec = 16 / tokens.element_size();
    TORCH_CHECK(tokens.size(2) % vec == 0, "dim must be a multiple of ", vec, " for ",
                tokens.scalar_type(), " (got ", tokens.size(2), ")");
  }

  static at::Tensor workspace_of(const at::Tensor& t, bool backward) {
    const int64_t n = fpscan_cl_workspace_bytes(t.size(0), t.size(1), t.size(2), dtype_code(t), backward);
    return at::empty({std::max<int64_t>(n, 256)}, t.options().dtype(at::kByte).requires_grad(false));
  }

  // keep: a backward pass can follow
  static Variable forward(AutogradContext* ctx, const Variable& gates, const Variable& tokens, bool keep) {
    check(gates, tokens);
    const c10::cuda::CUDAGuard guard(tokens.device());
    const int64_t b = tokens.size(0), l = tokens.size(1), d = tokens.size(2);
    const auto opts = tokens.options().requires_grad(false);
    at::Tensor out = at::empty_like(tokens);
    if (!keep) {
      if (b && d) {
        const at::Tensor ws = workspace_of(tokens, false);
        raise_on(fpscan_scan_fwd_cl(gates.data_ptr(), tokens.data_ptr(), out.data_ptr(), b, l, d,
                                    dtype_code(tokens), 0, ws.data_ptr(), ws.numel(),
                                    at::cuda::getCurrentCUDAStream().stream()),
                 "fpscan_scan_fwd_cl");
      }
      return out;
    }
    // rows of codes start on 16-byte boundaries, as the kernels' tile copies need
    at::Tensor codes = at::empty({b, l, (d + 15) / 16 * 16}, opts.dtype(at::kChar));
    at::Tensor steps = at::empty({b, (l + 7) / 8, d * tokens.element_size() / 16}, opts.dtype(at::kFloat));
    if (b && d) {
      const at::Tensor ws = workspace_of(tokens, false);
      raise_on(fpscan_scan_fwd_cl8(gates.data_ptr(), tokens.data_ptr(), out.data_ptr(),
                                   codes.data_ptr(), steps.data_ptr<float>(), b, l, d,
                                   dtype_code(tokens), ws.data_ptr(), ws.numel(),
                                   at::cuda::getCurrentCUDAStream().stream()),
               "fpscan_scan_fwd_cl8");
    }
    ctx->save_for_backward({gates, codes, steps});
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const at::Tensor gates = kept[0];
    const at::Tensor go = aligned(grads[0].contiguous());
    check(gates, go);
    const c10::cuda::CUDAGuard guard(go.device());
    at::Tensor dgates = at::empty_like(go), dtokens = at::empty_like(go);
    if (go.size(0) && go.size(2)) {
      const at::Tensor ws = workspace_of(go, true);
      raise_on(fpscan_scan_bwd_cl8(gates.data_ptr(), kept[1].data_ptr(), kept[2].data_ptr<float>(),
                                   go.data_ptr(), dgates.data_ptr(), dtokens.data_ptr(), go.size(0),
                                   go.size(1), go.size(2), dtype_code(go), ws.data_ptr(), ws.numel(),
                                   at::cuda::getCurrentCUDAStream().stream()),
               "fpscan_scan_bwd_cl8");
    }
    return once({dgates, dtokens, at::Tensor()}, "pscan_channels_last with checkpoint8");
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("fullscan_forward", &fullscan_forward,
        "fullscan_forward(gates, tokens, out, reverse) -> out (the reference extension's contract)");
  m.def("scan_forward", &scan_forward, "scan_forward(gates, tokens, reverse) -> out");
  m.def("scan_backward", &scan_backward,
        "scan_backward(gates, y, grad_out) -> (dgates, dtokens), the fused PScan backward");
  m.def("delta_step", &delta_step, "delta_step(q, k, v, log_decay, beta, state, scale, out) -> out");
  m.def("delta_forward", &delta_forward,
        "delta_forward(q, k, v, log_decay, beta, initial, scale, return_state, out) -> (out, final)");
  m.def("delta_backward", &delta_backward,
        "delta_backward(q, k, v, log_decay, beta, grad_out, initial, grad_final, scale, need_initial)"
        " -> (dq, dk, dv, dlog_decay, dbeta, dinitial)");
  m.def("gated_delta", &gated_delta,
        "gated_delta(q, k, v, log_decay, beta, state, scale, return_state, checkpoint8) -> (out, final),"
        " differentiable");
  m.def("pscan_channels_last8",
        [](const at::Tensor& gates, const at::Tensor& tokens) {
          return Scan8::apply(gates, tokens, wanted({&gates, &tokens}));
        },
        "pscan_channels_last8(gates, tokens) -> out, differentiable, the output kept in 8 bits");
  m.def("quantize8", &quantize8, "quantize8(x) -> (codes, steps)");
  m.def("dequantize8", [](const at::Tensor& codes, const at::Tensor& steps, py::object dtype) {
    return dequantize8(codes, steps, torch::python::detail::py_object_to_dtype(dtype));
  });
  m.def("abi_version", []() { return fpscan_abi_version(); });
}
