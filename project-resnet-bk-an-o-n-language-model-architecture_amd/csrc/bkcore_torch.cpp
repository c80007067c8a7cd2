// The layer operators as differentiable tensor functions: allocation, saved tensors and the launches of the C ABI
// (include/bkcore.h) in native code.  A layer norm's training step spends 42 us of host time this way (29 for a function that
// does nothing; 120 with the same steps written in Python, whose backward has to fetch the interpreter lock on the autograd
// engine's thread); the norms, convolutions and small attentions of this package are shorter than that on the GPU.
// Arguments are checked by the Python entry points (bkcore/norm.py, selective.py, attention.py), the only callers.
// `stream` is the current stream's handle at the forward; the engine runs the backward on that stream again.
#include <torch/extension.h>

#include "../../include/bkcore.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

int dtype_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return BKCORE_F32;
    case at::kBFloat16: return BKCORE_BF16;
    case at::kHalf: return BKCORE_F16;
    default: TORCH_CHECK_TYPE(false, "bkcore: unsupported element type ", t.scalar_type());
  }
}

void check(int rc, const char *what) {
  TORCH_CHECK(rc == 0, "bkcore: ", what, " failed: ", bkcore_error_string(rc), " (code ", rc, ", hip error ",
              bkcore_last_hip_error(), ")");
}

void first_derivatives_only(const char *what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "bkcore: ", what,
              " has first derivatives only (create_graph is not supported)");
}

// Strides between positions from here on are beyond the kernels' 32-bit offsets inside a tile.
constexpr int64_t FAR_STRIDE = 1 << 24;

// The tensor itself when its last dimension has unit stride and its positions lie near enough, else a contiguous copy.
Tensor inner(const Tensor &t) {
  if (!t.defined()) return t;
  const int64_t n = t.dim();
  if ((t.size(n - 1) <= 1 || t.stride(n - 1) == 1) && (n < 2 || t.stride(n - 2) < FAR_STRIDE)) return t;
  return t.contiguous();
}
Tensor dense(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *fptr(const Tensor &t) { return (float *)ptr(t); }
const int *iptr(const Tensor &t) { return (const int *)ptr(t); }
int64_t str(const Tensor &t, int64_t d) { return t.defined() ? t.stride(d) : 0; }
Tensor floats(const Tensor &like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor bytes(const Tensor &like, size_t n) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
// A caller's buffer was written through its pointer: functions that saved it for their backward have to notice, as they do
// after the tensor library's own in-place operations.
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// Calls without a derivative refuse forward-mode tangents, which would be lost without a word.
void no_tangent(const char *what, std::initializer_list<Tensor> operands) {
  for (const Tensor &t : operands)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "bkcore: ", what, " has no derivative, and an operand carries a "
                "forward-mode tangent");
}
using Optional = std::optional<Tensor>;
// An absent operand has no place among a node's edges, so a later operand's edge is counted over those that are there.
Tensor opt(const std::optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }
void *handle(int64_t stream) { return (void *)(uintptr_t)stream; }

// ------------------------------------------------------------------------------------------------------- layer norm

struct LayerNorm : Function<LayerNorm> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Optional &weight, const Optional &bias_, double eps,
                        bool keep, int64_t stream) {
    const int64_t D = x.size(-1);
    const Tensor x2 = inner(x.dim() == 2 ? x : x.reshape({-1, D})), w = dense(opt(weight)), bias = opt(bias_), b = dense(bias);
    const int64_t rows = x2.size(0);
    Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
    Tensor stats = keep ? floats(x, {2 * rows}) : Tensor();
    const Tensor &p = w.defined() ? w : b.defined() ? b : x2;
    check(bkcore_layer_norm(x2.data_ptr(), x2.stride(0), dtype_of(x), ptr(w), ptr(b), dtype_of(p), (float)eps, rows, D,
                            y.data_ptr(), fptr(stats), handle(stream)),
          "bkcore_layer_norm");
    if (keep) {
      ctx->save_for_backward({x2, w, stats});
      ctx->saved_data["shape"] = x.sizes().vec();
      ctx->saved_data["bias"] = bias.defined() ? (int64_t)bias.scalar_type() : -1;
      ctx->saved_data["stream"] = stream;
    }
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    first_derivatives_only("layer_norm");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x2 = saved[0], &w = saved[1], &stats = saved[2];
    const bool need_w = w.defined() && ctx->needs_input_grad(1);
    const int64_t bias = ctx->saved_data["bias"].toInt();
    const bool need_b = bias >= 0 && ctx->needs_input_grad(w.defined() ? 2 : 1);
    const int64_t rows = x2.size(0), D = x2.size(1);
    const Tensor g2 = inner(grads[0].dim() == 2 ? grads[0] : grads[0].reshape({-1, D}));
    Tensor dx = at::empty({rows, D}, x2.options()), gp, ws;
    size_t n = 0;
    if (need_w || need_b) {
      gp = floats(x2, {2, D});
      n = bkcore_layer_norm_backward_workspace_bytes(rows, D);
      ws = bytes(x2, n);
      if (rows == 0) gp.zero_();
    }
    check(bkcore_layer_norm_backward(g2.data_ptr(), g2.stride(0), x2.data_ptr(), x2.stride(0), dtype_of(x2), ptr(w),
                                     dtype_of(w.defined() ? w : x2), fptr(stats), rows, D, dx.data_ptr(), fptr(gp), ptr(ws),
                                     n, handle(ctx->saved_data["stream"].toInt())),
          "bkcore_layer_norm_backward");
    return {dx.view(ctx->saved_data["shape"].toIntVector()), need_w ? gp[0].to(w.scalar_type()) : Tensor(),
            need_b ? gp[1].to((at::ScalarType)bias) : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor layer_norm(const Tensor &x, const Optional &w, const Optional &b, double eps, bool keep,
                  int64_t stream) {
  return LayerNorm::apply(x, w, b, eps, keep, stream);
}

// ------------------------------------------------------------------------------------------------------ convolution

struct CausalConv : Function<CausalConv> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x_, const Tensor &weight, const Optional &bias,
                               const Optional &state, const Optional &lengths_, int64_t silu, bool keep, bool want_state,
                               int64_t stream) {
    const Tensor x = inner(x_), w = dense(weight), b = dense(opt(bias)), st = dense(opt(state)), lengths = opt(lengths_);
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), K = w.size(1);
    Tensor y = at::empty({B, T, C}, x.options());
    Tensor fin = want_state ? at::empty({B, K - 1, C}, x.options()) : Tensor();
    check(bkcore_causal_conv(x.data_ptr(), x.stride(0), x.stride(1), dtype_of(x), w.data_ptr(), ptr(b), dtype_of(w), ptr(st),
                             iptr(lengths), B, T, C, K, (int)silu, y.data_ptr(), ptr(fin), handle(stream)),
          "bkcore_causal_conv");
    if (keep) {
      ctx->save_for_backward({x, w, b, st, lengths});
      ctx->saved_data["silu"] = silu;
      ctx->saved_data["stream"] = stream;
      ctx->set_materialize_grads(false);
    }
    return want_state ? variable_list{y, fin} : variable_list{y};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    first_derivatives_only("causal_conv");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &st = saved[3], &lengths = saved[4];
    const bool need_w = ctx->needs_input_grad(1), need_b = b.defined() && ctx->needs_input_grad(2);
    const bool need_st = st.defined() && ctx->needs_input_grad(b.defined() ? 3 : 2);
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), K = w.size(1);
    const Tensor dy = grads[0].defined() ? inner(grads[0]) : at::zeros({B, T, C}, x.options());
    const Tensor dfin = grads.size() > 1 ? dense(grads[1]) : Tensor();
    Tensor dx = at::empty({B, T, C}, x.options()), dst = need_st ? at::empty_like(st) : Tensor(), gp, ws;
    size_t n = 0;
    if (need_w || need_b) {
      gp = floats(x, {C * (K + 1)});
      n = bkcore_causal_conv_backward_workspace_bytes(B, T, C, K);
      ws = bytes(x, n);
    }
    if (B == 0 || T == 0 || C == 0) {  // nothing runs: no position, and the state passes through unchanged
      if (gp.defined()) gp.zero_();
      if (dst.defined()) {
        if (dfin.defined()) dst.copy_(dfin);
        else dst.zero_();
      }
    }
    check(bkcore_causal_conv_backward(dy.data_ptr(), dy.stride(0), dy.stride(1), x.data_ptr(), x.stride(0), x.stride(1),
                                      dtype_of(x), w.data_ptr(), ptr(b), dtype_of(w), ptr(st), ptr(dfin), iptr(lengths), B,
                                      T, C, K, (int)ctx->saved_data["silu"].toInt(), dx.data_ptr(), fptr(gp), ptr(dst),
                                      ptr(ws), n, handle(ctx->saved_data["stream"].toInt())),
          "bkcore_causal_conv_backward");
    return {dx, need_w ? gp.narrow(0, 0, C * K).view({C, K}).to(w.scalar_type()) : Tensor(),
            need_b ? gp.narrow(0, C * K, C).to(b.scalar_type()) : Tensor(), dst, Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

variable_list causal_conv(const Tensor &x, const Tensor &w, const Optional &b, const Optional &state,
                          const Optional &lengths, int64_t silu, bool keep, bool want_state, int64_t stream) {
  return CausalConv::apply(x, w, b, state, lengths, silu, keep, want_state, stream);
}

Tensor causal_conv_step(const Tensor &x_, const Tensor &state, const Tensor &weight, const Optional &bias,
                        int64_t silu, int64_t stream) {
  no_tangent("causal_conv_step", {x_, state, weight, opt(bias)});
  const Tensor x = inner(x_), w = dense(weight), b = dense(opt(bias));
  const int64_t B = x.size(0), C = x.size(1), K = w.size(1);
  Tensor y = at::empty({B, C}, x.options());
  check(bkcore_causal_conv_step(x.data_ptr(), x.stride(0), dtype_of(x), state.data_ptr(), w.data_ptr(), ptr(b), dtype_of(w), B,
                                C, K, (int)silu, y.data_ptr(), handle(stream)),
        "bkcore_causal_conv_step");
  written(state);
  return y;
}

// --------------------------------------------------------------------------------------------------- selective scan

struct SelectiveScan : Function<SelectiveScan> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x_, const Tensor &delta_, const Tensor &A_,
                               const Tensor &B_, const Tensor &C_, const Optional &D_, const Optional &z_,
                               const Optional &bias_, const Optional &state_, const Optional &lengths_, int64_t softplus, bool keep, bool want_state,
                               int64_t stream) {
    const Tensor x = inner(x_), delta = inner(delta_), Bm = inner(B_), Cm = inner(C_), z = inner(opt(z_));
    const Tensor A = dense(A_), D = dense(opt(D_)), bias = dense(opt(bias_)), state = dense(opt(state_)), lengths = opt(lengths_);
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), N = A.size(1);
    Tensor y = at::empty({B, T, C}, x.options());
    Tensor fin = want_state ? floats(x, {B, C, N}) : Tensor();
    if (want_state && T == 0) {
      if (state.defined()) fin.copy_(state);
      else fin.zero_();
    }
    Tensor ckpt;
    if (keep) ckpt = at::empty({(int64_t)bkcore_selective_scan_checkpoint_bytes(B, T, C, N)}, x.options().dtype(at::kByte));
    const size_t n = bkcore_selective_scan_workspace_bytes(B, T, C, N);
    const Tensor ws = bytes(x, n);
    check(bkcore_selective_scan(x.data_ptr(), x.stride(0), x.stride(1), delta.data_ptr(), delta.stride(0), delta.stride(1),
                                fptr(A), Bm.data_ptr(), Bm.stride(0), Bm.stride(1), Cm.data_ptr(), Cm.stride(0),
                                Cm.stride(1), fptr(D), ptr(z), str(z, 0), str(z, 1), fptr(bias), (int)softplus, dtype_of(x),
                                iptr(lengths), fptr(state), B, T, C, N, y.data_ptr(), fptr(fin), fptr(ckpt), ptr(ws), n,
                                handle(stream)),
          "bkcore_selective_scan");
    if (keep) {
      ctx->save_for_backward({x, delta, A, Bm, Cm, D, z, bias, lengths, ckpt});
      ctx->saved_data["softplus"] = softplus;
      ctx->saved_data["state"] = state.defined();
      ctx->saved_data["stream"] = stream;
      ctx->set_materialize_grads(false);
    }
    return want_state ? variable_list{y, fin} : variable_list{y};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    first_derivatives_only("selective_scan");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &delta = saved[1], &A = saved[2], &Bm = saved[3], &Cm = saved[4], &D = saved[5], &z = saved[6],
                 &bias = saved[7], &lengths = saved[8], &ckpt = saved[9];
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), N = A.size(1);
    const Tensor dy = grads[0].defined() ? inner(grads[0]) : at::zeros({B, T, C}, x.options());
    const Tensor dfin = grads.size() > 1 ? dense(grads[1]) : Tensor();
    Tensor dx = at::empty({B, T, C}, x.options()), dd = at::empty({B, T, C}, x.options());
    Tensor dz = z.defined() ? at::empty({B, T, C}, x.options()) : Tensor();
    Tensor dB = at::empty({B, T, N}, x.options()), dC = at::empty({B, T, N}, x.options());
    Tensor gp = floats(x, {C * N + 2 * C});
    const bool need_state =
        ctx->saved_data["state"].toBool() && ctx->needs_input_grad(5 + D.defined() + z.defined() + bias.defined());
    Tensor dh0 = need_state ? floats(x, {B, C, N}) : Tensor();
    if (B == 0 || T == 0 || C == 0) {  // nothing runs: no position, and the state passes through unchanged
      gp.zero_();
      dB.zero_();
      dC.zero_();
      if (dh0.defined()) {
        if (dfin.defined()) dh0.copy_(dfin);
        else dh0.zero_();
      }
    }
    const size_t n = bkcore_selective_scan_backward_workspace_bytes(B, T, C, N);
    const Tensor ws = bytes(x, n);
    check(bkcore_selective_scan_backward(
              dy.data_ptr(), dy.stride(0), dy.stride(1), fptr(dfin), x.data_ptr(), x.stride(0), x.stride(1),
              delta.data_ptr(), delta.stride(0), delta.stride(1), fptr(A), Bm.data_ptr(), Bm.stride(0), Bm.stride(1),
              Cm.data_ptr(), Cm.stride(0), Cm.stride(1), fptr(D), ptr(z), str(z, 0), str(z, 1), fptr(bias),
              (int)ctx->saved_data["softplus"].toInt(), dtype_of(x), iptr(lengths), fptr(ckpt), B, T, C, N, dx.data_ptr(),
              dd.data_ptr(), fptr(gp), dB.data_ptr(), dC.data_ptr(), ptr(dz), fptr(dh0), ptr(ws), n,
              handle(ctx->saved_data["stream"].toInt())),
          "bkcore_selective_scan_backward");
    return {dx, dd, gp.narrow(0, 0, C * N).view({C, N}), dB, dC, D.defined() ? gp.narrow(0, C * N, C) : Tensor(), dz,
            bias.defined() ? gp.narrow(0, C * N + C, C) : Tensor(), dh0, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

variable_list selective_scan(const Tensor &x, const Tensor &delta, const Tensor &A, const Tensor &B, const Tensor &C,
                             const Optional &D, const Optional &z, const Optional &bias,
                             const Optional &state, const Optional &lengths, int64_t softplus,
                             bool keep, bool want_state, int64_t stream) {
  return SelectiveScan::apply(x, delta, A, B, C, D, z, bias, state, lengths, softplus, keep,
                              want_state, stream);
}

Tensor selective_scan_step(const Tensor &x_, const Tensor &state, const Tensor &delta_, const Tensor &A_, const Tensor &B_,
                           const Tensor &C_, const Optional &D_, const Optional &z_,
                           const Optional &bias_, int64_t softplus, int64_t stream) {
  no_tangent("selective_scan_step", {x_, state, delta_, A_, B_, C_, opt(D_), opt(z_), opt(bias_)});
  const Tensor x = inner(x_), delta = inner(delta_), Bm = inner(B_), Cm = inner(C_), z = inner(opt(z_));
  const Tensor D = dense(opt(D_)), bias = dense(opt(bias_));
  Tensor A = dense(A_);
  if ((uintptr_t)A.data_ptr() % 16) A = A.clone();
  const int64_t B = x.size(0), C = x.size(1), N = A.size(1);
  Tensor y = at::empty({B, C}, x.options());
  check(bkcore_selective_scan_step(x.data_ptr(), x.stride(0), fptr(state), delta.data_ptr(), delta.stride(0), fptr(A),
                                   Bm.data_ptr(), Bm.stride(0), Cm.data_ptr(), Cm.stride(0), fptr(D), ptr(z), str(z, 0),
                                   fptr(bias), (int)softplus, dtype_of(x), B, C, N, y.data_ptr(), handle(stream)),
        "bkcore_selective_scan_step");
  written(state);
  return y;
}

// --------------------------------------------------------------------------------------------------------- attention

struct SlidingAttention : Function<SlidingAttention> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q_, const Tensor &k_, const Tensor &v_, const Optional &lengths_,
                        int64_t window, int64_t sinks, double scale, bool keep, int64_t stream) {
    const Tensor q = inner(q_), k = inner(k_), v = inner(v_), lengths = opt(lengths_);
    const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3), Hk = k.size(1);
    Tensor o = at::empty({B, T, H, D}, q.options());
    Tensor lo = keep && q.scalar_type() != at::kFloat ? at::empty({B, T, H, D}, q.options()) : Tensor();
    Tensor lse = keep ? floats(q, {B * H * T}) : Tensor();
    check(bkcore_sliding_attention(q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.data_ptr(), k.stride(0),
                                   k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2),
                                   dtype_of(q), iptr(lengths), B, H, Hk, T, D, window, sinks, (float)scale, o.data_ptr(),
                                   ptr(lo), fptr(lse), handle(stream)),
          "bkcore_sliding_attention");
    if (keep) {
      ctx->save_for_backward({q, k, v, o, lo, lse, lengths});
      ctx->saved_data["window"] = window;
      ctx->saved_data["sinks"] = sinks;
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["stream"] = stream;
    }
    return o.transpose(1, 2);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    first_derivatives_only("sliding_attention");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &lo = saved[4], &lse = saved[5],
                 &lengths = saved[6];
    const Tensor g = inner(grads[0]);
    const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3), Hk = k.size(1);
    const int64_t window = ctx->saved_data["window"].toInt(), sinks = ctx->saved_data["sinks"].toInt();
    Tensor dq = at::empty({B, T, H, D}, q.options()), dk = at::empty({B, T, Hk, D}, q.options());
    Tensor dv = at::empty({B, T, Hk, D}, q.options());
    const size_t n = bkcore_sliding_attention_backward_workspace_bytes(B, H, Hk, T, D, window, sinks);
    const Tensor ws = bytes(q, n);
    check(bkcore_sliding_attention_backward(
              g.data_ptr(), g.stride(0), g.stride(1), g.stride(2), q.data_ptr(), q.stride(0), q.stride(1), q.stride(2),
              k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2),
              o.data_ptr(), ptr(lo), fptr(lse), dtype_of(q), iptr(lengths), B, H, Hk, T, D, window, sinks,
              (float)ctx->saved_data["scale"].toDouble(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), ptr(ws), n,
              handle(ctx->saved_data["stream"].toInt())),
          "bkcore_sliding_attention_backward");
    return {dq.transpose(1, 2), dk.transpose(1, 2), dv.transpose(1, 2), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};

Tensor sliding_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Optional &lengths,
                         int64_t window, int64_t sinks, double scale, bool keep, int64_t stream) {
  return SlidingAttention::apply(q, k, v, lengths, window, sinks, scale, keep, stream);
}

Tensor sliding_attention_step(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &kc, const Tensor &vc,
                              const Tensor &positions_, int64_t window, int64_t sinks, double scale, int64_t stream) {
  no_tangent("sliding_attention_step", {q_, k_, v_, kc, vc});
  const Tensor q = inner(q_), k = inner(k_), v = inner(v_), positions = positions_.contiguous();
  const int64_t B = q.size(0), H = q.size(1), D = q.size(2), Hk = k.size(1), cap = kc.size(2);
  Tensor o = at::empty({B, H, D}, q.options());
  const size_t n = bkcore_sliding_attention_step_workspace_bytes(B, H, Hk, cap, D, window, sinks);
  const Tensor ws = bytes(q, n);
  check(bkcore_sliding_attention_step(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                                      v.data_ptr(), v.stride(0), v.stride(1), kc.data_ptr(), kc.stride(0), kc.stride(1),
                                      kc.stride(2), vc.data_ptr(), vc.stride(0), vc.stride(1), vc.stride(2),
                                      iptr(positions), dtype_of(q), B, H, Hk, cap, D, window, sinks, (float)scale,
                                      o.data_ptr(), ptr(ws), n, handle(stream)),
        "bkcore_sliding_attention_step");
  written(kc);
  written(vc);
  return o;
}

void sliding_cache_fill(const Tensor &k_, const Tensor &v_, const Tensor &kc, const Tensor &vc,
                        const Optional &lengths_, int64_t sinks, int64_t stream) {
  no_tangent("sliding_cache_fill", {k_, v_, kc, vc});
  const Tensor k = inner(k_), v = inner(v_), lengths = opt(lengths_);
  check(bkcore_sliding_cache_fill(k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0),
                                  v.stride(1), v.stride(2), kc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2),
                                  vc.data_ptr(), vc.stride(0), vc.stride(1), vc.stride(2), iptr(lengths), dtype_of(k),
                                  k.size(0), k.size(1), k.size(2), kc.size(2), k.size(3), sinks, handle(stream)),
        "bkcore_sliding_cache_fill");
  written(kc);
  written(vc);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("abi_version", &bkcore_abi_version);
  m.def("layer_norm", &layer_norm);
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("sliding_attention", &sliding_attention);
  m.def("sliding_attention_step", &sliding_attention_step);
  m.def("sliding_cache_fill", &sliding_cache_fill);
}
