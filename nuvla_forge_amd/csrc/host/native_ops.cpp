// The host side of the fused ops in C++: argument checks, output and workspace
// allocation, kernel launches and the autograd node of one call, without the
// Python frames of the general path (kernels/*.py).  At the sizes of a small
// model the ops are bound by that host work: the adaLN seam at B 8 T 6 N 384,
// forward + backward, takes ~75 us of it in Python (seven allocations on
// autograd's thread, two ctypes calls, the Function's own machinery) and the
// kernels 17.
//
// Each entry takes the plain call only -- strided device tensors of one
// device, the shapes and types the kernels take, no tracing, no dispatch or
// function mode, no functorch transform, no forward-mode tangent -- and
// answers None to any other, which then runs the general path: it raises
// what it always raised, and stays visible to the tracer or mode.  Saved
// tensors go through save_for_backward, so saved-tensor hooks see them and
// autograd frees them after the backward.  Nothing is kept between calls.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/torch.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include "nuvla_forge_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxRow = 16384;  // widest adaLN row the kernels take
constexpr int64_t kMaxHead = 128;   // widest attention head
constexpr int64_t kMaxPairs = 256, kMaxTurned = 1024;  // most rotary pairs, widest rotary head

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return NF_DTYPE_F32;
    case at::kBFloat16: return NF_DTYPE_BF16;
    case at::kHalf: return NF_DTYPE_F16;
    default: return -1;
  }
}
int code_of(const Tensor &t) { return code_of(t.scalar_type()); }

void check(int rc, const char *what) {
  TORCH_CHECK(rc == 0, what, " failed (status ", rc, "): ", nf_last_error());
}

void *stream_of(const Tensor &t) {
  return static_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor bytes(size_t n, const Tensor &like) {
  return at::empty({(int64_t)(n > 0 ? n : 1)}, like.options().dtype(at::kByte));
}

// What a backward returns, `recording`: under create_graph.  The kernels record nothing, so a
// derivative taken through their results would leave terms out without a word; the results get a
// node that raises when one reaches it.  Its edges are the backward's own and those of the
// upstream gradients, so that it is reached by whichever of them the derivative is taken.
variable_list first_order_only(const char *op, bool recording, const variable_list &grads,
                               variable_list out) {
  if (!recording) return out;
  torch::autograd::edge_list edges;
  if (const auto here = torch::autograd::get_current_node()) edges = here->next_edges();
  for (const Tensor &g : grads)
    if (g.defined() && g.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(g));
  const std::shared_ptr<torch::autograd::Node> node(
      new torch::autograd::Error(
          std::string(op) + ": second derivatives are not supported on the device",
          std::move(edges)),
      torch::autograd::deleteNode);
  for (Tensor &t : out)
    if (t.defined()) {
      t = t.detach();
      torch::autograd::set_history(t, node);
    }
  return out;
}

// Nothing that could see or replace the ops of the general path is active.
bool quiet() {
  return !torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !at::impl::torch_function_mode_enabled() &&
         !c10::impl::tls_is_dispatch_key_included(
             c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// A strided device tensor with memory of its own kind.
bool plain(const Tensor &t, c10::Device dev) {
  if (!t.defined() || !dev.is_cuda() || t.device() != dev || t.layout() != at::kStrided) return false;
  const c10::DispatchKeySet ks = t.key_set();
  for (c10::DispatchKey k :
       {c10::DispatchKey::Python, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative,
        c10::DispatchKey::ZeroTensor, c10::DispatchKey::Functionalize,
        c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
        c10::DispatchKey::NestedTensor})
    if (ks.has(k)) return false;
  return !t._fw_grad(0).defined();
}

// ---------------------------------------------------------------------------
// adaLN seam
// ---------------------------------------------------------------------------
struct Seam : torch::autograd::Function<Seam> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &y,
                               const Tensor &gate, const Tensor &weight, const Tensor &scale,
                               const Tensor &shift, int64_t t, double eps) {
    const c10::DeviceGuard guard(x.device());
    const int64_t m = x.size(0), n = x.size(1);
    Tensor h = at::empty({m, n}, x.options()), out = at::empty({m, n}, x.options());
    Tensor rstd = at::empty({m}, x.options().dtype(at::kFloat));
    check(nf_adaln_fwd(x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), gate.data_ptr(),
                       gate.stride(0), weight.data_ptr(), scale.data_ptr(), scale.stride(0),
                       shift.data_ptr(), shift.stride(0), h.data_ptr(), out.data_ptr(),
                       rstd.data_ptr<float>(), m, n, t, (float)eps, code_of(x), code_of(y),
                       code_of(gate), code_of(weight), code_of(scale), code_of(shift),
                       stream_of(x)),
          "nf_adaln_fwd");
    ctx->save_for_backward({x, y, gate, weight, scale, rstd});
    ctx->saved_data["t"] = t;
    ctx->saved_data["shift"] = (int64_t)shift.scalar_type();
    ctx->set_materialize_grads(false);
    return {h, out};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list res(8);
    if (!grads[0].defined() && !grads[1].defined()) return res;
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &y = s[1], &gate = s[2], &weight = s[3], &scale = s[4], &rstd = s[5];
    const c10::DeviceGuard guard(x.device());
    const int64_t m = x.size(0), n = x.size(1), t = ctx->saved_data["t"].toInt(), b = m / t;
    const auto dt_shift = (at::ScalarType)ctx->saved_data["shift"].toInt();
    Tensor dh, dout;
    if (grads[0].defined()) dh = grads[0].to(x.scalar_type()).contiguous();
    if (grads[1].defined()) dout = grads[1].to(x.scalar_type()).contiguous();
    for (const Tensor *g : {&dh, &dout})
      TORCH_CHECK_VALUE(!g->defined() || g->device() == x.device(),
                        "fused_adaln_residual_rmsnorm backward: an upstream gradient is not on "
                        "the forward's device");
    Tensor dx = at::empty({m, n}, x.options()), dy = at::empty({m, n}, y.options());
    Tensor dgate, dweight, dscale, dshift;
    if (ctx->needs_input_grad(2)) dgate = at::empty({b, n}, gate.options());
    if (ctx->needs_input_grad(3)) dweight = at::empty({n}, weight.options());
    if (ctx->needs_input_grad(4)) dscale = at::empty({b, n}, scale.options());
    if (ctx->needs_input_grad(5)) dshift = at::empty({b, n}, scale.options().dtype(dt_shift));
    const size_t nbytes = nf_adaln_bwd_workspace(m, n, t);
    Tensor ws = bytes(nbytes, x);
    check(nf_adaln_bwd_full(ptr(dh), ptr(dout), x.data_ptr(), x.stride(0), y.data_ptr(),
                            y.stride(0), gate.data_ptr(), gate.stride(0), weight.data_ptr(),
                            scale.data_ptr(), scale.stride(0), rstd.data_ptr<float>(),
                            dx.data_ptr(), dy.data_ptr(), ptr(dgate), ptr(dweight), ptr(dscale),
                            ptr(dshift), ws.data_ptr(), nbytes, m, n, t, code_of(x), code_of(y),
                            code_of(gate), code_of(weight), code_of(scale), code_of(dt_shift),
                            stream_of(x)),
          "nf_adaln_bwd_full");
    if (ctx->needs_input_grad(0)) res[0] = dx;
    if (ctx->needs_input_grad(1)) res[1] = dy;
    res[2] = dgate;
    res[3] = dweight;
    res[4] = dscale;
    res[5] = dshift;
    return first_order_only("fused_adaln_residual_rmsnorm", at::GradMode::is_enabled(), grads,
                            std::move(res));
  }
};

// (x, y) element types the row kernels take: equal, or fp32 x with 16-bit y
bool seam_types(const Tensor &x, const Tensor &y) {
  const int cx = code_of(x), cy = code_of(y);
  return cx >= 0 && cy >= 0 && (cx == cy || cx == NF_DTYPE_F32);
}

bool seam_plain(const Tensor &x, const Tensor &y, const Tensor &gate, const Tensor &weight,
                const Tensor &scale, const Tensor &shift, int64_t t) {
  const c10::Device dev = x.device();
  for (const Tensor *v : {&x, &y, &gate, &weight, &scale, &shift})
    if (!plain(*v, dev) || code_of(*v) < 0) return false;
  if (x.dim() != 2 || y.dim() != 2 || x.size(0) == 0 || x.size(1) == 0 ||
      x.size(1) > kMaxRow || y.sizes() != x.sizes() || !seam_types(x, y))
    return false;
  const int64_t m = x.size(0), n = x.size(1);
  if (t <= 0 || m % t != 0 || x.stride(1) != 1 || y.stride(1) != 1) return false;
  for (const Tensor *v : {&gate, &scale, &shift})
    if (v->dim() != 2 || v->size(0) != m / t || v->size(1) != n || v->stride(1) != 1)
      return false;
  return weight.dim() == 1 && weight.size(0) == n && weight.is_contiguous();
}

// ---------------------------------------------------------------------------
// SwiGLU
// ---------------------------------------------------------------------------
struct SwiGLU : torch::autograd::Function<SwiGLU> {
  static Tensor forward(AutogradContext *ctx, const Tensor &a_in, const Tensor &b_in) {
    const c10::DeviceGuard guard(a_in.device());
    const Tensor a = a_in.contiguous(), b = b_in.contiguous();
    Tensor out = at::empty(a.sizes(), a.options());
    check(nf_swiglu_fwd(a.data_ptr(), b.data_ptr(), out.data_ptr(), a.numel(), code_of(a),
                        stream_of(a)),
          "nf_swiglu_fwd");
    ctx->save_for_backward({a, b});
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &a = s[0], &b = s[1];
    const c10::DeviceGuard guard(a.device());
    const Tensor g = grads[0].contiguous().to(a.scalar_type());
    TORCH_CHECK_VALUE(g.device() == a.device(),
                      "fused_swiglu backward: dout is not on the forward's device");
    Tensor da = at::empty(a.sizes(), a.options()), db = at::empty(b.sizes(), b.options());
    check(nf_swiglu_bwd(g.data_ptr(), a.data_ptr(), b.data_ptr(), da.data_ptr(), db.data_ptr(),
                        a.numel(), code_of(a), stream_of(a)),
          "nf_swiglu_bwd");
    return first_order_only("fused_swiglu", at::GradMode::is_enabled(), grads, {da, db});
  }
};

// ---------------------------------------------------------------------------
// gate/up projection with the SwiGLU in its epilogue
// ---------------------------------------------------------------------------
// bf16 with unit-stride rows
Tensor rows_bf16(const Tensor &t) {
  const Tensor r = t.to(at::kBFloat16);
  return r.stride(-1) == 1 ? r : r.contiguous();
}

// `t` with rows of whole 16-byte vectors (its width is a multiple of 8): a copy of a
// view whose base or row stride is not.  Every tile of the backward would read it
// element by element: x[:, 1:385] of M 9408 D 384 H 1536, forward + backward,
// 485 us, 231 with the copy.
Tensor vector_rows(const Tensor &t) {
  const bool whole = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && t.stride(0) % 8 == 0;
  return whole ? t : t.clone(at::MemoryFormat::Contiguous);
}

// act = silu(x wg^T) * (x wu^T); a and b (the two products) are written where
// `save`, for the backward.
Tensor gate_up_forward(const Tensor &x, const Tensor &wg, const Tensor &wu, bool save, Tensor &a,
                       Tensor &b) {
  const int64_t m = x.size(0), d = x.size(1), h = wg.size(0);
  if (save) a = at::empty({m, h}, x.options());
  if (save) b = at::empty({m, h}, x.options());
  Tensor act = at::empty({m, h}, x.options());
  check(nf_gemm_swiglu(x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(),
                       wu.stride(0), ptr(a), ptr(b), act.data_ptr(), h, m, d, h, NF_DTYPE_BF16,
                       stream_of(x)),
        "nf_gemm_swiglu");
  return act;
}

struct GateUp : torch::autograd::Function<GateUp> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x_in, const Tensor &g_in,
                        const Tensor &u_in) {
    const c10::DeviceGuard guard(x_in.device());
    const Tensor x = rows_bf16(x_in), wg = rows_bf16(g_in), wu = rows_bf16(u_in);
    Tensor a, b;
    const Tensor act = gate_up_forward(x, wg, wu, true, a, b);
    ctx->save_for_backward({x, wg, wu, a, b});
    ctx->saved_data["dt"] = std::vector<int64_t>{(int64_t)x_in.scalar_type(),
                                                 (int64_t)g_in.scalar_type(),
                                                 (int64_t)u_in.scalar_type()};
    return act;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    Tensor x = s[0], wg = s[1], wu = s[2];
    const Tensor &a = s[3], &b = s[4];
    const c10::DeviceGuard guard(x.device());
    const bool recording = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const auto dt = ctx->saved_data["dt"].toIntVector();
    const Tensor dact = grads[0].to(at::kBFloat16).contiguous();
    TORCH_CHECK_VALUE(dact.device() == x.device(),
                      "fused_gate_up_swiglu backward: dact is not on the forward's device");
    const int64_t m = x.size(0), d = x.size(1), h = a.size(1);
    Tensor da = at::empty({m, h}, a.options()), db = at::empty({m, h}, a.options());
    void *const st = stream_of(x);
    check(nf_swiglu_bwd(dact.data_ptr(), a.data_ptr(), b.data_ptr(), da.data_ptr(),
                        db.data_ptr(), a.numel(), NF_DTYPE_BF16, st),
          "nf_swiglu_bwd");
    // both weight gradients leave the kernel in one type: theirs, or fp32 where
    // two are wanted and differ (neither may round the other's gradient)
    const auto tx = (at::ScalarType)dt[0], tg = (at::ScalarType)dt[1], tu = (at::ScalarType)dt[2];
    const bool need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2);
    const auto tw = need_g && need_u && tg != tu ? at::kFloat : need_g ? tg : tu;
    Tensor dx, dg, du;
    bool one_x = ctx->needs_input_grad(0), one_w = need_g || need_u;  // left to the one launch
    if (need_g) dg = at::empty({h, d}, x.options().dtype(tw));
    if (need_u) du = at::empty({h, d}, x.options().dtype(tw));
    if (tx == at::kBFloat16 && tg == tx && tu == tx &&
        !nf_gemm_swiglu_bwd_wins(m, d, h, one_w)) {
      if (one_x) {
        const c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::autocast_dispatch_keyset);
        dx = at::addmm(at::mm(da, wg), db, wu);
        one_x = false;
      }
      if (need_g && need_u) {
        const size_t nb = nf_gemm_swiglu_wgrad_workspace(m, d, h);
        Tensor ws = bytes(nb, x);
        check(nf_gemm_swiglu_wgrad(da.data_ptr(), db.data_ptr(), h, x.data_ptr(), x.stride(0),
                                   dg.data_ptr(), du.data_ptr(), d, m, d, h, NF_DTYPE_BF16,
                                   ws.data_ptr(), nb, st),
              "nf_gemm_swiglu_wgrad");
        one_w = false;
      }
    }
    if (one_x) dx = at::empty({m, d}, x.options().dtype(tx));
    if (one_x || one_w) {
      if (d % 8 == 0 && h % 8 == 0) {  // other widths are copied to padded rows in the call
        x = vector_rows(x);
        wg = vector_rows(wg);
        wu = vector_rows(wu);
      }
      void *const pg = one_w ? ptr(dg) : nullptr, *const pu = one_w ? ptr(du) : nullptr;
      const size_t nb = nf_gemm_swiglu_bwd_workspace(m, d, h, one_x, pg != nullptr, pu != nullptr);
      Tensor ws = bytes(nb, x);
      check(nf_gemm_swiglu_bwd(da.data_ptr(), db.data_ptr(), h, x.data_ptr(), x.stride(0),
                               wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0),
                               one_x ? dx.data_ptr() : nullptr, code_of(tx), pg, pu, code_of(tw),
                               m, d, h, NF_DTYPE_BF16, ws.data_ptr(), nb, st),
            "nf_gemm_swiglu_bwd");
    }
    return first_order_only("fused_gate_up_swiglu", recording, grads,
                            {dx, need_g ? dg.to(tg) : dg, need_u ? du.to(tu) : du});
  }
};

// ---------------------------------------------------------------------------
// chunked cross entropy
// ---------------------------------------------------------------------------
struct ChunkedCE : torch::autograd::Function<ChunkedCE> {
  static Tensor forward(AutogradContext *ctx, const Tensor &hidden, const Tensor &weight,
                        const Tensor &targets, int64_t chunk_rows, int64_t ignore_index,
                        int64_t compute) {
    const c10::DeviceGuard guard(hidden.device());
    const auto cdt = (at::ScalarType)compute;
    const int64_t m = hidden.size(0), d = hidden.size(1), v = weight.size(0);
    const int code = code_of(cdt);
    const Tensor h = hidden.to(cdt).contiguous(), w = weight.to(cdt).contiguous();
    const Tensor tg = targets.to(at::kLong).contiguous();
    Tensor loss = at::empty({}, hidden.options().dtype(at::kFloat));
    const size_t ns = nf_ce_state_bytes(m, d, v, chunk_rows, code);
    const size_t nw = nf_ce_fwd_workspace(m, d, v, chunk_rows, code);
    TORCH_CHECK_VALUE(ns && nw, "chunked_cross_entropy: shape M=", m, " D=", d, " V=", v,
                      " is beyond the kernels");
    Tensor state = bytes(ns, hidden), ws = bytes(nw, hidden);
    check(nf_ce_fwd(h.data_ptr(), w.data_ptr(), tg.data_ptr<int64_t>(), m, d, v, ignore_index,
                    chunk_rows, code, loss.data_ptr<float>(), nullptr, state.data_ptr(), ns,
                    ws.data_ptr(), nw, stream_of(hidden)),
          "nf_ce_fwd");
    ctx->save_for_backward({state});
    ctx->saved_data["s"] = std::vector<int64_t>{m, d, v, chunk_rows, code,
                                                (int64_t)hidden.scalar_type(),
                                                (int64_t)weight.scalar_type()};
    return loss;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &state = saved[0];
    const c10::DeviceGuard guard(state.device());
    const auto s = ctx->saved_data["s"].toIntVector();
    const int64_t m = s[0], d = s[1], v = s[2], chunk_rows = s[3];
    const int code = (int)s[4];
    const auto th = (at::ScalarType)s[5], tw = (at::ScalarType)s[6];
    const Tensor g = grads[0].to(at::kFloat).contiguous();
    TORCH_CHECK_VALUE(g.device() == state.device(),
                      "chunked_cross_entropy backward: grad_output is not on the forward's device");
    Tensor dh = at::empty({m, d}, state.options().dtype(th));
    Tensor dw = at::empty({v, d}, state.options().dtype(tw));
    const size_t nw = nf_ce_bwd_workspace(m, d, v, chunk_rows, code);
    Tensor ws = bytes(nw, state);
    check(nf_ce_bwd(m, d, v, chunk_rows, code, state.data_ptr(), (size_t)state.numel(),
                    g.data_ptr<float>(), dh.data_ptr(), code_of(th), dw.data_ptr(), code_of(tw),
                    ws.data_ptr(), nw, stream_of(state)),
          "nf_ce_bwd");
    return first_order_only("chunked_cross_entropy", at::GradMode::is_enabled(), grads,
                            {dh, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// ---------------------------------------------------------------------------
// token log probabilities
// ---------------------------------------------------------------------------
// `t` ([R, D], contiguous) from a whole 16-byte vector on: a copy of a view that begins between
// two, which every kernel of the call would read element by element.  Forward and backward, bf16,
// V 32000, weight off by one element: 100 rows, D 2048 926 us, 296 with the copy (215 aligned), 5
// rows 555, 241 and 163, 200 rows, D 1024 414, 148 and 125.
Tensor from_vector(const Tensor &t) {
  const bool whole = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ||
                     t.size(1) * t.element_size() % 16 != 0;
  return whole ? t : t.clone();
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  // {logprobs, entropy, top_logprobs, top_ids}; `keep` what the backward reads
  static variable_list run(const Tensor &hidden, const Tensor &weight, const Tensor &targets,
                           int64_t top_k, int64_t chunk_rows, int64_t ignore_index,
                           at::ScalarType cdt, bool keep, Tensor &w, Tensor &state) {
    const int64_t m = hidden.size(0), d = hidden.size(1), v = weight.size(0);
    const int code = code_of(cdt);
    const Tensor h = from_vector(hidden.to(cdt).contiguous()), tg = targets.contiguous();
    w = from_vector(weight.to(cdt).contiguous());
    const auto f32 = hidden.options().dtype(at::kFloat).requires_grad(false);
    Tensor lp = at::empty({m}, f32), ent = at::empty({m}, f32), top = at::empty({m, top_k}, f32);
    Tensor ids = at::empty({m, top_k}, f32.dtype(at::kLong));
    const size_t ns = nf_token_logprobs_state_bytes(m, d, v, chunk_rows, keep, code);
    const size_t nw = nf_token_logprobs_fwd_workspace(m, d, v, chunk_rows, (int)top_k, code);
    TORCH_CHECK_VALUE(ns && nw, "chunked_token_logprobs: shape M=", m, " D=", d, " V=", v,
                      " is beyond the kernels");
    state = bytes(ns, hidden);
    Tensor ws = bytes(nw, hidden);
    check(nf_token_logprobs_fwd(h.data_ptr(), w.data_ptr(), tg.data_ptr<int64_t>(), m, d, v,
                                ignore_index, chunk_rows, (int)top_k, keep, code, lp.data_ptr<float>(),
                                ent.data_ptr<float>(), top.data_ptr<float>(),
                                ids.data_ptr<int64_t>(), state.data_ptr(), ns, ws.data_ptr(), nw,
                                stream_of(hidden)),
          "nf_token_logprobs_fwd");
    return {lp, ent, top, ids};
  }
  static variable_list forward(AutogradContext *ctx, const Tensor &hidden, const Tensor &weight,
                               const Tensor &targets, int64_t top_k, int64_t chunk_rows,
                               int64_t ignore_index, int64_t compute) {
    const c10::DeviceGuard guard(hidden.device());
    const auto cdt = (at::ScalarType)compute;
    Tensor w, state;
    const variable_list out =
        run(hidden, weight, targets, top_k, chunk_rows, ignore_index, cdt, true, w, state);
    ctx->save_for_backward({w, state});
    ctx->saved_data["s"] = std::vector<int64_t>{hidden.size(0), hidden.size(1), weight.size(0),
                                                chunk_rows, code_of(cdt),
                                                (int64_t)hidden.scalar_type(),
                                                (int64_t)weight.scalar_type()};
    ctx->mark_non_differentiable({out[2], out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list res(7);
    if (!grads[0].defined() && !grads[1].defined()) return res;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &w = saved[0], &state = saved[1];
    const c10::DeviceGuard guard(w.device());
    const auto s = ctx->saved_data["s"].toIntVector();
    const int64_t m = s[0], d = s[1], v = s[2], chunk_rows = s[3];
    const int code = (int)s[4];
    const auto th = (at::ScalarType)s[5], tw = (at::ScalarType)s[6];
    Tensor g[2];
    for (int i = 0; i < 2; ++i) {
      if (!grads[i].defined()) continue;
      TORCH_CHECK_VALUE(grads[i].device() == w.device(), "chunked_token_logprobs backward: an "
                        "upstream gradient is not on the forward's device");
      g[i] = grads[i].to(at::kFloat).contiguous();
    }
    if (ctx->needs_input_grad(0)) res[0] = at::empty({m, d}, w.options().dtype(th));
    if (ctx->needs_input_grad(1)) res[1] = at::empty({v, d}, w.options().dtype(tw));
    const size_t nw = nf_token_logprobs_bwd_workspace(m, d, v, chunk_rows, code);
    Tensor ws = bytes(nw, state);
    check(nf_token_logprobs_bwd(w.data_ptr(), m, d, v, chunk_rows, 1, code, state.data_ptr(),
                                (size_t)state.numel(), (const float *)ptr(g[0]),
                                (const float *)ptr(g[1]), ptr(res[0]), code_of(th), ptr(res[1]),
                                code_of(tw), ws.data_ptr(), nw, stream_of(w)),
          "nf_token_logprobs_bwd");
    return first_order_only("chunked_token_logprobs", at::GradMode::is_enabled(), grads,
                            std::move(res));
  }
};

// ---------------------------------------------------------------------------
// embedding lookup
// ---------------------------------------------------------------------------
// The lookup's gradient as an operator of its own: linear in dout, its gradient the lookup again.
struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Tensor run(const Tensor &dout, const Tensor &ids, int64_t v, double scale, int64_t pad,
                    at::ScalarType table_t) {
    const int64_t m = ids.numel(), d = dout.size(-1);
    const Tensor g = dout.contiguous();
    Tensor dtable = at::empty({v, d}, g.options().dtype(table_t).requires_grad(false));
    const size_t nw = nf_embedding_bwd_workspace(m, d, v);
    Tensor ws = bytes(nw, ids);
    check(nf_embedding_bwd(g.data_ptr(), ids.data_ptr<int64_t>(), pad, (float)scale, m, d, v,
                           dtable.data_ptr(), code_of(g), code_of(table_t), ws.data_ptr(), nw,
                           stream_of(g)),
          "nf_embedding_bwd");
    return dtable;
  }
  static Tensor forward(AutogradContext *ctx, const Tensor &dout, const Tensor &ids, int64_t v,
                        double scale, int64_t pad, int64_t table_t);
  static variable_list backward(AutogradContext *ctx, variable_list grads);
};

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor run(const Tensor &ids, const Tensor &table, double scale, at::ScalarType out_t) {
    const int64_t m = ids.numel(), v = table.size(0), d = table.size(1);
    std::vector<int64_t> sizes = ids.sizes().vec();
    sizes.push_back(d);
    Tensor out = at::empty(sizes, table.options().dtype(out_t).requires_grad(false));
    check(nf_embedding_fwd(ids.data_ptr<int64_t>(), table.data_ptr(), table.stride(0),
                           (float)scale, m, d, v, out.data_ptr(), code_of(table), code_of(out_t),
                           stream_of(table)),
          "nf_embedding_fwd");
    return out;
  }
  static Tensor forward(AutogradContext *ctx, const Tensor &ids, const Tensor &table,
                        double scale, int64_t pad, int64_t out_t) {
    const c10::DeviceGuard guard(table.device());
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["s"] =
        std::vector<int64_t>{table.size(0), pad, (int64_t)table.scalar_type()};
    return run(ids, table, scale, (at::ScalarType)out_t);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &ids = saved[0];
    const c10::DeviceGuard guard(ids.device());
    const auto s = ctx->saved_data["s"].toIntVector();
    const double scale = ctx->saved_data["scale"].toDouble();
    TORCH_CHECK_VALUE(grads[0].device() == ids.device(),
                      "embedding_lookup backward: dout is not on the forward's device");
    const bool recording = at::GradMode::is_enabled() && grads[0].requires_grad();
    const Tensor dtable =
        recording ? EmbeddingGrad::apply(grads[0], ids, s[0], scale, s[1], s[2])
                  : EmbeddingGrad::run(grads[0], ids, s[0], scale, s[1], (at::ScalarType)s[2]);
    return {Tensor(), dtable, Tensor(), Tensor(), Tensor()};
  }
};

Tensor EmbeddingGrad::forward(AutogradContext *ctx, const Tensor &dout, const Tensor &ids,
                              int64_t v, double scale, int64_t pad, int64_t table_t) {
  const c10::DeviceGuard guard(ids.device());
  ctx->save_for_backward({ids});
  ctx->saved_data["scale"] = scale;
  ctx->saved_data["s"] = std::vector<int64_t>{pad, (int64_t)dout.scalar_type()};
  return run(dout, ids, v, scale, pad, (at::ScalarType)table_t);
}
variable_list EmbeddingGrad::backward(AutogradContext *ctx, variable_list grads) {
  const variable_list saved = ctx->get_saved_variables();
  const c10::DeviceGuard guard(saved[0].device());
  const auto s = ctx->saved_data["s"].toIntVector();
  // the padding id's rows, which gave nothing, get nothing: as those outside the table
  const Tensor ids = s[0] < 0 ? saved[0] : saved[0].masked_fill(saved[0].eq(s[0]), -1);
  TORCH_CHECK_VALUE(grads[0].device() == ids.device(),
                    "embedding_lookup backward: a gradient is not on the forward's device");
  const Tensor g = grads[0].contiguous();
  const double scale = ctx->saved_data["scale"].toDouble();
  const bool recording = at::GradMode::is_enabled() && g.requires_grad();
  const Tensor ddout = recording ? Embedding::apply(ids, g, scale, -1, s[1])
                                 : Embedding::run(ids, g, scale, (at::ScalarType)s[1]);
  return {ddout, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
}

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------
struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor run(const Tensor &x, const Tensor &res, at::ScalarType out_t, int64_t threshold,
                    const Tensor &seed_t, int64_t seed, int64_t offset) {
    Tensor out = at::empty(x.sizes(), x.options().dtype(out_t).requires_grad(false));
    check(nf_dropout(x.data_ptr(), ptr(res), out.data_ptr(), x.numel(), (int32_t)threshold,
                     (const int64_t *)ptr(seed_t), seed, offset, code_of(x), code_of(out_t),
                     stream_of(x)),
          "nf_dropout");
    return out;
  }
  static Tensor forward(AutogradContext *ctx, const Tensor &x,
                        const std::optional<Tensor> &residual,
                        const std::optional<Tensor> &seed_in, int64_t threshold, int64_t seed,
                        int64_t offset, int64_t out_t) {
    const c10::DeviceGuard guard(x.device());
    Tensor r, seed_t;
    if (residual) r = residual->contiguous();
    if (seed_in) seed_t = *seed_in;
    if (seed_in) ctx->save_for_backward({seed_t});
    ctx->saved_data["s"] =
        std::vector<int64_t>{threshold, seed, offset, (int64_t)x.scalar_type(), seed_t.defined(),
                             r.defined()};
    return run(x.contiguous(), r, (at::ScalarType)out_t, threshold, seed_t, seed, offset);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto s = ctx->saved_data["s"].toIntVector();
    variable_list res(7);
    // an argument that was left out has no edge: the residual's is the second, if there is one
    if (s[5] && ctx->needs_input_grad(1)) res[1] = grads[0];
    if (!ctx->needs_input_grad(0)) return res;
    Tensor seed_t;
    if (s[4]) {
      seed_t = ctx->get_saved_variables()[0];
      TORCH_CHECK_VALUE(grads[0].device() == seed_t.device(),
                        "fused_dropout backward: dout is not on the forward's device");
    }
    const c10::DeviceGuard guard(grads[0].device());
    if (at::GradMode::is_enabled() && grads[0].requires_grad())  // dx is linear in dout
      res[0] = Dropout::apply(grads[0], std::optional<Tensor>(),
                              s[4] ? std::optional<Tensor>(seed_t) : std::nullopt, s[0], s[1],
                              s[2], s[3]);
    else
      res[0] = run(grads[0].contiguous(), Tensor(), (at::ScalarType)s[3], s[0], seed_t, s[1], s[2]);
    return res;
  }
};

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// [B, T, heads, D] with the strides as nf_attention_* take them
struct Heads {
  Tensor t;
  int64_t b, s, h;
  explicit Heads(const Tensor &x) : t(x) {
    b = x.size(0) == 1 ? 0 : x.stride(0);
    s = x.size(1) == 1 ? 0 : x.stride(1);
    h = x.size(2) == 1 ? 0 : x.stride(2);
  }
};

// `t` where its rows are whole 16-byte vectors within the kernels' reach, else a copy (zeros past
// D up to the next vector).
Heads head_rows(const Tensor &t) {
  const int64_t e = 16 / t.element_size(), d = t.size(3);
  const int64_t far = ((int64_t)1 << 30) / t.element_size();
  const Heads v(t);
  const bool whole = d % e == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                     (t.stride(3) == 1 || d == 1) && v.b % e == 0 && v.s % e == 0 &&
                     v.h % e == 0 && v.s <= far / 512 && 130 * v.s + t.size(2) * v.h < far;
  if (whole) return v;
  // written out, not padded by the library: that keeps the order of t's axes, the tokens innermost
  // where they are
  Tensor c = at::empty({t.size(0), t.size(1), t.size(2), (d + e - 1) / e * e},
                       t.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
  c.narrow(3, 0, d).copy_(t);
  if (d % e) c.narrow(3, d, e - d % e).zero_();
  return Heads(c);
}

struct Attention : torch::autograd::Function<Attention> {
  struct Sizes {
    int64_t B, Tq, Tk, H, Hk, D;
  };
  static Sizes sizes(const Tensor &q, const Tensor &k) {
    return {q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3)};
  }
  // the mask with its keys side by side
  static Tensor bytes_of(const Tensor &mask) {
    if (!mask.defined() || mask.stride(1) == 1 || mask.size(1) == 1) return mask;
    return mask.contiguous();
  }
  static int64_t step_of(const Tensor &mask) {
    return mask.defined() && mask.size(0) > 1 ? mask.stride(0) : 0;
  }
  static Tensor run(const Sizes &z, const Heads &q, const Heads &k, const Heads &v,
                    const Tensor &mask, bool causal, double scale, bool keep, Tensor &state) {
    const int dt = code_of(q.t);
    Tensor out = at::empty({z.B, z.Tq, z.H, z.D}, q.t.options().requires_grad(false));
    const size_t n_state =
        keep ? nf_attention_state_bytes(z.B, z.Tq, z.Tk, z.H, z.Hk, z.D, dt) : 0;
    const size_t n_ws = nf_attention_fwd_workspace(z.B, z.Tq, z.Tk, z.H, z.Hk, z.D, causal, dt);
    Tensor ws;
    if (n_state) state = bytes(n_state, out);
    if (n_ws) ws = bytes(n_ws, out);
    check(nf_attention_fwd(q.t.data_ptr(), q.b, q.s, q.h, k.t.data_ptr(), k.b, k.s, k.h,
                           v.t.data_ptr(), v.b, v.s, v.h, (const uint8_t *)ptr(mask),
                           step_of(mask), z.B, z.Tq, z.Tk, z.H, z.Hk, z.D, causal, (float)scale,
                           dt, out.data_ptr(), ptr(state), n_state, ptr(ws), n_ws, stream_of(out)),
          "nf_attention_fwd");
    return out;
  }
  static Tensor forward(AutogradContext *ctx, const Tensor &q_in, const Tensor &k_in,
                        const Tensor &v_in, const std::optional<Tensor> &mask_in, bool causal,
                        double scale) {
    const c10::DeviceGuard guard(q_in.device());
    const Heads q = head_rows(q_in), k = head_rows(k_in), v = head_rows(v_in);
    const Tensor mask = bytes_of(mask_in ? *mask_in : Tensor());
    Tensor state;
    const Tensor out = run(sizes(q_in, k_in), q, k, v, mask, causal, scale, true, state);
    variable_list kept = {q.t, k.t, v.t, out, state};
    if (mask.defined()) kept.push_back(mask);
    ctx->save_for_backward(kept);
    ctx->saved_data["s"] = std::vector<int64_t>{causal, q_in.size(3)};
    ctx->saved_data["f"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list res(6);
    const variable_list t = ctx->get_saved_variables();
    const auto s = ctx->saved_data["s"].toIntVector();
    // what a saved-tensor hook gives back may lie in memory in another way
    const Tensor out = t[3].contiguous(), state = t[4].contiguous();
    const Tensor mask = t.size() > 5 ? bytes_of(t[5]) : Tensor();
    const c10::DeviceGuard guard(out.device());
    TORCH_CHECK_VALUE(grads[0].device() == out.device(),
                      "fused_attention backward: dout is not on the forward's device");
    const Heads q = head_rows(t[0]), k = head_rows(t[1]), v = head_rows(t[2]);
    const Heads g = head_rows(grads[0].to(out.scalar_type()));
    Sizes z = sizes(q.t, k.t);
    z.D = s[1];
    const int causal = (int)s[0], dt = code_of(out);
    const auto opts = out.options().requires_grad(false);
    if (ctx->needs_input_grad(0)) res[0] = at::empty({z.B, z.Tq, z.H, z.D}, opts);
    for (int i : {1, 2})
      if (ctx->needs_input_grad(i)) res[i] = at::empty({z.B, z.Tk, z.Hk, z.D}, opts);
    const size_t n_ws = nf_attention_bwd_workspace(z.B, z.Tq, z.Tk, z.H, z.Hk, z.D, causal, dt);
    Tensor ws = bytes(n_ws, out);
    check(nf_attention_bwd(q.t.data_ptr(), q.b, q.s, q.h, k.t.data_ptr(), k.b, k.s, k.h,
                           v.t.data_ptr(), v.b, v.s, v.h, (const uint8_t *)ptr(mask),
                           step_of(mask), out.data_ptr(), g.t.data_ptr(), g.b, g.s, g.h, z.B, z.Tq,
                           z.Tk, z.H, z.Hk, z.D, causal, (float)ctx->saved_data["f"].toDouble(),
                           dt, state.data_ptr(), (size_t)state.numel(), ptr(res[0]), ptr(res[1]),
                           ptr(res[2]), ws.data_ptr(), n_ws, stream_of(out)),
          "nf_attention_bwd");
    return first_order_only("fused_attention", at::GradMode::is_enabled(), grads, std::move(res));
  }
};

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
struct Rotary : torch::autograd::Function<Rotary> {
  // q and k turned; either may be undefined.  call: joint, interleaved, then the sections
  static variable_list run(const Tensor &q_in, const Tensor &k_in, const Tensor &pos,
                           const std::vector<int64_t> &call, double base, bool inverse) {
    const Tensor &like = q_in.defined() ? q_in : k_in;
    Tensor x[2] = {q_in, k_in}, y[2];
    int64_t st[2][3] = {}, heads[2] = {0, 0};
    for (int i = 0; i < 2; ++i) {
      if (!x[i].defined()) continue;
      if (x[i].stride(3) != 1 && x[i].size(3) != 1) x[i] = x[i].contiguous();
      y[i] = at::empty(x[i].sizes(), x[i].options().requires_grad(false));
      for (int j = 0; j < 3; ++j) st[i][j] = x[i].stride(j);
      heads[i] = x[i].size(2);
    }
    const int axes = (int)call.size() - 2;
    int32_t sections[4];
    for (int i = 0; i < axes; ++i) sections[i] = (int32_t)call[2 + i];
    const int64_t B = like.size(0), T = like.size(1);
    const bool shared = pos.dim() == 2 || pos.size(0) == 1;
    const int kind = pos.scalar_type() == at::kLong ? 0 : pos.scalar_type() == at::kInt ? 1 : 2;
    check(nf_rotary(ptr(x[0]), st[0][0], st[0][1], st[0][2], ptr(y[0]), heads[0], ptr(x[1]),
                    st[1][0], st[1][1], st[1][2], ptr(y[1]), heads[1], pos.data_ptr(),
                    shared ? 0 : T * axes, kind, B, T, like.size(3), sections, axes, base,
                    (int)call[0], (int)call[1], inverse, code_of(like), stream_of(like)),
          "nf_rotary");
    return {y[0], y[1]};
  }
  // the tensors that are there, turned; what_of: 1 q, 2 k, 3 both
  static variable_list forward(AutogradContext *ctx, const std::optional<Tensor> &q,
                               const std::optional<Tensor> &k, const Tensor &pos,
                               const std::vector<int64_t> &call, double base, bool inverse) {
    const c10::DeviceGuard guard(pos.device());
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({pos});
    ctx->saved_data["c"] = call;
    ctx->saved_data["b"] = base;
    ctx->saved_data["i"] = inverse;
    ctx->saved_data["q"] = q.has_value();
    ctx->saved_data["k"] = k.has_value();
    variable_list y = run(q ? *q : Tensor(), k ? *k : Tensor(), pos, call, base, inverse);
    variable_list there;
    for (Tensor &t : y)
      if (t.defined()) there.push_back(t);
    return there;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    // an argument that was left out has neither an output nor an edge
    const bool has[2] = {ctx->saved_data["q"].toBool(), ctx->saved_data["k"].toBool()};
    Tensor g[2];
    for (int i = 0, at = 0; i < 2; ++i) {
      if (!has[i]) continue;
      if (ctx->needs_input_grad(at)) g[i] = grads[at];
      ++at;
    }
    variable_list res(6);
    if (!g[0].defined() && !g[1].defined()) return res;
    const Tensor pos = ctx->get_saved_variables()[0].contiguous();  // a hook may have moved it
    const auto call = ctx->saved_data["c"].toIntVector();
    const double base = ctx->saved_data["b"].toDouble();
    const bool inverse = ctx->saved_data["i"].toBool();
    bool recording = false;
    for (const Tensor &t : g) {
      TORCH_CHECK_VALUE(!t.defined() || t.device() == pos.device(),
                        "fused_rotary backward: a gradient is not on the forward's device");
      recording |= at::GradMode::is_enabled() && t.defined() && t.requires_grad();
    }
    const c10::DeviceGuard guard(pos.device());
    if (!recording) {
      const variable_list y = run(g[0], g[1], pos, call, base, !inverse);
      res[0] = y[0];
      res[1] = y[1];
    } else {  // linear in the gradients
      auto given = [](const Tensor &v) {
        return v.defined() ? std::optional<Tensor>(v) : std::nullopt;
      };
      const variable_list y = Rotary::apply(given(g[0]), given(g[1]), pos, call, base, !inverse);
      size_t at = 0;
      for (int i = 0; i < 2; ++i)
        if (g[i].defined()) res[i] = y[at++];
    }
    return res;
  }
};

// ---------------------------------------------------------------------------
// entries
// ---------------------------------------------------------------------------
// The call's leading `n` arguments as tensors; false when one is not.
template <int N>
bool tensors(PyObject *const *args, Py_ssize_t nargs, Py_ssize_t want, Tensor (&t)[N]) {
  if (nargs != want) return false;
  for (int i = 0; i < N; ++i) {
    if (!THPVariable_CheckExact(args[i])) return false;  // a subclass may have its own rules
    t[i] = THPVariable_Unpack(args[i]);
  }
  return true;
}

// The call without the interpreter lock, which other threads take meanwhile (an
// allocation or a launch may wait); what calls into Python, such as a
// saved-tensor hook, takes it for itself.
template <class F>
auto unlocked(F &&f) {
  const pybind11::gil_scoped_release no_gil;
  return f();
}

PyObject *py_seam(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor a[6];
  if (!tensors(args, nargs, 8, a) || !quiet()) Py_RETURN_NONE;
  const int64_t t = PyLong_Check(args[6]) ? PyLong_AsLongLong(args[6]) : 0;
  const double eps = PyFloat_AsDouble(args[7]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!seam_plain(a[0], a[1], a[2], a[3], a[4], a[5], t)) Py_RETURN_NONE;
  const variable_list r =
      unlocked([&] { return Seam::apply(a[0], a[1], a[2], a[3], a[4], a[5], t, eps); });
  PyObject *h = THPVariable_Wrap(r[0]), *out = THPVariable_Wrap(r[1]);
  PyObject *pair = PyTuple_Pack(2, h, out);
  Py_XDECREF(h);
  Py_XDECREF(out);
  return pair;
  END_HANDLE_TH_ERRORS
}

PyObject *py_swiglu(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor t[2];
  if (!tensors(args, nargs, 2, t) || !quiet()) Py_RETURN_NONE;
  const c10::Device dev = t[0].device();
  if (!plain(t[0], dev) || !plain(t[1], dev) || t[0].sizes() != t[1].sizes() ||
      t[0].scalar_type() != t[1].scalar_type() || code_of(t[0]) < 0 || t[0].numel() == 0)
    Py_RETURN_NONE;
  return THPVariable_Wrap(unlocked([&] { return SwiGLU::apply(t[0], t[1]); }));
  END_HANDLE_TH_ERRORS
}

// x [M, D], w_gate, w_up [H, D]
PyObject *py_gate_up(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor t[3];
  if (!tensors(args, nargs, 3, t) || !quiet()) Py_RETURN_NONE;
  const c10::Device dev = t[0].device();
  for (const Tensor &v : t)
    if (!plain(v, dev) || code_of(v) < 0 || v.dim() != 2 || v.numel() == 0) Py_RETURN_NONE;
  if (t[1].sizes() != t[2].sizes() || t[0].size(1) != t[1].size(1)) Py_RETURN_NONE;
  if (!at::GradMode::is_enabled() ||
      !(t[0].requires_grad() || t[1].requires_grad() || t[2].requires_grad())) {
    // no backward: two of the three [M, H] outputs are not written
    return THPVariable_Wrap(unlocked([&] {
      const c10::DeviceGuard guard(dev);
      const at::NoGradGuard no_grad;
      Tensor a, b;
      return gate_up_forward(rows_bf16(t[0]), rows_bf16(t[1]), rows_bf16(t[2]), false, a, b);
    }));
  }
  return THPVariable_Wrap(unlocked([&] { return GateUp::apply(t[0], t[1], t[2]); }));
  END_HANDLE_TH_ERRORS
}

// hidden [M, D], lm_weight [V, D], targets [M], chunk rows, ignore index,
// compute type (0 fp32, 1 bf16)
PyObject *py_ce(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor t[3];
  if (!tensors(args, nargs, 6, t) || !quiet()) Py_RETURN_NONE;
  int64_t v[3];
  for (int i = 0; i < 3; ++i) {
    if (!PyLong_Check(args[3 + i])) Py_RETURN_NONE;  // the general path converts it
    v[i] = PyLong_AsLongLong(args[3 + i]);
  }
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const c10::Device dev = t[0].device();
  for (const Tensor &x : t)
    if (!plain(x, dev)) Py_RETURN_NONE;
  if (t[0].dim() != 2 || t[1].dim() != 2 || t[0].size(1) != t[1].size(1) || t[0].numel() == 0 ||
      t[1].numel() == 0 || t[2].dim() != 1 || t[2].size(0) != t[0].size(0) ||
      code_of(t[0]) < 0 || code_of(t[1]) < 0 || t[2].scalar_type() != at::kLong || v[0] <= 0)
    Py_RETURN_NONE;
  const at::ScalarType cdt = v[2] == NF_DTYPE_BF16 ? at::kBFloat16 : at::kFloat;
  return THPVariable_Wrap(unlocked(
      [&] { return ChunkedCE::apply(t[0], t[1], t[2], v[0], v[1], (int64_t)cdt); }));
  END_HANDLE_TH_ERRORS
}

bool wants_grad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Python ints from args[at ..]; false when one is not, or does not fit.
template <int N>
bool ints(PyObject *const *args, int at, int64_t (&v)[N]) {
  for (int i = 0; i < N; ++i) {
    if (!PyLong_CheckExact(args[at + i])) return false;
    v[i] = PyLong_AsLongLong(args[at + i]);
    if (v[i] == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
  }
  return true;
}

// hidden [M, D], lm_weight [V, D], targets [M], top_k, chunk rows, ignore index, compute type
// (0 fp32, 1 bf16) -> (logprobs, entropy, top_logprobs, top_ids)
PyObject *py_token_logprobs(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor t[3];
  int64_t v[4];
  if (!tensors(args, nargs, 7, t) || !quiet() || !ints(args, 3, v)) Py_RETURN_NONE;
  const c10::Device dev = t[0].device();
  for (const Tensor &x : t)
    if (!plain(x, dev)) Py_RETURN_NONE;
  if (t[0].dim() != 2 || t[1].dim() != 2 || t[0].size(1) != t[1].size(1) || t[0].numel() == 0 ||
      t[1].numel() == 0 || t[2].dim() != 1 || t[2].size(0) != t[0].size(0) ||
      code_of(t[0]) < 0 || code_of(t[1]) < 0 || t[2].scalar_type() != at::kLong || v[0] < 0 ||
      v[0] > 32 || v[0] > t[1].size(0) || v[1] <= 0)
    Py_RETURN_NONE;
  const at::ScalarType cdt = v[3] == NF_DTYPE_BF16 ? at::kBFloat16 : at::kFloat;
  const variable_list r = unlocked([&]() -> variable_list {
    if (wants_grad({&t[0], &t[1]}))
      return TokenLogprobs::apply(t[0], t[1], t[2], v[0], v[1], v[2], (int64_t)cdt);
    const c10::DeviceGuard guard(dev);
    const at::NoGradGuard no_grad;
    Tensor w, state;
    return TokenLogprobs::run(t[0], t[1], t[2], v[0], v[1], v[2], cdt, false, w, state);
  });
  PyObject *tuple = PyTuple_New(4);
  if (!tuple) return nullptr;
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(tuple, i, THPVariable_Wrap(r[i]));
  return tuple;
  END_HANDLE_TH_ERRORS
}

// ids, table [V, D], scale, padding id (-1: none), out's type (NF_DTYPE_*)
PyObject *py_embedding(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor t[2];
  if (!tensors(args, nargs, 5, t) || !quiet()) Py_RETURN_NONE;
  int64_t v[2];
  if (!PyFloat_CheckExact(args[2]) || !ints(args, 3, v)) Py_RETURN_NONE;
  const double scale = PyFloat_AS_DOUBLE(args[2]);
  const c10::Device dev = t[1].device();
  if (!plain(t[0], dev) || !plain(t[1], dev) || t[0].scalar_type() != at::kLong ||
      !t[0].is_contiguous() || t[0].numel() == 0 || t[1].dim() != 2 || t[1].numel() == 0 ||
      code_of(t[1]) < 0 || t[1].stride(1) != 1 || t[1].stride(0) < t[1].size(1))
    Py_RETURN_NONE;
  const at::ScalarType out_t = v[1] == NF_DTYPE_F32    ? at::kFloat
                               : v[1] == NF_DTYPE_BF16 ? at::kBFloat16
                                                       : at::kHalf;
  if (out_t != t[1].scalar_type() && t[1].scalar_type() != at::kFloat) Py_RETURN_NONE;
  return THPVariable_Wrap(unlocked([&]() -> Tensor {
    if (wants_grad({&t[1]})) return Embedding::apply(t[0], t[1], scale, v[0], (int64_t)out_t);
    const c10::DeviceGuard guard(dev);
    return Embedding::run(t[0], t[1], scale, out_t);
  }));
  END_HANDLE_TH_ERRORS
}

// x, residual or None, threshold, seed (int, or an int64 tensor of one element), offset
PyObject *py_dropout(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5 || !quiet() || !THPVariable_CheckExact(args[0])) Py_RETURN_NONE;
  const Tensor x = THPVariable_Unpack(args[0]);
  const c10::Device dev = x.device();
  Tensor r, seed_t;
  int64_t threshold[1], seed[1] = {0}, offset[1];
  if (args[1] != Py_None) {
    if (!THPVariable_CheckExact(args[1])) Py_RETURN_NONE;
    r = THPVariable_Unpack(args[1]);
    if (!plain(r, dev) || r.sizes() != x.sizes() ||
        (r.scalar_type() != x.scalar_type() && r.scalar_type() != at::kFloat))
      Py_RETURN_NONE;
  }
  if (THPVariable_CheckExact(args[3])) {
    seed_t = THPVariable_Unpack(args[3]);
    if (!plain(seed_t, dev) || seed_t.scalar_type() != at::kLong || seed_t.numel() != 1)
      Py_RETURN_NONE;
  } else if (!ints(args, 3, seed)) {
    Py_RETURN_NONE;
  }
  if (!plain(x, dev) || code_of(x) < 0 || x.numel() == 0 || !ints(args, 2, threshold) ||
      !ints(args, 4, offset) || threshold[0] < 0 || threshold[0] > 65536 || offset[0] < 0)
    Py_RETURN_NONE;
  const at::ScalarType out_t = r.defined() ? r.scalar_type() : x.scalar_type();
  auto given = [](const Tensor &v) { return v.defined() ? std::optional<Tensor>(v) : std::nullopt; };
  return THPVariable_Wrap(unlocked([&]() -> Tensor {
    if (wants_grad({&x, &r}))
      return Dropout::apply(x, given(r), given(seed_t), threshold[0], seed[0], offset[0],
                            (int64_t)out_t);
    const c10::DeviceGuard guard(dev);
    const Tensor rc = r.defined() ? r.contiguous() : r;
    return Dropout::run(x.contiguous(), rc, out_t, threshold[0], seed_t, seed[0], offset[0]);
  }));
  END_HANDLE_TH_ERRORS
}

// q [B, Tq, H, D], k, v [B, Tk, Hk, D], key_mask [B, Tk] or None, causal, scale
PyObject *py_attention(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor t[3], mask;
  if (!tensors(args, nargs, 6, t) || !quiet() || !PyFloat_CheckExact(args[5])) Py_RETURN_NONE;
  const c10::Device dev = t[0].device();
  for (const Tensor &x : t)
    if (!plain(x, dev) || x.dim() != 4 || x.numel() == 0 || code_of(x) < 0 ||
        x.scalar_type() != t[0].scalar_type())
      Py_RETURN_NONE;
  if (t[1].sizes() != t[2].sizes() || t[1].size(0) != t[0].size(0) ||
      t[1].size(3) != t[0].size(3) || t[0].size(2) % t[1].size(2) || t[0].size(3) > kMaxHead)
    Py_RETURN_NONE;
  if (args[3] != Py_None) {
    if (!THPVariable_CheckExact(args[3])) Py_RETURN_NONE;
    mask = THPVariable_Unpack(args[3]);
    if (!plain(mask, dev) || mask.scalar_type() != at::kBool || mask.dim() != 2 ||
        mask.size(0) != t[1].size(0) || mask.size(1) != t[1].size(1))
      Py_RETURN_NONE;
  }
  const bool causal = args[4] == Py_True;
  const double scale = PyFloat_AS_DOUBLE(args[5]);
  if (!(std::fabs(scale) <= 0x1p127)) Py_RETURN_NONE;
  return THPVariable_Wrap(unlocked([&]() -> Tensor {
    if (wants_grad({&t[0], &t[1], &t[2]}))
      return Attention::apply(t[0], t[1], t[2],
                              mask.defined() ? std::optional<Tensor>(mask) : std::nullopt, causal,
                              scale);
    const c10::DeviceGuard guard(dev);
    const at::NoGradGuard no_grad;
    Tensor state;
    return Attention::run(Attention::sizes(t[0], t[1]), head_rows(t[0]), head_rows(t[1]),
                          head_rows(t[2]), Attention::bytes_of(mask), causal, scale, false, state);
  }));
  END_HANDLE_TH_ERRORS
}

// q [B, T, H, D], k [B, T, Hk, D] or None, positions [B, T, axes] or [T, axes], sections (a tuple
// of ints), base, ladder, interleaved -> (q, k)
PyObject *py_rotary(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7 || !quiet() || !THPVariable_CheckExact(args[0]) ||
      !THPVariable_CheckExact(args[2]) || !PyTuple_CheckExact(args[3]) ||
      !PyFloat_CheckExact(args[4]) || !PyUnicode_CheckExact(args[5]))
    Py_RETURN_NONE;
  const Tensor q = THPVariable_Unpack(args[0]), pos = THPVariable_Unpack(args[2]);
  Tensor k;
  const c10::Device dev = q.device();
  if (!plain(q, dev) || q.dim() != 4 || q.numel() == 0 || code_of(q) < 0 || !plain(pos, dev) ||
      !pos.is_contiguous() || pos.requires_grad())
    Py_RETURN_NONE;
  const int64_t B = q.size(0), T = q.size(1), D = q.size(3);
  if (args[1] != Py_None) {
    if (!THPVariable_CheckExact(args[1])) Py_RETURN_NONE;
    k = THPVariable_Unpack(args[1]);
    if (!plain(k, dev) || k.dim() != 4 || k.numel() == 0 || k.scalar_type() != q.scalar_type() ||
        k.size(0) != B || k.size(1) != T || k.size(3) != D)
      Py_RETURN_NONE;
  }
  const Py_ssize_t axes = PyTuple_GET_SIZE(args[3]);
  if (axes < 1 || axes > 4) Py_RETURN_NONE;
  std::vector<int64_t> call(2 + axes);
  const bool joint = PyUnicode_CompareWithASCIIString(args[5], "joint") == 0;
  if (!joint && PyUnicode_CompareWithASCIIString(args[5], "axis") != 0) Py_RETURN_NONE;
  call[0] = joint;
  call[1] = args[6] == Py_True;
  int64_t pairs = 0;
  for (Py_ssize_t i = 0; i < axes; ++i) {
    PyObject *const o = PyTuple_GET_ITEM(args[3], i);
    if (!PyLong_CheckExact(o)) Py_RETURN_NONE;
    const int64_t n = PyLong_AsLongLong(o);
    if (n == -1 && PyErr_Occurred()) PyErr_Clear();
    if (n < 0 || n > kMaxPairs) Py_RETURN_NONE;
    call[2 + i] = n;
    pairs += n;
  }
  const double base = PyFloat_AS_DOUBLE(args[4]);
  const at::ScalarType pt = pos.scalar_type();
  if (pairs < 1 || pairs > kMaxPairs || 2 * pairs > D || D > kMaxTurned || !(base > 0.0) ||
      !std::isfinite(base) || (pt != at::kLong && pt != at::kInt && pt != at::kFloat) ||
      pos.dim() < 2 || pos.dim() > 3 || pos.size(-1) != axes || pos.size(-2) != T ||
      (pos.dim() == 3 && pos.size(0) != B && pos.size(0) != 1))
    Py_RETURN_NONE;
  const variable_list r = unlocked([&]() -> variable_list {
    if (wants_grad({&q, &k}))
      return Rotary::apply(std::optional<Tensor>(q),
                           k.defined() ? std::optional<Tensor>(k) : std::nullopt, pos, call, base,
                           false);
    const c10::DeviceGuard guard(dev);
    const at::NoGradGuard no_grad;
    return Rotary::run(q, k, pos, call, base, false);
  });
  PyObject *tuple = PyTuple_New(2);
  if (!tuple) return nullptr;
  for (int i = 0; i < 2; ++i)
    PyTuple_SET_ITEM(tuple, i, THPVariable_Wrap((size_t)i < r.size() ? r[i] : Tensor()));
  return tuple;
  END_HANDLE_TH_ERRORS
}

// op's name, the upstream gradients and the results of a backward in Python (tuples of tensors and
// Nones) -> the results under create_graph (see first_order_only above)
PyObject *py_first_order_only(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(nargs == 3 && PyUnicode_Check(args[0]) && PyTuple_Check(args[1]) &&
                       PyTuple_Check(args[2]),
                   "first_order_only: (name, gradients, results) expected");
  variable_list v[2];
  for (int k = 0; k < 2; ++k)
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[1 + k]); ++i) {
      PyObject *const o = PyTuple_GET_ITEM(args[1 + k], i);
      v[k].push_back(THPVariable_Check(o) ? THPVariable_Unpack(o) : Tensor());
    }
  const variable_list r = first_order_only(PyUnicode_AsUTF8(args[0]), true, v[0], v[1]);
  PyObject *tuple = PyTuple_New((Py_ssize_t)r.size());
  if (!tuple) return nullptr;
  for (size_t i = 0; i < r.size(); ++i) PyTuple_SET_ITEM(tuple, (Py_ssize_t)i, THPVariable_Wrap(r[i]));
  return tuple;
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"first_order_only", (PyCFunction)(void (*)(void))py_first_order_only, METH_FASTCALL, nullptr},
    {"seam", (PyCFunction)(void (*)(void))py_seam, METH_FASTCALL, nullptr},
    {"swiglu", (PyCFunction)(void (*)(void))py_swiglu, METH_FASTCALL, nullptr},
    {"gate_up", (PyCFunction)(void (*)(void))py_gate_up, METH_FASTCALL, nullptr},
    {"ce", (PyCFunction)(void (*)(void))py_ce, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void (*)(void))py_token_logprobs, METH_FASTCALL, nullptr},
    {"embedding", (PyCFunction)(void (*)(void))py_embedding, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))py_attention, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void (*)(void))py_rotary, METH_FASTCALL, nullptr},
    {"dropout", (PyCFunction)(void (*)(void))py_dropout, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&kModule); }
