// Host adapters of the transformer-block operators: shape, type and device checks, then
// the C ABI of include/laplacianformer_amd.h on the tensors' device and current stream; and
// their autograd nodes, in C++ because a small call's time is its host time (a training
// step of softmax attention at B2 H2 N196 d32: 89 us with nodes in Python).
#include "Block.h"

#include <ATen/ATen.h>
#include <torch/csrc/autograd/custom_function.h>

#include "torch_common.h"

namespace laplace {

namespace {

using at::Tensor;
using OptTensor = std::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// Rows of `width` elements at one stride: the tensor itself where its leading
// dimensions collapse, else a contiguous copy. Returns the row stride.
int64_t row_view(Tensor& t) {
  const int nd = (int)t.dim();
  const int64_t w = t.size(nd - 1);
  if (t.stride(nd - 1) != 1 && w != 1) t = t.contiguous();
  int64_t stride = 0, span = 1;
  for (int i = nd - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (span == 1) stride = t.stride(i);
    else if (t.stride(i) != stride * span) {
      t = t.contiguous();
      return w;
    }
    span *= t.size(i);
  }
  return span == 1 ? w : stride;
}

struct NormIn {
  Tensor x, res;
  int64_t xs = 0, rs = 0, rows = 0, width = 0;
  int dt = 0, wt = 0;
};

NormIn norm_in(const char* op, const Tensor& x, const Tensor& weight, const OptTensor& residual) {
  TORCH_CHECK(x.is_cuda(), op, ": tensors must be on GPU");
  TORCH_CHECK(x.dim() >= 1, op, ": x needs at least one dimension");
  NormIn n;
  n.dt = detail::abi_dtype(x, op);
  n.wt = detail::abi_dtype(weight, op);
  TORCH_CHECK(weight.is_cuda() && weight.device() == x.device(), op, ": weight must be on the same GPU as x");
  TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1), op, ": weight must have x's last size, ", x.size(-1));
  n.width = x.size(-1);
  n.rows = n.width ? x.numel() / n.width : 0;
  n.x = x;
  n.xs = row_view(n.x);
  if (given(residual)) {
    TORCH_CHECK(residual->sizes() == x.sizes(), op, ": residual and x must have the same shape");
    detail::same_type(x, *residual, "residual");
    n.res = *residual;
    n.rs = row_view(n.res);
  }
  return n;
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

const Tensor* if_given(const OptTensor& t) { return given(t) ? &*t : nullptr; }

// The kernels carry no tangents: a dual tensor's would be dropped, which says that the derivative is zero.
void no_tangent(const char* op, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t || !t->defined() || !t->_fw_grad(0).defined(), op, " has no forward-mode derivative");
}

}  // namespace

std::vector<Tensor> AddRmsNorm_forward(const Tensor x, const Tensor weight, const OptTensor residual, double eps,
                                       bool need_rstd) {
  const Tensor w = weight.contiguous();
  NormIn n = norm_in("add_rms_norm", x, weight, residual);
  at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options()), sum, rstd;
  if (n.res.defined()) sum = at::empty(x.sizes(), x.options());
  if (need_rstd) rstd = at::empty({n.rows}, x.options().dtype(at::kFloat));
  detail::check_status(lfamd_add_rms_norm(n.dt, ptr(n.x), n.xs, ptr(n.res), n.rs, n.wt, ptr(w), ptr(y), ptr(sum),
                                          (float*)ptr(rstd), n.rows, n.width, (float)eps, detail::stream_of(x)));
  return {y, sum.defined() ? sum : x, rstd};
}

std::vector<Tensor> AddRmsNorm_forward_fp8(const Tensor x, const Tensor weight, const OptTensor residual, double eps) {
  no_tangent("add_rms_norm_fp8", {&x, &weight, if_given(residual)});
  const Tensor w = weight.contiguous();
  NormIn n = norm_in("add_rms_norm_fp8", x, weight, residual);
  at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  std::vector<int64_t> ss(x.sizes().begin(), x.sizes().end());
  ss.back() = 1;
  Tensor y = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), scale = at::empty(ss, x.options().dtype(at::kFloat)), sum;
  if (n.res.defined()) sum = at::empty(x.sizes(), x.options());
  detail::check_status(lfamd_add_rms_norm_fp8(n.dt, ptr(n.x), n.xs, ptr(n.res), n.rs, n.wt, ptr(w), ptr(y),
                                              (float*)ptr(scale), ptr(sum), n.rows, n.width, (float)eps,
                                              detail::stream_of(x)));
  return {y, scale, sum.defined() ? sum : x};
}

std::vector<Tensor> AddRmsNorm_backward(const Tensor grad_y, const OptTensor grad_sum, const Tensor x,
                                        const Tensor weight, const OptTensor residual, const Tensor rstd, bool need_weight) {
  const char* op = "add_rms_norm backward";
  const Tensor w = weight.contiguous();
  NormIn n = norm_in(op, x, weight, residual);
  TORCH_CHECK(grad_y.sizes() == x.sizes(), op, ": grad_y and x must have the same shape");
  detail::same_type(x, grad_y, "grad_y");
  TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.numel() == n.rows && rstd.is_contiguous() && rstd.device() == x.device(),
              op, ": rstd must be the forward's");
  Tensor gy = grad_y, gs;
  const int64_t gys = row_view(gy);
  int64_t gss = 0;
  if (given(grad_sum)) {
    TORCH_CHECK(grad_sum->sizes() == x.sizes(), op, ": grad_sum and x must have the same shape");
    detail::same_type(x, *grad_sum, "grad_sum");
    gs = *grad_sum;
    gss = row_view(gs);
  }
  at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor dx = at::empty(x.sizes(), x.options()), dw, ws;
  size_t wsb = 0;
  if (need_weight) {
    dw = at::empty_like(w);
    wsb = lfamd_add_rms_norm_backward_workspace_size(n.dt, n.rows, n.width);
    ws = at::empty({(int64_t)wsb}, x.options().dtype(at::kByte));
  }
  detail::check_status(lfamd_add_rms_norm_backward(n.dt, ptr(gy), gys, ptr(gs), gss, ptr(n.x), n.xs, ptr(n.res), n.rs,
                                                   n.wt, ptr(w), rstd.data_ptr<float>(), ptr(dx), ptr(dw), n.rows,
                                                   n.width, ptr(ws), wsb, detail::stream_of(x)));
  return {dx, need_weight ? dw : Tensor()};
}

namespace {

struct GatedIn {
  NormIn n;
  Tensor w, wp, gate;
  lfamd_gated_norm d{};
};

GatedIn gated_in(const char* op, const Tensor& x, const Tensor& weight, const Tensor& residual, const OptTensor& post_weight,
                 const OptTensor& gate, double scale, double eps) {
  GatedIn in;
  in.w = weight.contiguous();
  in.n = norm_in(op, x, weight, residual);
  lfamd_gated_norm& d = in.d;
  d.rows = in.n.rows, d.width = in.n.width, d.x_stride = in.n.xs, d.residual_stride = in.n.rs;
  d.weight_dtype = in.n.wt, d.post_weight_dtype = d.gate_dtype = in.n.dt;
  d.scale = (float)scale, d.eps = (float)eps;
  if (given(post_weight)) {
    TORCH_CHECK(post_weight->is_cuda() && post_weight->device() == x.device(), op, ": post_weight must be on the same GPU as x");
    TORCH_CHECK(post_weight->dim() == 1 && post_weight->size(0) == x.size(-1), op, ": post_weight must have x's last size, ",
                x.size(-1));
    d.post_weight_dtype = detail::abi_dtype(*post_weight, op);
    in.wp = post_weight->contiguous();
  }
  if (given(gate)) {
    TORCH_CHECK(gate->is_cuda() && gate->device() == x.device(), op, ": gate must be on the same GPU as x");
    const int64_t nd = x.dim();
    int64_t same = 0;  // leading dimensions that the gate has in full; behind them it has ones
    bool fits = (gate->dim() == 1 || gate->dim() == nd) && gate->size(-1) == x.size(-1);
    if (fits && gate->dim() == nd) {
      while (same < nd - 1 && gate->size(same) == x.size(same)) ++same;
      for (int64_t i = same; i < nd - 1; ++i) fits = fits && gate->size(i) == 1;
    }
    TORCH_CHECK(fits, op, ": gate must be [", x.size(-1), "], or of x's dimensions with ones behind some of the leading ones, got ",
                gate->sizes(), " for x ", x.sizes());
    d.gate_dtype = detail::abi_dtype(*gate, op);
    in.gate = *gate;
    d.gate_stride = row_view(in.gate);
    if (same) {
      d.gate_rows = 1;
      for (int64_t i = same; i < nd - 1; ++i) d.gate_rows *= x.size(i);
    }
  }
  return in;
}

}  // namespace

std::vector<Tensor> GatedAddRmsNorm_forward(const Tensor x, const Tensor weight, const Tensor residual,
                                            const OptTensor post_weight, const OptTensor gate, double scale, double eps,
                                            bool need_rstd) {
  GatedIn in = gated_in("gated_add_rms_norm", x, weight, residual, post_weight, gate, scale, eps);
  at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options()), sum = at::empty(x.sizes(), x.options()), rstd, post;
  if (need_rstd) {
    rstd = at::empty({in.n.rows}, x.options().dtype(at::kFloat));
    if (in.wp.defined()) post = at::empty({in.n.rows}, x.options().dtype(at::kFloat));
  }
  detail::check_status(lfamd_gated_add_rms_norm(in.n.dt, &in.d, ptr(in.n.x), ptr(in.n.res), ptr(in.w), ptr(in.wp), ptr(in.gate),
                                                ptr(y), ptr(sum), (float*)ptr(rstd), (float*)ptr(post), detail::stream_of(x)));
  return {y, sum, rstd, post};
}

std::vector<Tensor> GatedAddRmsNorm_backward(const Tensor grad_y, const OptTensor grad_sum, const Tensor x, const Tensor weight,
                                             const Tensor residual, const OptTensor post_weight, const OptTensor gate,
                                             const Tensor rstd, const OptTensor post_rstd, double scale, double eps,
                                             bool need_weight, bool need_post_weight, bool need_gate) {
  const char* op = "gated_add_rms_norm backward";
  GatedIn in = gated_in(op, x, weight, residual, post_weight, gate, scale, eps);
  TORCH_CHECK(grad_y.sizes() == x.sizes(), op, ": grad_y and x must have the same shape");
  detail::same_type(x, grad_y, "grad_y");
  for (const Tensor* t : {&rstd, if_given(post_rstd)})
    TORCH_CHECK(t ? t->scalar_type() == at::kFloat && t->numel() == in.n.rows && t->is_contiguous() && t->device() == x.device()
                  : !in.wp.defined(),
                op, ": the statistics must be the forward's");
  Tensor gy = grad_y, gs;
  const int64_t gys = row_view(gy);
  int64_t gss = 0;
  if (given(grad_sum)) {
    TORCH_CHECK(grad_sum->sizes() == x.sizes(), op, ": grad_sum and x must have the same shape");
    detail::same_type(x, *grad_sum, "grad_sum");
    gs = *grad_sum;
    gss = row_view(gs);
  }
  at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor dx = at::empty(x.sizes(), x.options()), dr = at::empty(x.sizes(), x.options()), dw, dwp, dg;
  if (need_weight) dw = at::empty(in.w.sizes(), in.w.options());
  if (need_post_weight) dwp = at::empty(in.wp.sizes(), in.wp.options());
  if (need_gate) dg = in.n.rows ? at::empty(gate->sizes(), gate->options()) : at::zeros(gate->sizes(), gate->options());
  const size_t wsb = lfamd_gated_add_rms_norm_backward_workspace_size(in.n.dt, &in.d);
  const Tensor ws = at::empty({(int64_t)wsb}, x.options().dtype(at::kByte));
  detail::check_status(lfamd_gated_add_rms_norm_backward(in.n.dt, &in.d, ptr(gy), gys, ptr(gs), gss, ptr(in.n.x), ptr(in.n.res),
                                                         ptr(in.w), ptr(in.wp), ptr(in.gate), rstd.data_ptr<float>(),
                                                         given(post_rstd) ? post_rstd->data_ptr<float>() : nullptr, ptr(dx), ptr(dr),
                                                         ptr(dw), ptr(dwp), in.n.rows ? ptr(dg) : nullptr, ptr(ws), wsb,
                                                         detail::stream_of(x)));
  return {dx, dr, dw, dwp, dg};
}

namespace {

// [B, heads, tokens, channels] with adjacent channels.
Tensor unit_last(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// An output in t's order of dimensions, its channels adjacent: empty_like alone takes the channels of windows
// into one row (tokens and channels both one element apart, fewer tokens than channels) for the outer dimension.
Tensor output_like(const Tensor& t) {
  const Tensor out = at::empty_like(t);
  return out.size(-1) <= 1 || out.stride(-1) == 1 ? out : at::empty(t.sizes(), t.options());
}

}  // namespace

std::vector<Tensor> Rotary(const Tensor q, const OptTensor k, const Tensor positions, const std::vector<int64_t> sections,
                           double base, bool interleaved, bool inverse) {
  const char* op = "rotary";
  TORCH_CHECK(q.is_cuda(), op, ": tensors must be on GPU");
  TORCH_CHECK(q.dim() == 4, op, ": q must be [batch, heads, tokens, channels]");
  const int dt = detail::abi_dtype(q, op);
  const int64_t B = q.size(0), N = q.size(2), D = q.size(3);
  const bool has_k = given(k);
  if (has_k) {
    TORCH_CHECK(k->dim() == 4 && k->size(0) == B && k->size(2) == N && k->size(3) == D, op,
                ": q and k may differ in their heads only, got ", q.sizes(), " and ", k->sizes());
    detail::same_type(q, *k, "k");
  }
  const int64_t A = (int64_t)sections.size();
  TORCH_CHECK(positions.is_cuda() && positions.device() == q.device(), op, ": positions must be on the same GPU as q");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, op,
              ": positions must be int32 or int64");
  TORCH_CHECK((positions.dim() == 2 && positions.size(0) == A && positions.size(1) == N) ||
                  (positions.dim() == 3 && positions.size(0) == A && positions.size(1) == B && positions.size(2) == N),
              op, ": positions must be [axes, tokens] or [axes, batch, tokens] with ", A, " axes and ", N, " tokens, got ",
              positions.sizes());
  const int64_t ps[3] = {positions.stride(0), positions.dim() == 3 ? positions.stride(1) : 0, positions.stride(-1)};
  at::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const Tensor qi = unit_last(q), ki = has_k ? unit_last(*k) : Tensor();
  Tensor qo = output_like(qi), ko = has_k ? output_like(ki) : Tensor();
  detail::check_status(lfamd_rotary(dt, ptr(qi), qi.strides().data(), ptr(qo), qo.strides().data(), q.size(1), ptr(ki),
                                    has_k ? ki.strides().data() : nullptr, ptr(ko), has_k ? ko.strides().data() : nullptr,
                                    has_k ? k->size(1) : 0, B, N, D, ptr(positions), positions.scalar_type() == at::kLong,
                                    ps, (int)A, sections.data(), base, interleaved, inverse, detail::stream_of(q)));
  return {qo, ko};
}

namespace {

struct AttnIn {
  Tensor q, k, v, mask;
  lfamd_attention d{};
  int dt = 0;
};

const int32_t* per_batch(const char* op, const Tensor& q, const OptTensor& t, const char* name) {
  if (!given(t)) return nullptr;
  TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == q.size(0) && t->is_contiguous(), op, ": ", name,
              " must be a contiguous int32 tensor of one value per sequence");
  TORCH_CHECK(t->is_cuda() && t->device() == q.device(), op, ": ", name, " must be on the same GPU as q");
  return t->data_ptr<int32_t>();
}

void set_strides(int64_t* to, const Tensor& t) {
  for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

AttnIn attn_in(const char* op, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& mask, bool causal,
               const OptTensor& k_lengths, const OptTensor& q_lengths, const OptTensor& q_starts, double scale) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), op, ": tensors must be on GPU");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, op, ": q, k and v must be [batch, heads, tokens, channels]");
  AttnIn in;
  in.dt = detail::abi_dtype(q, op);
  detail::same_type(q, k, "k");
  detail::same_type(q, v, "v");
  TORCH_CHECK(k.sizes() == v.sizes(), op, ": k and v must have the same shape, got ", k.sizes(), " and ", v.sizes());
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3), op, ": q ", q.sizes(), " and k ", k.sizes(),
              " differ in batch or channels");
  in.q = unit_last(q), in.k = unit_last(k), in.v = unit_last(v);
  lfamd_attention& d = in.d;
  d.batch = q.size(0), d.heads = q.size(1), d.kv_heads = k.size(1), d.q_len = q.size(2), d.k_len = k.size(2);
  d.head_dim = q.size(3);
  set_strides(d.q_strides, in.q);
  set_strides(d.k_strides, in.k);
  set_strides(d.v_strides, in.v);
  d.k_lengths = per_batch(op, q, k_lengths, "k_lengths");
  d.q_lengths = per_batch(op, q, q_lengths, "q_lengths");
  d.q_starts = per_batch(op, q, q_starts, "q_starts");
  if (given(mask)) {
    TORCH_CHECK(mask->is_cuda() && mask->device() == q.device(), op, ": mask must be on the same GPU as q");
    switch (mask->scalar_type()) {
      case at::kBool: d.mask_kind = LFAMD_MASK_BOOL; break;
      case at::kFloat: d.mask_kind = LFAMD_MASK_F32; break;
      case at::kHalf: d.mask_kind = LFAMD_MASK_F16; break;
      case at::kBFloat16: d.mask_kind = LFAMD_MASK_BF16; break;
      default: TORCH_CHECK(false, op, ": mask must be bool, float32, float16 or bfloat16");
    }
    const int64_t full[4] = {d.batch, d.heads, d.q_len, d.k_len};
    TORCH_CHECK(mask->dim() <= 4, op, ": mask must broadcast to [batch, heads, queries, keys]");
    for (int i = 0; i < 4; ++i) {
      const int j = i - (4 - (int)mask->dim());
      const int64_t size = j < 0 ? 1 : mask->size(j);
      TORCH_CHECK(size == full[i] || size == 1, op, ": mask ", mask->sizes(), " does not broadcast to [", d.batch, ", ", d.heads,
                  ", ", d.q_len, ", ", d.k_len, "]");
      d.mask_strides[i] = size == 1 ? 0 : mask->stride(j);
    }
    in.mask = *mask;
    d.mask = mask->data_ptr();
  }
  d.causal = causal;
  d.scale = (float)scale;
  return in;
}

}  // namespace

std::vector<Tensor> SoftmaxAttention_forward(const Tensor q, const Tensor k, const Tensor v, const OptTensor mask,
                                             bool causal, const OptTensor k_lengths, const OptTensor q_lengths,
                                             const OptTensor q_starts, double scale, bool need_stats) {
  AttnIn in = attn_in("softmax_attention", q, k, v, mask, causal, k_lengths, q_lengths, q_starts, scale);
  at::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor out = output_like(in.q), stats, ws;
  set_strides(in.d.out_strides, out);
  if (need_stats)
    stats = at::empty({(int64_t)lfamd_softmax_attention_stats_size(in.dt, &in.d) / 4}, q.options().dtype(at::kFloat));
  const size_t wsb = lfamd_softmax_attention_workspace_size(in.dt, &in.d);
  if (wsb) ws = at::empty({(int64_t)wsb}, q.options().dtype(at::kByte));
  detail::check_status(lfamd_softmax_attention(in.dt, &in.d, ptr(in.q), ptr(in.k), ptr(in.v), ptr(out),
                                               (float*)ptr(stats), ptr(ws), wsb, detail::stream_of(q)));
  return {out, stats};
}

std::vector<Tensor> SoftmaxAttention_backward(const Tensor grad_out, const Tensor q, const Tensor k, const Tensor v,
                                              const Tensor out, const Tensor stats, const OptTensor mask, bool causal,
                                              const OptTensor k_lengths, const OptTensor q_lengths,
                                              const OptTensor q_starts, double scale, bool need_q, bool need_kv) {
  const char* op = "softmax_attention backward";
  AttnIn in = attn_in(op, q, k, v, mask, causal, k_lengths, q_lengths, q_starts, scale);
  TORCH_CHECK(grad_out.sizes() == q.sizes() && out.sizes() == q.sizes(), op, ": grad_out, out and q must have the same shape");
  detail::same_type(q, grad_out, "grad_out");
  detail::same_type(q, out, "out");
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.device() == q.device() &&
                  stats.numel() * 4 == (int64_t)lfamd_softmax_attention_stats_size(in.dt, &in.d),
              op, ": stats must be the forward's");
  at::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const Tensor o = unit_last(out), g = unit_last(grad_out);
  set_strides(in.d.out_strides, o);
  Tensor dq, dk, dv;
  lfamd_attention_grads gr{};
  if (need_q) dq = output_like(in.q);
  if (need_kv) dk = output_like(in.k), dv = output_like(in.v);
  gr.grad_out = ptr(g);
  set_strides(gr.grad_out_strides, g);
  if (need_q) gr.grad_q = ptr(dq), set_strides(gr.grad_q_strides, dq);
  if (need_kv) {
    gr.grad_k = ptr(dk), gr.grad_v = ptr(dv);
    set_strides(gr.grad_k_strides, dk);
    set_strides(gr.grad_v_strides, dv);
  }
  const size_t wsb = lfamd_softmax_attention_backward_workspace_size(in.dt, &in.d);
  const Tensor ws = at::empty({(int64_t)wsb}, q.options().dtype(at::kByte));
  detail::check_status(lfamd_softmax_attention_backward(in.dt, &in.d, ptr(in.q), ptr(in.k), ptr(in.v), ptr(o),
                                                        stats.data_ptr<float>(), &gr, ptr(ws), wsb, detail::stream_of(q)));
  return {dq, dk, dv};
}

namespace {

struct DecayIn {
  Tensor q, k, v, state;
  lfamd_decay d{};
  int dt = 0;
};

void check_state(const char* op, const Tensor& q, const Tensor& t, const lfamd_decay& d, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), op, ": ", name, " must be on the same GPU as q");
  TORCH_CHECK(t.scalar_type() == at::kFloat, op, ": ", name, " must be float32");
  TORCH_CHECK(t.dim() == 4 && t.size(0) == d.batch && t.size(1) == d.heads && t.size(2) == d.key_dim && t.size(3) == d.value_dim,
              op, ": ", name, " must be [", d.batch, ", ", d.heads, ", ", d.key_dim, ", ", d.value_dim, "], got ", t.sizes());
}

DecayIn decay_in(const char* op, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                 const OptTensor& state, const OptTensor& lengths, double scale) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), op, ": tensors must be on GPU");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, op, ": q, k and v must be [batch, heads, tokens, channels]");
  DecayIn in;
  in.dt = detail::abi_dtype(q, op);
  detail::same_type(q, k, "k");
  detail::same_type(q, v, "v");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2) && k.size(3) == q.size(3), op, ": q ", q.sizes(), " and k ",
              k.sizes(), " may differ in their heads only");
  TORCH_CHECK(v.size(0) == k.size(0) && v.size(1) == k.size(1) && v.size(2) == k.size(2), op, ": k ", k.sizes(), " and v ",
              v.sizes(), " may differ in their channels only");
  TORCH_CHECK(log_decay.scalar_type() == at::kFloat && log_decay.dim() == 1 && log_decay.size(0) == q.size(1) &&
                  log_decay.is_contiguous(),
              op, ": log_decay must be a contiguous float32 tensor of one value per query head");
  TORCH_CHECK(log_decay.is_cuda() && log_decay.device() == q.device(), op, ": log_decay must be on the same GPU as q");
  in.q = unit_last(q), in.k = unit_last(k), in.v = unit_last(v);
  lfamd_decay& d = in.d;
  d.batch = q.size(0), d.heads = q.size(1), d.kv_heads = k.size(1), d.tokens = q.size(2), d.key_dim = q.size(3);
  d.value_dim = v.size(3);
  set_strides(d.q_strides, in.q);
  set_strides(d.k_strides, in.k);
  set_strides(d.v_strides, in.v);
  d.log_decay = log_decay.data_ptr<float>();
  d.lengths = per_batch(op, q, lengths, "lengths");
  d.scale = (float)scale;
  if (given(state)) {
    check_state(op, q, *state, d, "state");
    in.state = state->contiguous();
  }
  return in;
}

// The values' channels in q's order of dimensions.
Tensor decay_output(const DecayIn& in) {
  if (in.d.key_dim == in.d.value_dim) return output_like(in.q);
  const bool tokens_first = in.q.dim() == 4 && in.q.stride(1) < in.q.stride(2);
  const auto o = in.q.options();
  return tokens_first ? at::empty({in.d.batch, in.d.tokens, in.d.heads, in.d.value_dim}, o).transpose(1, 2)
                      : at::empty({in.d.batch, in.d.heads, in.d.tokens, in.d.value_dim}, o);
}

}  // namespace

std::vector<Tensor> DecayAttention_forward(const Tensor q, const Tensor k, const Tensor v, const Tensor log_decay,
                                           const OptTensor state, const OptTensor lengths, double scale, bool need_last) {
  DecayIn in = decay_in("decay_attention", q, k, v, log_decay, state, lengths, scale);
  at::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor out = decay_output(in), last, ws;
  set_strides(in.d.out_strides, out);
  if (need_last) last = at::empty({in.d.batch, in.d.heads, in.d.key_dim, in.d.value_dim}, q.options().dtype(at::kFloat));
  const size_t wsb = lfamd_decay_attention_workspace_size(in.dt, &in.d);
  if (wsb) ws = at::empty({(int64_t)wsb}, q.options().dtype(at::kByte));
  detail::check_status(lfamd_decay_attention(in.dt, &in.d, ptr(in.q), ptr(in.k), ptr(in.v), (const float*)ptr(in.state), ptr(out),
                                             (float*)ptr(last), ptr(ws), wsb, detail::stream_of(q)));
  return {out, last};
}

std::vector<Tensor> DecayAttention_backward(const OptTensor grad_out, const OptTensor grad_last, const Tensor q, const Tensor k,
                                            const Tensor v, const Tensor log_decay, const OptTensor state,
                                            const OptTensor lengths, double scale, bool need_q, bool need_kv, bool need_state) {
  const char* op = "decay_attention backward";
  DecayIn in = decay_in(op, q, k, v, log_decay, state, lengths, scale);
  const lfamd_decay& d = in.d;
  at::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor g, gl;
  if (given(grad_out)) {
    TORCH_CHECK(grad_out->dim() == 4 && grad_out->size(0) == d.batch && grad_out->size(1) == d.heads &&
                    grad_out->size(2) == d.tokens && grad_out->size(3) == d.value_dim,
                op, ": grad_out must have the output's shape");
    detail::same_type(q, *grad_out, "grad_out");
    g = unit_last(*grad_out);
  } else {
    g = at::zeros({d.batch, d.heads, d.tokens, d.value_dim}, q.options());
  }
  if (given(grad_last)) {
    check_state(op, q, *grad_last, d, "the last state's gradient");
    gl = grad_last->contiguous();
  }
  need_kv = need_kv || need_state;
  Tensor dq, dk, dv, ds;
  lfamd_decay_grads gr{};
  gr.grad_out = ptr(g), gr.grad_last_state = (const float*)ptr(gl);
  set_strides(gr.grad_out_strides, g);
  if (need_q) {
    dq = output_like(in.q);
    gr.grad_q = ptr(dq), set_strides(gr.grad_q_strides, dq);
  }
  if (need_kv) {
    dk = output_like(in.k), dv = output_like(in.v);
    gr.grad_k = ptr(dk), gr.grad_v = ptr(dv);
    set_strides(gr.grad_k_strides, dk);
    set_strides(gr.grad_v_strides, dv);
  }
  if (need_state) {
    ds = at::empty({d.batch, d.heads, d.key_dim, d.value_dim}, q.options().dtype(at::kFloat));
    gr.grad_state = (float*)ptr(ds);
  }
  const size_t wsb = lfamd_decay_attention_backward_workspace_size(in.dt, &in.d);
  const Tensor ws = at::empty({(int64_t)wsb}, q.options().dtype(at::kByte));
  detail::check_status(lfamd_decay_attention_backward(in.dt, &in.d, ptr(in.q), ptr(in.k), ptr(in.v), (const float*)ptr(in.state),
                                                      &gr, ptr(ws), wsb, detail::stream_of(q)));
  return {dq, dk, dv, ds};
}

Tensor DecayAttentionStep(const Tensor q, const Tensor k, const Tensor v, const Tensor log_decay, const Tensor state,
                          double scale) {
  const char* op = "decay_attention_step";
  no_tangent(op, {&q, &k, &v, &log_decay, &state});
  DecayIn in = decay_in(op, q, k, v, log_decay, std::nullopt, std::nullopt, scale);
  const lfamd_decay& d = in.d;
  TORCH_CHECK(d.tokens == 1, op, ": takes one token, not ", d.tokens);
  check_state(op, q, state, d, "state");
  const int64_t size = d.key_dim * d.value_dim, sb = state.stride(0), sh = state.stride(1);
  TORCH_CHECK(state.numel() == 0 || ((d.value_dim == 1 || state.stride(3) == 1) && (d.key_dim == 1 || state.stride(2) == d.value_dim)),
              op, ": each head's state must be contiguous");
  TORCH_CHECK((d.heads <= 1 || sh >= size) && (d.batch <= 1 || sb >= size) &&
                  (d.heads <= 1 || d.batch <= 1 || sb >= d.heads * sh || sh >= d.batch * sb),
              op, ": the states of sequences or heads overlap");
  at::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor out = decay_output(in);
  set_strides(in.d.out_strides, out);
  const int64_t ss[2] = {sb, sh};
  state.unsafeGetTensorImpl()->bump_version();
  detail::check_status(lfamd_decay_attention_step(in.dt, &in.d, ptr(in.q), ptr(in.k), ptr(in.v), ptr(out), (float*)ptr(state), ss,
                                                  detail::stream_of(q)));
  return out;
}

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The backward passes are kernels without a derivative of their own.
void once(const char* op, const variable_list& grads) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, " has no second derivative: call backward without create_graph");
  for (const Tensor& g : grads) no_tangent(op, {&g});
}

struct AddRmsNormNode : torch::autograd::Function<AddRmsNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual,
                               double eps) {
    ctx->set_materialize_grads(false);
    const auto r = AddRmsNorm_forward(x, weight, residual, eps, true);
    // In 16-bit types the addends, whose sum has not been rounded; in fp32 the sum, one tensor less.
    const bool addends = given(residual) && x.element_size() == 2;
    ctx->save_for_backward({addends ? x : r[1], weight, r[2], addends ? *residual : Tensor()});
    if (given(residual)) return {r[0], r[1]};
    return {r[0]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("add_rms_norm", g);
    const auto saved = ctx->get_saved_variables();
    const Tensor gs = g.size() > 1 ? g[1] : Tensor();
    if (!g[0].defined() && !gs.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor gy = g[0].defined() ? g[0] : at::zeros_like(saved[0]);
    const auto d = AddRmsNorm_backward(gy, gs.defined() ? OptTensor(gs) : std::nullopt, saved[0], saved[1],
                                       saved[3].defined() ? OptTensor(saved[3]) : std::nullopt, saved[2],
                                       ctx->needs_input_grad(1));
    return {d[0], d[1], g.size() > 1 ? d[0] : Tensor(), Tensor()};
  }
};

struct GatedAddRmsNormNode : torch::autograd::Function<GatedAddRmsNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& residual,
                               const OptTensor& post_weight, const OptTensor& gate, double scale, double eps) {
    ctx->set_materialize_grads(false);
    const auto r = GatedAddRmsNorm_forward(x, weight, residual, post_weight, gate, scale, eps, true);
    auto or_none = [](const OptTensor& t) { return given(t) ? *t : Tensor(); };
    ctx->save_for_backward({x, weight, residual, or_none(post_weight), or_none(gate), r[2], r[3]});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("gated_add_rms_norm", g);
    variable_list out(7);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    const Tensor gy = g[0].defined() ? g[0] : at::zeros_like(s[0]);
    const size_t gate_at = s[3].defined() ? 4 : 3;  // needs_input_grad counts the tensors that are given
    const auto d = GatedAddRmsNorm_backward(gy, opt(g[1]), s[0], s[1], s[2], opt(s[3]), opt(s[4]), s[5], opt(s[6]),
                                            ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble(),
                                            ctx->needs_input_grad(1), s[3].defined() && ctx->needs_input_grad(3),
                                            s[4].defined() && ctx->needs_input_grad(gate_at));
    out[0] = d[0], out[1] = d[2], out[2] = d[1], out[3] = d[3], out[4] = d[4];
    return out;
  }
};

struct RotaryNode : torch::autograd::Function<RotaryNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions,
                               std::vector<int64_t> sections, double base, bool interleaved) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["base"] = base;
    ctx->saved_data["interleaved"] = interleaved;
    auto r = Rotary(q, k, positions, sections, base, interleaved, false);
    if (!given(k)) r.pop_back();
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("rotary", g);
    const Tensor positions = ctx->get_saved_variables()[0];
    const auto sections = ctx->saved_data["sections"].toIntVector();
    const double base = ctx->saved_data["base"].toDouble();
    const bool inter = ctx->saved_data["interleaved"].toBool();
    variable_list out(6);
    const bool has_k = g.size() > 1 && g[1].defined();
    if (g[0].defined()) {
      const auto r = Rotary(g[0], has_k ? OptTensor(g[1]) : std::nullopt, positions, sections, base, inter, true);
      out[0] = r[0], out[1] = r[1];
    } else if (has_k) {
      out[1] = Rotary(g[1], std::nullopt, positions, sections, base, inter, true)[0];
    }
    return out;
  }
};

struct SoftmaxAttentionNode : torch::autograd::Function<SoftmaxAttentionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& mask,
                        bool causal, const OptTensor& k_lengths, const OptTensor& q_lengths, const OptTensor& q_starts,
                        double scale) {
    const auto r = SoftmaxAttention_forward(q, k, v, mask, causal, k_lengths, q_lengths, q_starts, scale, true);
    auto or_none = [](const OptTensor& t) { return given(t) ? *t : Tensor(); };
    ctx->save_for_backward({q, k, v, r[0], r[1], or_none(mask), or_none(k_lengths), or_none(q_lengths), or_none(q_starts)});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("softmax_attention", g);
    const auto s = ctx->get_saved_variables();
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    const bool need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2);
    const auto d = SoftmaxAttention_backward(g[0], s[0], s[1], s[2], s[3], s[4], opt(s[5]), ctx->saved_data["causal"].toBool(),
                                             opt(s[6]), opt(s[7]), opt(s[8]), ctx->saved_data["scale"].toDouble(),
                                             ctx->needs_input_grad(0), need_k || need_v);
    variable_list out(9);
    out[0] = d[0];
    if (need_k) out[1] = d[1];
    if (need_v) out[2] = d[2];
    return out;
  }
};

struct DecayAttentionNode : torch::autograd::Function<DecayAttentionNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                               const OptTensor& state, const OptTensor& lengths, double scale, bool return_state) {
    ctx->set_materialize_grads(false);
    auto r = DecayAttention_forward(q, k, v, log_decay, state, lengths, scale, return_state);
    auto or_none = [](const OptTensor& t) { return given(t) ? *t : Tensor(); };
    ctx->save_for_backward({q, k, v, log_decay, or_none(state), or_none(lengths)});
    ctx->saved_data["scale"] = scale;
    if (!return_state) r.pop_back();
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("decay_attention", g);
    const auto s = ctx->get_saved_variables();
    auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    variable_list out(8);
    const Tensor gl = g.size() > 1 ? g[1] : Tensor();
    if (!g[0].defined() && !gl.defined()) return out;
    const bool need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2);
    const bool need_s = s[4].defined() && ctx->needs_input_grad(4);
    const auto d = DecayAttention_backward(opt(g[0]), opt(gl), s[0], s[1], s[2], s[3], opt(s[4]), opt(s[5]),
                                           ctx->saved_data["scale"].toDouble(), ctx->needs_input_grad(0), need_k || need_v, need_s);
    out[0] = d[0];
    if (need_k) out[1] = d[1];
    if (need_v) out[2] = d[2];
    out[4] = d[3];
    return out;
  }
};

bool records(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}

}  // namespace

std::vector<Tensor> AddRmsNorm(const Tensor x, const Tensor weight, const OptTensor residual, double eps) {
  no_tangent("add_rms_norm", {&x, &weight, if_given(residual)});
  if (records({&x, &weight, if_given(residual)})) return AddRmsNormNode::apply(x, weight, residual, eps);
  auto r = AddRmsNorm_forward(x, weight, residual, eps, false);
  r.resize(given(residual) ? 2 : 1);
  return r;
}

std::vector<Tensor> GatedAddRmsNorm(const Tensor x, const Tensor weight, const Tensor residual, const OptTensor post_weight,
                                    const OptTensor gate, double scale, double eps) {
  no_tangent("gated_add_rms_norm", {&x, &weight, &residual, if_given(post_weight), if_given(gate)});
  if (records({&x, &weight, &residual, if_given(post_weight), if_given(gate)}))
    return GatedAddRmsNormNode::apply(x, weight, residual, post_weight, gate, scale, eps);
  auto r = GatedAddRmsNorm_forward(x, weight, residual, post_weight, gate, scale, eps, false);
  r.resize(2);
  return r;
}

std::vector<Tensor> RotaryPositions(const Tensor q, const OptTensor k, const Tensor positions,
                                    const std::vector<int64_t> sections, double base, bool interleaved) {
  no_tangent("rotary", {&q, if_given(k)});
  if (records({&q, if_given(k)})) {
    auto r = RotaryNode::apply(q, k, positions, sections, base, interleaved);
    r.resize(2);
    return r;
  }
  return Rotary(q, k, positions, sections, base, interleaved, false);
}

Tensor SoftmaxAttention(const Tensor q, const Tensor k, const Tensor v, const OptTensor mask, bool causal,
                        const OptTensor k_lengths, const OptTensor q_lengths, const OptTensor q_starts, double scale) {
  TORCH_CHECK(!given(mask) || !mask->requires_grad(), "softmax_attention: the mask has no gradient");
  no_tangent("softmax_attention", {&q, &k, &v, if_given(mask)});
  if (records({&q, &k, &v}))
    return SoftmaxAttentionNode::apply(q, k, v, mask, causal, k_lengths, q_lengths, q_starts, scale);
  return SoftmaxAttention_forward(q, k, v, mask, causal, k_lengths, q_lengths, q_starts, scale, false)[0];
}

std::vector<Tensor> DecayAttention(const Tensor q, const Tensor k, const Tensor v, const Tensor log_decay, const OptTensor state,
                                   const OptTensor lengths, double scale, bool return_state) {
  TORCH_CHECK(!records({&log_decay}), "decay_attention: log_decay has no gradient");
  no_tangent("decay_attention", {&q, &k, &v, &log_decay, if_given(state)});
  if (records({&q, &k, &v, if_given(state)}))
    return DecayAttentionNode::apply(q, k, v, log_decay, state, lengths, scale, return_state);
  auto r = DecayAttention_forward(q, k, v, log_decay, state, lengths, scale, return_state);
  if (!return_state) r.pop_back();
  return r;
}

}  // namespace laplace
