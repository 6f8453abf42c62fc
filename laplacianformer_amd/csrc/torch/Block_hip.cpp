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

}  // namespace laplace
