// C entries of softmax_attention: argument checks, and the call as the kernels take it.
#include <math.h>

#include <algorithm>

#include "attn_common.h"

namespace lfamd {

namespace {

constexpr int64_t kMostRows = (int64_t)1 << 29;  // sums of a query's and a key's position stay 32-bit

// How a streamed tensor is read (LoadMode): by the alignment of every row's start and end, for row
// strides that keep a tile of at most 128 rows within 2^31 bytes.
int load_mode(const void* p, const int64_t* strides, int64_t d, int64_t size, bool keyMask) {
  auto all = [&](int64_t bytes) {
    return (int64_t)((uintptr_t)p % bytes) == 0 && d * size % bytes == 0 && strides[0] * size % bytes == 0 &&
           strides[1] * size % bytes == 0 && strides[2] * size % bytes == 0;
  };
  if (strides[2] < 0 || strides[2] >= ((int64_t)1 << 22)) return kPlain;
  return all(16) ? kAsync : all(4) && !keyMask ? kAsync4 : kPlain;
}

// Sizes, types and what else needs no tensor pointer. *empty: there is no head.
int check_desc(const char* who, int dtype, const lfamd_attention* d, bool* empty) {
  if (dtype != LFAMD_F32 && dtype != LFAMD_F16 && dtype != LFAMD_BF16)
    return fail(LFAMD_ERR_DTYPE, "%s: unsupported dtype %d", who, dtype);
  if (!d) return fail(LFAMD_ERR_ARG, "%s: null description", who);
  if (d->batch < 0 || d->heads < 0 || d->kv_heads < 0 || d->q_len < 0 || d->k_len < 0 || d->head_dim < 0)
    return fail(LFAMD_ERR_ARG, "%s: negative size", who);
  if (d->head_dim < 1 || d->head_dim > 128)
    return fail(LFAMD_ERR_UNSUPPORTED, "%s: head size %lld is outside 1 .. 128", who, (long long)d->head_dim);
  if (d->heads ? !d->kv_heads || d->heads % d->kv_heads : d->kv_heads)
    return fail(LFAMD_ERR_ARG, "%s: %lld query heads do not share %lld key heads evenly", who, (long long)d->heads,
                (long long)d->kv_heads);
  if (!(d->scale > 0.0f) || !isfinite(d->scale)) return fail(LFAMD_ERR_ARG, "%s: scale must be positive and finite", who);
  if (d->mask_kind < LFAMD_MASK_NONE || d->mask_kind > LFAMD_MASK_BF16)
    return fail(LFAMD_ERR_ARG, "%s: unknown mask kind %d", who, d->mask_kind);
  const int64_t g = d->kv_heads ? d->heads / d->kv_heads : 0;
  if (d->q_len > kMostRows || d->k_len > kMostRows || (g && d->q_len > kMostRows / g))
    return fail(LFAMD_ERR_UNSUPPORTED, "%s: at most 2^29 keys, and queries per key head, are taken", who);
  if (d->batch > INT32_MAX || d->heads > INT32_MAX || (d->heads && d->batch > INT32_MAX / d->heads))
    return fail(LFAMD_ERR_UNSUPPORTED, "%s: batch * heads must be below 2^31", who);
  *empty = d->batch == 0 || d->heads == 0;
  return LFAMD_OK;
}

AttnArgs make_args(const lfamd_attention* d) {
  AttnArgs a{};
  a.B = (int)d->batch, a.H = (int)d->heads, a.Hk = (int)d->kv_heads, a.G = a.Hk ? a.H / a.Hk : 1;
  a.N = (int)d->q_len, a.M = (int)d->k_len, a.D = (int)d->head_dim;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = d->q_strides[i], a.ks[i] = d->k_strides[i], a.vs[i] = d->v_strides[i], a.os[i] = d->out_strides[i];
  }
  a.klen = d->k_lengths, a.qlen = d->q_lengths, a.qstart = d->q_starts;
  // Without a query or a key no mask is read, not even for which keys take part: its pointer may be null.
  const int kind = a.N && a.M ? d->mask_kind : LFAMD_MASK_NONE;
  a.mask = d->mask, a.maskKind = kind, a.causal = d->causal != 0;
  for (int i = 0; i < 4; ++i) a.ms[i] = d->mask_strides[i];
  a.keyMask = kind && d->mask_strides[1] == 0 && d->mask_strides[2] == 0;
  a.scale = d->scale, a.c = d->scale * kLog2e;
  a.divN = FastDiv((uint32_t)std::max(a.N, 1));
  return a;
}

}  // namespace

}  // namespace lfamd

using namespace lfamd;

extern "C" {

size_t lfamd_softmax_attention_workspace_size(int dtype, const lfamd_attention* desc) {
  bool empty = false;
  if (check_desc("softmax_attention", dtype, desc, &empty) || empty || desc->q_len == 0) return 0;
  return attn_fwd_workspace(dtype, make_args(desc));
}

size_t lfamd_softmax_attention_stats_size(int dtype, const lfamd_attention* desc) {
  bool empty = false;
  if (check_desc("softmax_attention", dtype, desc, &empty) || empty) return 0;
  const AttnArgs a = make_args(desc);
  const size_t rest = dtype == LFAMD_F32 ? 0 : (size_t)a.B * a.H * a.N * a.D * dtype_size(dtype);
  return (size_t)stat_planes(a) * sizeof(float) + (rest + 3) / 4 * 4;
}

int lfamd_softmax_attention(int dtype, const lfamd_attention* desc, const void* q, const void* k, const void* v, void* out,
                            float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "softmax_attention";
  bool empty = false;
  if (int e = check_desc(who, dtype, desc, &empty)) return e;
  if (empty || desc->q_len == 0) return ok();
  if (!q || !out || (desc->k_len && (!k || !v)) || (desc->mask_kind && desc->k_len && !desc->mask))
    return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
  AttnArgs a = make_args(desc);
  const size_t need = attn_fwd_workspace(dtype, a);
  if (need && (!workspace || workspace_bytes < need)) return fail(LFAMD_ERR_ARG, "%s: workspace too small", who);
  if (need && ((uintptr_t)workspace & 15)) return fail(LFAMD_ERR_ARG, "%s: workspace must be 16-byte aligned", who);
  const int64_t size = (int64_t)dtype_size(dtype);
  a.q = q, a.k = k, a.v = v, a.out = out, a.stat = stats;
  a.modeK = load_mode(k, a.ks, a.D, size, a.keyMask), a.modeV = load_mode(v, a.vs, a.D, size, a.keyMask);
  return attn_fwd(dtype, a, workspace, (hipStream_t)stream);
}

size_t lfamd_softmax_attention_backward_workspace_size(int dtype, const lfamd_attention* desc) {
  bool empty = false;
  if (check_desc("softmax_attention backward", dtype, desc, &empty) || empty) return 0;
  return attn_bwd_workspace(dtype, make_args(desc));
}

int lfamd_softmax_attention_backward(int dtype, const lfamd_attention* desc, const void* q, const void* k, const void* v,
                                     const void* out, const float* stats, const lfamd_attention_grads* grads,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "softmax_attention backward";
  bool empty = false;
  if (int e = check_desc(who, dtype, desc, &empty)) return e;
  if (!grads) return fail(LFAMD_ERR_ARG, "%s: null gradients", who);
  if ((grads->grad_k == nullptr) != (grads->grad_v == nullptr))
    return fail(LFAMD_ERR_ARG, "%s: grad_k and grad_v come together", who);
  if (empty || (desc->q_len == 0 && desc->k_len == 0)) return ok();
  if ((desc->q_len && (!q || !out || !stats || !grads->grad_out)) || (desc->k_len && (!k || !v)) ||
      (desc->mask_kind && desc->q_len && desc->k_len && !desc->mask))
    return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
  AttnArgs a = make_args(desc);
  const size_t need = attn_bwd_workspace(dtype, a);
  if (need && !workspace) return fail(LFAMD_ERR_ARG, "%s: null workspace", who);
  if (workspace_bytes < need) return fail(LFAMD_ERR_ARG, "%s: workspace too small", who);
  if ((uintptr_t)workspace & 15) return fail(LFAMD_ERR_ARG, "%s: workspace must be 16-byte aligned", who);
  for (int i = 0; i < 3; ++i) {
    a.gs[i] = grads->grad_out_strides[i], a.dqs[i] = grads->grad_q_strides[i];
    a.dks[i] = grads->grad_k_strides[i], a.dvs[i] = grads->grad_v_strides[i];
  }
  const int64_t size = (int64_t)dtype_size(dtype);
  a.q = q, a.k = k, a.v = v, a.o = out, a.g = grads->grad_out, a.stat = (float*)stats;
  a.dq = a.N ? grads->grad_q : nullptr, a.dk = a.M ? grads->grad_k : nullptr, a.dv = a.M ? grads->grad_v : nullptr;
  a.modeQ = load_mode(q, a.qs, a.D, size, false), a.modeG = load_mode(a.g, a.gs, a.D, size, false);
  a.modeK = load_mode(k, a.ks, a.D, size, a.keyMask), a.modeV = load_mode(v, a.vs, a.D, size, a.keyMask);
  return attn_bwd(dtype, a, workspace, (hipStream_t)stream);
}

}  // extern "C"
