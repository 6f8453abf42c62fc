// C entries of decay_attention and decay_attention_step: argument checks, the plan of a call's segments, and
// the kernels around the tiles' (decay_common.h): the segments' states joined, gradients of shared heads
// added, and the single token.
#include <math.h>

#include <algorithm>

#include "decay_common.h"

namespace lfamd {

namespace {

// The segments' own states become the states in front of them (behind them, if reverse), in place and in
// order: S(s + 1) = a^tokens(s) S(s) + own(s). One thread per element, its loads eight segments ahead.
__global__ void __launch_bounds__(256) decay_join_kernel(const DecayArgs a) {
  const DecayJob& jb = a.job[blockIdx.z];
  const int size = jb.dk * jb.dv, e = blockIdx.y * 256 + threadIdx.x, bh = blockIdx.x;
  if (e >= size) return;
  const int b = bh / a.H, len = decay_length(a, b), span = a.segTiles * kDecayTile;
  const float lg = a.logDecay[bh % a.H];
  float low;
  const float full = decay_pow64(lg, span, &low);
  float* p = jb.seg + (int64_t)bh * a.nseg * size + e;
  float s = 0.0f;
  if (jb.first) {
    const int d = e / jb.dv, c = e - d * jb.dv;
    s = jb.first[(int64_t)bh * size + (jb.firstT ? c * jb.dk + d : e)];
  }
  for (int n0 = 0; n0 < a.nseg; n0 += 8) {
    float own[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int n = min(n0 + u, a.nseg - 1);
      own[u] = p[(int64_t)(jb.reverse ? a.nseg - 1 - n : n) * size];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int n = n0 + u, at = jb.reverse ? a.nseg - 1 - n : n;
      if (n >= a.nseg) break;
      int begin, end;
      decay_segment(a, len, at, jb.reverse, &begin, &end);
      p[(int64_t)at * size] = s;
      s = end - begin == span ? fmaf(full, s, fmaf(low, s, own[u])) : fmaf(decay_pow64(lg, end - begin), s, own[u]);
    }
  }
}

// out[b][hk][n] = sum over the heads that share hk, in order, of part[b][h][n] (fp32), rounded once: dk and dv.
struct ShareArgs {
  const float* part[2];
  void* out[2];
  int64_t s[2][3];
  int D[2];
  int B, Hk, G, N;
};
template <typename T> __global__ void __launch_bounds__(256) decay_share_kernel(const ShareArgs a) {
  const int z = blockIdx.y, D = a.D[z], packs = (D + 3) / 4;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= (int64_t)a.B * a.Hk * a.N * packs) return;
  const int64_t row = at / packs;
  const int c = (int)(at - row * packs) * 4;
  const int64_t bh = row / a.N, n = row - bh * a.N;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int g = 0; g < a.G; ++g) {
    const float* p = a.part[z] + ((bh * a.G + g) * a.N + n) * D + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < D) x[j] += p[j];
  }
  store4<T>((T*)a.out[z] + (bh / a.Hk) * a.s[z][0] + (bh % a.Hk) * a.s[z][1] + n * a.s[z][2], c, D, x[0], x[1], x[2], x[3]);
}

struct StepArgs {
  const void *q, *k, *v;
  void* out;
  float* state;
  const float* logDecay;
  int64_t qs[2], ks[2], vs[2], os[2], ss[2];  // strides of batch and head
  int B, H, G, dk, dv, blocks;
  float scale;
};

// e^x - 1 for |x| < 0.5, its series up to x^9 / 9! (the rest is below 2^-9 / 10! = 2^-30 of it).
__device__ __forceinline__ float small_expm1(float x) {
  float y = 1.0f;
#pragma unroll
  for (int n = 9; n > 1; --n) y = fmaf(x * (1.0f / (float)n), y, 1.0f);
  return x * y;
}

// One token: S <- a S + k v^T in place, out = scale S^T q. Slow heads take it as S + ((a - 1) S + k v^T): an a that is rounded to 32 bits is
// off by the same 2^-25 at every token, which over the 1 / (1 - a) tokens that the state holds adds up to up to 2e-5 of it at a = 1 - 2^-10,
// where the roundings themselves come to 6e-7; a - 1 is off by 2^-24 of itself. (Fast heads would cancel S in it.) Memory-bound by the state, read and written once:
// a workgroup takes 32 value columns of a head's state, a thread four of them (16 bytes) in every 32nd row,
// all of its rows in flight at once; the rows' shares of out are added in a fixed order. 2048 states of 128 x 128: 56 us,
// 4.8 TB/s (one that the last level of cache still holds half of: 42); four of 32 x 32: 3.0.
template <typename T> __global__ void __launch_bounds__(256) decay_step_kernel(const StepArgs a) {
  __shared__ float share[4][32];
  const int block = blockIdx.x % a.blocks, bh = blockIdx.x / a.blocks, b = bh / a.H, hq = bh % a.H;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c0 = 32 * block + 4 * (threadIdx.x & 7), row0 = threadIdx.x >> 3;
  const float lg = a.logDecay[hq];
  const bool slow = fabsf(lg) < 0.5f;
  const T* q = (const T*)a.q + b * a.qs[0] + hq * a.qs[1];
  const T* k = (const T*)a.k + b * a.ks[0] + (hq / a.G) * a.ks[1];
  const T* v = (const T*)a.v + b * a.vs[0] + (hq / a.G) * a.vs[1];
  float* s = a.state + b * a.ss[0] + hq * a.ss[1];
  f32x4 x[4];
  float kr[4], qr[4], vc[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = row0 + 32 * u;
    x[u] = __builtin_bit_cast(f32x4, load_chunk<float>(s + (int64_t)r * a.dv, r < a.dk, c0, a.dv));
    kr[u] = r < a.dk ? to_acc(k[r]) : 0.0f;
    qr[u] = r < a.dk ? to_acc(q[r]) : 0.0f;
    vc[u] = c0 + u < a.dv ? to_acc(v[c0 + u]) : 0.0f;
  }
  const float factor = slow ? small_expm1(lg) : expf(lg);
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = row0 + 32 * u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[u][j] = fmaf(x[u][j], factor, kr[u] * vc[j]) + (slow ? x[u][j] : 0.0f);
      o[j] = fmaf(qr[u], x[u][j], o[j]);
    }
    if (r < a.dk) store4<float>(s + (int64_t)r * a.dv, c0, a.dv, x[u][0], x[u][1], x[u][2], x[u][3]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int d = 8; d < 64; d <<= 1) o[j] += __shfl_xor(o[j], d);
    if (lane < 8) share[wave][4 * lane + j] = o[j];
  }
  __syncthreads();
  const int c = 32 * block + (int)threadIdx.x;
  if (threadIdx.x < 32 && c < a.dv) {
    const float y = share[0][threadIdx.x] + share[1][threadIdx.x] + share[2][threadIdx.x] + share[3][threadIdx.x];
    ((T*)a.out)[b * a.os[0] + hq * a.os[1] + c] = from_acc<T>(y * a.scale);
  }
}

constexpr int64_t kMostTokens = (int64_t)1 << 29, kMostHeads = kMostWorkgroups / 4;

int check_desc(const char* who, int dtype, const lfamd_decay* d, bool* empty) {
  if (dtype != LFAMD_F32 && dtype != LFAMD_F16 && dtype != LFAMD_BF16)
    return fail(LFAMD_ERR_DTYPE, "%s: unsupported dtype %d", who, dtype);
  if (!d) return fail(LFAMD_ERR_ARG, "%s: null description", who);
  if (d->batch < 0 || d->heads < 0 || d->kv_heads < 0 || d->tokens < 0 || d->key_dim < 0 || d->value_dim < 0)
    return fail(LFAMD_ERR_ARG, "%s: negative size", who);
  if (d->key_dim < 1 || d->key_dim > 128 || d->value_dim < 1 || d->value_dim > 128)
    return fail(LFAMD_ERR_UNSUPPORTED, "%s: head sizes %lld and %lld are outside 1 .. 128", who, (long long)d->key_dim,
                (long long)d->value_dim);
  if (d->heads ? !d->kv_heads || d->heads % d->kv_heads : d->kv_heads)
    return fail(LFAMD_ERR_ARG, "%s: %lld query heads do not share %lld key heads evenly", who, (long long)d->heads,
                (long long)d->kv_heads);
  if (!(d->scale > 0.0f) || !isfinite(d->scale)) return fail(LFAMD_ERR_ARG, "%s: scale must be positive and finite", who);
  if (d->tokens > kMostTokens) return fail(LFAMD_ERR_UNSUPPORTED, "%s: at most 2^29 tokens are taken", who);
  *empty = d->batch == 0 || d->heads == 0;
  if (!*empty && (d->batch > kMostHeads || d->heads > kMostHeads || d->batch > kMostHeads / d->heads))
    return fail(LFAMD_ERR_UNSUPPORTED, "%s: batch * heads is above %lld", who, (long long)kMostHeads);
  if (!*empty && !d->log_decay) return fail(LFAMD_ERR_ARG, "%s: null log_decay", who);
  return LFAMD_OK;
}

int load_mode(const void* p, const int64_t* strides, int64_t d, int64_t size) {
  auto whole = [](int64_t bytes) { return bytes % 16 == 0; };
  return (uintptr_t)p % 16 == 0 && whole(d * size) && whole(strides[0] * size) && whole(strides[1] * size) &&
                 whole(strides[2] * size) && strides[2] >= 0 && strides[2] < ((int64_t)1 << 22)
             ? kAsync
             : kPlain;
}

// Into how many segments the sequences of `runs` (runs of the operator times sequences times heads) are cut, and
// how their states are found: the least of what the busiest SIMD takes. A wave alone takes tf us for a tile (one
// segment of 15 tiles against one of 1, one head, 32 and 128 key channels: bf16 1.3 and 2.2, fp16 1.5 and 2.45, fp32 3.1 and
// 8.1), ts for its state alone (15 tiles in 15 segments: bf16 0.74 and 1.1, fp16 0.76 and 1.15, fp32 1.3 and 3.3), and
// 3 us to begin; the constants below are within a tenth of those, but for fp32's (tf a tenth, ts a quarter less, of kernels before
// they lost their reads ahead). A SIMD holds two waves, which take one and a half times as long together (fp32, whose products
// fill it alone, 1.9). Segments joined in launches of their own cost two more, 10 us, and four passes
// over their states at 4 TB/s; the join's chain is not in it. At most 64 segments, which bounds the workspace and that chain: 256
// would be faster for few heads and very long sequences (one head, 131072 tokens, 128 channels, bf16: 243 us against 122, fp32 764 against 255; four,
// 64 channels: 185 against 131) and in fp32 (one head, 32768 tokens, 64 channels: 133 against 87), not for that head in bf16 (66 against 72).
void plan_segments(int dtype, DecayArgs& a, int64_t runs, int dk, int dv) {
  const bool f32 = dtype == LFAMD_F32;
  const int64_t tiles = ((int64_t)a.N + kDecayTile - 1) / kDecayTile;
  const double width = decay_key_dim(dk);
  const double tf = f32 ? 1.3 + 0.047 * width : (dtype == LFAMD_F16 ? 1.3 : 0.85) + 0.0095 * width;
  const double ts = (f32 ? 0.35 : 0.58) * tf;
  const double waves = (double)runs * (decay_value_dim(f32, dk, dv) / 32) / (4.0 * num_cus());
  double least = 0.0;
  for (int64_t n = 1; n <= 64 && n <= std::max<int64_t>(tiles, 1); ++n) {
    const int64_t seg = std::max<int64_t>(1, (tiles + n - 1) / n);
    if (n > 1 && (tiles + seg - 1) / seg != n) continue;  // fewer segments do the same
    const int64_t w = std::max<int64_t>(1, (int64_t)ceil(waves * (double)n));
    const double share = (double)(w / 2) * (f32 ? 1.9 : 1.5) + (double)(w % 2);
    // The last segment has most in front of it.
    const double prefix = ((double)(tiles - seg) * ts + (double)seg * tf + 3.0) * share;
    const double joined = n == 1 ? prefix : ((double)seg * (tf + ts) + 6.0) * share + 10.0 + (double)(runs * n * dk * dv) * 16.0 / 4e6;
    if (n > 1 && std::min(prefix, joined) >= least) continue;
    least = std::min(prefix, joined);
    a.nseg = (int)n, a.segTiles = (int)seg, a.prefix = n > 1 && prefix <= joined;
  }
}

DecayArgs base_args(const lfamd_decay* d) {
  DecayArgs a{};
  a.logDecay = d->log_decay, a.lengths = d->lengths;
  a.B = (int)d->batch, a.H = (int)d->heads, a.N = (int)d->tokens;
  return a;
}

int run_tiles(int dtype, const DecayArgs& a, int out, hipStream_t st) {
  return dtype == LFAMD_F32 ? decay_run_f32(a, out, st) : dtype == LFAMD_F16 ? decay_run_f16(a, out, st) : decay_run_bf16(a, out, st);
}

// The jobs of `a`, whose channels computed with agree, through their segments.
int run_jobs(int dtype, const DecayArgs& a, hipStream_t st) {
  if (a.nseg > 1 && !a.prefix) {
    DecayArgs s = a;  // the jobs whose states are formed
    s.jobs = 0;
    int most = 0;
    for (int j = 0; j < a.jobs; ++j)
      if (!a.job[j].segT) {
        s.job[s.jobs++] = a.job[j];
        most = std::max(most, a.job[j].dk * a.job[j].dv);
      }
    if (int e = run_tiles(dtype, s, 0, st)) return e;
    decay_join_kernel<<<dim3(s.B * s.H, (most + 255) / 256, s.jobs), dim3(256), 0, st>>>(s);
    if (int e = check_launch("decay_attention")) return e;
  }
  return run_tiles(dtype, a, 1, st);
}

void set3(int64_t* to, const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

// The three runs of a backward pass, in one launch where their channels computed with agree.
struct BackwardPlan {
  DecayArgs both, own;  // dq and dk (keys as wide as the values); dv by itself, if the widths differ
  bool split, shared;
  size_t segs[3], part[2], total;  // bytes of each run's segments (dq, dk, dv), of the shared heads' parts of dk and dv
};

BackwardPlan plan_backward(int dtype, const lfamd_decay* d) {
  BackwardPlan p{};
  p.split = decay_key_dim((int)d->key_dim) != decay_key_dim((int)d->value_dim);
  p.shared = d->kv_heads != d->heads;
  p.both = p.own = base_args(d);
  const int64_t bh = d->batch * d->heads;
  plan_segments(dtype, p.both, bh * (p.split ? 2 : 3), (int)d->value_dim, (int)d->key_dim);
  if (p.split) plan_segments(dtype, p.own, bh, (int)d->key_dim, (int)d->value_dim);
  else p.own.nseg = p.both.nseg, p.own.segTiles = p.both.segTiles, p.own.prefix = p.both.prefix;
  const size_t state = (size_t)bh * d->key_dim * d->value_dim * sizeof(float);
  for (int j = 0; j < 3; ++j) {
    const DecayArgs& a = j == 2 ? p.own : p.both;
    // dk takes the states that dv forms, transposed, where the two are in one launch.
    p.segs[j] = a.nseg > 1 && !a.prefix && !(j == 1 && !p.split) ? round16(state * a.nseg) : 0;
    p.total += p.segs[j];
  }
  const size_t rows = (size_t)bh * d->tokens * sizeof(float);
  p.part[0] = p.shared ? round16(rows * d->key_dim) : 0;
  p.part[1] = p.shared ? round16(rows * d->value_dim) : 0;
  p.total += p.part[0] + p.part[1];
  return p;
}

int check_workspace(const char* who, const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need)) return fail(LFAMD_ERR_ARG, "%s: workspace too small", who);
  if (need && ((uintptr_t)ws & 15)) return fail(LFAMD_ERR_ARG, "%s: workspace must be 16-byte aligned", who);
  return LFAMD_OK;
}

}  // namespace

}  // namespace lfamd

using namespace lfamd;

extern "C" {

size_t lfamd_decay_attention_workspace_size(int dtype, const lfamd_decay* desc) {
  bool empty = false;
  if (check_desc("decay_attention", dtype, desc, &empty) || empty) return 0;
  DecayArgs a = base_args(desc);
  plan_segments(dtype, a, desc->batch * desc->heads, (int)desc->key_dim, (int)desc->value_dim);
  return a.nseg > 1 && !a.prefix ? (size_t)desc->batch * desc->heads * a.nseg * desc->key_dim * desc->value_dim * sizeof(float) : 0;
}

int lfamd_decay_attention(int dtype, const lfamd_decay* desc, const void* q, const void* k, const void* v, const float* state,
                          void* out, float* last_state, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "decay_attention";
  bool empty = false;
  if (int e = check_desc(who, dtype, desc, &empty)) return e;
  if (empty || (desc->tokens == 0 && !last_state)) return ok();
  // Segments read the first state while another writes the last one.
  if (last_state && last_state == state) return fail(LFAMD_ERR_ARG, "%s: last_state must not be state", who);
  if (desc->tokens && (!q || !k || !v || !out)) return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
  if (int e = check_workspace(who, workspace, workspace_bytes, lfamd_decay_attention_workspace_size(dtype, desc))) return e;
  DecayArgs a = base_args(desc);
  plan_segments(dtype, a, desc->batch * desc->heads, (int)desc->key_dim, (int)desc->value_dim);
  const int64_t size = (int64_t)dtype_size(dtype);
  DecayJob& j = a.job[0];
  a.jobs = 1;
  j.q = q, j.k = k, j.v = v, j.first = state, j.out = out, j.last = last_state, j.seg = (float*)workspace;
  set3(j.qs, desc->q_strides), set3(j.ks, desc->k_strides), set3(j.vs, desc->v_strides), set3(j.os, desc->out_strides);
  j.qg = 1, j.kg = j.vg = (int)(desc->heads / desc->kv_heads);
  j.dk = (int)desc->key_dim, j.dv = (int)desc->value_dim;
  j.modeQ = load_mode(q, j.qs, j.dk, size), j.modeK = load_mode(k, j.ks, j.dk, size), j.modeV = load_mode(v, j.vs, j.dv, size);
  j.sp = j.so = desc->scale, j.sk = 1.0f;
  return run_jobs(dtype, a, (hipStream_t)stream);
}

size_t lfamd_decay_attention_backward_workspace_size(int dtype, const lfamd_decay* desc) {
  bool empty = false;
  if (check_desc("decay_attention backward", dtype, desc, &empty) || empty) return 0;
  return plan_backward(dtype, desc).total;
}

int lfamd_decay_attention_backward(int dtype, const lfamd_decay* desc, const void* q, const void* k, const void* v,
                                   const float* state, const lfamd_decay_grads* grads, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const char* who = "decay_attention backward";
  bool empty = false;
  if (int e = check_desc(who, dtype, desc, &empty)) return e;
  if (!grads) return fail(LFAMD_ERR_ARG, "%s: null gradients", who);
  const bool kv = grads->grad_k != nullptr;
  if (kv != (grads->grad_v != nullptr)) return fail(LFAMD_ERR_ARG, "%s: grad_k and grad_v come together", who);
  if (desc->tokens && grads->grad_state && !kv) return fail(LFAMD_ERR_ARG, "%s: grad_state comes with grad_k and grad_v", who);
  if (grads->grad_state && grads->grad_state == grads->grad_last_state)
    return fail(LFAMD_ERR_ARG, "%s: grad_state must not be grad_last_state", who);
  if (empty || (!kv && !grads->grad_q && !grads->grad_state)) return ok();
  if (desc->tokens == 0 && !grads->grad_state) return ok();
  if (desc->tokens && (!q || !k || !v || !grads->grad_out)) return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
  BackwardPlan p = plan_backward(dtype, desc);
  if (int e = check_workspace(who, workspace, workspace_bytes, p.total)) return e;
  char* ws = (char*)workspace;
  auto take = [&](size_t n) {
    char* x = ws;
    ws += n;
    return (float*)x;
  };
  float* segs[3];
  for (int j = 0; j < 3; ++j) segs[j] = take(p.segs[j]);
  float* part[2] = {take(p.part[0]), take(p.part[1])};
  const int64_t size = (int64_t)dtype_size(dtype);
  const int G = (int)(desc->heads / desc->kv_heads);
  const int dk = (int)desc->key_dim, dv = (int)desc->value_dim;
  struct Role {
    const void* p;
    const int64_t* s;
    int g, d;
  };
  const Role Q{q, desc->q_strides, 1, dk}, K{k, desc->k_strides, G, dk}, V{v, desc->v_strides, G, dv},
      O{grads->grad_out, grads->grad_out_strides, 1, dv};
  auto job = [&](const Role& x, const Role& y, const Role& z, void* out, const int64_t* os, float* seg) {
    DecayJob j{};
    j.q = x.p, j.k = y.p, j.v = z.p, j.out = out, j.seg = seg;
    set3(j.qs, x.s), set3(j.ks, y.s), set3(j.vs, z.s), set3(j.os, os);
    j.qg = x.g, j.kg = y.g, j.vg = z.g, j.dk = x.d, j.dv = z.d;
    j.modeQ = load_mode(x.p, x.s, x.d, size), j.modeK = load_mode(y.p, y.s, y.d, size), j.modeV = load_mode(z.p, z.s, z.d, size);
    j.sp = desc->scale;
    return j;
  };
  DecayArgs& a = p.both;
  DecayArgs& o = p.split ? p.own : p.both;
  if (grads->grad_q && desc->tokens) {
    DecayJob j = job(O, V, K, grads->grad_q, grads->grad_q_strides, segs[0]);
    j.first = state, j.firstT = 1, j.so = desc->scale, j.sk = 1.0f;
    a.job[a.jobs++] = j;
  }
  const int64_t rows[2][3] = {{desc->heads * desc->tokens * dk, desc->tokens * dk, dk},
                              {desc->heads * desc->tokens * dv, desc->tokens * dv, dv}};
  if (kv && desc->tokens) {
    DecayJob j = job(V, O, Q, p.shared ? part[0] : grads->grad_k, p.shared ? rows[0] : grads->grad_k_strides, segs[1]);
    j.first = grads->grad_last_state, j.firstT = 1, j.reverse = 1, j.outF32 = p.shared, j.so = 1.0f, j.sk = desc->scale;
    if (!p.split) j.seg = segs[2], j.segT = 1;
    a.job[a.jobs++] = j;
  }
  if (kv || grads->grad_state) {
    DecayJob j = job(K, Q, O, p.shared ? part[1] : grads->grad_v, p.shared ? rows[1] : grads->grad_v_strides, segs[2]);
    j.first = grads->grad_last_state, j.reverse = 1, j.outF32 = p.shared, j.so = 1.0f, j.sk = desc->scale;
    j.last = grads->grad_state;
    o.job[o.jobs++] = j;
  }
  hipStream_t st = (hipStream_t)stream;
  if (a.jobs)
    if (int e = run_jobs(dtype, a, st)) return e;
  if (p.split && o.jobs)
    if (int e = run_jobs(dtype, o, st)) return e;
  if (p.shared && kv && desc->tokens) {
    ShareArgs h{};
    h.part[0] = part[0], h.part[1] = part[1], h.out[0] = grads->grad_k, h.out[1] = grads->grad_v;
    set3(h.s[0], grads->grad_k_strides), set3(h.s[1], grads->grad_v_strides);
    h.D[0] = dk, h.D[1] = dv, h.B = (int)desc->batch, h.Hk = (int)desc->kv_heads, h.G = G, h.N = (int)desc->tokens;
    const int64_t packs = desc->batch * desc->kv_heads * desc->tokens * ((std::max(dk, dv) + 3) / 4);
    const dim3 grid((unsigned)((packs + 255) / 256), 2), t(256);
    switch (dtype) {
      case LFAMD_F32: decay_share_kernel<float><<<grid, t, 0, st>>>(h); break;
      case LFAMD_F16: decay_share_kernel<f16s><<<grid, t, 0, st>>>(h); break;
      default: decay_share_kernel<bf16s><<<grid, t, 0, st>>>(h); break;
    }
    return check_launch(who);
  }
  return ok();
}

int lfamd_decay_attention_step(int dtype, const lfamd_decay* desc, const void* q, const void* k, const void* v, void* out,
                               float* state, const int64_t* state_strides, void* stream) {
  const char* who = "decay_attention_step";
  bool empty = false;
  if (int e = check_desc(who, dtype, desc, &empty)) return e;
  if (desc->tokens != 1) return fail(LFAMD_ERR_ARG, "%s: takes one token, not %lld", who, (long long)desc->tokens);
  if (empty) return ok();
  if (!q || !k || !v || !out || !state || !state_strides) return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
  StepArgs a{};
  a.q = q, a.k = k, a.v = v, a.out = out, a.state = state, a.logDecay = desc->log_decay, a.scale = desc->scale;
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = desc->q_strides[i], a.ks[i] = desc->k_strides[i], a.vs[i] = desc->v_strides[i], a.os[i] = desc->out_strides[i];
    a.ss[i] = state_strides[i];
  }
  a.B = (int)desc->batch, a.H = (int)desc->heads, a.G = (int)(desc->heads / desc->kv_heads);
  a.dk = (int)desc->key_dim, a.dv = (int)desc->value_dim, a.blocks = (a.dv + 31) / 32;
  const dim3 g((unsigned)((int64_t)a.B * a.H * a.blocks)), t(256);
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case LFAMD_F32: decay_step_kernel<float><<<g, t, 0, st>>>(a); break;
    case LFAMD_F16: decay_step_kernel<f16s><<<g, t, 0, st>>>(a); break;
    default: decay_step_kernel<bf16s><<<g, t, 0, st>>>(a); break;
  }
  return check_launch(who);
}

}  // extern "C"
