// gated_add_rms_norm: a block's output x through its own norm, a gate and a scale onto the residual, and the norm
// of that sum,
//   m = x rx (rx = 1 / sqrt(mean(x^2) + eps); without post_weight m = x),  z = m wp,
//   s = residual + c g z,   rs = 1 / sqrt(mean(s^2) + eps),   n = s rs,   y = n w,
// and its backward pass
//   ds = gs + rs (gn - n mean(gn n)), gn = gy w;   d residual = ds;   dg = c ds z;   dw = sum over rows of gy n
//   dm = c g ds wp;   dx = rx (dm - m mean(dm m))  (without post_weight c g ds);   dwp = sum over rows of c g ds m
// where dg is summed over the rows that share a gate row.
//
// Memory-bound: x and the residual are read once and y and the sum written once, where the norm, the gated
// addition and the second norm by themselves read five tensors and write four; backward x, the residual, gy and gs
// in and two gradients out. A row stays in the registers of the threads that own it (one wave,
// or 256, 512 or 1024 threads: at most 8 elements each, so that the backward's weights and sums fit beside
// it) through both of its reductions. s is formed again in the backward from the unrounded addends.
//
// The sums over rows share their factors: with A = sum of ds m, a gate that all rows share (or none) has
// dg = c wp A and dwp = c g A, one sum for both. Workgroups (for narrow rows, waves) walk pieces of the rows
// that share a gate row in a fixed order, and a second kernel adds what they found in order: the same
// call gives the same bits.
// Measured on one MI355X: 8 x 2048 x 4096 bf16, a gate per sequence, 113 us forward (537 MB, 4.8 TB/s), 166 backward (805 MB,
// 4.85 TB/s) and 15 for the partial rows; 64 x 196 x 333 fp32, a gate per channel, 17, 32 and 4 us (rows of 84 vectors
// in a wave each: their own latencies).
#include <math.h>

#include <algorithm>

#include "norm_common.h"

namespace lfamd {

namespace {

struct GatedArgs {
  const void *x, *res, *gy, *gs, *w, *wp, *gate;
  void *y, *sum, *dx, *dres, *dgate;
  float *rstd, *rpost;                 // 1 / root mean square of the sum and of x, by row
  float *pw, *pa, *pg;                 // partial rows: of dw; of A or dwp; of A for each piece of a gate's rows
  int64_t xs, rs, gys, gss, gts;       // row strides of x, residual, gy, gs, gate
  int rows, width, share;              // share: rows that read the same gate row
  int pieces, span;                    // a gate's rows are walked in `pieces` pieces of `span` rows
  int wf32, wpf32, gf32;
  float scale, eps;
};

template <typename T> __device__ __forceinline__ void load_floats(const void* row, int f32, int c, int width, float* v) {
  constexpr int V = Pack<T>::V;
  if (f32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const Pack<float> p = Pack<float>::load((const float*)row, c + j, width);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j + i] = p.e[i];
    }
  } else {
    const Pack<T> p = Pack<T>::load((const T*)row, c, width);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_acc(p.e[j]);
  }
}

// To the row that begins at element `at`, in fp32 or T.
template <typename T>
__device__ __forceinline__ void store_floats(void* to, int f32, int64_t at, int c, int width, const float* v) {
  constexpr int V = Pack<T>::V;
  if (c >= width) return;
  if (f32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const Pack<float> p = {{v[j], v[j + 1], v[j + 2], v[j + 3]}};
      if (c + j < width) p.store((float*)to + at, c + j, width);
    }
  } else {
    Pack<T> p;
#pragma unroll
    for (int j = 0; j < V; ++j) p.e[j] = from_acc<T>(v[j]);
    p.store((T*)to + at, c, width);
  }
}

template <typename T> __device__ __forceinline__ const void* gate_row(const GatedArgs& a, int64_t g) {
  return (const char*)a.gate + g * a.gts * (a.gf32 ? 4 : (int)sizeof(T));
}

// GATE: what a row's gate is, as a call describes it. Without a gate that the description has rows for it is 1 in every kind.
enum GateKind { kGateAll = 0, kGateGroup = 1, kGateRow = 2 };  // none or one for all rows; one for some; one each

template <typename T, int TPR, int NV, bool POST>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) gated_add_rms_norm_kernel(const GatedArgs a) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR, V = Pack<T>::V;
  __shared__ float lds[16];
  const int t = threadIdx.x % TPR;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole waves, and whole workgroups where they meet at barriers (RPB = 1)
  const void* gate = a.gate ? gate_row<T>(a, (uint32_t)row / (uint32_t)a.share) : nullptr;
  float s[NV][V], sq = 0.0f;
  Pack<T> pr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * V;
    if (c < a.width) {
      const Pack<T> px = Pack<T>::load((const T*)a.x + row * a.xs, c, a.width);
      pr[i] = Pack<T>::load((const T*)a.res + row * a.rs, c, a.width);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[i][j] = to_acc(px.e[j]);
        sq = fmaf(s[i][j], s[i][j], sq);
      }
    }
  }
  float rx = 1.0f;
  if constexpr (POST) {
    sq = row_reduce<TPR, false>(sq, lds);
    rx = 1.0f / sqrtf(sq / (float)a.width + a.eps);
    if (t == 0 && a.rpost) a.rpost[row] = rx;
  }
  sq = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * V;
    if (c < a.width) {
      float f[V], g[V];
      if constexpr (POST) {
        load_floats<T>(a.wp, a.wpf32, c, a.width, f);
#pragma unroll
        for (int j = 0; j < V; ++j) s[i][j] = s[i][j] * rx * f[j];
      }
      if (gate) {
        load_floats<T>(gate, a.gf32, c, a.width, g);
#pragma unroll
        for (int j = 0; j < V; ++j) s[i][j] *= g[j];
      }
      Pack<T> ps;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[i][j] = fmaf(a.scale, s[i][j], to_acc(pr[i].e[j]));
        ps.e[j] = from_acc<T>(s[i][j]);
        sq = fmaf(s[i][j], s[i][j], sq);
      }
      ps.store((T*)a.sum + row * a.width, c, a.width);
    }
  }
  sq = row_reduce<TPR, false>(sq, lds);
  const float r = 1.0f / sqrtf(sq / (float)a.width + a.eps);
  if (t == 0 && a.rstd) a.rstd[row] = r;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * V;
    if (c < a.width) {
      float w[V];
      load_floats<T>(a.w, a.wf32, c, a.width, w);
      Pack<T> py;
#pragma unroll
      for (int j = 0; j < V; ++j) py.e[j] = from_acc<T>(s[i][j] * r * w[j]);
      py.store((T*)a.y + row * a.width, c, a.width);
    }
  }
}

// Walkers (workgroups, or the four waves of one) take pieces of rows with one gate in turn. Behind the walk dw's
// share goes to pw[workgroup] and A's (kGateAll), or dwp's, to pa[workgroup].
template <typename T, int TPR, int NV, int GATE, bool POST>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) gated_add_rms_norm_bwd_kernel(const GatedArgs a) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR, V = Pack<T>::V;
  __shared__ float lds[16];
  const int t = threadIdx.x % TPR;
  float w[NV][V], wp[NV][V], g[NV][V], dw[NV][V], sa[NV][V], dwp[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) w[i][j] = dw[i][j] = sa[i][j] = dwp[i][j] = 0.0f, wp[i][j] = g[i][j] = 1.0f;
    if (c < a.width) {
      load_floats<T>(a.w, a.wf32, c, a.width, w[i]);
      if constexpr (POST) load_floats<T>(a.wp, a.wpf32, c, a.width, wp[i]);
      if (GATE == kGateAll && a.gate) load_floats<T>(a.gate, a.gf32, c, a.width, g[i]);
    }
  }
  const int groups = a.rows / a.share, units = groups * a.pieces;
  for (int u = blockIdx.x * RPB + threadIdx.x / TPR; u < units; u += gridDim.x * RPB) {
    const int group = u / a.pieces, first = group * a.share + (u - group * a.pieces) * a.span;
    const int end = min(first + a.span, (group + 1) * a.share);
    if constexpr (GATE == kGateGroup) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) sa[i][j] = 0.0f;
        if (a.gate && c < a.width) load_floats<T>(gate_row<T>(a, group), a.gf32, c, a.width, g[i]);
      }
    }
    // The next row's elements are loaded in front of this row's reductions (bf16 8 x 2048 x 4096: 221 -> 169 us), but
    // for 1024 threads, whose 128 registers do not hold two rows. A piece's last row, and so every row with a gate of its
    // own, has none behind it and loads itself again, from the cache: with gates by token the step's time is the same without
    // that load (8 x 2048 x 4096 bf16 417 -> 412 us, 1024 wide 154 -> 158) and in longer pieces (414 and 154; 16 x 1024 x 2048
    // fp32 330 -> 342).
    constexpr bool EARLY = TPR < 1024;
    Pack<T> nx[NV], nr[NV], ny[NV], ng[NV];
    float next_rx = 1.0f, next_r = 0.0f;
    auto load = [&](int64_t row) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
        if (c < a.width) {
          nx[i] = Pack<T>::load((const T*)a.x + row * a.xs, c, a.width);
          nr[i] = Pack<T>::load((const T*)a.res + row * a.rs, c, a.width);
          ny[i] = Pack<T>::load((const T*)a.gy + row * a.gys, c, a.width);
          if (a.gs) ng[i] = Pack<T>::load((const T*)a.gs + row * a.gss, c, a.width);
        }
      }
      if constexpr (POST) next_rx = a.rpost[row];
      next_r = a.rstd[row];
    };
    if (EARLY) load(first);
    for (int64_t row = first; row < end; ++row) {
      if (!EARLY) load(row);
      Pack<T> px[NV], pr[NV], py[NV], pg[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        px[i] = nx[i], pr[i] = nr[i], py[i] = ny[i], pg[i] = ng[i];
        const int c = (t + i * TPR) * V;
        if (GATE == kGateRow && a.gate && c < a.width) load_floats<T>(gate_row<T>(a, row), a.gf32, c, a.width, g[i]);
      }
      const float rx = next_rx, r = next_r;
      if (EARLY) load(min(row + 1, (int64_t)end - 1));
      float n[NV][V], m[NV][V], dot = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if ((t + i * TPR) * V < a.width)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            m[i][j] = to_acc(px[i].e[j]) * rx;
            n[i][j] = fmaf(a.scale, m[i][j] * wp[i][j] * g[i][j], to_acc(pr[i].e[j])) * r;
            const float gy = to_acc(py[i].e[j]);
            dw[i][j] = fmaf(gy, n[i][j], dw[i][j]);
            dot = fmaf(gy * w[i][j], n[i][j], dot);
          }
      dot = row_reduce<TPR, false>(dot, lds) / (float)a.width;
      float back = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
        if (c < a.width) {
          Pack<T> pd;
          float dg[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float d = r * fmaf(-n[i][j], dot, to_acc(py[i].e[j]) * w[i][j]);
            if (a.gs) d += to_acc(pg[i].e[j]);
            pd.e[j] = from_acc<T>(d);
            const float dm = d * m[i][j];
            if constexpr (GATE == kGateRow) {
              dg[j] = a.scale * dm * wp[i][j];
              dwp[i][j] = fmaf(a.scale * g[i][j], dm, dwp[i][j]);
            } else {
              sa[i][j] += dm;
            }
            n[i][j] = a.scale * g[i][j] * wp[i][j] * d;  // the gradient of m
            back = fmaf(n[i][j], m[i][j], back);
          }
          pd.store((T*)a.dres + row * a.width, c, a.width);
          if constexpr (GATE == kGateRow) {
            if (a.dgate) store_floats<T>(a.dgate, a.gf32, row * a.width, c, a.width, dg);
          }
        }
      }
      if constexpr (POST) back = row_reduce<TPR, false>(back, lds) / (float)a.width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
        if (c < a.width) {
          Pack<T> pd;
#pragma unroll
          for (int j = 0; j < V; ++j) pd.e[j] = from_acc<T>(POST ? rx * fmaf(-m[i][j], back, n[i][j]) : n[i][j]);
          pd.store((T*)a.dx + row * a.width, c, a.width);
        }
      }
    }
    if constexpr (GATE == kGateGroup) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (t + i * TPR) * V;
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          Pack<float> p;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            dwp[i][j + k] = fmaf(a.scale * g[i][j + k], sa[i][j + k], dwp[i][j + k]);
            p.e[k] = sa[i][j + k];
          }
          if (a.pg && c + j < a.width) p.store(a.pg + (int64_t)u * a.width, c + j, a.width);
        }
        if (a.dgate && !a.pg) {  // the gate's only piece
#pragma unroll
          for (int j = 0; j < V; ++j) sa[i][j] *= a.scale * wp[i][j];
          store_floats<T>(a.dgate, a.gf32, (int64_t)group * a.width, c, a.width, sa[i]);
        }
      }
    }
  }
  float* to[2] = {a.pw ? a.pw + (int64_t)blockIdx.x * a.width : nullptr, a.pa ? a.pa + (int64_t)blockIdx.x * a.width : nullptr};
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    if (!to[z]) continue;
    const float(&from)[NV][V] = z == 0 ? dw : GATE == kGateAll ? sa : dwp;
    if constexpr (RPB > 1) {
      // The four waves' shares, added in their order.
      extern __shared__ float share[];  // [width]
      for (int k = 0; k < RPB; ++k) {
        if ((int)threadIdx.x / TPR == k) {
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const int c = (t + i * TPR) * V;
#pragma unroll
            for (int j = 0; j < V; ++j)
              if (c + j < a.width) share[c + j] = k ? share[c + j] + from[i][j] : from[i][j];
          }
        }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < a.width; c += THREADS) to[z][c] = share[c];
      __syncthreads();
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const Pack<float> p = {{from[i][j], from[i][j + 1], from[i][j + 2], from[i][j + 3]}};
          const int c = (t + i * TPR) * V + j;
          if (c < a.width) p.store(to[z], c, a.width);
        }
    }
  }
}

// What the walkers' partial rows add up to, 16 columns x 64 row groups per workgroup, the groups' sums in their
// order. blockIdx.y 0: dw. 1: dwp and, where one gate row serves all (or none), its gradient, from A.
// From 2 on: the gradient of gate row blockIdx.y - 2, from the pieces of its rows.
struct SumArgs {
  const float *pw, *pa, *pg;
  const void *wp, *gate;
  void *dw, *dwp, *dgate;
  int n, pieces, width, kind;
  int wf32, wpf32, gf32;
  float scale;
};
template <typename T> __device__ __forceinline__ float one_float(const void* p, int f32, int64_t c) {
  return f32 ? ((const float*)p)[c] : to_acc(((const T*)p)[c]);
}
template <typename T> __device__ __forceinline__ void one_store(void* p, int f32, int64_t c, float x) {
  if (f32) ((float*)p)[c] = x;
  else ((T*)p)[c] = from_acc<T>(x);
}
template <typename T> __global__ void __launch_bounds__(1024) gated_norm_sum_kernel(const SumArgs a) {
  __shared__ float s[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4, what = blockIdx.y;
  const float* part = what == 0 ? a.pw : what == 1 ? a.pa : a.pg + (int64_t)(what - 2) * a.pieces * a.width;
  const int n = what < 2 ? a.n : a.pieces;
  if (!part) return;
  float x = 0.0f;
  if (c < a.width) {
#pragma unroll 8
    for (int i = k; i < n; i += 64) x += part[(int64_t)i * a.width + c];
  }
  s[k][threadIdx.x & 15] = x;
  __syncthreads();
  if (k != 0 || c >= a.width) return;
  x = 0.0f;
#pragma unroll
  for (int i = 0; i < 64; ++i) x += s[i][threadIdx.x];
  const float wp = a.wp ? one_float<T>(a.wp, a.wpf32, c) : 1.0f;
  if (what == 0) {
    one_store<T>(a.dw, a.wf32, c, x);
  } else if (what == 1) {
    if (a.dwp) one_store<T>(a.dwp, a.wpf32, c, a.kind == kGateAll ? a.scale * (a.gate ? one_float<T>(a.gate, a.gf32, c) : 1.0f) * x : x);
    if (a.kind == kGateAll && a.dgate) one_store<T>(a.dgate, a.gf32, c, a.scale * wp * x);
  } else {
    one_store<T>(a.dgate, a.gf32, (int64_t)(what - 2) * a.width + c, a.scale * wp * x);
  }
}

constexpr int kGatedMaxWidth = 8192;

struct GatedPlan {
  int tpr, nv, grid, pieces, span, kind;
};

GatedPlan gated_plan(int dtype, const lfamd_gated_norm* d) {
  const int V = dtype == LFAMD_F32 ? 4 : 8, most = 8 / V, units = ((int)d->width + V - 1) / V;
  GatedPlan p{1024, most, 1, 1, 1, kGateAll};
  for (int tpr : {64, 256, 512, 1024})
    if (units <= tpr * most) {
      p.tpr = tpr;
      break;
    }
  p.nv = units <= p.tpr ? 1 : most;
  const int64_t share = d->gate_rows > 0 ? d->gate_rows : d->rows;
  const int64_t groups = share ? d->rows / share : 0;
  p.kind = groups <= 1 ? kGateAll : share == 1 ? kGateRow : kGateGroup;
  // Eight waves per CU, what its registers hold (64 x 196 x 333 fp32: 41 us with twice as many), or two workgroups; a
  // walker takes at least four rows of a gate.
  const int rpb = p.tpr < 256 ? 256 / p.tpr : 1;
  const int64_t most_groups = (int64_t)num_cus() * (p.tpr == 1024 ? 1 : 2), walkers = most_groups * rpb;
  const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>((walkers + groups - 1) / std::max<int64_t>(groups, 1), (share + 3) / 4));
  p.span = (int)std::max<int64_t>(1, (share + pieces - 1) / pieces);
  p.pieces = (int)std::max<int64_t>(1, (share + p.span - 1) / p.span);
  p.grid = (int)std::max<int64_t>(1, std::min<int64_t>((groups * p.pieces + rpb - 1) / rpb, most_groups));
  return p;
}

int check_sizes(const char* who, int dtype, const lfamd_gated_norm* d) {
  if (dtype != LFAMD_F32 && dtype != LFAMD_F16 && dtype != LFAMD_BF16)
    return fail(LFAMD_ERR_DTYPE, "%s: unsupported dtype %d", who, dtype);
  if (!d) return fail(LFAMD_ERR_ARG, "%s: null description", who);
  for (int t : {d->weight_dtype, d->post_weight_dtype, d->gate_dtype})
    if (t != dtype && t != LFAMD_F32)
      return fail(LFAMD_ERR_DTYPE, "%s: weights and gate must have the input's dtype or fp32", who);
  if (d->rows < 0 || d->width < 0 || d->gate_rows < 0) return fail(LFAMD_ERR_ARG, "%s: negative size", who);
  if (d->width < 1 || d->width > kGatedMaxWidth)
    return fail(LFAMD_ERR_UNSUPPORTED, "%s: width %lld is outside 1 .. %d", who, (long long)d->width, kGatedMaxWidth);
  if (d->rows > INT32_MAX / 2) return fail(LFAMD_ERR_UNSUPPORTED, "%s: too many rows", who);
  if (d->gate_rows && d->rows % d->gate_rows)
    return fail(LFAMD_ERR_ARG, "%s: %lld rows do not share gates of %lld rows evenly", who, (long long)d->rows, (long long)d->gate_rows);
  if (!isfinite(d->scale)) return fail(LFAMD_ERR_ARG, "%s: scale must be finite", who);
  return LFAMD_OK;
}

GatedArgs base_args(const lfamd_gated_norm* d, const void* x, const void* res, const void* w, const void* wp, const void* gate) {
  GatedArgs a{};
  a.x = x, a.res = res, a.w = w, a.wp = wp, a.gate = gate;
  a.xs = d->x_stride, a.rs = d->residual_stride, a.gts = d->gate_stride;
  a.rows = (int)d->rows, a.width = (int)d->width, a.share = (int)(d->gate_rows > 0 ? d->gate_rows : std::max<int64_t>(d->rows, 1));
  a.wf32 = d->weight_dtype == LFAMD_F32, a.wpf32 = d->post_weight_dtype == LFAMD_F32, a.gf32 = d->gate_dtype == LFAMD_F32;
  a.scale = d->scale, a.eps = d->eps;
  return a;
}

// f.template go<TPR, NV>() for a plan.
template <typename T, int TPR, typename F> int with_nv(const GatedPlan& p, F&& f) {
  if constexpr (sizeof(T) == 2) return f.template go<TPR, 1>();
  else if constexpr (TPR > 256) return f.template go<TPR, 2>();  // wider workgroups begin at two vectors
  else return p.nv == 1 ? f.template go<TPR, 1>() : f.template go<TPR, 2>();
}
template <typename T, typename F> int with_plan(const GatedPlan& p, F&& f) {
  switch (p.tpr) {
    case 64: return with_nv<T, 64>(p, f);
    case 256: return with_nv<T, 256>(p, f);
    case 512: return with_nv<T, 512>(p, f);
    default: return with_nv<T, 1024>(p, f);
  }
}

template <typename T> struct Forward {
  GatedArgs a;
  hipStream_t st;
  template <int TPR, int NV> int go() {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    // A grid's axis has below 2^32 threads: the workgroups beyond 2^21 go along the second.
    const int64_t n = ((int64_t)a.rows + RPB - 1) / RPB, x = std::min<int64_t>(n, 1 << 21);
    const dim3 g((unsigned)x, (unsigned)((n + x - 1) / x)), b(TPR < 256 ? 256 : TPR);
    if (a.wp) gated_add_rms_norm_kernel<T, TPR, NV, true><<<g, b, 0, st>>>(a);
    else gated_add_rms_norm_kernel<T, TPR, NV, false><<<g, b, 0, st>>>(a);
    return check_launch("gated_add_rms_norm");
  }
};

template <typename T> struct Backward {
  GatedArgs a;
  GatedPlan p;
  hipStream_t st;
  template <int TPR, int NV, int GATE> int kind() {
    const size_t lds = TPR < 256 ? (size_t)a.width * sizeof(float) : 0;
    const dim3 g(p.grid), b(TPR < 256 ? 256 : TPR);
    if (a.wp) gated_add_rms_norm_bwd_kernel<T, TPR, NV, GATE, true><<<g, b, lds, st>>>(a);
    else gated_add_rms_norm_bwd_kernel<T, TPR, NV, GATE, false><<<g, b, lds, st>>>(a);
    return check_launch("gated_add_rms_norm backward");
  }
  template <int TPR, int NV> int go() {
    switch (p.kind) {
      case kGateAll: return kind<TPR, NV, kGateAll>();
      case kGateGroup: return kind<TPR, NV, kGateGroup>();
      default: return kind<TPR, NV, kGateRow>();
    }
  }
};

// The partial rows: dw's, A's (or dwp's), and A's of each piece of a gate's rows where it has several.
size_t partial_rows(const GatedPlan& p, const lfamd_gated_norm* d) {
  return 2 * (size_t)p.grid + (p.kind == kGateGroup && p.pieces > 1 ? (size_t)(d->rows / d->gate_rows) * p.pieces : 0);
}

}  // namespace

}  // namespace lfamd

using namespace lfamd;

extern "C" {

int lfamd_gated_add_rms_norm(int dtype, const lfamd_gated_norm* desc, const void* x, const void* residual, const void* weight,
                             const void* post_weight, const void* gate, void* y, void* sum, float* rstd, float* post_rstd,
                             void* stream) {
  const char* who = "gated_add_rms_norm";
  if (int e = check_sizes(who, dtype, desc)) return e;
  if (desc->rows == 0) return ok();
  if (!x || !residual || !weight || !y || !sum) return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
  GatedArgs a = base_args(desc, x, residual, weight, post_weight, gate);
  a.y = y, a.sum = sum, a.rstd = rstd, a.rpost = post_rstd;
  const GatedPlan p = gated_plan(dtype, desc);
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case LFAMD_F32: return with_plan<float>(p, Forward<float>{a, st});
    case LFAMD_F16: return with_plan<f16s>(p, Forward<f16s>{a, st});
    default: return with_plan<bf16s>(p, Forward<bf16s>{a, st});
  }
}

size_t lfamd_gated_add_rms_norm_backward_workspace_size(int dtype, const lfamd_gated_norm* desc) {
  if (check_sizes("gated_add_rms_norm backward", dtype, desc) || desc->rows == 0) return 0;
  return partial_rows(gated_plan(dtype, desc), desc) * desc->width * sizeof(float);
}

int lfamd_gated_add_rms_norm_backward(int dtype, const lfamd_gated_norm* desc, const void* grad_y, int64_t grad_y_stride,
                                      const void* grad_sum, int64_t grad_sum_stride, const void* x, const void* residual,
                                      const void* weight, const void* post_weight, const void* gate, const float* rstd,
                                      const float* post_rstd, void* grad_x, void* grad_residual, void* grad_weight,
                                      void* grad_post_weight, void* grad_gate, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const char* who = "gated_add_rms_norm backward";
  if (int e = check_sizes(who, dtype, desc)) return e;
  if ((grad_post_weight && !post_weight) || (grad_gate && !gate))
    return fail(LFAMD_ERR_ARG, "%s: a gradient without what it is of", who);
  hipStream_t st = (hipStream_t)stream;
  GatedArgs a = base_args(desc, x, residual, weight, post_weight, gate);
  // Without rows there are no gate rows either, unless one serves all.
  if (desc->rows == 0 && desc->gate_rows) grad_gate = nullptr;
  const bool sums = grad_weight || grad_post_weight || grad_gate;
  GatedPlan p{};
  int groups = 0;
  if (desc->rows > 0) {
    if (!grad_y || !x || !residual || !weight || !rstd || !grad_x || !grad_residual || (post_weight && !post_rstd))
      return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
    const size_t need = lfamd_gated_add_rms_norm_backward_workspace_size(dtype, desc);
    if (!workspace || workspace_bytes < need) return fail(LFAMD_ERR_ARG, "%s: workspace too small", who);
    if ((uintptr_t)workspace & 3) return fail(LFAMD_ERR_ARG, "%s: workspace must be 4-byte aligned", who);
    p = gated_plan(dtype, desc);
    groups = (int)(desc->rows / a.share);
    a.gy = grad_y, a.gs = grad_sum, a.gys = grad_y_stride, a.gss = grad_sum_stride;
    a.rstd = (float*)rstd, a.rpost = (float*)post_rstd, a.dx = grad_x, a.dres = grad_residual, a.dgate = grad_gate;
    a.pieces = p.pieces, a.span = p.span;
    a.pw = grad_weight ? (float*)workspace : nullptr;
    a.pa = grad_post_weight || (grad_gate && p.kind == kGateAll) ? (float*)workspace + (size_t)p.grid * desc->width : nullptr;
    a.pg = grad_gate && p.kind == kGateGroup && p.pieces > 1 ? (float*)workspace + 2 * (size_t)p.grid * desc->width : nullptr;
    int e;
    switch (dtype) {
      case LFAMD_F32: e = with_plan<float>(p, Backward<float>{a, p, st}); break;
      case LFAMD_F16: e = with_plan<f16s>(p, Backward<f16s>{a, p, st}); break;
      default: e = with_plan<bf16s>(p, Backward<bf16s>{a, p, st}); break;
    }
    if (e) return e;
  }
  if (!sums) return ok();
  SumArgs s{};
  // Without rows the sums are of none, from any pointer.
  s.pw = grad_weight ? (desc->rows ? a.pw : (const float*)grad_weight) : nullptr;
  s.pa = desc->rows ? a.pa : grad_post_weight ? (const float*)grad_post_weight : (const float*)grad_gate;
  s.pg = a.pg, s.wp = post_weight, s.gate = gate, s.dw = grad_weight, s.dwp = grad_post_weight, s.dgate = grad_gate;
  s.n = desc->rows ? p.grid : 0, s.pieces = p.pieces, s.width = (int)desc->width, s.kind = p.kind;
  s.wf32 = a.wf32, s.wpf32 = a.wpf32, s.gf32 = a.gf32, s.scale = desc->scale;
  const dim3 b(1024);
  const unsigned cols = (unsigned)((desc->width + 15) / 16);
  // Gates of several pieces are fewer than the walkers.
  const dim3 g(cols, (unsigned)(2 + (a.pg ? groups : 0)));
  switch (dtype) {
    case LFAMD_F32: gated_norm_sum_kernel<float><<<g, b, 0, st>>>(s); break;
    case LFAMD_F16: gated_norm_sum_kernel<f16s><<<g, b, 0, st>>>(s); break;
    default: gated_norm_sum_kernel<bf16s><<<g, b, 0, st>>>(s); break;
  }
  return check_launch(who);
}

}  // extern "C"
