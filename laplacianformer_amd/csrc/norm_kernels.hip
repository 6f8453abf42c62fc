// add_rms_norm: s = x + residual, rstd = 1 / sqrt(mean(s^2) + eps), y = s rstd w, and its backward pass
//   gn = gy w,  n = s rstd,  ds = gs + rstd (gn - n mean(gn n)),  dw = sum over rows of gy n.
//
// Memory-bound: every element is read and written once. A row stays in the registers
// of the threads that own it (one wave, or a workgroup of 256 or 1024 threads, chosen
// by the width so that a thread holds at most 16 elements) between the sum of squares
// and the scaling. Rows may begin and end anywhere: the 16-byte accesses need no alignment. The forward normalises the
// fp32 sum, not its stored rounding, and so does the backward where the two addends are
// given (16-bit types: a quarter more to move, and gradients 1.4 times as exact, as the stored
// sum's half step would enter n beside the gradients' own rounding: dw of 2048 x 16000 bf16
// 93 us and 1.6e-3 off, from the stored sum 72 us and 2.4e-3; equal times at 4096 x 4096).
// gn is formed twice rather than held: beyond 8192 columns, where 1024 threads have 128 registers each, fewer
// values go through scratch (104 -> 93 us, fp32 159 -> 145; fp32 still keeps 60 bytes a thread there, 128 from
// addends, and fp16 and bf16 from addends 44 and 12). The backward's workgroups walk the rows with a
// fixed stride, keep their share of dw in registers, and write one fp32 partial row
// each; a second kernel adds those in their order, so the same call gives the same bits.
// Measured on one MI355X: 16384 x 4096 bf16 to 8 bits 88 us (470 MB, 5.3 TB/s, the rate of a large copy); 12544 x 333
// fp32 14 us forward, 19 + 4 backward (67 MB each way: the rows' own latencies, three rows per wave).
#include <algorithm>

#include "norm_common.h"

namespace lfamd {

namespace {

struct NormArgs {
  const void *x, *res, *w, *gy, *gs;
  void *y, *sum, *dx;
  float *rstd, *scale, *part;
  int64_t xs, rs, gys, gss;  // row strides of x, residual, gy, gs (y, sum, dx: contiguous)
  int64_t rows;
  int width, wf32, e4m3;
  float eps;
};

template <typename T> __device__ __forceinline__ void load_weight(const NormArgs& a, int c, float* w) {
  constexpr int V = Pack<T>::V;
  if (a.wf32) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const Pack<float> p = Pack<float>::load((const float*)a.w, c + j, a.width);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[j + i] = p.e[i];
    }
  } else {
    const Pack<T> p = Pack<T>::load((const T*)a.w, c, a.width);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = to_acc(p.e[j]);
  }
}

template <typename T, int TPR, int NV, bool F8>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) add_rms_norm_kernel(const NormArgs a) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR, V = Pack<T>::V;
  __shared__ float lds[16];
  const int t = threadIdx.x % TPR;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole waves, and whole workgroups where they meet at barriers (RPB = 1)
  float s[NV][V], sq = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * V;
    if (c < a.width) {
      const Pack<T> px = Pack<T>::load((const T*)a.x + row * a.xs, c, a.width);
      if (a.res) {
        const Pack<T> pr = Pack<T>::load((const T*)a.res + row * a.rs, c, a.width);
        Pack<T> ps;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s[i][j] = to_acc(px.e[j]) + to_acc(pr.e[j]);
          ps.e[j] = from_acc<T>(s[i][j]);
        }
        ps.store((T*)a.sum + row * a.width, c, a.width);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) s[i][j] = to_acc(px.e[j]);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sq = fmaf(s[i][j], s[i][j], sq);
    }
  }
  sq = row_reduce<TPR, false>(sq, lds);
  const float r = 1.0f / sqrtf(sq / (float)a.width + a.eps);
  if (t == 0 && a.rstd) a.rstd[row] = r;
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * V;
    if (c < a.width) {
      float w[V];
      load_weight<T>(a, c, w);
      Pack<T> py;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[i][j] = s[i][j] * r * w[j];
        if constexpr (F8) top = fmaxf(top, fabsf(s[i][j]));
        else py.e[j] = from_acc<T>(s[i][j]);
      }
      if constexpr (!F8) py.store((T*)a.y + row * a.width, c, a.width);
    }
  }
  if constexpr (F8) {
    top = row_reduce<TPR, true>(top, lds);
    // Below 2^-117 the scale would be subnormal: such a row, all zeros among them, keeps 1 and becomes zeros.
    const float scale = top < 6.0185310762101e-36f ? 1.0f : top / 448.0f;
    if (t == 0) a.scale[row] = scale;
    uint8_t* y = (uint8_t*)a.y + row * a.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * V;
      if (c < a.width) {
        // |y / scale| <= 448 (1 + 2^-23), which rounds to at most 448: nothing saturates.
        uint32_t o[V / 4];
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
          const float* z = &s[i][4 * j];
          const int p = __builtin_amdgcn_cvt_pk_fp8_f32(z[0] / scale, z[1] / scale, 0, false);
          o[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2] / scale, z[3] / scale, p, true);
        }
        if (c + V <= a.width) {
          if constexpr (V == 8) {
            const uint64_t both = (uint64_t)o[1] << 32 | o[0];
            __builtin_memcpy(y + c, &both, 8);
          } else {
            __builtin_memcpy(y + c, o, 4);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (c + j < a.width) y[c + j] = (uint8_t)(o[j >> 2] >> (8 * (j & 3)));
        }
      }
    }
  }
}

// ADD: a.x and a.res are the addends; otherwise a.x is their sum. part: [gridDim.x][width].
template <typename T, int TPR, int NV, bool ADD>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) add_rms_norm_bwd_kernel(const NormArgs a) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR, V = Pack<T>::V;
  __shared__ float lds[16];
  const int t = threadIdx.x % TPR;
  float w[NV][V], dw[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (t + i * TPR) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) w[i][j] = dw[i][j] = 0.0f;
    if (c < a.width) load_weight<T>(a, c, w[i]);
  }
  // Without barriers in the loop (RPB > 1) the waves of a workgroup walk their rows alone.
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    Pack<T> ps[NV], pr[ADD ? NV : 1], py[NV], pg[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * V;
      if (c < a.width) {
        ps[i] = Pack<T>::load((const T*)a.x + row * a.xs, c, a.width);
        if constexpr (ADD) pr[i] = Pack<T>::load((const T*)a.res + row * a.rs, c, a.width);
        py[i] = Pack<T>::load((const T*)a.gy + row * a.gys, c, a.width);
        if (a.gs) pg[i] = Pack<T>::load((const T*)a.gs + row * a.gss, c, a.width);
      }
    }
    const float r = a.rstd[row];
    float n[NV][V], dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((t + i * TPR) * V < a.width)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float s = to_acc(ps[i].e[j]);
          if constexpr (ADD) s += to_acc(pr[i].e[j]);
          n[i][j] = s * r;
          const float gy = to_acc(py[i].e[j]);
          dw[i][j] = fmaf(gy, n[i][j], dw[i][j]);
          dot = fmaf(gy * w[i][j], n[i][j], dot);
        }
    dot = row_reduce<TPR, false>(dot, lds) / (float)a.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * TPR) * V;
      if (c < a.width) {
        Pack<T> pd;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float d = r * fmaf(-n[i][j], dot, to_acc(py[i].e[j]) * w[i][j]);
          if (a.gs) d += to_acc(pg[i].e[j]);
          pd.e[j] = from_acc<T>(d);
        }
        pd.store((T*)a.dx + row * a.width, c, a.width);
      }
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * a.width;
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
            if (c + j < a.width) share[c + j] = k ? share[c + j] + dw[i][j] : dw[i][j];
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.width; c += THREADS) part[c] = share[c];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        Pack<float> p;
#pragma unroll
        for (int k = 0; k < 4; ++k) p.e[k] = dw[i][j + k];
        const int c = (t + i * TPR) * V + j;
        if (c < a.width) p.store(part, c, a.width);
      }
  }
}

// dw[c] = sum over the partial rows: 16 columns x 64 row groups per workgroup, then the
// groups' sums in their order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* part, int n, int width, T* dw, int f32) {
  __shared__ float s[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4;
  float x = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int i = k; i < n; i += 64) x += part[(int64_t)i * width + c];
  }
  s[k][threadIdx.x & 15] = x;
  __syncthreads();
  if (k == 0 && c < width) {
    x = 0.0f;
#pragma unroll
    for (int i = 0; i < 64; ++i) x += s[i][threadIdx.x];
    if (f32) ((float*)dw)[c] = x;
    else dw[c] = from_acc<T>(x);
  }
}

constexpr int kNormMaxWidth = 16384;

struct NormPlan {
  int tpr, nv;
};

// Threads per row and 16-byte vectors per thread, for at most 16 elements each (the backward
// holds the weight, dw and n of each in fp32, and its inputs packed). One wave per row while that holds the row, as a wave
// reduces without barriers; then the smallest workgroup that does.
NormPlan norm_plan(int dtype, int width) {
  const int V = dtype == LFAMD_F32 ? 4 : 8, most = 16 / V, units = (width + V - 1) / V;
  NormPlan p{1024, 1};
  for (int tpr : {64, 256, 1024})
    if (units <= tpr * most) {
      p.tpr = tpr;
      break;
    }
  const int need = (units + p.tpr - 1) / p.tpr;
  p.nv = need <= 1 ? 1 : need <= 2 ? 2 : 4;
  return p;
}

// Calls f.template go<TPR, NV>() for a plan. (fp32: wider workgroups begin at two vectors.)
template <typename T, int TPR, typename F> int with_nv(const NormPlan& p, F&& f) {
  if constexpr (sizeof(T) == 2) return p.nv == 1 ? f.template go<TPR, 1>() : f.template go<TPR, 2>();
  else if constexpr (TPR == 64) return p.nv == 1 ? f.template go<TPR, 1>() : p.nv == 2 ? f.template go<TPR, 2>() : f.template go<TPR, 4>();
  else return p.nv == 2 ? f.template go<TPR, 2>() : f.template go<TPR, 4>();
}
template <typename T, typename F> int with_plan(const NormPlan& p, F&& f) {
  return p.tpr == 64 ? with_nv<T, 64>(p, f) : p.tpr == 256 ? with_nv<T, 256>(p, f) : with_nv<T, 1024>(p, f);
}

template <typename T, bool F8> struct NormFwd {
  NormArgs a;
  hipStream_t st;
  template <int TPR, int NV> int go() {
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
    // A grid's axis has below 2^32 threads: the workgroups beyond 2^21 go along the second.
    const int64_t n = (a.rows + RPB - 1) / RPB, x = std::min<int64_t>(n, 1 << 21);
    add_rms_norm_kernel<T, TPR, NV, F8>
        <<<dim3((unsigned)x, (unsigned)((n + x - 1) / x)), dim3(TPR < 256 ? 256 : TPR), 0, st>>>(a);
    return check_launch("add_rms_norm");
  }
};

int bwd_grid(const NormPlan& p, int64_t rows) {
  const int rpb = p.tpr < 256 ? 256 / p.tpr : 1;
  // Four workgroups of 256 threads per CU, two of 1024.
  const int64_t most = (int64_t)num_cus() * (p.tpr > 256 ? 2 : 4);
  return (int)std::max<int64_t>(1, std::min<int64_t>((rows + rpb - 1) / rpb, most));
}

template <typename T> struct NormBwd {
  NormArgs a;
  hipStream_t st;
  int grid;
  template <int TPR, int NV> int go() {
    const size_t lds = TPR < 256 && a.part ? (size_t)a.width * sizeof(float) : 0;
    const dim3 g(grid), b(TPR < 256 ? 256 : TPR);
    if (a.res) add_rms_norm_bwd_kernel<T, TPR, NV, true><<<g, b, lds, st>>>(a);
    else add_rms_norm_bwd_kernel<T, TPR, NV, false><<<g, b, lds, st>>>(a);
    return check_launch("add_rms_norm backward");
  }
};

int check_sizes(const char* who, int dtype, int w_dtype, int64_t rows, int64_t width) {
  if (dtype != LFAMD_F32 && dtype != LFAMD_F16 && dtype != LFAMD_BF16)
    return fail(LFAMD_ERR_DTYPE, "%s: unsupported dtype %d", who, dtype);
  if (w_dtype != dtype && w_dtype != LFAMD_F32)
    return fail(LFAMD_ERR_DTYPE, "%s: the weight must have the input's dtype or fp32", who);
  if (rows < 0 || width < 0) return fail(LFAMD_ERR_ARG, "%s: negative size", who);
  if (width < 1 || width > kNormMaxWidth)
    return fail(LFAMD_ERR_UNSUPPORTED, "%s: width %lld is outside 1 .. %d", who, (long long)width, kNormMaxWidth);
  if (rows > INT32_MAX) return fail(LFAMD_ERR_UNSUPPORTED, "%s: too many rows", who);
  return LFAMD_OK;
}

template <bool F8> int norm_forward(int dtype, const NormArgs& a, hipStream_t st) {
  const NormPlan p = norm_plan(dtype, a.width);
  switch (dtype) {
    case LFAMD_F32: return with_plan<float>(p, NormFwd<float, F8>{a, st});
    case LFAMD_F16: return with_plan<f16s>(p, NormFwd<f16s, F8>{a, st});
    default: return with_plan<bf16s>(p, NormFwd<bf16s, F8>{a, st});
  }
}

}  // namespace

}  // namespace lfamd

using namespace lfamd;

extern "C" {

int lfamd_add_rms_norm(int dtype, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                       int w_dtype, const void* weight, void* y, void* sum, float* rstd, int64_t rows, int64_t width,
                       float eps, void* stream) {
  if (int e = check_sizes("add_rms_norm", dtype, w_dtype, rows, width)) return e;
  if (rows == 0) return ok();
  if (!x || !weight || !y || (residual && !sum)) return fail(LFAMD_ERR_ARG, "add_rms_norm: null pointer");
  NormArgs a{};
  a.x = x, a.res = residual, a.w = weight, a.y = y, a.sum = sum, a.rstd = rstd;
  a.xs = x_stride, a.rs = residual_stride, a.rows = rows, a.width = (int)width, a.wf32 = w_dtype == LFAMD_F32, a.eps = eps;
  return norm_forward<false>(dtype, a, (hipStream_t)stream);
}

int lfamd_add_rms_norm_fp8(int dtype, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                           int w_dtype, const void* weight, void* y, float* scale, void* sum, int64_t rows,
                           int64_t width, float eps, void* stream) {
  if (int e = check_sizes("add_rms_norm_fp8", dtype, w_dtype, rows, width)) return e;
  if (rows == 0) return ok();
  if (!x || !weight || !y || !scale || (residual && !sum)) return fail(LFAMD_ERR_ARG, "add_rms_norm_fp8: null pointer");
  NormArgs a{};
  a.x = x, a.res = residual, a.w = weight, a.y = y, a.sum = sum, a.scale = scale;
  a.xs = x_stride, a.rs = residual_stride, a.rows = rows, a.width = (int)width, a.wf32 = w_dtype == LFAMD_F32, a.eps = eps;
  return norm_forward<true>(dtype, a, (hipStream_t)stream);
}

size_t lfamd_add_rms_norm_backward_workspace_size(int dtype, int64_t rows, int64_t width) {
  if (rows <= 0 || width < 1 || width > kNormMaxWidth || rows > INT32_MAX) return 0;
  const int grid = bwd_grid(norm_plan(dtype, (int)width), rows);
  return (size_t)grid * width * sizeof(float);
}

int lfamd_add_rms_norm_backward(int dtype, const void* grad_y, int64_t grad_y_stride, const void* grad_sum,
                                int64_t grad_sum_stride, const void* x, int64_t x_stride, const void* residual,
                                int64_t residual_stride, int w_dtype, const void* weight, const float* rstd,
                                void* grad_x, void* grad_weight, int64_t rows, int64_t width, void* workspace,
                                size_t workspace_bytes, void* stream) {
  const char* who = "add_rms_norm backward";
  if (int e = check_sizes(who, dtype, w_dtype, rows, width)) return e;
  hipStream_t st = (hipStream_t)stream;
  if (rows > 0 && (!grad_y || !x || !weight || !rstd || !grad_x)) return fail(LFAMD_ERR_ARG, "%s: null pointer", who);
  if (rows == 0 && !grad_weight) return ok();
  NormArgs a{};
  a.gy = grad_y, a.gs = grad_sum, a.x = x, a.res = residual, a.w = weight, a.rstd = (float*)rstd, a.dx = grad_x;
  a.gys = grad_y_stride, a.gss = grad_sum_stride, a.xs = x_stride, a.rs = residual_stride;
  a.rows = rows, a.width = (int)width;
  a.wf32 = w_dtype == LFAMD_F32;
  int grid = 0;
  if (rows > 0) {
    const NormPlan p = norm_plan(dtype, (int)width);
    grid = bwd_grid(p, rows);
    if (grad_weight) {
      if (!workspace || workspace_bytes < lfamd_add_rms_norm_backward_workspace_size(dtype, rows, width))
        return fail(LFAMD_ERR_ARG, "%s: workspace too small", who);
      if ((uintptr_t)workspace & 3) return fail(LFAMD_ERR_ARG, "%s: workspace must be 4-byte aligned", who);
      a.part = (float*)workspace;
    }
    int e;
    switch (dtype) {
      case LFAMD_F32: e = with_plan<float>(p, NormBwd<float>{a, st, grid}); break;
      case LFAMD_F16: e = with_plan<f16s>(p, NormBwd<f16s>{a, st, grid}); break;
      default: e = with_plan<bf16s>(p, NormBwd<bf16s>{a, st, grid}); break;
    }
    if (e) return e;
  }
  if (grad_weight) {
    const dim3 g((unsigned)((width + 15) / 16)), b(1024);
    switch (w_dtype) {
      case LFAMD_F32: norm_dw_kernel<float><<<g, b, 0, st>>>(a.part, grid, (int)width, (float*)grad_weight, 1); break;
      case LFAMD_F16: norm_dw_kernel<f16s><<<g, b, 0, st>>>(a.part, grid, (int)width, (f16s*)grad_weight, 0); break;
      default: norm_dw_kernel<bf16s><<<g, b, 0, st>>>(a.part, grid, (int)width, (bf16s*)grad_weight, 0); break;
    }
    return check_launch(who);
  }
  return ok();
}

}  // extern "C"
