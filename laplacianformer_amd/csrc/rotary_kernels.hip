// Rotary positions over several axes. The rotated channels of a head are pairs; pairs
// are dealt to the axes in order, axis a taking n_a of them, and pair j of axis a turns by
//   angle = position_a * base^(-j / n_a).
// Channels behind the pairs pass through. The backward pass is the rotation by -angle.
//
// The angle is reduced in integers: base^(-j / n) / (2 pi) is held as a 96-bit fraction of a
// turn (rotary_turns.h), and position * fraction modulo 2^96 is the turn's fractional part: a position of
// 63 bits moves it by 2^-33 turns at most. Its upper 32 bits go through sincospi in fp32.
//
// Memory-bound. A workgroup takes 16 tokens of a sequence: it computes their cosines
// and sines into LDS once, then walks the heads of q and of k with 16-byte accesses
// (single elements where strides or head size leave no vectors). 16 tokens: enough work per workgroup to
// hide the table behind other workgroups' loads, few enough for small grids. 671 MB (20 heads of 16 x 32 x 32 tokens
// at 128 channels) take 127 to 138 us, the rate of a large copy; single elements take 2.7 to 3.2 times their
// share of that (heads of 40, 50 and 72 channels over two axes).
#include <math.h>

#include "lf_common.h"
#include "lf_internal.h"
#include "rotary_turns.h"

namespace lfamd {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxPairs = 128, kTokens = 16, kMaxAxes = 8;

struct RotaryArgs {
  const void *x[2];
  void *y[2];
  int64_t xs[2][3], ys[2][3];  // batch, head, token
  int heads[2];
  const void* pos;
  int64_t ps[3];               // axis, batch, token
  int pos64, N, D, pairs, headsPerBlock;
  float sign;                  // -1: the inverse rotation
  uint64_t turn[kMaxPairs];    // the fraction's upper 64 bits
  uint32_t low[kMaxPairs];     // its next 32
  uint8_t axis[kMaxPairs];
};

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  __shared__ float2 cs[kTokens * kMaxPairs];
  const int tok0 = blockIdx.x * kTokens, b = blockIdx.y, tokens = min(kTokens, a.N - tok0);
  const int P = a.pairs;
  for (int i = threadIdx.x; i < tokens * P; i += 256) {
    const int t = i / P, p = i - t * P;
    const int64_t off = a.axis[p] * a.ps[0] + b * a.ps[1] + (int64_t)(tok0 + t) * a.ps[2];
    const int64_t pos = a.pos64 ? ((const int64_t*)a.pos)[off] : (int64_t)((const int32_t*)a.pos)[off];
    // Bits 32 .. 95 of the signed position times the fraction.
    const uint64_t up = (uint64_t)pos * a.turn[p] + ((uint64_t)(uint32_t)pos * a.low[p] >> 32) + (uint64_t)((pos >> 32) * (int64_t)a.low[p]);
    const int32_t f = (int32_t)(up >> 32);                           // of a turn, times 2^32
    float s, c;
    sincospif((float)f * 4.656612873077393e-10f, &s, &c);            // 2^-31: half turns
    cs[i] = make_float2(c, s * a.sign);
  }
  __syncthreads();

  // Work items of one token and head: V pairs (INTER: V / 2), or V channels that pass.
  constexpr int PV = INTER ? (V == 1 ? 1 : V / 2) : V;
  const int rot = P / PV, items = rot + (a.D - 2 * P) / V;
  const int first = blockIdx.z * a.headsPerBlock, total = a.heads[0] + a.heads[1];
  const int last = min(first + a.headsPerBlock, total);
  const int perHead = tokens * items;
  for (int i = threadIdx.x; i < (last - first) * perHead; i += 256) {
    const int hd = i / perHead, r = i - hd * perHead, t = r / items, it = r - t * items;
    int head = first + hd;
    const int w = head >= a.heads[0];
    if (w) head -= a.heads[0];
    const T* x = (const T*)a.x[w] + b * a.xs[w][0] + head * a.xs[w][1] + (int64_t)(tok0 + t) * a.xs[w][2];
    T* y = (T*)a.y[w] + b * a.ys[w][0] + head * a.ys[w][1] + (int64_t)(tok0 + t) * a.ys[w][2];
    if (it >= rot) {
      const int c = 2 * P + (it - rot) * V;
      if constexpr (V == 1) y[c] = x[c];
      else *(u32x4*)(y + c) = *(const u32x4*)(x + c);
      continue;
    }
    const float2* tcs = cs + t * P + it * PV;
    if constexpr (INTER) {
      const int c = 2 * it * PV;
      T e[2 * PV], o[2 * PV];
      if constexpr (V == 1) e[0] = x[c], e[1] = x[c + 1];
      else *(u32x4*)e = *(const u32x4*)(x + c);
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        const float2 k = tcs[j];
        const float u = to_acc(e[2 * j]), v = to_acc(e[2 * j + 1]);
        o[2 * j] = from_acc<T>(fmaf(u, k.x, -(v * k.y)));
        o[2 * j + 1] = from_acc<T>(fmaf(u, k.y, v * k.x));
      }
      if constexpr (V == 1) y[c] = o[0], y[c + 1] = o[1];
      else *(u32x4*)(y + c) = *(const u32x4*)o;
    } else {
      const int c = it * PV;
      T e[PV], f[PV], o[PV], p[PV];
      if constexpr (V == 1) {
        e[0] = x[c], f[0] = x[c + P];
      } else {
        *(u32x4*)e = *(const u32x4*)(x + c);
        *(u32x4*)f = *(const u32x4*)(x + c + P);
      }
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        const float2 k = tcs[j];
        const float u = to_acc(e[j]), v = to_acc(f[j]);
        o[j] = from_acc<T>(fmaf(u, k.x, -(v * k.y)));
        p[j] = from_acc<T>(fmaf(u, k.y, v * k.x));
      }
      if constexpr (V == 1) {
        y[c] = o[0], y[c + P] = p[0];
      } else {
        *(u32x4*)(y + c) = *(const u32x4*)o;
        *(u32x4*)(y + c + P) = *(const u32x4*)p;
      }
    }
  }
}

template <typename T> int rotary_launch(const RotaryArgs& a, int64_t B, bool vec, bool inter, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const int heads = a.heads[0] + a.heads[1];
  const dim3 grid((unsigned)((a.N + kTokens - 1) / kTokens), (unsigned)B,
                  (unsigned)((heads + a.headsPerBlock - 1) / a.headsPerBlock));
  if (vec && inter) rotary_kernel<T, V, true><<<grid, 256, 0, st>>>(a);
  else if (vec) rotary_kernel<T, V, false><<<grid, 256, 0, st>>>(a);
  else if (inter) rotary_kernel<T, 1, true><<<grid, 256, 0, st>>>(a);
  else rotary_kernel<T, 1, false><<<grid, 256, 0, st>>>(a);
  return check_launch("rotary");
}

}  // namespace

}  // namespace lfamd

using namespace lfamd;

extern "C" int lfamd_rotary(int dtype, const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides,
                            int64_t q_heads, const void* k, const int64_t* k_strides, void* k_out,
                            const int64_t* k_out_strides, int64_t k_heads, int64_t batch, int64_t tokens, int64_t head_dim,
                            const void* positions, int positions_64, const int64_t* position_strides, int num_axes,
                            const int64_t* sections, double base, int interleaved, int inverse, void* stream) {
  if (dtype != LFAMD_F32 && dtype != LFAMD_F16 && dtype != LFAMD_BF16)
    return fail(LFAMD_ERR_DTYPE, "rotary: unsupported dtype %d", dtype);
  if (batch < 0 || tokens < 0 || head_dim < 0 || q_heads < 0 || k_heads < 0) return fail(LFAMD_ERR_ARG, "rotary: negative size");
  if (num_axes < 1 || num_axes > kMaxAxes || !sections)
    return fail(LFAMD_ERR_UNSUPPORTED, "rotary: %d axes, 1 to %d are taken", num_axes, kMaxAxes);
  if (!(base > 0.0) || !isfinite(base)) return fail(LFAMD_ERR_ARG, "rotary: base must be positive and finite");
  RotaryArgs a{};
  int64_t pairs = 0;
  for (int i = 0; i < num_axes; ++i) {
    if (sections[i] < 0 || sections[i] > kMaxPairs) return fail(LFAMD_ERR_ARG, "rotary: section %d has %lld pairs", i, (long long)sections[i]);
    turn128 turns[kMaxPairs];
    rotary_turns(base, (int)sections[i], turns);
    for (int64_t j = 0; j < sections[i] && pairs + j < kMaxPairs; ++j) {
      a.turn[pairs + j] = (uint64_t)(turns[j] >> 64), a.low[pairs + j] = (uint32_t)(turns[j] >> 32);
      a.axis[pairs + j] = (uint8_t)i;
    }
    pairs += sections[i];
  }
  if (pairs < 1 || pairs > kMaxPairs || 2 * pairs > head_dim)
    return fail(LFAMD_ERR_ARG, "rotary: the sections hold %lld pairs, head size %lld has room for %lld (at most %d)",
                (long long)pairs, (long long)head_dim, (long long)(head_dim / 2), kMaxPairs);
  const int64_t heads = q_heads + k_heads;
  if (batch == 0 || tokens == 0 || heads == 0) return ok();
  if ((q_heads && (!q || !q_out || !q_strides || !q_out_strides)) || (k_heads && (!k || !k_out || !k_strides || !k_out_strides)) ||
      !positions || !position_strides)
    return fail(LFAMD_ERR_ARG, "rotary: null pointer");
  if (batch > 65535 || tokens > (1 << 27) || heads > 65535 || head_dim > 1024)
    return fail(LFAMD_ERR_UNSUPPORTED, "rotary: batch, heads <= 65535, tokens <= 2^27 and head size <= 1024 are taken");
  const int V = dtype == LFAMD_F32 ? 4 : 8;
  bool vec = head_dim % V == 0 && (interleaved ? 2 * pairs : pairs) % V == 0;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  const int64_t* is[2] = {q_strides, k_strides};
  const int64_t* os[2] = {q_out_strides, k_out_strides};
  const int64_t nh[2] = {q_heads, k_heads};
  for (int w = 0; w < 2; ++w) {
    if (!nh[w]) continue;
    a.x[w] = in[w], a.y[w] = out[w], a.heads[w] = (int)nh[w];
    if (((uintptr_t)in[w] | (uintptr_t)out[w]) & 15) vec = false;
    for (int i = 0; i < 3; ++i) {
      a.xs[w][i] = is[w][i], a.ys[w][i] = os[w][i];
      if (is[w][i] % V || os[w][i] % V) vec = false;
    }
  }
  a.pos = positions, a.pos64 = positions_64;
  for (int i = 0; i < 3; ++i) a.ps[i] = position_strides[i];
  a.N = (int)tokens, a.D = (int)head_dim, a.pairs = (int)pairs, a.sign = inverse ? -1.0f : 1.0f;
  // All heads of 16 tokens in one workgroup share its cosines and sines; fewer per
  // workgroup where that leaves CUs without one.
  const int64_t blocks = batch * ((tokens + kTokens - 1) / kTokens), want = 2 * (int64_t)num_cus();
  int64_t groups = blocks >= want ? 1 : (want + blocks - 1) / blocks;
  if (groups > heads) groups = heads;
  a.headsPerBlock = (int)((heads + groups - 1) / groups);
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case LFAMD_F32: return rotary_launch<float>(a, batch, vec, interleaved, st);
    case LFAMD_F16: return rotary_launch<f16s>(a, batch, vec, interleaved, st);
    default: return rotary_launch<bf16s>(a, batch, vec, interleaved, st);
  }
}
