// softmax_attention, forward:  o_i = sum_j p_ij v_j,  p_i = softmax_j(scale q_i . k_j + mask_ij).
//
// One pass over the keys with the running maximum and sum of each row. The query
// heads that share a key head are laid end to end, so that a workgroup's rows are
// taken from G * N rows, whatever their number. Scores are formed as S^T = K Q^T
// and the output as O^T = V^T P^T: a lane owns one query in both, so that the
// softmax needs one exchange between lane halves per tile and P goes from the one
// product's accumulators to the other's operand within the lane's registers.
//
// Units: without an additive mask the scores stay unscaled in the accumulators and the row
// reference m is in log2 units, p = exp2(c S - m) with c = scale log2 e (one fma and
// one exp2 per score). With one, x = scale S + mask in natural units, as an
// additive mask may hold the type's lowest value, and p = exp2((x - m) log2 e). A mask of truth
// values is packed into bits first (attn_bits_kernel), whatever its strides: a lane then takes its
// keys of a tile by one load, a tile ahead, and the scores stay in the units of no mask.
// P is rounded to the element type for the product with V; its sum is of the
// unrounded values.
//
// Row statistics for the backward pass, [B][H][N] planes: without an additive mask one plane,
// m + log2(sum) (+inf for a row without keys: its p is then 0); with one two, m
// and 1 / sum, since m + log(sum) loses the sum where m is the type's lowest value. For the
// 16-bit types what the output's rounding took off follows, so that the backward's
// delta = rowsum(g o) is of the fp32 output: where few keys weigh in, o is of the size of v, and
// its half step in delta was the third that the gradients of q and k carried (2.8e-3 against 2.4e-3 in bf16).
//
// What bounds it (one MI355X, bf16): 8192 x 8192 causal at 128 channels and 32 heads runs 544 us, 1.01 PFLOP/s at
// the power-limited 1.6 GHz with the matrix cores busy half the cycles and the VALU (an fma, an exp2, an add,
// half a maximum and half a rounding per score) the other half, 85 % of a large library product's rate;
// 4096 x 4096 at 64 channels and 64 heads 326 us, VALU issue 75 %. 128 rows per workgroup (32 per wave) keep two
// (64 channels: three) waves per SIMD, whose products and softmaxes overlap; a 64-key tile is what four waves load
// while they compute on the other. One token over 8192 keys (16 sequences, 8 key heads, 128 channels): 81 us
// for 403 MB, 4.97 TB/s, the rate of a large copy.
#include "attn_common.h"

namespace lfamd {

namespace {

template <int KS> constexpr int key_tile() { return KS == 1 ? 64 : 128; }

template <typename T, int DP, int KS> constexpr int num_buffers() {
  return 4 * key_tile<KS>() * DP * (int)sizeof(T) <= 128 * 1024 ? 2 : 1;
}

// 32 queries per wave. KS: 1, the four waves take different queries; 4,
// they take different keys of each tile and their results are joined at the end.
template <typename T, int DC, int KS, int FORM>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && DC >= 96 ? 1 : 2) attn_fwd_kernel(const AttnArgs a) {
  constexpr bool MASK = FORM == kAdd;
  constexpr int DP = row_pitch(DC), KT = key_tile<KS>(), NBUF = num_buffers<T, DP, KS>(), NT = DC / 16, ND = DC / 32;
  constexpr int KB = KS == 1 ? KT / 32 : 1;  // 32-key blocks per wave and tile
  constexpr int ROWS = KS == 1 ? 128 : 32;
  using L = Tile<T, DP>;
  constexpr int TB = KT * L::ROW;  // bytes of one tile
  extern __shared__ __align__(16) char smem[];

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t place = xcd_place(blockIdx.x, gridDim.x);
  const int split = place % a.nsplit, t0 = place / a.nsplit;
  const int bh = t0 / a.tiles, tile = a.tiles - 1 - t0 % a.tiles;  // the longest rows of a causal mask first
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int R = a.G * a.N, row0 = tile * ROWS + (KS == 1 ? wave * 32 : 0);
  const int klen = key_count(a, b), qlen = query_count(a, b), qstart = query_start(a, b);

  // Bounds of the keys that any row of the workgroup, or every row of the wave, sees.
  auto last_key = [&](int first, int count) {
    if (!a.causal) return klen;
    const int end = min(first + count, R) - 1;
    const int n = end < first || a.divN.div(end) != a.divN.div(first) ? a.N - 1 : end - (int)a.divN.div(end) * a.N;
    return min(klen, qstart + n + 1);
  };
  const int kendAll = max(last_key(tile * ROWS, ROWS), 0);
  const int kbeg = split * a.chunk * KT, kend = min(kendAll, kbeg + a.chunk * KT);
  const int wend = row0 < R ? min(kend, last_key(row0, 32)) : 0;

  // This lane's queries.
  const bool stored = row0 + (lane & 31) < R;
  const int qrow = stored ? row0 + (lane & 31) : 0;
  const int g = a.divN.div(qrow), n = qrow - g * a.N, hq = hk * a.G + g;
  const bool alive = stored && n < qlen;
  const int lim = !alive ? 0 : a.causal ? min(klen, qstart + n + 1) : klen;
  const int64_t qoff = (int64_t)b * a.qs[0] + (int64_t)hq * a.qs[1] + (int64_t)n * a.qs[2];
  const int64_t ooff = (int64_t)b * a.os[0] + (int64_t)hq * a.os[1] + (int64_t)n * a.os[2];
  const int64_t soff = ((int64_t)b * a.H + hq) * a.N + n;
  const int64_t moff = FORM == kBits ? (int64_t)b * a.bs[0] + (int64_t)hq * a.bs[1] + (int64_t)n * a.bs[2]
                                     : (int64_t)b * a.ms[0] + (int64_t)hq * a.ms[1] + (int64_t)n * a.ms[2];
  int full = klen;  // every row of the wave sees the keys in front of it
  if (a.causal) {   // a row behind R or qlen needs no check: what it computes is not used
    int f = alive ? lim : klen;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) f = min(f, __shfl_xor(f, s));
    full = uniform(f);
  }

  Frag<T> qf[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) qf[t] = global_frag<T>((const T*)a.q + qoff, alive, t, h, a.D);

  f32x16 o[ND];
  float m = kNegInf, l = 0.0f;
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x16{};

  // The next tile to fill.
  const T* knext = (const T*)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[1] + (int64_t)kbeg * a.ks[2];
  const T* vnext = (const T*)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[1] + (int64_t)kbeg * a.vs[2];
  using LD = Loader<T, DP, DC, KT>;
  // Keys that a mask takes from every query are not read either: what they hold is nobody's.
  const bool byKey = FORM != kNoMask && a.keyMask;
  auto fill = [&](int buf, int key0, uint32_t live) {
    LD::fill(smem + buf * 2 * TB, knext, a.ks[2], key0, kend, a.D, a.modeK, live);
    LD::fill(smem + buf * 2 * TB + TB, vnext, a.vs[2], key0, kend, a.D, a.modeV, live);
    knext += KT * a.ks[2];
    vnext += KT * a.vs[2];
  };

  // A row's bits of the wave's keys of one tile.
  auto load_bits = [&](int key0) {
    const uint32_t* p = a.bits + moff + key0 / 32;
    if constexpr (KS == 4) return (uint64_t)p[wave];
    else return *(const uint64_t*)p;
  };
  uint64_t bits = 0;
  uint32_t live = ~0u;  // of the next tile to fill
  if (kbeg < kend) {
    if constexpr (FORM == kBits) bits = load_bits(kbeg);
    if (byKey) live = live_keys<LD>(a, b, kbeg);
    fill(0, kbeg, live);
    if (NBUF == 2 && byKey) live = live_keys<LD>(a, b, kbeg + KT);
  }
  land();
  __syncthreads();
  const int rl0 = L::row_lane(lane), cl0 = L::col_lane(lane);
  int buf = 0;
  for (int key0 = kbeg; key0 < kend; key0 += KT) {
    const bool more = key0 + KT < kend;
    if (NBUF == 2 && more) fill(buf ^ 1, key0 + KT, live);
    if (byKey) live = live_keys<LD>(a, b, key0 + (NBUF == 2 ? 2 : 1) * KT);
    const uint64_t now = bits;
    if constexpr (FORM == kBits)
      if (more) bits = load_bits(key0 + KT);
    const int rl = launder(rl0), cl = launder(cl0);
    const char* tk = smem + buf * 2 * TB;
    const char* tv = tk + TB;
    const int wkey = key0 + (KS == 1 ? 0 : 32 * wave);
    if (wkey < wend) {
      f32x16 bias[MASK ? KB : 1];
      if constexpr (MASK) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) mask_of_keys(a, moff, wkey + 32 * kb, h, bias[kb]);
      }
      f32x16 s[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[kb] = f32x16{};
      // At two waves per SIMD (DC >= 96) the one in its products goes first: 8192 causal keys at 128 channels
      // 658 -> 646 us, but 332 -> 352 us for 4096 x 4096 at 64, where three waves share a SIMD.
      if constexpr (DC >= 96) __builtin_amdgcn_s_setprio(1);
      const char* tkw = tk + (KS == 1 ? 0 : 32 * wave) * L::ROW;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const Frag<T> kf = L::row_frag(tkw + 32 * kb * L::ROW, rl, t);
          s[kb] = mma<T>(kf, qf[t], s[kb]);
        }
      if constexpr (sizeof(T) == 2) reads_ahead<KB * NT, (KB * NT < 4 ? KB * NT : 4)>();
      if constexpr (DC >= 96) __builtin_amdgcn_s_setprio(0);
      // The mask, and what lies behind the row's last key.
      if constexpr (FORM == kBits) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const uint32_t w = ((uint32_t)(now >> (32 * kb)) & bits_below(lim, wkey + 32 * kb)) >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = w & (1u << (8 * (r >> 2) + (r & 3))) ? s[kb][r] : kNegInf;
        }
      } else if (MASK || wkey + 32 * KB > full) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = wkey + 32 * kb + 8 * (r >> 2) + 4 * h + (r & 3);
            if constexpr (MASK) {
              s[kb][r] = j < lim ? masked_score(a, s[kb][r], bias[kb][r]) : kNegInf;
            } else {
              s[kb][r] = j < lim ? s[kb][r] : kNegInf;
            }
          }
      }
      float mx = s[0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
      mx = half_max(mx);
      if (!MASK) mx *= a.c;
      // The reference follows the maximum only when that has grown by 2^8: p stays
      // below 2^8, which every element type holds at full precision, and the
      // accumulators are rescaled in few tiles.
      const float slack = MASK ? 8.0f / kLog2e : 8.0f;
      if (__any(mx > m + slack)) {
        const float mn = fmaxf(m, mx), ms = mn == kNegInf ? 0.0f : mn;
        const float alpha = exp2_fast(MASK ? (m - ms) * kLog2e : m - ms);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      }
      const float ref = m == kNegInf ? 0.0f : m;
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = exp2_fast(MASK ? (s[kb][r] - ref) * kLog2e : fmaf(s[kb][r], a.c, -ref));
          s[kb][r] = p;
          sum += p;
        }
      l += sum;
      if constexpr (DC >= 96) __builtin_amdgcn_s_setprio(1);
      const char* tvw = tv + (KS == 1 ? 0 : 32 * wave) * L::ROW;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const Frag<T> pf = acc_frag<T>(s[kb], st);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const Frag<T> vf = L::col_frag(tvw + 32 * kb * L::ROW, cl, st, d);
            o[d] = mma<T>(vf, pf, o[d]);
          }
        }
      if constexpr (DC >= 96) __builtin_amdgcn_s_setprio(0);
    }
    if (NBUF == 1) {
      __syncthreads();
      if (more) fill(0, key0 + KT, live);
    } else {
      buf ^= 1;
    }
    land();
    __syncthreads();
  }

  l = half_sum(l);

  constexpr float kUnit = MASK ? kLog2e : 1.0f;
  if constexpr (KS == 4) {
    // Join the four waves' results through LDS (the loop's last barrier has passed).
    constexpr int PS = DC + 4;  // floats per row: rows start four banks apart
    static_assert(4 * 32 * (PS + 2) * 4 <= 2 * NBUF * TB, "the tiles' LDS holds the partial results");
    float* po = (float*)smem;
    float* pm = po + 4 * 32 * PS;
    float* pl = pm + 128;
    const int q = lane & 31;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        *(f32x4*)(po + (wave * 32 + q) * PS + 32 * d + 8 * gq + 4 * h) =
            (f32x4){o[d][4 * gq], o[d][4 * gq + 1], o[d][4 * gq + 2], o[d][4 * gq + 3]};
    if (h == 0) {
      pm[wave * 32 + q] = m;
      pl[wave * 32 + q] = l;
    }
    __syncthreads();
    // Wave w takes columns 8 w + 4 h of every 32.
    float mt = kNegInf;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, pm[w * 32 + q]);
    const float ref = mt == kNegInf ? 0.0f : mt;
    float lt = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = exp2_fast((pm[w * 32 + q] - ref) * kUnit);
      lt += f[w] * pl[w * 32 + q];
    }
    if (!stored) return;
    const float inv = a.nsplit > 1 ? 1.0f : lt == 0.0f ? 0.0f : 1.0f / lt;
    const bool live = alive;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int c0 = 32 * d + 8 * wave + 4 * h;
      f32x4 x = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) x += f[w] * *(const f32x4*)(po + (w * 32 + q) * PS + c0);
      x *= inv;
      if (!live) x = f32x4{0, 0, 0, 0};
      if (a.nsplit > 1) {
        *(f32x4*)(a.part + (((int64_t)split * a.B * a.Hk + bh) * R + qrow) * DC + c0) = x;
      } else {
        store4<T>((T*)a.out + ooff, c0, a.D, x[0], x[1], x[2], x[3]);
        if constexpr (sizeof(T) == 2)
          if (a.stat) store4_rest<T>(rest_row<T>(a, soff), c0, a.D, x[0], x[1], x[2], x[3]);
      }
    }
    if (wave == 0 && h == 0) {
      if (a.nsplit > 1) {
        float* ps = a.part + (int64_t)a.nsplit * a.B * a.Hk * R * DC + (((int64_t)split * a.B * a.Hk + bh) * R + qrow) * 2;
        ps[0] = live ? mt : kNegInf;
        ps[1] = live ? lt : 0.0f;
      } else if (a.stat) {
        const bool none = !live || lt == 0.0f;
        if (MASK) {
          a.stat[soff] = none ? 0.0f : mt;
          a.stat[(int64_t)a.B * a.H * a.N + soff] = none ? 0.0f : 1.0f / lt;
        } else {
          a.stat[soff] = none ? __builtin_inff() : mt + log2f(lt);
        }
      }
    }
  } else {
    if (!stored) return;
    const bool none = !alive || l == 0.0f;
    const float inv = a.nsplit > 1 ? 1.0f : none ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        const int c0 = 32 * d + 8 * gq + 4 * h;
        f32x4 x = {o[d][4 * gq], o[d][4 * gq + 1], o[d][4 * gq + 2], o[d][4 * gq + 3]};
        x *= inv;
        if (none) x = f32x4{0, 0, 0, 0};
        if (a.nsplit > 1) {
          *(f32x4*)(a.part + (((int64_t)split * a.B * a.Hk + bh) * R + qrow) * DC + c0) = x;
        } else {
          store4<T>((T*)a.out + ooff, c0, a.D, x[0], x[1], x[2], x[3]);
          if constexpr (sizeof(T) == 2)
            if (a.stat) store4_rest<T>(rest_row<T>(a, soff), c0, a.D, x[0], x[1], x[2], x[3]);
        }
      }
    if (h == 0) {
      if (a.nsplit > 1) {
        float* ps = a.part + (int64_t)a.nsplit * a.B * a.Hk * R * DC +
                    (((int64_t)split * a.B * a.Hk + bh) * R + qrow) * 2;
        ps[0] = none ? kNegInf : m;
        ps[1] = none ? 0.0f : l;
      } else if (a.stat) {
        if (MASK) {
          a.stat[soff] = none ? 0.0f : m;
          a.stat[(int64_t)a.B * a.H * a.N + soff] = none ? 0.0f : 1.0f / l;
        } else {
          a.stat[soff] = none ? __builtin_inff() : m + log2f(l);
        }
      }
    }
  }
}

// Joins the key splits' partial results. DC / 4 threads (32 for 96) take a row's columns, four
// each; SHARE: a workgroup has one row, whose splits its groups of threads divide (few rows),
// else each group has a row of its own.
template <typename T, int DC, bool MASK, bool SHARE>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
  constexpr int TPR = DC == 96 ? 32 : DC / 4, GROUPS = 256 / TPR;
  constexpr float kUnit = MASK ? kLog2e : 1.0f;
  const int64_t R = (int64_t)a.G * a.N, total = (int64_t)a.B * a.Hk * R;
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR, c0 = t * 4, lane0 = (threadIdx.x & 63) - t;
  const int64_t at = SHARE ? blockIdx.x : (int64_t)blockIdx.x * GROUPS + grp, row = at < total ? at : total - 1;
  const float* ps = a.part + (int64_t)a.nsplit * total * DC;
  const int first = SHARE ? grp : 0, step = SHARE ? GROUPS : 1;
  const int mine = (a.nsplit - first + step - 1) / step;  // splits of this group: first + i step
  float m = kNegInf;
  for (int s = t; s < a.nsplit; s += TPR) m = fmaxf(m, ps[(s * total + row) * 2]);
#pragma unroll
  for (int i = 1; i < TPR; i <<= 1) m = fmaxf(m, __shfl_xor(m, i));
  const float ref = m == kNegInf ? 0.0f : m;
  float l = 0.0f;
  f32x4 x = {0, 0, 0, 0};
  for (int i0 = 0; i0 < mine; i0 += TPR) {
    const int own = first + min(i0 + t, mine - 1) * step;
    const f32x2 st = *(const f32x2*)(ps + (own * total + row) * 2);
    const float f = i0 + t < mine ? exp2_fast((st[0] - ref) * kUnit) : 0.0f;
    l += f * st[1];
    const int n = min(TPR, mine - i0);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const f32x4 y = *(const f32x4*)(a.part + ((first + (i0 + i) * step) * total + row) * DC + min(c0, DC - 4));
      x += __shfl(f, lane0 + i) * y;
    }
  }
#pragma unroll
  for (int i = 1; i < TPR; i <<= 1) l += __shfl_xor(l, i);
  if constexpr (SHARE) {
    __shared__ float sx[256][4], sl[GROUPS];
    *(f32x4*)sx[threadIdx.x] = x;
    if (t == 0) sl[grp] = l;
    __syncthreads();
    if (grp) return;
    l = 0.0f;
    x = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      l += sl[g];
      x += *(const f32x4*)sx[g * TPR + t];
    }
  }
  if (at >= total || c0 >= DC) return;
  const bool none = l == 0.0f;
  x *= none ? 0.0f : 1.0f / l;
  if (none) x = f32x4{0, 0, 0, 0};
  const int bh = (int)(row / R), r = (int)(row % R), b = bh / a.Hk, hk = bh % a.Hk;
  const int g = a.divN.div(r), n = r - g * a.N, hq = hk * a.G + g;
  T* out = (T*)a.out + (int64_t)b * a.os[0] + (int64_t)hq * a.os[1] + (int64_t)n * a.os[2];
  store4<T>(out, c0, a.D, x[0], x[1], x[2], x[3]);
  const int64_t so = ((int64_t)b * a.H + hq) * a.N + n;
  if constexpr (sizeof(T) == 2)
    if (a.stat) store4_rest<T>(rest_row<T>(a, so), c0, a.D, x[0], x[1], x[2], x[3]);
  if (a.stat && c0 == 0) {
    if (MASK) {
      a.stat[so] = none ? 0.0f : m;
      a.stat[(int64_t)a.B * a.H * a.N + so] = none ? 0.0f : 1.0f / l;
    } else {
      a.stat[so] = none ? __builtin_inff() : m + log2f(l);
    }
  }
}

// A mask of truth values as bits: one word of 32 keys per thread, rows of `words` words; bytes that are not
// zero are ones, keys behind M zeros. The mask's own sizes (1 where it is broadcast): heads Hm, rows Nm.
__global__ void __launch_bounds__(256) attn_bits_kernel(const uint8_t* mask, int64_t s0, int64_t s1, int64_t s2, int64_t s3,
                                                        uint32_t* bits, int Hm, int Nm, int M, int words, int64_t total) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int w = (int)(id % words);
  const int64_t row = id / words, n = row % Nm, bh = row / Nm;
  const uint8_t* p = mask + bh / Hm * s0 + bh % Hm * s1 + n * s2;
  uint32_t out = 0;
  if (s3 == 1 && 32 * w + 32 <= M) {
    u32x4 x[2];
    __builtin_memcpy(x, p + 32 * w, 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t y = x[i >> 2][i & 3];
      const uint32_t t = ((((y & 0x7f7f7f7fu) + 0x7f7f7f7fu) | y) & 0x80808080u) >> 7;  // bits 0, 8, 16, 24
      out |= ((t | t >> 7 | t >> 14 | t >> 21) & 15u) << (4 * i);
    }
  } else {
    for (int i = 0; i < 32; ++i) {
      const int j = 32 * w + i;
      if (j < M) out |= (uint32_t)(p[j * s3] != 0) << i;
    }
  }
  bits[id] = out;
}

// How a call is laid over the chip.
struct FwdPlan {
  int ks, rows, kt, tiles, nsplit, chunk, dc;
};

FwdPlan fwd_plan(int dtype, const AttnArgs& a, int cus) {
  FwdPlan p;
  const int64_t R = (int64_t)a.G * a.N;
  p.dc = compute_dim(a.D);
  // Up to 32 rows per key head fill one wave's block: the four waves then share the
  // rows and divide each tile's keys.
  p.ks = R <= 32 ? 4 : 1;
  p.rows = p.ks == 4 ? 32 : 128;
  p.kt = p.ks == 4 ? 128 : 64;
  p.tiles = (int)((R + p.rows - 1) / p.rows);
  const int64_t wgs = (int64_t)a.B * a.Hk * p.tiles;
  const int steps = (a.M + p.kt - 1) / p.kt;
  // The keys are split where the rows alone leave CUs without work. A tile's throughput: its products at
  // the 3.5 TFLOP/s that a CU reaches (fp32: 0.5), its 8192 exponentials at least. Its latency as measured
  // where a CU has one workgroup; an additive mask's loads add to both.
  const double thr = std::max(0.5, 4.0 * (p.ks == 4 ? 32 * 128 : 128 * 64) * p.dc / (dtype == LFAMD_F32 ? 0.5e6 : 3.5e6)) +
                     (a.maskKind > kMaskBool ? 0.4 : 0.0);
  const double lat = std::max((p.ks == 4 ? 1.0 : p.dc <= 64 ? 1.5 : 2.0) + (a.maskKind > kMaskBool ? 1.5 : 0.0), thr);
  const int ns = best_split(wgs, steps, cus, lat, thr, (double)a.B * a.Hk * R * p.dc * sizeof(float));
  p.chunk = std::max(1, (steps + ns - 1) / ns);
  p.nsplit = std::max(1, (steps + p.chunk - 1) / p.chunk);
  return p;
}

template <typename T, int DC, int FORM> int fwd_launch(const AttnArgs& a, const FwdPlan& p, hipStream_t st) {
  constexpr int DP = row_pitch(DC);
  constexpr bool MASK = FORM == kAdd;
  const void* fn = p.ks == 4 ? (const void*)attn_fwd_kernel<T, DC, 4, FORM> : (const void*)attn_fwd_kernel<T, DC, 1, FORM>;
  const int nbuf = p.ks == 4 ? num_buffers<T, DP, 4>() : num_buffers<T, DP, 1>();
  const size_t lds = (size_t)2 * nbuf * p.kt * DP * sizeof(T);
  if (int e = set_dyn_lds(fn, lds, "softmax_attention")) return e;
  if (int e = check_fit(fn, 256, lds, "softmax_attention")) return e;
  const unsigned grid = (unsigned)((int64_t)a.B * a.Hk * p.tiles * p.nsplit);
  AttnArgs args = a;
  void* params[] = {&args};
  if (hipLaunchKernel(fn, dim3(grid), dim3(256), params, lds, st) != hipSuccess)
    return check_launch("softmax_attention");
  if (int e = check_launch("softmax_attention")) return e;
  if (p.nsplit > 1) {
    const int64_t rows = (int64_t)a.B * a.Hk * a.G * a.N;
    constexpr int RPB = 256 / (DC == 96 ? 32 : DC / 4);
    // Up to eight workgroups per CU, a row each: what counts is the depth of the loop over the splits.
    if (rows <= 8 * (int64_t)num_cus()) attn_join_kernel<T, DC, MASK, true><<<dim3((unsigned)rows), dim3(256), 0, st>>>(a);
    else attn_join_kernel<T, DC, MASK, false><<<dim3((unsigned)((rows + RPB - 1) / RPB)), dim3(256), 0, st>>>(a);
    return check_launch("softmax_attention (join)");
  }
  return ok();
}

template <typename T, int DC> int fwd_mask(const AttnArgs& a, const FwdPlan& p, hipStream_t st) {
  switch (a.maskKind) {
    case kMaskNone: return fwd_launch<T, DC, kNoMask>(a, p, st);
    case kMaskBool: return fwd_launch<T, DC, kBits>(a, p, st);
    default: return fwd_launch<T, DC, kAdd>(a, p, st);
  }
}

template <typename T> int fwd_dim(const AttnArgs& a, const FwdPlan& p, hipStream_t st) {
  switch (p.dc) {
    case 32: return fwd_mask<T, 32>(a, p, st);
    case 64: return fwd_mask<T, 64>(a, p, st);
    case 96: return fwd_mask<T, 96>(a, p, st);
    default: return fwd_mask<T, 128>(a, p, st);
  }
}

}  // namespace

namespace {

// The mask's own sizes, its broadcast dimensions taken once.
struct BitsShape {
  int64_t B, H, N, words;
};
BitsShape bits_shape(const AttnArgs& a) {
  return {a.ms[0] ? a.B : 1, a.ms[1] ? a.H : 1, a.ms[2] ? a.N : 1, (int64_t)(a.M + 127) / 128 * 4};
}

}  // namespace

size_t attn_bits_bytes(const AttnArgs& a) {
  if (a.maskKind != kMaskBool) return 0;
  const BitsShape s = bits_shape(a);
  return ((size_t)(s.B * s.H * s.N * s.words) * sizeof(uint32_t) + 255) / 256 * 256;
}

int attn_pack_bits(AttnArgs& a, void* workspace, hipStream_t st) {
  if (a.maskKind != kMaskBool) return LFAMD_OK;
  const BitsShape s = bits_shape(a);
  a.bits = (uint32_t*)workspace;
  a.bs[0] = s.B > 1 ? s.H * s.N * s.words : 0;
  a.bs[1] = s.H > 1 ? s.N * s.words : 0;
  a.bs[2] = s.N > 1 ? s.words : 0;
  const int64_t total = s.B * s.H * s.N * s.words;
  if ((total + 255) / 256 > kMostWorkgroups) return fail(LFAMD_ERR_UNSUPPORTED, "softmax_attention: the mask is too large");
  attn_bits_kernel<<<dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st>>>(
      (const uint8_t*)a.mask, a.ms[0], a.ms[1], a.ms[2], a.ms[3], a.bits, (int)s.H, (int)s.N, a.M, (int)s.words, total);
  return check_launch("softmax_attention (mask)");
}

size_t attn_fwd_workspace(int dtype, const AttnArgs& a) {
  const FwdPlan p = fwd_plan(dtype, a, num_cus());
  const size_t part = p.nsplit <= 1 ? 0 : (size_t)p.nsplit * a.B * a.Hk * a.G * a.N * (p.dc + 2) * sizeof(float);
  return attn_bits_bytes(a) + part;
}

int attn_fwd(int dtype, AttnArgs a, void* workspace, hipStream_t st) {
  const FwdPlan p = fwd_plan(dtype, a, num_cus());
  a.nsplit = p.nsplit;
  a.tiles = p.tiles;
  a.chunk = p.chunk;
  if ((int64_t)a.B * a.Hk * p.tiles * p.nsplit > kMostWorkgroups)
    return fail(LFAMD_ERR_UNSUPPORTED, "softmax_attention: too many workgroups");
  a.part = (float*)((char*)workspace + attn_bits_bytes(a));
  if (int e = attn_pack_bits(a, workspace, st)) return e;
  switch (dtype) {
    case LFAMD_F32: return fwd_dim<float>(a, p, st);
    case LFAMD_F16: return fwd_dim<f16s>(a, p, st);
    default: return fwd_dim<bf16s>(a, p, st);
  }
}

}  // namespace lfamd
