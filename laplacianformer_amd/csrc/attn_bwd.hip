// softmax_attention, backward. With p_ij recomputed from the forward's row statistics,
//   delta_i = g_i . o_i   (o_i in fp32: the stored output and what its rounding took off)
//   dv_j = sum_i p_ij g_i
//   dz_ij = p_ij (g_i . v_j - delta_i)
//   dk_j = scale sum_i dz_ij q_i,   dq_i = scale sum_j dz_ij k_j.
//
// Two kernels without atomics, each owning its outputs: attn_dkdv_kernel a block of
// keys (over every query of the heads that share them, so that shared heads' sums
// need no second pass), attn_dq_kernel a block of queries. The scores and g . v are
// formed in both: seven products instead of five, and the same bits on every run.
// Both form the scores with the owned rows as columns, so that p and dz leave the
// accumulators as the next product's operand (attn_common.h).
//
// fp16: dz follows the gradient's magnitude (a scaled loss overflows 65504, a mean
// over many keys falls below 2^-14), so it is rounded after a multiplication by a power of
// two f per key head, with |dz| <= |g_i| |v_j| + |delta_i| <= bound and f bound <= 2^14,
// which the result is divided by; p <= 1 likewise carries 2^15 into the product for
// dv. bf16 and fp32 have the exponents and take f = 1.
//
// What bounds it (one MI355X, bf16, 4096 x 4096 at 64 channels and 64 heads): dk/dv 663 us for four products, 0.83
// PFLOP/s, matrix cores busy 41 % and VALU 43 % of the cycles at 1.84 GHz, two waves per SIMD (accumulators 64,
// operands 32, scores 32 and reads in flight make 204 registers); dq 431 us for three, 0.96 PFLOP/s, three waves.
// Both run at the power limit, where a large library product reaches 1.18.
#include "attn_common.h"

namespace lfamd {

namespace {

constexpr float kPShift = 15.0f;

// Streamed rows per LDS tile, taken in blocks of 32: queries (dk, dv), keys (dq).
template <typename T, int DC> constexpr int query_tile() { return DC < 96 && (sizeof(T) == 2 || DC == 32) ? 64 : 32; }
template <typename T, int DC> constexpr int key_tile() { return sizeof(T) == 2 || DC == 32 ? 64 : 32; }

// At 128 channels the accumulators of dk and dv and both owned operands are more than a lane's
// registers at two waves per SIMD (128 + 64 + 64 with the scores): V is read from LDS then. That leaves the 16-bit
// forms still above the 256: 48 to 84 bytes a lane in scratch, part of them written and read in the loop (140 to 152
// with an additive mask, whose 16 values are held across the products, and 28 to 36 with one at 96 channels).
template <int DC> constexpr bool v_in_lds() { return DC >= 128; }

// Bytes of a streamed query's statistics: lse, delta, 1 / sum and last key, or its bits of the 128 keys.
template <int FORM> constexpr int row_stats() { return FORM == kBits ? 24 : 16; }

template <typename T, int DC, int FORM> constexpr size_t dkdv_lds() {
  constexpr int DP = row_pitch(DC);
  return (size_t)2 * query_tile<T, DC>() * (2 * DP * sizeof(T) + row_stats<FORM>()) + (v_in_lds<DC>() ? 128 * DP * sizeof(T) : 0);
}
template <typename T, int DC> constexpr size_t dq_lds() { return (size_t)2 * key_tile<T, DC>() * 2 * row_pitch(DC) * sizeof(T); }

// delta_i, and for fp16 the maxima over 64 rows of |g_i| and |delta_i|, or over 64
// keys of |v_j|. A workgroup takes 64 rows of one head: four threads per row.
template <typename T, bool BOUND>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnArgs a) {
  constexpr int CE = 16 / (int)sizeof(T);
  const int qt = (a.N + 63) / 64, kt = (a.M + 63) / 64;
  const int64_t nq = (int64_t)a.B * a.H * qt;
  const bool keys = BOUND && blockIdx.x >= nq;
  const int64_t id = keys ? blockIdx.x - nq : blockIdx.x;
  const int tiles = keys ? kt : qt, heads = keys ? a.Hk : a.H;
  const int64_t bh = id / tiles;
  const int tile = (int)(id % tiles), b = (int)(bh / heads), hd = (int)(bh % heads);
  const int row = tile * 64 + threadIdx.x / 4, part = threadIdx.x % 4;
  float dot = 0.0f, sq = 0.0f;
  if (keys) {
    const bool in = row < key_count(a, b);
    const T* p = (const T*)a.v + (int64_t)b * a.vs[0] + (int64_t)hd * a.vs[1] + (int64_t)row * a.vs[2];
    bool live = in;
    if (in && a.keyMask) {
      const int64_t off = (int64_t)b * a.ms[0] + (int64_t)row * a.ms[3];
      live = mask_bias(a, off) != kNegInf;
    }
    for (int c = part * CE; c < a.D; c += 4 * CE) {
      const u32x4 x = load_chunk<T>(p, live, c, a.D);
#pragma unroll
      for (int j = 0; j < CE; ++j) {
        const float v = to_acc(((const T*)&x)[j]);
        sq = fmaf(v, v, sq);
      }
    }
  } else {
    const bool in = row < query_count(a, b);
    const T* po = (const T*)a.o + (int64_t)b * a.os[0] + (int64_t)hd * a.os[1] + (int64_t)row * a.os[2];
    const T* pg = (const T*)a.g + (int64_t)b * a.gs[0] + (int64_t)hd * a.gs[1] + (int64_t)row * a.gs[2];
    for (int c = part * CE; c < a.D; c += 4 * CE) {
      const u32x4 x = load_chunk<T>(po, in, c, a.D), y = load_chunk<T>(pg, in, c, a.D);
      u32x4 z;
      if constexpr (sizeof(T) == 2) z = load_chunk<T>(rest_row<T>(a, bh * a.N + row), in, c, a.D);
#pragma unroll
      for (int j = 0; j < CE; ++j) {
        float u = to_acc(((const T*)&x)[j]);
        if constexpr (sizeof(T) == 2) u += to_acc(((const T*)&z)[j]);
        const float v = to_acc(((const T*)&y)[j]);
        dot = fmaf(u, v, dot);
        if (BOUND) sq = fmaf(v, v, sq);
      }
    }
  }
#pragma unroll
  for (int s = 1; s < 4; s <<= 1) {
    dot += __shfl_xor(dot, s);
    sq += __shfl_xor(sq, s);
  }
  if (!keys && part == 0 && row < a.N) a.delta[bh * a.N + row] = dot;
  if constexpr (BOUND) {
    __shared__ float w[2][4];
    float nrm = sqrtf(sq), del = fabsf(dot);
#pragma unroll
    for (int s = 4; s < 64; s <<= 1) {
      nrm = fmaxf(nrm, __shfl_xor(nrm, s));
      del = fmaxf(del, __shfl_xor(del, s));
    }
    if ((threadIdx.x & 63) == 0) {
      w[0][threadIdx.x >> 6] = nrm;
      w[1][threadIdx.x >> 6] = del;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      nrm = fmaxf(fmaxf(w[0][0], w[0][1]), fmaxf(w[0][2], w[0][3]));
      del = fmaxf(fmaxf(w[1][0], w[1][1]), fmaxf(w[1][2], w[1][3]));
      if (keys) {
        a.bounds[2 * nq + id] = nrm;
      } else {
        a.bounds[2 * id] = nrm;
        a.bounds[2 * id + 1] = del;
      }
    }
  }
}

// The power of two that dz of key head (b, hk) is multiplied by before it is rounded to fp16.
__device__ __forceinline__ float dz_factor(const AttnArgs& a, int b, int hk) {
  const int qt = (a.N + 63) / 64, kt = (a.M + 63) / 64, lane = threadIdx.x & 63;
  const int64_t q0 = ((int64_t)b * a.H + (int64_t)hk * a.G) * qt;
  float g = 0.0f, d = 0.0f, v = 0.0f;
  for (int64_t i = lane; i < (int64_t)a.G * qt; i += 64) {
    g = fmaxf(g, a.bounds[2 * (q0 + i)]);
    d = fmaxf(d, a.bounds[2 * (q0 + i) + 1]);
  }
  const float* vb = a.bounds + 2 * (int64_t)a.B * a.H * qt + ((int64_t)b * a.Hk + hk) * kt;
  for (int i = lane; i < kt; i += 64) v = fmaxf(v, vb[i]);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    g = fmaxf(g, __shfl_xor(g, s));
    d = fmaxf(d, __shfl_xor(d, s));
    v = fmaxf(v, __shfl_xor(v, s));
  }
  const float bound = fmaf(g, v, d);
  // A bound of zero, infinity or NaN leaves dz as it is.
  if (!(bound > 0.0f && bound < 1e37f)) return 1.0f;
  return exp2f(fminf(fmaxf(13.0f - floorf(log2f(bound)), -120.0f), 60.0f));
}

// p of one score. x0, x1: the row's statistics.
template <bool MASK> __device__ __forceinline__ float prob(float s, float c, float x0, float x1) {
  return MASK ? exp2_fast((s - x0) * kLog2e) * x1 : exp2_fast(fmaf(s, c, -x0));
}

// Whether key j of sequence b takes part at all.
template <int FORM> __device__ __forceinline__ bool key_live(const AttnArgs& a, int b, int j, int klen) {
  if (j >= klen) return false;
  if (FORM == kNoMask || !a.keyMask) return true;
  const int64_t off = (int64_t)b * a.ms[0] + (int64_t)j * a.ms[3];
  return mask_bias(a, off) != kNegInf;
}

// dk and dv of 128 keys, 32 per wave; queries stream through LDS in tiles of QT.
template <typename T, int DC, int FORM>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && DC >= 64 ? 1 : 2)
    __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 && DC >= 64 ? 1 : 2, 2))) attn_dkdv_kernel(const AttnArgs a) {
  constexpr bool MASK = FORM == kAdd;
  constexpr int DP = row_pitch(DC), QT = query_tile<T, DC>(), NT = DC / 16, ND = DC / 32;
  constexpr bool F16 = std::is_same<T, f16s>::value;
  using L = Tile<T, DP>;
  constexpr int TB = QT * L::ROW, SB = QT * row_stats<FORM>();  // bytes of a tile, and of its rows' statistics
  constexpr bool VL = v_in_lds<DC>();
  extern __shared__ __align__(16) char smem[];   // [2][q tile, g tile], [2][lse, delta, 1 / sum, last key], [v tile]

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t place = xcd_place(blockIdx.x, gridDim.x);
  const int split = place % a.nsplit, t0 = place / a.nsplit, bh = t0 / a.tiles, ktile = t0 % a.tiles;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int klen = key_count(a, b), qlen = query_count(a, b), qstart = query_start(a, b);
  const int key0 = ktile * 128, mykey = key0 + wave * 32 + (lane & 31);

  // Query tiles of one head that can see a key of the block.
  const int firstRow = a.causal ? min(max(key0 - qstart, 0), qlen) : 0;
  const int tb = key0 < klen ? firstRow / QT : 0, te = key0 < klen ? (qlen + QT - 1) / QT : 0;
  const int perHead = max(te - tb, 0), total = perHead * a.G;
  const int share = (total + a.nsplit - 1) / a.nsplit;
  const int beg = min(split * share, total), end = min(beg + share, total);

  const bool live = key_live<FORM>(a, b, mykey, klen);
  Frag<T> kf[NT], vf[VL ? 1 : NT];
  const char* tv = smem + 4 * TB + 2 * SB + wave * 32 * L::ROW;
  {
    const int kr = live ? mykey : 0;
    const T* kp = (const T*)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[1] + (int64_t)kr * a.ks[2];
    const T* vp = (const T*)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[1] + (int64_t)kr * a.vs[2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      kf[t] = global_frag<T>(kp, live, t, h, a.D);
      if constexpr (!VL) vf[t] = global_frag<T>(vp, live, t, h, a.D);
    }
    if constexpr (VL) {
      using LV = Loader<T, DP, DC, 128>;
      const uint32_t bits = FORM != kNoMask && a.keyMask && klen > 0 ? live_keys<LV>(a, b, key0) : ~0u;
      LV::fill(smem + 4 * TB + 2 * SB, (const T*)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[1] + (int64_t)key0 * a.vs[2],
               a.vs[2], key0, klen, a.D,
               a.modeV, bits);
    }
  }
  const float f = F16 ? dz_factor(a, b, hk) : 1.0f;
  // fp16: p carries 2^15 and dz the factor f: dz = (p 2^15) ((g.v) f' - delta f'), f' = f 2^-15.
  const float fd = F16 ? f * exp2f(-kPShift) : 1.0f;

  const int64_t moff = (int64_t)b * a.ms[0] + (int64_t)min(mykey, a.M - 1) * a.ms[3];
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};

  using LD = Loader<T, DP, DC, QT>;
  float st0 = 0.0f, st1 = 0.0f, st2 = 0.0f;
  int st3 = 0;
  u32x4 st4 = {0, 0, 0, 0};
  // The next tile to fill: its head, rows, and where they begin. Counted on, as a division per tile is
  // forty scalar instructions of each wave.
  int nextG = perHead ? beg / perHead : 0, nextT = perHead ? beg % perHead : 0, nextH = hk * a.G + nextG;
  int nextRow = (tb + nextT) * QT;
  const T *qnext, *gnext;
  auto settle = [&]() {
    nextH = hk * a.G + nextG;
    nextRow = (tb + nextT) * QT;
    qnext = (const T*)a.q + (int64_t)b * a.qs[0] + (int64_t)nextH * a.qs[1] + (int64_t)nextRow * a.qs[2];
    gnext = (const T*)a.g + (int64_t)b * a.gs[0] + (int64_t)nextH * a.gs[1] + (int64_t)nextRow * a.gs[2];
  };
  settle();
  auto advance = [&]() {
    if (++nextT == perHead) {
      nextT = 0;
      ++nextG;
      settle();
    } else {
      nextRow += QT;
      qnext += QT * a.qs[2];
      gnext += QT * a.gs[2];
    }
  };
  auto fill = [&](int buf) {
    const int row0 = nextRow, hq = nextH;
    LD::fill(smem + buf * 2 * TB, qnext, a.qs[2], row0, qlen, a.D, a.modeQ);
    LD::fill(smem + buf * 2 * TB + TB, gnext, a.gs[2], row0, qlen, a.D, a.modeG);
    if (threadIdx.x < QT) {
      const int n = row0 + threadIdx.x;
      const bool in = n < qlen;
      const int64_t so = ((int64_t)b * a.H + hq) * a.N + n;
      st0 = in ? a.stat[so] : MASK ? 0.0f : __builtin_inff();
      st1 = in ? a.delta[so] * fd : 0.0f;
      st2 = MASK && in ? a.stat[(int64_t)a.B * a.H * a.N + so] : 0.0f;
      st3 = !in ? 0 : a.causal ? min(klen, qstart + n + 1) : klen;
      if constexpr (FORM == kBits) {
        st4 = u32x4{0, 0, 0, 0};
        if (in)
          st4 = *(const u32x4*)(a.bits + (int64_t)b * a.bs[0] + (int64_t)hq * a.bs[1] + (int64_t)n * a.bs[2] + key0 / 32);
      }
      if (F16) {
        if (MASK) st2 *= exp2f(kPShift);
        else st0 -= kPShift;
      }
    }
  };
  auto store = [&](int buf) {  // the rows' statistics, through registers
    if (threadIdx.x < QT) {
      float* s = (float*)(smem + 4 * TB + buf * SB);
      s[threadIdx.x] = st0;
      s[QT + threadIdx.x] = st1;
      if constexpr (FORM == kBits) {  // by 32 keys, one wave's: what the mask and the row's last key leave
#pragma unroll
        for (int w = 0; w < 4; ++w)
          ((uint32_t*)s)[(2 + w) * QT + threadIdx.x] = st4[w] & bits_below(st3, key0 + 32 * w);
      } else {
        s[2 * QT + threadIdx.x] = st2;
        ((int*)s)[3 * QT + threadIdx.x] = st3;
      }
    }
  };

  if (beg < end) {
    fill(0);
    store(0);
  }
  land();
  __syncthreads();
  const int rl0 = L::row_lane(lane), cl0 = L::col_lane(lane);
  int buf = 0;
  for (int step = beg; step < end; ++step) {
    const bool more = step + 1 < end;
    const int row0 = nextRow, hq = nextH;
    if (more) {
      advance();
      fill(buf ^ 1);
    }
    const char* tq = smem + buf * 2 * TB;
    const char* tg = tq + TB;
    const float* stats = (const float*)(smem + 4 * TB + buf * SB);
#pragma unroll 1
    for (int qb = 0; qb < QT; qb += 32) {
      const int rl = launder(rl0), cl = launder(cl0);
      f32x16 s{}, dp{}, bias;
      if constexpr (MASK) mask_of_queries(a, moff + (int64_t)hq * a.ms[1], row0 + qb, h, bias);
      struct Pair { Frag<T> a, b; };
      {
        auto read = [&](auto n) {
          Pair p;
          p.a = L::row_frag((n < NT ? tq : tg) + qb * L::ROW, rl, n % NT);
          if constexpr (VL && n >= NT) p.b = L::row_frag(tv, rl, n % NT);
          return p;
        };
        Ring<Pair, (sizeof(T) == 4 ? 1 : VL ? 2 : 4)> ring;
        first_reads<2 * NT>(ring, read);
        read_and_use<2 * NT>(ring, read, [&](auto n, const Pair& p) {
          if constexpr (n < NT) s = mma<T>(p.a, kf[n], s);
          else if constexpr (VL) dp = mma<T>(p.a, p.b, dp);
          else dp = mma<T>(p.a, vf[n - NT], dp);
        });
      }
      // Every row sees every key of the wave: nothing to leave out.
      const int wlast = key0 + wave * 32 + 31;
      const bool check = FORM != kNoMask || wlast >= klen || row0 + qb + 32 > qlen || (a.causal && wlast > qstart + row0 + qb);
      // Pairs that are left out: score -inf, so that p = 0, and g.v = 0, so that dz = 0 (delta - 0).
      if (check) {
#pragma unroll
        for (int rq = 0; rq < 4; ++rq) {
          u32x4 w;
          if constexpr (FORM == kBits) w = *(const u32x4*)(stats + (2 + wave) * QT + qb + 8 * rq + 4 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 4 * rq + i;
            bool in;
            if constexpr (FORM == kBits) in = (int)(w[i] << (31 - (lane & 31))) < 0;
            else in = mykey < ((const int*)stats)[3 * QT + qb + 8 * rq + 4 * h + i];
            s[r] = !in ? kNegInf : MASK ? masked_score(a, s[r], bias[r]) : s[r];
            dp[r] = s[r] == kNegInf ? 0.0f : dp[r];
          }
        }
      }
      // The first columns of g and q are read while the exponentials run.
      auto cread = [&](auto n) {
        return Pair{L::col_frag(tg + qb * L::ROW, cl, n / ND, n % ND), L::col_frag(tq + qb * L::ROW, cl, n / ND, n % ND)};
      };
      Ring<Pair, (sizeof(T) == 2 && DC <= 64 ? 2 : 1)> cring;
      first_reads<2 * ND>(cring, cread);
#pragma unroll
      for (int rq = 0; rq < 4; ++rq) {
        const int rr = qb + 8 * rq + 4 * h;
        const f32x4 x0 = *(const f32x4*)(stats + rr), de = *(const f32x4*)(stats + QT + rr);
        f32x4 x1 = {1, 1, 1, 1};
        if constexpr (MASK) x1 = *(const f32x4*)(stats + 2 * QT + rr);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * rq + i;
          const float p = prob<MASK>(s[r], a.c, x0[i], x1[i]);
          s[r] = p;
          dp[r] = p * (F16 ? fmaf(dp[r], fd, -de[i]) : dp[r] - de[i]);
        }
      }
      Frag<T> pf, zf;
      read_and_use<2 * ND>(cring, cread, [&](auto n, const Pair& p) {
        if constexpr (n % ND == 0) pf = acc_frag<T>(s, n / ND), zf = acc_frag<T>(dp, n / ND);
        dv[n % ND] = mma<T>(p.a, pf, dv[n % ND]);
        dk[n % ND] = mma<T>(p.b, zf, dk[n % ND]);
      });
    }
    if (more) store(buf ^ 1);
    buf ^= 1;
    land();
    __syncthreads();
  }

  if (mykey >= a.M) return;
  const float kScale = a.scale / f, vScale = F16 ? exp2f(-kPShift) : 1.0f;
  T* dkp = (T*)a.dk + (int64_t)b * a.dks[0] + (int64_t)hk * a.dks[1] + (int64_t)mykey * a.dks[2];
  T* dvp = (T*)a.dv + (int64_t)b * a.dvs[0] + (int64_t)hk * a.dvs[1] + (int64_t)mykey * a.dvs[2];
  float* pk = a.part + ((((int64_t)split * 2) * a.B * a.Hk + bh) * a.M + mykey) * DC;
  float* pv = pk + (int64_t)a.B * a.Hk * a.M * DC;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const int c0 = 32 * d + 8 * gq + 4 * h;
      f32x4 x = {dk[d][4 * gq], dk[d][4 * gq + 1], dk[d][4 * gq + 2], dk[d][4 * gq + 3]};
      f32x4 y = {dv[d][4 * gq], dv[d][4 * gq + 1], dv[d][4 * gq + 2], dv[d][4 * gq + 3]};
      x *= kScale;
      y *= vScale;
      if (a.nsplit > 1) {
        *(f32x4*)(pk + c0) = x;
        *(f32x4*)(pv + c0) = y;
      } else {
        store4<T>(dkp, c0, a.D, x[0], x[1], x[2], x[3]);
        store4<T>(dvp, c0, a.D, y[0], y[1], y[2], y[3]);
      }
    }
}

// dq of 128 queries of one head, 32 per wave; keys stream through LDS in tiles of KT.
template <typename T, int DC, int FORM>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && DC >= 96 ? 1 : 2) attn_dq_kernel(const AttnArgs a) {
  constexpr bool MASK = FORM == kAdd;
  constexpr int DP = row_pitch(DC), KT = key_tile<T, DC>(), NT = DC / 16, ND = DC / 32;
  constexpr bool F16 = std::is_same<T, f16s>::value;
  using L = Tile<T, DP>;
  constexpr int TB = KT * L::ROW;
  extern __shared__ __align__(16) char smem[];  // [2][k tile, v tile]

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t place = xcd_place(blockIdx.x, gridDim.x);
  const int split = place % a.nsplit, t0 = place / a.nsplit, bhq = t0 / a.tiles, qtile = a.tiles - 1 - t0 % a.tiles;
  const int b = bhq / a.H, hq = bhq % a.H, hk = hq / a.G;
  const int klen = key_count(a, b), qlen = query_count(a, b), qstart = query_start(a, b);
  const int row0 = qtile * 128 + wave * 32, n = row0 + (lane & 31);
  const bool alive = n < qlen;
  const int nr = alive ? n : 0;
  const int lim = !alive ? 0 : a.causal ? min(klen, qstart + n + 1) : klen;
  const int lastAll = min(qtile * 128 + 128, qlen) - 1;
  const int kendAll = lastAll < qtile * 128 ? 0 : a.causal ? max(min(klen, qstart + lastAll + 1), 0) : klen;
  const int kbeg = split * a.chunk * KT, kend = min(kendAll, kbeg + a.chunk * KT);
  const int wend = row0 >= qlen ? 0 : a.causal ? min(kend, qstart + row0 + 32) : kend;
  const int full = a.causal ? min(klen, qstart + row0 + 1) : klen;

  Frag<T> qf[NT], gf[NT];
  {
    const T* qp = (const T*)a.q + (int64_t)b * a.qs[0] + (int64_t)hq * a.qs[1] + (int64_t)nr * a.qs[2];
    const T* gp = (const T*)a.g + (int64_t)b * a.gs[0] + (int64_t)hq * a.gs[1] + (int64_t)nr * a.gs[2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      qf[t] = global_frag<T>(qp, alive, t, h, a.D);
      gf[t] = global_frag<T>(gp, alive, t, h, a.D);
    }
  }
  const float f = F16 ? dz_factor(a, b, hk) : 1.0f;
  const int64_t so = ((int64_t)b * a.H + hq) * a.N + nr;
  const float x0 = alive ? a.stat[so] : MASK ? 0.0f : __builtin_inff();
  const float x1 = MASK && alive ? a.stat[(int64_t)a.B * a.H * a.N + so] : 0.0f;
  const float de = alive ? a.delta[so] * f : 0.0f;
  const int64_t moff = (int64_t)b * a.ms[0] + (int64_t)hq * a.ms[1] + (int64_t)nr * a.ms[2];

  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = f32x16{};

  // The next tile to fill.
  const T* knext = (const T*)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[1] + (int64_t)kbeg * a.ks[2];
  const T* vnext = (const T*)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[1] + (int64_t)kbeg * a.vs[2];
  using LD = Loader<T, DP, DC, KT>;
  const bool byKey = FORM != kNoMask && a.keyMask;
  auto fill = [&](int buf, int k0, uint32_t live) {
    LD::fill(smem + buf * 2 * TB, knext, a.ks[2], k0, kend, a.D, a.modeK, live);
    LD::fill(smem + buf * 2 * TB + TB, vnext, a.vs[2], k0, kend, a.D, a.modeV, live);
    knext += KT * a.ks[2];
    vnext += KT * a.vs[2];
  };
  // The row's bits of a tile's keys.
  const int64_t boff = (int64_t)b * a.bs[0] + (int64_t)hq * a.bs[1] + (int64_t)nr * a.bs[2];
  auto load_bits = [&](int k0) {
    const uint32_t* p = a.bits + boff + k0 / 32;
    if constexpr (KT == 32) return (uint64_t)*p;
    else return *(const uint64_t*)p;
  };
  uint64_t bits = 0;
  if constexpr (FORM == kBits)
    if (kbeg < kend) bits = load_bits(kbeg);
  uint32_t live = ~0u;  // of the next tile to fill
  if (kbeg < kend) {
    if (byKey) live = live_keys<LD>(a, b, kbeg);
    fill(0, kbeg, live);
    if (byKey) live = live_keys<LD>(a, b, kbeg + KT);
  }
  land();
  __syncthreads();
  const int rl0 = L::row_lane(lane), cl0 = L::col_lane(lane);
  int buf = 0;
  for (int key0 = kbeg; key0 < kend; key0 += KT) {
    const bool more = key0 + KT < kend;
    if (more) fill(buf ^ 1, key0 + KT, live);
    if (byKey) live = live_keys<LD>(a, b, key0 + 2 * KT);
    const uint64_t now = bits;
    if constexpr (FORM == kBits)
      if (more) bits = load_bits(key0 + KT);
    const char* tk = smem + buf * 2 * TB;
    const char* tv = tk + TB;
#pragma unroll 1
    for (int kb = 0; kb < KT; kb += 32) {
      if (key0 + kb >= wend) break;
      const int rl = launder(rl0), cl = launder(cl0);
      f32x16 s{}, dp{}, bias;
      if constexpr (MASK) mask_of_keys(a, moff, key0 + kb, h, bias);
      {
        auto read = [&](auto n) { return L::row_frag((n < NT ? tk : tv) + kb * L::ROW, rl, n % NT); };
        Ring<Frag<T>, (sizeof(T) == 4 ? 1 : 4)> ring;
        first_reads<2 * NT>(ring, read);
        read_and_use<2 * NT>(ring, read, [&](auto n, const Frag<T>& x) {
          if constexpr (n < NT) s = mma<T>(x, qf[n], s);
          else dp = mma<T>(x, gf[n - NT], dp);
        });
      }
      const bool check = FORM != kNoMask || key0 + kb + 32 > full;
      if (check) {
        const uint32_t w = FORM == kBits ? ((uint32_t)(now >> kb) & bits_below(lim, key0 + kb)) >> (4 * h) : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if constexpr (FORM == kBits) {
            s[r] = w & (1u << (8 * (r >> 2) + (r & 3))) ? s[r] : kNegInf;
          } else {
            const int j = key0 + kb + 8 * (r >> 2) + 4 * h + (r & 3);
            s[r] = j >= lim ? kNegInf : MASK ? masked_score(a, s[r], bias[r]) : s[r];
          }
          dp[r] = s[r] == kNegInf ? 0.0f : dp[r];
        }
      }
      // The first columns of k are read while the exponentials run.
      auto cread = [&](auto n) { return L::col_frag(tk + kb * L::ROW, cl, n / ND, n % ND); };
      Ring<Frag<T>, (sizeof(T) == 4 ? 1 : DC <= 64 ? 4 : 2)> cring;
      first_reads<2 * ND>(cring, cread);
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = prob<MASK>(s[r], a.c, x0, x1) * (F16 ? fmaf(dp[r], f, -de) : dp[r] - de);
      Frag<T> zf;
      read_and_use<2 * ND>(cring, cread, [&](auto n, const Frag<T>& x) {
        if constexpr (n % ND == 0) zf = acc_frag<T>(dp, n / ND);
        dq[n % ND] = mma<T>(x, zf, dq[n % ND]);
      });
    }
    buf ^= 1;
    land();
    __syncthreads();
  }

  if (n >= a.N) return;
  const float scale = a.scale / f;
  T* dqp = (T*)a.dq + (int64_t)b * a.dqs[0] + (int64_t)hq * a.dqs[1] + (int64_t)n * a.dqs[2];
  float* pq = a.part + (((int64_t)split * a.B * a.H + bhq) * a.N + n) * DC;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const int c0 = 32 * d + 8 * gq + 4 * h;
      f32x4 x = {dq[d][4 * gq], dq[d][4 * gq + 1], dq[d][4 * gq + 2], dq[d][4 * gq + 3]};
      x *= scale;
      if (a.nsplit > 1) *(f32x4*)(pq + c0) = x;
      else store4<T>(dqp, c0, a.D, x[0], x[1], x[2], x[3]);
    }
}

// One gradient whose splits' partial rows are to be added.
struct SumOf {
  const float* part;
  int64_t splitStride, s0, s1, s2, rows;  // rows: heads x batch x `len`
  void* out;
  int nsplit, heads, len;
};

// Adds the splits' partial gradients in their order: DC / 4 threads per row, up to three gradients.
template <typename T, int DC>
__global__ void __launch_bounds__(256) attn_sum_kernel(const SumOf a0, const SumOf a1, const SumOf a2, int D) {
  constexpr int TPR = DC == 96 ? 32 : DC / 4, RPB = 256 / TPR;
  int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const int which = row < a0.rows ? 0 : row < a0.rows + a1.rows ? 1 : 2;
  const SumOf& a = which == 0 ? a0 : which == 1 ? a1 : a2;
  if (which) row -= which == 1 ? a0.rows : a0.rows + a1.rows;
  const int c0 = (threadIdx.x % TPR) * 4;
  if (row >= a.rows || c0 >= DC) return;
  f32x4 x = {0, 0, 0, 0};
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) x += *(const f32x4*)(a.part + s * a.splitStride + row * DC + c0);
  const int64_t bh = row / a.len, n = row % a.len;
  store4<T>((T*)a.out + bh / a.heads * a.s0 + bh % a.heads * a.s1 + n * a.s2, c0, D, x[0], x[1], x[2], x[3]);
}

struct BwdPlan {
  int dc, ktiles, ksplit, qtiles, qsplit, qchunk;
  size_t deltaBytes, boundBytes, kpartBytes, partBytes;
};

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

BwdPlan bwd_plan(int dtype, const AttnArgs& a, int cus) {
  BwdPlan p{};
  p.dc = compute_dim(a.D);
  p.ktiles = (a.M + 127) / 128;
  p.qtiles = (a.N + 127) / 128;
  const int64_t kw = (int64_t)a.B * a.Hk * p.ktiles, qw = (int64_t)a.B * a.H * p.qtiles;
  const bool wide = dtype != LFAMD_F32 || p.dc == 32;
  const int qt = wide && p.dc < 96 ? 64 : 32, kt = wide ? 64 : 32;  // query_tile, key_tile
  const int64_t ksteps = (int64_t)a.G * ((a.N + qt - 1) / qt), qsteps = (a.M + kt - 1) / kt;
  // The other axis is split where a kernel's own blocks leave CUs without work. A tile's throughput: its
  // four (dq: three) products at the 3 TFLOP/s that a CU reaches (fp32: 0.45); its latency as measured
  // where a CU has one workgroup.
  const double rate = dtype == LFAMD_F32 ? 0.45e6 : 3e6, f32 = sizeof(float), add = a.maskKind > kMaskBool ? 1.5 : 0.0;
  const double kthr = 8.0 * 128 * qt * p.dc / rate, qthr = 6.0 * 128 * kt * p.dc / rate;
  const double klat = std::max(kthr, qt == 64 ? 2.5 : 1.5) + add, qlat = std::max(qthr, kt == 64 ? 2.0 : 1.2) + add;
  p.ksplit = kw && ksteps ? best_split(kw, ksteps, cus, klat, kthr + 0.3 * add, 2.0 * a.B * a.Hk * a.M * p.dc * f32) : 1;
  p.qsplit = qw && qsteps ? best_split(qw, qsteps, cus, qlat, qthr + 0.3 * add, 1.0 * a.B * a.H * a.N * p.dc * f32) : 1;
  p.qchunk = (int)std::max<int64_t>(1, (qsteps + p.qsplit - 1) / p.qsplit);
  p.deltaBytes = up256((size_t)a.B * a.H * a.N * sizeof(float));
  if (dtype == LFAMD_F16)
    p.boundBytes = up256(((size_t)a.B * a.H * ((a.N + 63) / 64) * 2 + (size_t)a.B * a.Hk * ((a.M + 63) / 64)) * sizeof(float));
  // Both kernels' partial results at once: one launch adds them all.
  const size_t kp = p.ksplit > 1 ? (size_t)p.ksplit * 2 * a.B * a.Hk * a.M * p.dc * sizeof(float) : 0;
  const size_t qp = p.qsplit > 1 ? (size_t)p.qsplit * a.B * a.H * a.N * p.dc * sizeof(float) : 0;
  p.kpartBytes = up256(kp);
  p.partBytes = p.kpartBytes + qp;
  return p;
}

int launch(const void* fn, int64_t grid, size_t lds, const AttnArgs& a, hipStream_t st) {
  const char* what = "softmax_attention backward";
  if (int e = set_dyn_lds(fn, lds, what)) return e;
  if (int e = check_fit(fn, 256, lds, what)) return e;
  AttnArgs args = a;
  void* params[] = {&args};
  if (hipLaunchKernel(fn, dim3((unsigned)grid), dim3(256), params, lds, st) != hipSuccess) return check_launch(what);
  return check_launch(what);
}

template <typename T, int DC, int FORM> int bwd_launch(AttnArgs a, const BwdPlan& p, hipStream_t st) {
  constexpr bool F16 = std::is_same<T, f16s>::value;
  const int qt = (a.N + 63) / 64, kt = (a.M + 63) / 64;
  int64_t grid = (int64_t)a.B * a.H * qt + (F16 ? (int64_t)a.B * a.Hk * kt : 0);
  if (grid)
    if (int e = launch((const void*)attn_delta_kernel<T, F16>, grid, 0, a, st)) return e;
  float* const part = a.part;
  SumOf sums[3] = {};
  if (a.dk) {
    a.nsplit = p.ksplit;
    a.tiles = p.ktiles;
    if (int e = launch((const void*)attn_dkdv_kernel<T, DC, FORM>, (int64_t)a.B * a.Hk * p.ktiles * p.ksplit,
                       dkdv_lds<T, DC, FORM>(), a, st))
      return e;
    if (p.ksplit > 1) {
      const int64_t rows = (int64_t)a.B * a.Hk * a.M;
      sums[0] = SumOf{part, 2 * rows * DC, a.dks[0], a.dks[1], a.dks[2], rows, a.dk, p.ksplit, a.Hk, a.M};
      sums[1] = SumOf{part + rows * DC, 2 * rows * DC, a.dvs[0], a.dvs[1], a.dvs[2], rows, a.dv, p.ksplit, a.Hk, a.M};
    }
  }
  if (a.dq) {
    a.nsplit = p.qsplit;
    a.tiles = p.qtiles;
    a.chunk = p.qchunk;
    a.part = (float*)((char*)part + p.kpartBytes);
    if (int e = launch((const void*)attn_dq_kernel<T, DC, FORM>, (int64_t)a.B * a.H * p.qtiles * p.qsplit, dq_lds<T, DC>(), a, st))
      return e;
    if (p.qsplit > 1) {
      const int64_t rows = (int64_t)a.B * a.H * a.N;
      sums[2] = SumOf{a.part, rows * DC, a.dqs[0], a.dqs[1], a.dqs[2], rows, a.dq, p.qsplit, a.H, a.N};
    }
  }
  const int64_t rows = sums[0].rows + sums[1].rows + sums[2].rows;
  if (!rows) return ok();
  constexpr int RPB = 256 / (DC == 96 ? 32 : DC / 4);
  attn_sum_kernel<T, DC><<<dim3((unsigned)((rows + RPB - 1) / RPB)), dim3(256), 0, st>>>(sums[0], sums[1], sums[2], a.D);
  return check_launch("softmax_attention backward (sums)");
}

template <typename T, int DC> int bwd_mask(const AttnArgs& a, const BwdPlan& p, hipStream_t st) {
  switch (a.maskKind) {
    case kMaskNone: return bwd_launch<T, DC, kNoMask>(a, p, st);
    case kMaskBool: return bwd_launch<T, DC, kBits>(a, p, st);
    default: return bwd_launch<T, DC, kAdd>(a, p, st);
  }
}

template <typename T> int bwd_dim(const AttnArgs& a, const BwdPlan& p, hipStream_t st) {
  switch (p.dc) {
    case 32: return bwd_mask<T, 32>(a, p, st);
    case 64: return bwd_mask<T, 64>(a, p, st);
    case 96: return bwd_mask<T, 96>(a, p, st);
    default: return bwd_mask<T, 128>(a, p, st);
  }
}

}  // namespace

size_t attn_bwd_workspace(int dtype, const AttnArgs& a) {
  const BwdPlan p = bwd_plan(dtype, a, num_cus());
  return attn_bits_bytes(a) + p.deltaBytes + p.boundBytes + p.partBytes;
}

int attn_bwd(int dtype, AttnArgs a, void* workspace, hipStream_t st) {
  const BwdPlan p = bwd_plan(dtype, a, num_cus());
  char* rest = (char*)workspace + attn_bits_bytes(a);
  a.delta = (float*)rest;
  a.bounds = (float*)(rest + p.deltaBytes);
  a.part = (float*)(rest + p.deltaBytes + p.boundBytes);
  const int64_t most = std::max({(int64_t)a.B * a.Hk * p.ktiles * p.ksplit, (int64_t)a.B * a.H * p.qtiles * p.qsplit,
                                 (int64_t)a.B * a.H * ((a.N + 63) / 64) + (int64_t)a.B * a.Hk * ((a.M + 63) / 64)});
  if (most > kMostWorkgroups) return fail(LFAMD_ERR_UNSUPPORTED, "softmax_attention backward: too many workgroups");
  if (int e = attn_pack_bits(a, workspace, st)) return e;
  switch (dtype) {
    case LFAMD_F32: return bwd_dim<float>(a, p, st);
    case LFAMD_F16: return bwd_dim<f16s>(a, p, st);
    default: return bwd_dim<bf16s>(a, p, st);
  }
}

}  // namespace lfamd
