// decay_attention: causal linear attention with a decay for each head,
//   S_t = a S_(t-1) + k_t v_t^T,   out_t = scale S_t^T q_t,   a = exp(log_decay).
//
// Tiles of 32 tokens. With S the state in front of a tile and i, j its tokens,
//   out_i = scale (a^(i+1) S^T q_i + sum over j <= i of a^(i-j) (q_i . k_j) v_j),
//   S'    = a^32 S + sum over j of a^(31-j) k_j v_j^T.
// A wave owns 32 value columns: their part of S stays in its accumulators from one tile to the
// next (rows: key channels), and every product is on matrix cores:
//   scores   P^T = K Q^T          rows j, columns i; every wave forms them, one 32 x 32 block
//   memory   O^T = S^T Q^T        S goes from accumulators to operand within the lane
//   inside   O^T += V^T P^T       likewise P
//   state    S  += K^T (a^(31-j) V)   V's operand of the product above, scaled
// so that nothing crosses lanes or waves, and the only barriers are those of the tiles' loads.
//
// Operands are of 16 bits where the inputs are, and whatever is rounded in front of a product (P, S,
// the scaled V) is carried in two pieces x = hi + lo (V in bf16 in three), whose products the
// accumulators add. Two pieces leave 2^-17 of each score and state that an output is formed of in bf16, 2^-23 in
// fp16, in front of the output's own rounding of 2^-8 or 2^-11; of the values that go into the state, which is fp32, three
// leave 2^-26 in bf16. In fp16 the pieces are scaled by powers of two that keep both ends of the type's range away: P
// for each query, S for each wave and tile, V for each column (a column of 1e-5 beside one of 600: its state 1e-3 off with one
// power for the wave, 1e-7 with its own; times the same).
//
// The gradients are the same operator on other operands: with g the gradient of out and S^T for S,
//   dq = run(g, v, k) forwards;   dk = run(v, g, q),  dv = run(k, q, g) backwards in time,
// the latter two from the gradient of the last state. Backwards, R stands behind a tile of c tokens,
//   out_i = a^(c-1-i) R^T q_i + sum over j >= i of a^(j-i) scale (q_i . k_j) v_j,
//   R'    = a^c R + scale sum over j of a^(j+1) k_j v_j^T.
//
// A run's first tile may be short, the others are whole: forwards the tiles end where the sequence does,
// backwards they begin where it does. Only a (c) and the query's power a^(c-1-i) or a^(i+1) know of it.
//
// Where heads are few, a sequence is cut into segments, in one of two ways. Long ones: the segments' own states first
// (the kernel without OUT), those joined in order (decay_join_kernel), then every segment from the state in front of
// it. Short ones: every segment runs through all tiles in front of it for the state alone, in the one launch.
//
// What bounds it (one MI355X, bf16): 32 heads over 8 key heads, 32768 tokens, 128 channels: 276 us for the outputs and
// 103 for the states (HBM alone: 133 and 26). A wave issues some 530 VALU instructions (192 make the state's pieces, 120
// the values', 48 the scores') and 52 matrix products for a tile, and the time is about the sum of 4 cycles for each of
// the former and 32 for each of the latter (the SIMDs' matrix cores are busy for 38 % of it, VALU issue for 52 %); why two waves on a SIMD
// overlap them so little is not known. 64 heads, 16384 tokens, 64 channels:
// 118 us forward (4.5 TB/s), 330 for the three gradients (1.4 GB, 4.2 TB/s): HBM. P and S in one piece instead of two
// took 365 instead of 418 us at the former and 2 % off the latter, for outputs 1.4 times as far off. In three bf16 pieces
// instead of two they take 455 instead of 401 us (whole call), and the latter's training step 709 instead of 652: outputs and gradients are as far
// off in 64 bits' eyes (1.7e-3, bf16's own rounding) and differ from plain fp32 arithmetic rounded to bf16 by 6e-5 in place of 1e-4 of their norm (what
// is off by 2^-17 rounds the other way now and then). Two are kept.
#pragma once

#include "attn_common.h"

namespace lfamd {

constexpr int kDecayTile = 32;
constexpr int kDecayJobs = 3;

// One run of the operator over every sequence and head.
struct DecayJob {
  const void *q, *k, *v;              // in their roles in this run
  const float* first;                 // state in front (behind, if reverse), or null: zero
  void* out;
  float* last;                        // the state that it ends with, or null
  float* seg;                         // [B H][nseg][dk][dv], see decay_join_kernel
  int64_t qs[3], ks[3], vs[3], os[3]; // element strides of batch, head, token
  int qg, kg, vg;                     // query heads per head of q, k, v
  int dk, dv;
  int reverse, outF32, firstT, segT;  // firstT, segT: first, seg is [dv][dk]; segT: and another job's
  int modeQ, modeK, modeV;            // LoadMode, kPlain or kAsync
  float sp, so, sk;                   // scales of the scores, of the state's part and of what is added to the state
};

struct DecayArgs {
  DecayJob job[kDecayJobs];
  const float* logDecay;
  const int32_t* lengths;
  int B, H, N, jobs, nseg, segTiles;
  int prefix;  // every segment forms the state in front of it by itself; otherwise decay_join_kernel has
};

// Pieces that a value is carried in.
template <typename T> struct DecayPieces { static constexpr int P = 2, S = 2, V = 2; };
template <> struct DecayPieces<bf16s> { static constexpr int P = 2, S = 2, V = 3; };
template <> struct DecayPieces<float> { static constexpr int P = 1, S = 1, V = 1; };

__device__ __forceinline__ int decay_length(const DecayArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;
}
// exp(lg n) for whole n >= 0, of a log_decay of -inf too.
__device__ __forceinline__ float decay_pow(float lg, int n) { return n == 0 ? 1.0f : expf(lg * (float)n); }
// The same in 64 bits: the factor of a whole tile or segment, which powers are taken of. A rounding of it to 32 bits would be made in
// each of them again (2^-25 of the state a tile, over all tiles that it holds), so that low takes what it leaves.
__device__ __forceinline__ float decay_pow64(float lg, int n, float* low = nullptr) {
  const double x = n == 0 ? 1.0 : exp((double)lg * (double)n);
  if (low) *low = (float)(x - (double)(float)x);
  return (float)x;
}

// The tokens of a segment of a sequence of len: cut from its end if it is run forwards, from its start if backwards.
__device__ __forceinline__ void decay_segment(const DecayArgs& a, int len, int seg, bool rev, int* begin, int* end) {
  const int64_t span = (int64_t)a.segTiles * kDecayTile;
  const int64_t at = rev ? seg * span : len - (a.nseg - seg) * span;
  *begin = (int)min(max(at, (int64_t)0), (int64_t)len);
  *end = (int)min(max(at + span, (int64_t)0), (int64_t)len);
}

template <typename T> __device__ __forceinline__ float low_half(uint32_t w);
template <typename T> __device__ __forceinline__ float high_half(uint32_t w);
template <> __device__ __forceinline__ float low_half<bf16s>(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
template <> __device__ __forceinline__ float high_half<bf16s>(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
template <> __device__ __forceinline__ float low_half<f16s>(uint32_t w) { return to_acc(f16s{(uint16_t)w}); }
template <> __device__ __forceinline__ float high_half<f16s>(uint32_t w) { return to_acc(f16s{(uint16_t)(w >> 16)}); }

// Keeps what computes x in front: products of which nothing in a step is read are moved behind all steps
// otherwise, and their operands wait in registers. There is no instruction in it that could read x early.
__device__ __forceinline__ void hold(f32x16& x) { asm volatile("" : "+v"(x)); }

// x y, but 0 where either is, of infinities and NaN too: v_mul_legacy_f32, one instruction like the product itself. (There is no builtin
// for it, and inline assembly would have to wait for matrix results by itself.)
extern "C" __device__ float lfamd_mul_zero(float x, float y) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float mul_zero(float x, float y) { return lfamd_mul_zero(x, y); }

// Eight values as NP pieces of an operand.
template <typename T, int NP> __device__ __forceinline__ void split_pieces(f32x8 x, Frag<T> (&f)[NP]) {
  if constexpr (sizeof(T) == 4) {
    f[0].v = x;
  } else {
    unrolled<4 * NP>([&](auto y) {
      constexpr int p = y / 4, j = y % 4;
      const uint32_t w = pack2<T>(x[2 * j], x[2 * j + 1]);
      f[p].v[j] = w;
      x[2 * j] -= low_half<T>(w);
      x[2 * j + 1] -= high_half<T>(w);
    });
  }
}

template <typename T> __device__ __forceinline__ f32x8 frag_values(const Frag<T>& f) {
  f32x8 x;
  if constexpr (sizeof(T) == 4) {
    x = f.v;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[2 * j] = low_half<T>(f.v[j]), x[2 * j + 1] = high_half<T>(f.v[j]);
  }
  return x;
}

// The largest of a wave's values, without the LDS that a shuffle goes through (three in a row for each tile in fp16): lanes turned
// round within 16, then the two exchanges of 16 and of 32 lanes.
template <int TURN> __device__ __forceinline__ float turned_max(float x) {
  return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + TURN, 0xf, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float x) {
  x = turned_max<1>(turned_max<2>(turned_max<4>(turned_max<8>(x))));
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return half_max(fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1])));
}

// The tile of tokens t0 .. into LDS: Tile<T, DP>'s layout by THREADS threads, whole waves at a time.
template <typename T, int DC, int THREADS> struct DecayLoader {
  static constexpr int DP = row_pitch(DC);
  using L = Tile<T, DP>;
  static constexpr int CHUNKS = kDecayTile * L::CPR, NIT = (CHUNKS + THREADS - 1) / THREADS;
  static_assert(CHUNKS % 64 == 0, "whole waves");

  // first: the tile's row 0 (uniform); rows from lo on and below hi exist.
  static __device__ __forceinline__ void fill(char* tile, const T* first, int64_t stride, int lo, int hi, int D, int mode) {
    const uint32_t rowBytes = (uint32_t)stride * (uint32_t)sizeof(T);
    const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)tile;
    const int wave = uniform(threadIdx.x >> 6);
    if (mode == kAsync) {
      // What is not loaded keeps the zeros that the kernel begins with: columns behind D never are, rows outside lack in a run's first
      // tile alone.
      const bool whole = hi - lo == kDecayTile;
      constexpr int STEPS = sizeof(T) == 4 && NIT > 2 ? 2 : NIT;  // more would hold an address each through the kernel
#pragma unroll STEPS
      for (int i = 0; i < NIT; ++i) {
        const int s = i * THREADS + (int)threadIdx.x;
        if (CHUNKS % THREADS != 0 && i * THREADS + wave * 64 >= CHUNKS) break;
        const int r = s / L::CPR, c = (s % L::CPR) ^ L::swz(r);
        if ((whole || (r >= lo && r < hi)) && (D == DP || c * L::CE < D))
          load_to_lds<16>(first, (uint32_t)r * rowBytes + (uint32_t)c * 16, to + (i * THREADS + wave * 64) * 16);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < NIT; ++i) {
        const int s = i * THREADS + (int)threadIdx.x;
        if (CHUNKS % THREADS != 0 && i * THREADS + wave * 64 >= CHUNKS) break;
        const int r = s / L::CPR, c = (s % L::CPR) ^ L::swz(r);
        *(u32x4*)(tile + s * 16) = load_chunk<T>(first + (int64_t)r * stride, r >= lo && r < hi, c * L::CE, D);
      }
    }
  }
};

// LDS addresses as numbers: a pointer to the workgroup's memory, whose place the compiler does not know, costs an
// addition for every read.
template <typename X> __device__ __forceinline__ __attribute__((address_space(3))) X* lds(int at) {
  return (__attribute__((address_space(3))) X*)(uint32_t)at;
}

// Row lane % 32 of a tile, the channels of step t as acc_frag deals them.
template <typename T, int DP> struct DealtRow {
  using L = Tile<T, DP>;
  static __device__ __forceinline__ int lane_offset(int lane) {
    const int r = lane & 31, h = lane >> 5;
    if constexpr (sizeof(T) == 2) return r * L::ROW + (L::swz(r) << 4) + 8 * h;
    else return r * L::ROW + ((h ^ L::swz(r)) << 4);
  }
  // dl: the lane's offset with the tile's LDS address.
  static __device__ __forceinline__ Frag<T> read(int dl, int t) {
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
      const u32x2 a = *lds<u32x2>(dl ^ ((2 * t) << 4));
      const u32x2 b = *lds<u32x2>(dl ^ ((2 * t + 1) << 4));
      f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3);
    } else {
      const f32x4 a = *lds<f32x4>(dl ^ ((4 * t) << 4));
      const f32x4 b = *lds<f32x4>(dl ^ ((4 * t + 2) << 4));
      f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }
};

// Column 32 db + lane % 32 of contraction step s of a tile (Tile::col_frag). cl: col_lane with the tile's LDS address; at: that alone.
template <typename T, int DP> __device__ __forceinline__ Frag<T> dealt_column(int at, int cl, int lane, int s, int db) {
  using L = Tile<T, DP>;
  if constexpr (sizeof(T) == 2) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<s16x4>((cl ^ (db << 6)) + 16 * s * L::ROW));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds<s16x4>((cl ^ (db << 6) ^ 32) + (16 * s + 8) * L::ROW));
    Frag<T> f;
    f.v = __builtin_shufflevector(__builtin_bit_cast(u32x2, a), __builtin_bit_cast(u32x2, b), 0, 1, 2, 3);
    return f;
  } else {
    return L::col_frag((const char*)lds<char>(at), lane, s, db);
  }
}

// Bytes of LDS: two buffers of the three tiles (of two, for the states alone).
template <typename T, int DK, int DV, bool OUT> constexpr size_t decay_lds() {
  return (size_t)2 * kDecayTile * ((OUT ? 2 : 1) * row_pitch(DK) + row_pitch(DV)) * sizeof(T);
}

// Grid: jobs x B H x segments. OUT: the outputs; otherwise the segments' own states only. DK, DV: channels
// computed with; a wave for every 32 of DV.
template <typename T, int DK, int DV, bool OUT>
__global__ void __launch_bounds__(DV * 2, sizeof(T) == 4 && (DK >= 96 || (DK == 64 && DV == 32)) ? 1 : 2) decay_kernel(const DecayArgs a) {
  constexpr int THREADS = DV * 2, NT = DK / 16, ND = DK / 32, TILE = kDecayTile;
  constexpr int NPP = DecayPieces<T>::P, NPS = DecayPieces<T>::S, NPV = DecayPieces<T>::V;
  constexpr bool F16 = std::is_same<T, f16s>::value;
  // Fragment reads in flight in front of their products (fp32: none, its products take long and their fragments registers).
  constexpr int AHEAD = sizeof(T) == 2 ? 3 : 0;
  using LK = DecayLoader<T, DK, THREADS>;
  using LV = DecayLoader<T, DV, THREADS>;
  using TK = typename LK::L;
  using TV = typename LV::L;
  using DR = DealtRow<T, LK::DP>;
  constexpr int BK = TILE * TK::ROW, BV = TILE * TV::ROW, BUF = (OUT ? 2 : 1) * BK + BV;
  extern __shared__ __align__(256) char smem[];

  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, i = lane & 31;
  // A segment's jobs side by side, on one XCD; the outputs from the last segment on, whose keys and values the
  // states' launch has read last.
  const uint32_t ahead_ = xcd_place(blockIdx.x, gridDim.x), place = OUT ? gridDim.x - 1 - ahead_ : ahead_;
  const int rest = uniform(place / a.jobs), seg = uniform(rest % a.nseg), bh = uniform(rest / a.nseg);
  const DecayJob& jb = a.job[uniform(place - rest * a.jobs)];
  const int b = uniform(bh / a.H), hq = bh - b * a.H;
  const bool rev = jb.reverse;
  const float lg = a.logDecay[hq];
  const int len = uniform(decay_length(a, b));
  int begin, end;
  decay_segment(a, len, seg, rev, &begin, &end);
  int pre = 0;  // tiles that are run for the state alone
  if (OUT && a.prefix && end > begin) {
    pre = (rev ? len - end : begin) / TILE + ((rev ? len - end : begin) % TILE != 0);
    if (rev) end = len;
    else begin = 0;
  }
  const int tiles = (end - begin + TILE - 1) / TILE;
  const int short_ = end - begin - (tiles - 1) * TILE;  // tokens of the tile that is run first
  const int dk = jb.dk, dv = jb.dv;
  const int c = 32 * wave + i;  // this lane's value column

  const T* kp = uniform_ptr((const T*)jb.k + (int64_t)b * jb.ks[0] + (int64_t)uniform(hq / jb.kg) * jb.ks[1]);
  const T* vp = uniform_ptr((const T*)jb.v + (int64_t)b * jb.vs[0] + (int64_t)uniform(hq / jb.vg) * jb.vs[1]);
  const T* qp = OUT ? uniform_ptr((const T*)jb.q + (int64_t)b * jb.qs[0] + (int64_t)uniform(hq / jb.qg) * jb.qs[1]) : nullptr;
  const int64_t ooff = (int64_t)b * jb.os[0] + (int64_t)hq * jb.os[1];

  // Row 0 of the n-th tile that is run; the first may lack rows in front (forwards) or behind.
  auto tile_at = [&](int n) { return rev ? begin + (tiles - 1 - n) * TILE : end - (tiles - n) * TILE; };
  auto fill = [&](int buf, int n) {
    const int at = tile_at(n), lo = n || rev ? 0 : TILE - short_, hi = n || !rev ? TILE : short_;
    char* to = smem + buf * BUF;
    LK::fill(to, kp + (int64_t)at * jb.ks[2], jb.ks[2], lo, hi, dk, jb.modeK);
    LV::fill(to + BK, vp + (int64_t)at * jb.vs[2], jb.vs[2], lo, hi, dv, jb.modeV);
    if (OUT && n >= pre) LK::fill(to + BK + BV, qp + (int64_t)at * jb.qs[2], jb.qs[2], lo, hi, dk, jb.modeQ);
  };
  if (tiles && (short_ < TILE || dk < LK::DP || dv < LV::DP)) {
    for (int x = threadIdx.x * 16; x < 2 * BUF; x += THREADS * 16) *(u32x4*)(smem + x) = (u32x4){0, 0, 0, 0};
    __syncthreads();
  }
  if (tiles) fill(0, 0);

  // The state's rows 32 m + 8 (r / 4) + 4 h + r % 4 of column c.
  f32x16 st[ND];
#pragma unroll
  for (int m = 0; m < ND; ++m) st[m] = f32x16{};
  const bool joined = a.nseg > 1 && !a.prefix;
  const float* from = !OUT ? nullptr : joined ? jb.seg + ((int64_t)bh * a.nseg + seg) * dk * dv
                                     : jb.first ? jb.first + (int64_t)bh * dk * dv : nullptr;
  if (from && c < dv) {
    const bool tr = joined ? jb.segT : jb.firstT;
#pragma unroll
    for (int m = 0; m < ND; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * m + 8 * (r >> 2) + 4 * h + (r & 3);
        if (d < dk) st[m][r] = from[tr ? c * dk + d : d * dv + c];
      }
  }

  // Powers of the decay: of a score's distance (0 outside the triangle), of a token's to the state that it goes
  // into, of the query's from the state in front, and of a whole tile. A lane forms one and asks the others for the
  // rest (33 exponentials in each lane took 1 us of a call's 8).
  const float power = decay_pow(lg, lane);
  auto power_of = [&](int n) { return __shfl(power, n); };
  auto row_of = [&](int r) { return 8 * (r >> 2) + 4 * h + (r & 3); };
  f32x16 pw, gam;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int j = row_of(r), n = rev ? j - i : i - j;
    gam[r] = jb.sk * power_of(rev ? j + 1 : TILE - 1 - j);
    if constexpr (OUT) {
      const float x = jb.sp * power_of(max(n, 0));
      pw[r] = n < 0 ? 0.0f : x;
    }
  }
  const int ahead = TILE - short_;  // rows that the first tile lacks
  float lam = jb.so * power_of(max(rev ? short_ - 1 - i : i + 1 - ahead, 0));
  const float lams = jb.so * power_of(rev ? TILE - 1 - i : i + 1);
  float low;  // what wholes leaves of a whole tile's factor; a first tile's is met once
  const float wholes = decay_pow64(lg, TILE, &low);
  float whole = short_ == TILE ? wholes : decay_pow64(lg, short_);

  const int kcl0 = TK::col_lane(lane), vcl0 = TV::col_lane(lane), dl0 = DR::lane_offset(lane);
  struct KQ {
    Frag<T> k, q;
  };
  const int base = (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  // The lane's four output columns of every eight, and where they go.
  const bool wide = 32 * wave + 32 <= dv;
  const int64_t step = (rev ? -TILE : TILE) * jb.os[2];
  int64_t off = ooff + (int64_t)(tile_at(0) + i) * jb.os[2] + 32 * wave + 4 * h;
  float due = 1.0f;
  int unit = 0;  // fp16: st holds the state's column times 2^unit as well
  land();
  __syncthreads();
  for (int n = 0; n < tiles; ++n) {
    const int buf = n & 1;
    if (n + 1 < tiles) fill(buf ^ 1, n + 1);
    // The buffer's place (a multiple of 256 bytes, which the exclusive-ors stay below) goes into the lane's offset. Two
    // addresses of one offset: reads of both tiles from one would be merged, and their halves copied apart.
    static_assert(BK % 256 == 0 && BV % 256 == 0, "tiles begin at a whole row of banks");
    const int dlk = launder(dl0 + base + buf * BUF), dlq = launder(dl0 + base + buf * BUF + BK + BV);
    const int kat = base + buf * BUF, vat = kat + BK, kcl = launder(kcl0 + kat), vcl = vcl0 + vat;
    Frag<T> vf[2];
    auto read_v = [&] {
#pragma unroll
      for (int s = 0; s < 2; ++s) vf[s] = dealt_column<T, LV::DP>(vat, vcl, lane, s, wave);
    };
    // Two of the state's row blocks at a time (the last alone if they are odd), so that neighbouring products do not
    // wait for one another.
    constexpr int PAIR = ND % 2 || sizeof(T) == 4 ? 1 : 2;
    struct KF {
      Frag<T> x[PAIR];
    };
    auto read_k = [&](auto y) {
      KF f;
      unrolled<PAIR>([&](auto e) { f.x[e] = dealt_column<T, LK::DP>(kat, kcl, lane, y & 1, (y >> 1) * PAIR + e); });
      return f;
    };
    constexpr int KAHEAD = PAIR == 2 ? 1 : AHEAD;
    Ring<KF, KAHEAD> kring;

    f32x16 o = f32x16{};
    float back = 1.0f;  // fp16: what takes the output out of its unit
    const bool full = OUT && n >= pre;
    if (full) {
      Ring<KQ, AHEAD> ring;
      auto read_kq = [&](auto t) { return KQ{DR::read(dlk, t), DR::read(dlq, t)}; };
      first_reads<NT, AHEAD>(ring, read_kq);
      f32x16 p = f32x16{};
      float mul = 1.0f, front = lam * due;
      if constexpr (F16) {
        float top = 0.0f;
#pragma unroll
        for (int m = 0; m < ND; ++m)
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(st[m][r]));
        // Columns have units of their own, outputs add over key channels alone: one power of two for the wave.
        const float column = top > 0.0f ? (float)(__builtin_amdgcn_frexp_expf(top) - unit) : -1000.0f;
        const int e = 15 - min(max((int)wave_max(column), -60), 120);
        mul = __builtin_amdgcn_ldexpf(1.0f, e - unit);
        front = __builtin_amdgcn_ldexpf(front, -e);
      }
      // Scores and memory by 16 channels: the pieces of one step's state are made while the products of the
      // step before it run.
      read_and_use<NT, AHEAD>(ring, read_kq, [&](auto t, const KQ& f) {
        constexpr int m = t >> 1, e = 8 * (t & 1);
        f32x8 x = __builtin_shufflevector(st[m], st[m], e, e + 1, e + 2, e + 3, e + 4, e + 5, e + 6, e + 7);
        if constexpr (F16) x *= mul;
        Frag<T> sf[NPS];
        split_pieces<T, NPS>(x, sf);
        // Neighbours do not wait for one another.
        if constexpr (NPS > 1) o = mma<T>(sf[NPS - 1], f.q, o);
        p = mma<T>(f.k, f.q, p);
        o = mma<T>(sf[0], f.q, o);
        if constexpr (sizeof(T) == 2) hold(o);
      });
      read_v();
      first_reads<2 * ND / PAIR, KAHEAD>(kring, read_k);
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] = mul_zero(p[r], pw[r]);
      if constexpr (F16) {
        float top = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(p[r]));
        const int e = 15 - min(max(__builtin_amdgcn_frexp_expf(half_max(top)), -25), 60);
        const float f = __builtin_amdgcn_ldexpf(1.0f, e);
        back = __builtin_amdgcn_ldexpf(1.0f, -e);
        front *= f;
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] *= f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) o[r] *= front;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        Frag<T> pf[NPP];
        split_pieces<T, NPP>(s ? __builtin_shufflevector(p, p, 8, 9, 10, 11, 12, 13, 14, 15)
                               : __builtin_shufflevector(p, p, 0, 1, 2, 3, 4, 5, 6, 7), pf);
#pragma unroll
        for (int z = NPP - 1; z >= 0; --z) o = mma<T>(vf[s], pf[z], o);
      }
    } else {
      read_v();
      first_reads<2 * ND / PAIR, KAHEAD>(kring, read_k);
    }

    // The state behind the tile. st holds it over `due`, the decay that it has not been multiplied with yet:
    // that is done when it falls below 2^-20, and what is added in between is divided by it.
    f32x8 x[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      x[s] = frag_values<T>(vf[s]);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[s][j] *= gam[8 * s + j];
    }
    float keep = fmaf(due, whole, n ? due * low : 0.0f), f = 1.0f;
    bool now = keep < 0x1p-20f;
    if constexpr (F16) {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[s][j]));
      // The lane pair's column: its largest value times 2^unit is to be of 2^8 to 2^15, so that the second piece's step,
      // 2^-24, is 2^-32 of it or less; a new unit makes it one of 2^11, between the two, if the column's state has room for it.
      top = half_max(top);
      const int over = __builtin_amdgcn_frexp_expf(top / keep) + unit;
      now = __any(now || (top > 0.0f && (over > 15 || over < 9)));
      if (now) {
        float most = 0.0f;
#pragma unroll
        for (int m = 0; m < ND; ++m)
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(st[m][r]));
        const int room = 100 + unit - __builtin_amdgcn_frexp_expf(half_max(most) * keep);
        const int to = top > 0.0f ? min(12 - min(max(__builtin_amdgcn_frexp_expf(top), -80), 60), room) : unit;
        keep = __builtin_amdgcn_ldexpf(keep, to - unit), unit = to;
      }
      f = __builtin_amdgcn_ldexpf(1.0f, unit);
    }
    if (now) {
#pragma unroll
      for (int m = 0; m < ND; ++m) st[m] *= keep;
      due = 1.0f;
    } else {
      due = keep;
      f /= keep;
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) x[s] *= f;
    Frag<T> xf[2][NPV];
#pragma unroll
    for (int s = 0; s < 2; ++s) split_pieces<T, NPV>(x[s], xf[s]);
    read_and_use<2 * ND / PAIR, KAHEAD>(kring, read_k, [&](auto y, const KF& kf) {
      constexpr int m = (y >> 1) * PAIR, s = y & 1;
      unrolled<NPV * PAIR>([&](auto z) {
        constexpr int e = z % PAIR;
        st[m + e] = mma<T>(kf.x[e], xf[s][NPV - 1 - z / PAIR], st[m + e]);
      });
    });

    land();  // the next tile; in front of the stores, so that they are not waited for
    if constexpr (OUT) {
      if (full && (n || (rev ? i < short_ : i >= ahead))) {
        if (wide && !jb.outF32) {
          T* to = (T*)jb.out + off;
          if constexpr (sizeof(T) == 2) {
            // The halves of a lane pair exchange four channels of every sixteen: 16 adjacent bytes each.
#pragma unroll
            for (int u = 0; u < 4; u += 2) {
              u32x4 w;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const auto y = __builtin_amdgcn_permlane32_swap(pack2<T>(o[4 * u + 2 * e] * back, o[4 * u + 2 * e + 1] * back),
                                                                pack2<T>(o[4 * u + 4 + 2 * e] * back, o[4 * u + 5 + 2 * e] * back), false, false);
                w[e] = y[0], w[2 + e] = y[1];
              }
              __builtin_memcpy(to + 8 * u + 4 * h, &w, 16);
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) store4<T>(to + 8 * u, 0, 4, o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
          }
        } else {
          const int left = dv - 32 * wave - 4 * h;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (jb.outF32) store4<float>((float*)jb.out + off, 8 * u, left, o[4 * u] * back, o[4 * u + 1] * back, o[4 * u + 2] * back, o[4 * u + 3] * back);
            else store4<T>((T*)jb.out + off, 8 * u, left, o[4 * u] * back, o[4 * u + 1] * back, o[4 * u + 2] * back, o[4 * u + 3] * back);
          }
        }
      }
      off += step;
    }
    lam = lams, whole = wholes;
    __syncthreads();
  }

  float* to = nullptr;
  if constexpr (OUT) {
    if (jb.last && seg == (rev ? 0 : a.nseg - 1)) to = jb.last + (int64_t)bh * dk * dv;
  } else {
    to = jb.seg + ((int64_t)bh * a.nseg + seg) * dk * dv;
  }
  if (to && c < dv) {
    const float f = F16 ? __builtin_amdgcn_ldexpf(due, -unit) : due;
#pragma unroll
    for (int m = 0; m < ND; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * m + row_of(r);
        if (d < dk) to[d * dv + c] = st[m][r] * f;
      }
  }
  if constexpr (OUT) {
    // Tokens behind the sequence's length are zero.
    constexpr int RPP = THREADS / 32;
    for (int64_t t = (int64_t)len + seg * RPP + (int)threadIdx.x / 32; t < a.N; t += a.nseg * RPP) {
      const int64_t row = ooff + t * jb.os[2];
      for (int y = threadIdx.x & 31; y < dv; y += 32) {
        if (jb.outF32) ((float*)jb.out)[row + y] = 0.0f;
        else ((T*)jb.out)[row + y] = T{};
      }
    }
  }
}

template <typename T, int DK, int DV, bool OUT> int decay_launch(const DecayArgs& a, hipStream_t st) {
  constexpr size_t lds = decay_lds<T, DK, DV, OUT>();
  const void* fn = (const void*)decay_kernel<T, DK, DV, OUT>;
  if (int e = set_dyn_lds(fn, lds, "decay_attention")) return e;
  const int64_t n = (int64_t)a.jobs * a.B * a.H * a.nseg;
  decay_kernel<T, DK, DV, OUT><<<dim3((unsigned)n), dim3(DV * 2), lds, st>>>(a);
  return check_launch("decay_attention");
}

// Channels computed with for `d`: of keys, of values.
inline int decay_key_dim(int d) { return compute_dim(d); }
// (In fp32 few value columns of 128 key channels would take more registers than a workgroup of few waves may be given:
// its waves for the other columns run empty.)
inline int decay_value_dim(bool f32, int dk, int dv) {
  return f32 && decay_key_dim(dk) == 128 ? 128 : dv <= 32 ? 32 : dv <= 64 ? 64 : 128;
}

template <typename T, bool OUT> int decay_dispatch(const DecayArgs& a, hipStream_t st) {
  auto values = [&](auto dk) {
    constexpr int DK = decltype(dk)::value;
    if constexpr (sizeof(T) == 2 || DK < 128) {
      switch (decay_value_dim(sizeof(T) == 4, DK, a.job[0].dv)) {
        case 32: return decay_launch<T, DK, 32, OUT>(a, st);
        case 64: return decay_launch<T, DK, 64, OUT>(a, st);
        default: break;
      }
    }
    return decay_launch<T, DK, 128, OUT>(a, st);
  };
  switch (decay_key_dim(a.job[0].dk)) {
    case 32: return values(std::integral_constant<int, 32>{});
    case 64: return values(std::integral_constant<int, 64>{});
    case 96: return values(std::integral_constant<int, 96>{});
    default: return values(std::integral_constant<int, 128>{});
  }
}

// Jobs whose channels computed with agree, on a filled-in call: the segments' own states (out == 0) or the outputs.
int decay_run_f32(const DecayArgs& a, int out, hipStream_t st);
int decay_run_f16(const DecayArgs& a, int out, hipStream_t st);
int decay_run_bf16(const DecayArgs& a, int out, hipStream_t st);

}  // namespace lfamd
