// Shared by the softmax-attention kernels: matrix-core fragments, the LDS tile
// and its loader, and the arguments of a call.
//
// Every product runs on 32 x 32 accumulators (v_mfma_f32_32x32x16 for the 16-bit
// types, eight v_mfma_f32_32x32x2_f32 for fp32, which take the same fragments: the
// contraction index may be dealt to the lanes in any order that both operands
// share). With h = lane / 32 and i = lane % 32:
//   operand     row (A) or column (B) i, contraction elements 8h .. 8h+7 of 16
//   accumulator column i, rows 8 (r / 4) + 4 h + r % 4 for r = 0 .. 15
// The scores are formed transposed where their columns are to be a product's
// right operand: the eight accumulator values r = 8s .. 8s+7 of a lane are then
// already its operand for contraction step s, if that step's rows are dealt as
//   slot j of half h  <->  row 16 s + 8 (j / 4) + 4 h + j % 4,
// which col_frag() reads the other operand by. No value crosses lanes.
#pragma once

#include <algorithm>

#include "lf_common.h"
#include "lf_internal.h"

namespace lfamd {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Frag { u32x4 v; };       // eight 16-bit elements
template <> struct Frag<float> { f32x8 v; };

template <typename T> __device__ __forceinline__ f32x16 mma(const Frag<T>& a, const Frag<T>& b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mma<f16s>(const Frag<f16s>& a, const Frag<f16s>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a.v), __builtin_bit_cast(h16x8, b.v), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mma<bf16s>(const Frag<bf16s>& a, const Frag<bf16s>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a.v), __builtin_bit_cast(b16x8, b.v), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mma<float>(const Frag<float>& a, const Frag<float>& b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// Two fp32 values rounded to nearest even and packed.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<f16s>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, h16x2));
}
template <> __device__ __forceinline__ uint32_t pack2<bf16s>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, b16x2));
}

// Accumulator values 8s .. 8s+7 as an operand of contraction step s.
template <typename T> __device__ __forceinline__ Frag<T> acc_frag(const f32x16& c, int s) {
  Frag<T> f;
#pragma unroll
  for (int j = 0; j < 4; ++j) f.v[j] = pack2<T>(c[8 * s + 2 * j], c[8 * s + 2 * j + 1]);
  return f;
}
template <> __device__ __forceinline__ Frag<float> acc_frag<float>(const f32x16& c, int s) {
  Frag<float> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = c[8 * s + j];
  return f;
}

// The other half's value of a lane pair (lane, lane ^ 32), combined.
__device__ __forceinline__ float half_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (uint32_t)p[0]) + __builtin_bit_cast(float, (uint32_t)p[1]);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int64_t kMostWorkgroups = (1 << 24) - 1;  // of 256 threads: a grid has below 2^32

constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// Channels that a kernel computes with for heads of D, and elements from one LDS row to the next.
inline int compute_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
__host__ __device__ constexpr int row_pitch(int dc) { return dc == 96 ? 128 : dc; }

// A tile of rows of DP elements in LDS, in 16-byte chunks. A row's chunks are
// exchanged (xor with f(row)) so that both ways it is read spread over the 64
// banks: row_frag (32 rows, one chunk each) and col_frag (four rows x 32 bytes
// for every 16 lanes: rows that share banks differ in f's upper bits first).
template <typename T, int DP> struct Tile {
  static constexpr int CE = 16 / (int)sizeof(T);         // elements per chunk
  static constexpr int CPR = DP / CE;                    // chunks per row
  static constexpr int ROW = DP * (int)sizeof(T);        // bytes per row
  static constexpr int RPB = ROW >= 256 ? 1 : 256 / ROW; // rows per pass over the banks

  static __device__ __forceinline__ int swz(int row) {
    const int x = row / RPB;
    if constexpr (CPR >= 16) return ((x & 3) << 2) | ((x >> 2) & 3);
    else if constexpr (CPR == 8) return ((x & 1) << 2) | ((x >> 1) & 3);
    else return x & (CPR - 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * ROW + ((chunk ^ swz(row)) << 4); }

  // A lane's byte offset into a tile for row_frag and col_frag; the terms of t, db, s and the
  // block of rows are exclusive-ors and sums of constants on it (`tile` may point at any multiple
  // of 16 rows). Kernels pass it through launder() once per tile: one exclusive-or in front of a
  // read costs less than the registers that its hoisted address would hold.
  static __device__ __forceinline__ int row_lane(int lane) {
    const int r = lane & 31, h = lane >> 5;
    return r * ROW + (((sizeof(T) == 2 ? h : 2 * h) ^ swz(r)) << 4);
  }
  static __device__ __forceinline__ int col_lane(int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, row = 4 * h + (i >> 2);
      return row * ROW + (((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ swz(row)) << 4) + (i & 1) * 8;
    } else {
      return lane;
    }
  }

  // Elements 16 t + 8 h .. + 7 of row lane % 32.
  static __device__ __forceinline__ Frag<T> row_frag(const char* tile, int rl, int t) {
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
      f.v = *(const u32x4*)(tile + (rl ^ (t << 5)));
    } else {
      const f32x4 a = *(const f32x4*)(tile + (rl ^ (t << 6)));
      const f32x4 b = *(const f32x4*)(tile + (rl ^ (t << 6) ^ 16));
      f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }

  // Column 32 db + lane % 32 of the rows of contraction step s (rows 16 s .. 16 s + 15, dealt as
  // acc_frag deals them). 16-bit: the transposing LDS read, which gives lane i of 16 the i-th
  // element of four rows; rows 8 further on differ by 2 in the exchange.
  static __device__ __forceinline__ Frag<T> col_frag(const char* tile, int cl, int s, int db) {
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(tile + (cl ^ (db << 6) ^ (u << 5)) + (16 * s + 8 * u) * ROW));
        const u32x2 y = __builtin_bit_cast(u32x2, x);
        f.v[2 * u] = y[0];
        f.v[2 * u + 1] = y[1];
      }
    } else {
      const int lane = cl, h = lane >> 5, d = 32 * db + (lane & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 16 * s + 8 * (j >> 2) + 4 * h + (j & 3);
        f.v[j] = *(const float*)(tile + at(row, d / CE) + (d % CE) * 4);
      }
    }
    return f;
  }
};

// Hides a value's origin from the compiler.
__device__ __forceinline__ int launder(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Keeps the order of what stands before and behind: left alone the scheduler puts every fragment's read
// right in front of its product, and waits there, to save registers that are free.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// The weaker form for a row of N reads and products in one block: AHEAD reads in front, then one by one.
template <int N, int AHEAD> __device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// use(i, x) for i = 0 .. N - 1 on what read(i) gives, AHEAD reads in flight. ring: the first AHEAD reads,
// which first_reads() has issued earlier (in front of other work that they then overlap).
template <typename F, int AHEAD> struct Ring { F x[AHEAD + 1]; };
template <int N, int AHEAD, typename F, typename R> __device__ __forceinline__ void first_reads(Ring<F, AHEAD>& ring, R&& read) {
  unrolled<(AHEAD < N ? AHEAD : N)>([&](auto i) { ring.x[i] = read(i); });
  fence();
}
template <int N, int AHEAD, typename F, typename R, typename U>
__device__ __forceinline__ void read_and_use(Ring<F, AHEAD>& ring, R&& read, U&& use) {
  unrolled<N>([&](auto i) {
    if constexpr (i + AHEAD < N) ring.x[(i + AHEAD) % (AHEAD + 1)] = read(std::integral_constant<int, i + AHEAD>{});
    fence();
    use(i, ring.x[i % (AHEAD + 1)]);
  });
}

// How a tensor's rows are read: kAsync, to LDS directly by 16 bytes (rows 16-byte aligned, D a multiple of
// 16 bytes); kAsync4, to LDS directly by 4 bytes (the same with 4); kPlain, through registers by 16 bytes at
// any alignment. The first two keep a tile's offsets within 32 bits.
enum LoadMode { kPlain = 0, kAsync4 = 1, kAsync = 2 };

// 16 bytes of a row from element c0 on at any alignment, zero where row or column is outside.
template <typename T> __device__ __forceinline__ u32x4 load_chunk(const T* row, bool inside, int c0, int D) {
  constexpr int CE = 16 / (int)sizeof(T);
  u32x4 r = {0, 0, 0, 0};
  if (!inside || c0 >= D) return r;
  if (c0 + CE <= D) {
    __builtin_memcpy(&r, row + c0, 16);
    return r;
  }
#pragma unroll
  for (int j = 0; j < CE - 1; ++j)
    if (c0 + j < D) {
      if constexpr (sizeof(T) == 2) r[j >> 1] |= (uint32_t)((const uint16_t*)(row + c0))[j] << (16 * (j & 1));
      else r[j] = ((const uint32_t*)(row + c0))[j];
    }
  return r;
}

// 16 (or 4) bytes per lane from base + off (base uniform) to LDS at lds + 16 (or 4) lane, without registers in
// between. In asm because the compiler puts a wait for every such load in front of the next transposing LDS
// read, whichever tile that reads; there is no output register that it could reuse early, and land() is the
// wait. M0 takes the LDS address, one wait state in front of its use, and gets its value back (the compiler
// does not take it as a clobber).
template <int BYTES> __device__ __forceinline__ void load_to_lds(const void* base, uint32_t off, uint32_t lds) {
  uint32_t m0;
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
  else
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
}

// Rows of a matrix into an LDS tile by a workgroup of 256 threads. Thread t fills the
// tile's t-th chunk of every 4 KiB (kAsync4: the t-th word of every 1 KiB), whose place in
// the row the tile's exchange gives: a wave's loads land side by side. Rows at or behind
// `limit`, columns from D to DC (what the kernel computes with) and rows whose bit in `live`
// is 0 are zero and not read. fill() issues; land() waits for this wave's loads, before the
// barrier behind which the tile may be read.
template <typename T, int DP, int DC, int ROWS> struct Loader {
  using L = Tile<T, DP>;
  static constexpr int RPI = 256 / L::CPR, NIT = ROWS / RPI;
  static_assert(256 % L::CPR == 0 && ROWS % RPI == 0 && NIT <= 32, "tile shape");

  static __device__ __forceinline__ int row_of(int i) { return (int)threadIdx.x / L::CPR + i * RPI; }

  // first: row row0 (uniform).
  static __device__ __forceinline__ void fill(char* tile, const T* first, int64_t stride, int row0, int limit, int D,
                                              int mode, uint32_t live = ~0u) {
    const int slot = threadIdx.x % L::CPR;
    const char* from = (const char*)first;
    const uint32_t rowBytes = (uint32_t)stride * (uint32_t)sizeof(T);
    const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)tile;
    const int wave = uniform(threadIdx.x >> 6);
    if (__builtin_expect(mode == kAsync && row0 + ROWS <= limit && live == ~0u, 1)) {
      // A whole tile of rows, the loop's ordinary case: no branch between its loads at D = DP.
      if (D == DP) {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          const int r = row_of(i), c = slot ^ L::swz(r);
          load_to_lds<16>(from, (uint32_t)r * rowBytes + (uint32_t)c * 16, to + wave * 1024 + i * 4096);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NIT; ++i) {
          const int r = row_of(i), c = slot ^ L::swz(r);
          if (c * L::CE < D) load_to_lds<16>(from, (uint32_t)r * rowBytes + (uint32_t)c * 16, to + wave * 1024 + i * 4096);
          else if (c * L::CE < DC) *(u32x4*)(tile + i * 4096 + threadIdx.x * 16) = (u32x4){0, 0, 0, 0};
        }
      }
    } else if (mode == kAsync) {
#pragma unroll 1
      for (int i = 0; i < NIT; ++i) {
        const int r = row_of(i), c = slot ^ L::swz(r);
        if (row0 + r < limit && c * L::CE < D && (live >> i & 1))
          load_to_lds<16>(from, (uint32_t)r * rowBytes + (uint32_t)c * 16, to + wave * 1024 + i * 4096);
        else if (c * L::CE < DC)
          *(u32x4*)(tile + i * 4096 + threadIdx.x * 16) = (u32x4){0, 0, 0, 0};
      }
    } else if (mode == kAsync4) {
      // `live` belongs to the rows of row_of: a call with a mask over keys takes kPlain instead.
#pragma unroll 4
      for (int i = 0; i < 4 * NIT; ++i) {
        const int byte = i * 1024 + (int)threadIdx.x * 4, r = byte / L::ROW;
        const int c = (byte % L::ROW / 16 ^ L::swz(r)) * L::CE + byte % 16 / (int)sizeof(T);
        if (row0 + r < limit && c < D)
          load_to_lds<4>(from, (uint32_t)r * rowBytes + (uint32_t)c * (uint32_t)sizeof(T), to + wave * 256 + i * 1024);
        else if (c < DC)
          *(uint32_t*)(tile + byte) = 0;
      }
    } else {
      // Not unrolled: few registers beside the kernel's accumulators.
#pragma unroll 1
      for (int i = 0; i < NIT; ++i) {
        const int r = row_of(i), c = slot ^ L::swz(r);
        *(u32x4*)(tile + i * 4096 + threadIdx.x * 16) =
            load_chunk<T>(first + (int64_t)r * stride, row0 + r < limit && (live >> i & 1), c * L::CE, D);
      }
    }
  }
};
// Waits for every load into LDS that the wave has issued .
// The builtin, so that the compiler knows its own loads to have landed as well (0x0f70: vmcnt(0) alone).
__device__ __forceinline__ void land() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);
  asm volatile("" ::: "memory");
}

// The eight elements 16 t + 8 h .. + 7 of a row in memory.
template <typename T>
__device__ __forceinline__ Frag<T> global_frag(const T* row, bool inside, int t, int h, int D) {
  Frag<T> f;
  const int c0 = 16 * t + 8 * h;
  if constexpr (sizeof(T) == 2) {
    f.v = load_chunk<T>(row, inside, c0, D);
  } else {
    const f32x4 a = __builtin_bit_cast(f32x4, load_chunk<T>(row, inside, c0, D));
    const f32x4 b = __builtin_bit_cast(f32x4, load_chunk<T>(row, inside, c0 + 4, D));
    f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// Four consecutive elements of a row from c0 on, rounded from fp32, at any alignment.
template <typename T>
__device__ __forceinline__ void store4(T* row, int c0, int D, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 2) {
    const u32x2 w = {pack2<T>(a, b), pack2<T>(c, d)};
    if (c0 + 4 <= D) {
      __builtin_memcpy(row + c0, &w, 8);
      return;
    }
    uint16_t* p = (uint16_t*)(row + c0);
    if (c0 < D) p[0] = (uint16_t)w[0];
    if (c0 + 1 < D) p[1] = (uint16_t)(w[0] >> 16);
    if (c0 + 2 < D) p[2] = (uint16_t)w[1];
  } else {
    const f32x4 w = {a, b, c, d};
    if (c0 + 4 <= D) {
      __builtin_memcpy(row + c0, &w, 16);
      return;
    }
    if (c0 < D) row[c0] = a;
    if (c0 + 1 < D) row[c0 + 1] = b;
    if (c0 + 2 < D) row[c0 + 2] = c;
  }
}

// What store4 rounds off its four values, rounded itself (16-bit types).
template <typename T>
__device__ __forceinline__ void store4_rest(T* row, int c0, int D, float a, float b, float c, float d) {
  const float x[4] = {a, b, c, d};
  float r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = x[i] - to_acc(from_acc<T>(x[i]));
  store4<T>(row, c0, D, r[0], r[1], r[2], r[3]);
}

// n / d for 0 <= n < 2^31 by a multiplication (d >= 1).
struct FastDiv {
  uint32_t mul = 0, shift = 0, d = 1;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1u << shift) < div && shift < 31) ++shift;
    mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - div)) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    const uint32_t t = __umulhi(n, mul);
    return (uint32_t)(((uint64_t)t + n) >> shift);
  }
};

enum MaskKind { kMaskNone = 0, kMaskBool = 1, kMaskF32 = 2, kMaskF16 = 3, kMaskBF16 = 4 };

struct AttnArgs {
  const void *q, *k, *v, *o, *g;       // o: forward output (backward reads it); g: its gradient
  void *out, *dq, *dk, *dv;
  float *stat;                         // forward statistics of each row, see attn_fwd.hip
  float *part;                         // fp32 partial results of split work
  float *delta;                        // rowsum(g o), [B][H][N]
  float *bounds;                       // fp16: per 64 rows max |g_i| and max |delta_i|; per 64 keys max |v_j|
  const void* mask;
  const int32_t *klen, *qlen, *qstart;
  int64_t qs[3], ks[3], vs[3], os[3], gs[3], dqs[3], dks[3], dvs[3];  // element strides of batch, head, row
  int64_t ms[4];                       // mask strides: batch, head, row, key (0 where broadcast)
  int B, H, Hk, G, N, M, D;
  int maskKind, causal, keyMask;       // keyMask: the mask is the same for every head and row
  uint32_t* bits;                      // a truth-value mask packed by attn_bits_kernel, strides bs in words
  int64_t bs[3];
  int modeQ, modeK, modeV, modeG;      // LoadMode where the tensor streams through LDS
  int nsplit, tiles, chunk;            // work split along the other axis; tiles along the own one; steps per split
  float scale, c;                      // c = scale * log2(e)
  FastDiv divN;
};

// Row statistics: planes of [B][H][N] fp32 (two with an additive mask), then for the 16-bit types what the
// output's rounding took off, [B][H][N][D].
__host__ __device__ inline int64_t stat_planes(const AttnArgs& a) {
  return (a.maskKind > kMaskBool ? 2 : 1) * (int64_t)a.B * a.H * a.N;
}
template <typename T> __device__ __forceinline__ T* rest_row(const AttnArgs& a, int64_t row) {
  return (T*)(a.stat + stat_planes(a)) + row * a.D;
}

// Keys of sequence b that exist, and queries.
__device__ __forceinline__ int key_count(const AttnArgs& a, int b) {
  return a.klen ? min(max(a.klen[b], 0), a.M) : a.M;
}
__device__ __forceinline__ int query_count(const AttnArgs& a, int b) {
  return a.qlen ? min(max(a.qlen[b], 0), a.N) : a.N;
}
// The key position of query 0.
__device__ __forceinline__ int query_start(const AttnArgs& a, int b) {
  return a.qstart ? min(max(a.qstart[b], -a.N), a.M) : a.M - a.N;
}

// A mask element as an additive term in natural units.
__device__ __forceinline__ float mask_bias(const AttnArgs& a, int64_t off) {
  if (a.maskKind == kMaskBool) return ((const uint8_t*)a.mask)[off] ? 0.0f : kNegInf;
  if (a.maskKind == kMaskF32) return ((const float*)a.mask)[off];
  if (a.maskKind == kMaskF16) return to_acc(((const f16s*)a.mask)[off]);
  return to_acc(((const bf16s*)a.mask)[off]);
}

// What a kernel does about a mask: nothing, an additive term per score, a bit per score.
enum MaskForm { kNoMask = 0, kAdd = 1, kBits = 2 };

// Bits of the keys in front of a row's last one: 32 keys from j0 on.
__device__ __forceinline__ uint32_t bits_below(int lim, int j0) {
  const int n = lim - j0;
  return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
}

// The additive mask of a lane's 16 scores of one query: keys j0 + 8 (r / 4) + 4 h + r % 4. off: the
// query's row. Keys at or behind M give -inf and are not read. Four adjacent keys are one
// (unaligned) load where the mask's keys are adjacent.
__device__ __forceinline__ void mask_of_keys(const AttnArgs& a, int64_t off, int j0, int h, f32x16& x) {
  if (a.ms[3] == 1 && j0 + 32 <= a.M) {
    const int64_t at = off + j0 + 4 * h;
    if (a.maskKind == kMaskF32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 y;
        __builtin_memcpy(&y, (const float*)a.mask + at + 8 * q, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * q + i] = y[i];
      }
    } else {
      u32x2 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) __builtin_memcpy(&w[q], (const uint16_t*)a.mask + at + 8 * q, 8);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint16_t bits = (uint16_t)(w[r >> 2][(r >> 1) & 1] >> (16 * (r & 1)));
        x[r] = a.maskKind == kMaskF16 ? to_acc(f16s{bits}) : to_acc(bf16s{bits});
      }
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int j = j0 + 8 * (r >> 2) + 4 * h + (r & 3);
    x[r] = j < a.M ? mask_bias(a, off + (int64_t)j * a.ms[3]) : kNegInf;
  }
}

// The same for one key and the queries n0 + 8 (r / 4) + 4 h + r % 4; off: the key's column.
__device__ __forceinline__ void mask_of_queries(const AttnArgs& a, int64_t off, int n0, int h, f32x16& x) {
  const int64_t at = off + (int64_t)(n0 + 4 * h) * a.ms[2];
  if (n0 + 32 <= a.N) {
    if (a.maskKind == kMaskF32) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = ((const float*)a.mask)[at + (8 * (r >> 2) + (r & 3)) * a.ms[2]];
    } else {
      uint16_t w[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = ((const uint16_t*)a.mask)[at + (8 * (r >> 2) + (r & 3)) * a.ms[2]];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = a.maskKind == kMaskF16 ? to_acc(f16s{w[r]}) : to_acc(bf16s{w[r]});
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int n = n0 + 8 * (r >> 2) + 4 * h + (r & 3);
    x[r] = n < a.N ? mask_bias(a, off + (int64_t)n * a.ms[2]) : kNegInf;
  }
}

// A score under a mask in natural units; -inf removes the key, whatever its score.
__device__ __forceinline__ float masked_score(const AttnArgs& a, float s, float bias) {
  return bias == kNegInf ? kNegInf : fmaf(s, a.scale, bias);
}

// Bit i: row row0 + row_of(i) of the keys takes part, as far as a mask over keys alone says.
template <typename LD> __device__ __forceinline__ uint32_t live_keys(const AttnArgs& a, int b, int row0) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < LD::NIT; ++i) {
    const int j = min(row0 + LD::row_of(i), a.M - 1);
    bits |= (uint32_t)(mask_bias(a, (int64_t)b * a.ms[0] + (int64_t)j * a.ms[3]) != kNegInf) << i;
  }
  return LD::NIT == 32 || bits != (1u << (LD::NIT & 31)) - 1 ? bits : ~0u;
}

// How many pieces to cut the streamed axis of `steps` tiles into, for `wgs` workgroups on `cus` CUs: the
// least of what the busiest CU takes and of joining. A workgroup alone takes `lat` us per tile (one wave
// per SIMD waits for its own reads, products and exponentials in turn), workgroups that share a CU `thr`
// each, and 4 us go to a start and an end; n pieces of `bytes` are written and read at 4 TB/s, behind a
// launch of 6 us. At most 64 pieces, which bounds the workspace; a call of one workgroup then uses 64 CUs
// (one token over 131072 keys of 128 channels: 31 us). `steps` are the buffer's: lengths are known to the device alone, and the pieces behind
// a short sequence's end are written and joined empty.
inline int best_split(int64_t wgs, int64_t steps, int cus, double lat, double thr, double bytes) {
  int best = 1;
  double least = 0;
  for (int64_t n = 1; n <= 64 && n <= steps; ++n) {
    const int64_t chunk = (steps + n - 1) / n, each = (wgs * n + cus - 1) / cus;
    if ((steps + chunk - 1) / chunk != n) continue;  // fewer pieces do the same
    const double cost = std::max(lat, thr * (double)each) * (double)chunk + 4.0 * (double)((each + 1) / 2) +
                        (n > 1 ? 6.0 + (double)n * 2.0 * bytes / 4e6 : 0.0);
    if (n == 1 || cost < least) best = (int)n, least = cost;
  }
  return best;
}

// The workgroup's place: consecutive places on one XCD (workgroups are dealt to
// the eight XCDs in turn), so that a head's keys stay in one XCD's L2.
__device__ __forceinline__ uint32_t xcd_place(uint32_t id, uint32_t n) {
  const uint32_t q = n / 8, r = n % 8, x = id % 8, y = id / 8;
  return x * q + min(x, r) + y;
}

}  // namespace lfamd
