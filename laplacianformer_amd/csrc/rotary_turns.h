// The turns of rotary positions per unit of position, base^(-j / n) / (2 pi) modulo 1, as 128-bit
// fractions (host code). They are good to 2^-110 of the frequency: at a position of 63 bits and frequencies
// up to 1 (base >= 1) the angle is good to 2^-47 turns, far below fp32's rounding of it. (Fractions of
// 64 bits would leave half a turn there; formed in doubles they were 1.4e-6 rad off at 2^31.)
#pragma once

#include <math.h>
#include <stdint.h>

namespace lfamd {

typedef unsigned __int128 turn128;

// m 2^(e - 128), the upper bit of m set. Products are cut off, at most 2^-125 of them lost.
struct Wide {
  turn128 m;
  int e;
};

inline Wide wide(double x) {
  int e;
  const double f = frexp(x, &e);
  return {(turn128)(uint64_t)ldexp(f, 64) << 64, e};
}

inline Wide operator*(const Wide& a, const Wide& b) {
  const uint64_t ah = (uint64_t)(a.m >> 64), al = (uint64_t)a.m, bh = (uint64_t)(b.m >> 64), bl = (uint64_t)b.m;
  Wide r{(turn128)ah * bh + ((turn128)ah * bl >> 64) + ((turn128)al * bh >> 64), a.e + b.e};
  if (!(r.m >> 127)) r.m <<= 1, --r.e;
  return r;
}

// out[j] = floor(2^128 frac(base^(-j / n) / (2 pi))), j = 0 .. n - 1. base: positive and finite.
inline void rotary_turns(double base, int n, turn128* out) {
  // q = base^(-1 / n): base q^n = 1 by Newton's iteration from a double, 52 -> 100 -> more than 110 bits. A
  // step is so small that a double holds it.
  Wide q = wide(1.0);
  if (n > 1) {
    q = wide(pow(base, -1.0 / n));
    const Wide b = wide(base);
    for (int it = 0; it < 2; ++it) {
      Wide p = b, sq = q;
      for (int k = n; k; k >>= 1, sq = sq * sq)
        if (k & 1) p = p * sq;
      const turn128 one = (turn128)1 << 127;  // of p.e = 1
      const double left = p.e == 1 ? (double)(p.m - one) * -0x1p-127 : (double)((turn128)0 - p.m) * 0x1p-128;  // 1 - p
      const turn128 was = q.m;
      q.m += (turn128)(__int128)((double)q.m * (left / n));
      if (left > 0 && q.m < was) q.m = one | q.m >> 1, ++q.e;
      else if (!(q.m >> 127)) q.m <<= 1, --q.e;
    }
  }
  // 1 / (2 pi) = 0x0.28BE60DB9391054A7F09D5F47D4D377036D8..., its first digits shifted up
  Wide f{(turn128)0xA2F9836E4E441529ULL << 64 | 0xFC2757D1F534DDC0ULL, -2};
  for (int j = 0; j < n; ++j, f = f * q)  // whole turns go: a base below 1 has frequencies above 1
    out[j] = f.e <= -128 || f.e >= 128 ? 0 : f.e < 0 ? f.m >> -f.e : f.m << f.e;
}

}  // namespace lfamd
