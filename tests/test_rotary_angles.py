"""Rotary angles at far positions, against angles formed in 80 decimal digits: the turns per unit of
position (csrc/rotary_turns.h, built with the host compiler) and what the kernel makes of them."""
import decimal
import math
import os
import shutil
import subprocess

import pytest
import torch

from lfcheck import gen

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
D = decimal.Decimal
CTX = decimal.Context(prec=80, Emax=10 ** 6, Emin=-10 ** 6)
# Machin: pi = 16 atan(1/5) - 4 atan(1/239)
_atan = lambda x: sum(D((-1) ** k) / ((2 * k + 1) * D(x) ** (2 * k + 1)) for k in range(70))
with decimal.localcontext(CTX):
    TWO_PI = 2 * (16 * _atan(5) - 4 * _atan(239))


def turns(base, n):
    """base^(-j / n) / (2 pi) for j < n."""
    with decimal.localcontext(CTX):
        return [D(base) ** (-D(j) / n) / TWO_PI for j in range(n)]


def angle(pos, turn):
    """The angle in (-pi, pi] of a whole position, as a float."""
    with decimal.localcontext(CTX):
        t = D(pos) * turn % 1
        return float((t - (1 if t > D("0.5") else -1 if t < D("-0.5") else 0)) * TWO_PI)


PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "rotary_turns.h"
int main(int argc, char** argv) {
  lfamd::turn128 t[128];
  for (int i = 1; i + 1 < argc; i += 2) {
    const int n = atoi(argv[i + 1]);
    lfamd::rotary_turns(strtod(argv[i], nullptr), n, t);
    for (int j = 0; j < n; ++j) printf("%016llx%016llx\n", (unsigned long long)(t[j] >> 64), (unsigned long long)t[j]);
  }
}
"""


def test_turns(tmp_path):
    """Each fraction is within 2^-110 of its frequency and 2^-127 of the exact one, modulo whole turns: a product
    loses up to 2^-125 of itself, base q^n (at most 16 products) and so q about 2^-121, and q enters 127 times."""
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-O2", "-std=c++17", "-Wall", "-I", os.path.join(ROOT, "laplacianformer_amd", "csrc"),
                    str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    cases = [(10000.0, 32), (10000.0, 128), (500.0, 13), (1.0, 5), (1e9, 64), (1.7e308, 128), (7.0, 1), (1.5, 2),
             (0.5, 4), (1e-3, 16), (1e-30, 3), (4.0, 2), (2.0 ** 40, 40), (math.nextafter(16.0, 0), 4), (math.nextafter(16.0, 17), 4),
             (math.nextafter(1.0, 2), 128), (math.nextafter(1.0, 0), 128), (5e-324, 1), (5e-324, 7), (math.pi, 100)]
    args = [x for base, n in cases for x in (repr(base), str(n))]
    out = subprocess.run([str(tmp_path / "t"), *args], check=True, capture_output=True, text=True).stdout.split()
    at = 0
    with decimal.localcontext(CTX):
        for base, n in cases:
            for j, want in enumerate(turns(base, n)):
                got = D(int(out[at], 16)) / 2 ** 128
                at += 1
                if want > D(2) ** 100:  # nothing behind the point is held
                    continue
                off = abs(got - want % 1)
                assert min(off, 1 - off) <= want * D(2) ** -110 + D(2) ** -127, (base, n, j)
    assert at == len(out)


FAR = [0, 1, -1, 1000003, 2 ** 31 - 1, -2 ** 31, 10 ** 12 + 7, -10 ** 15 - 3, 2 ** 53 + 1, 2 ** 62 + 12345, 2 ** 63 - 1, -2 ** 63]


@pytest.mark.gpu
@pytest.mark.parametrize("base,n", [(10000.0, 32), (10000.0, 128), (1e6, 20), (1.0, 3), (0.5, 8)])
def test_far_positions(gpu, base, n):
    """(x, 0) turns to x (cos, sin) of the exact angle. The angle is off by 2^-32 turns (the bits that the kernel
    drops) and by half a step of fp32 at up to one half turn, 2^-25 of it; cosine and sine by 4 of 2^-24, the
    two products and their sum by 2 of 2^-24."""
    import laplacianformer_amd as lf

    print(f"rotary far {base} {n}", flush=True)
    x = torch.zeros(1, 1, len(FAR), 2 * n)
    x[..., :n] = 1.0
    for pos, many in ((torch.tensor([FAR], dtype=torch.int64), FAR),
                      (torch.tensor([[max(min(p, 2 ** 31 - 1), -2 ** 31) for p in FAR]], dtype=torch.int32), None)):
        many = many or pos[0].tolist()
        y, _ = lf.rotary(x.to(gpu), None, pos.to(gpu), [n], base=base)
        back, _ = lf.rotary(y, None, -pos.to(gpu), [n], base=base)
        t = turns(base, n)
        want = torch.tensor([[angle(p, u) for u in t] for p in many], dtype=torch.float64)
        tol = 2 * math.pi * 2.0 ** -32 + math.pi * 2.0 ** -25 + 6 * 2.0 ** -24
        got = y[0, 0].cpu().double()
        for part, ref in ((got[:, :n], want.cos()), (got[:, n:], want.sin())):
            off = (part - ref).abs().amax(1)
            assert bool((off <= tol).all()), list(zip(many, off.tolist()))
        # the lowest value of a type is its own negative: it does not turn back
        keep = [i for i, p in enumerate(many) if p != torch.iinfo(pos.dtype).min]
        assert (back.cpu() - x)[:, :, keep].abs().max() <= 4 * tol
