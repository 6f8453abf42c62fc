"""decay_attention's and gated_add_rms_norm's checks that need no GPU: refusals of the C entries before any device call, CPU
tensors at the public entry points, the ctypes layout of the call structs, and the kernels' registers."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from test_kernel_resources_cpu import _kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL, DUMMY = ctypes.c_void_p(0), ctypes.c_void_p(16)


@pytest.fixture(scope="module")
def lib():
    import laplacianformer_amd as lf

    return lf.capi()


def decay(**kw):
    import laplacianformer_amd._lib as L

    d = L.Decay(batch=1, heads=4, kv_heads=2, tokens=8, key_dim=16, value_dim=24, log_decay=16, scale=0.25)
    for n, x in kw.items():
        setattr(d, n, x)
    return d


def norm(**kw):
    import laplacianformer_amd._lib as L

    d = L.GatedNorm(rows=12, width=8, x_stride=8, residual_stride=8, gate_rows=4, gate_stride=8, scale=1.0, eps=1e-6)
    for n, x in kw.items():
        setattr(d, n, x)
    return d


def test_struct_layout(tmp_path):
    import laplacianformer_amd._lib as L

    src = ['#include <stddef.h>', '#include <stdio.h>', '#include "laplacianformer_amd.h"', "int main(void) {"]
    want = []
    for name, cls in (("lfamd_decay", L.Decay), ("lfamd_decay_grads", L.DecayGrads), ("lfamd_gated_norm", L.GatedNorm)):
        src.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            src.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src.append("return 0; }")
    (tmp_path / "s.c").write_text("\n".join(src))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def test_decay_refusals(lib):
    import laplacianformer_amd._lib as L

    def f(d, dt=0, q=DUMMY, out=DUMMY, last=NULL, ws=NULL, n=0):
        return lib.lfamd_decay_attention(dt, ctypes.byref(d) if d else None, q, DUMMY, DUMMY, NULL, out, last, ws, n, NULL)

    assert f(decay(), 3) == 2 and b"dtype" in lib.lfamd_last_error()
    assert f(None) == 1
    for kw in ({"batch": -1}, {"tokens": -1}, {"kv_heads": 3}, {"kv_heads": 0}, {"heads": 0}, {"scale": 0.0}, {"scale": float("nan")},
               {"scale": float("inf")}, {"log_decay": 0}):
        assert f(decay(**kw)) == 1, kw
    for kw in ({"key_dim": 129}, {"key_dim": 0}, {"value_dim": 129}, {"value_dim": 0}, {"tokens": 2 ** 29 + 1}, {"batch": 2 ** 21},
               {"batch": 2 ** 62}):
        assert f(decay(**kw)) == 3, kw
    assert f(decay(), q=NULL) == 1 and f(decay(), out=NULL) == 1
    assert f(decay(batch=0)) == 0 and f(decay(tokens=0)) == 0 and f(decay(heads=0, kv_heads=0)) == 0
    size = lib.lfamd_decay_attention_workspace_size
    long = decay(tokens=100000)
    need = size(0, ctypes.byref(long))
    assert need > 0 and need % (4 * 16 * 24 * 4) == 0 and size(0, ctypes.byref(decay())) == 0 and size(3, ctypes.byref(long)) == 0
    assert f(long) == 1 and b"workspace" in lib.lfamd_last_error()
    assert f(long, ws=DUMMY, n=need - 1) == 1
    assert f(long, ws=ctypes.c_void_p(24), n=need) == 1 and b"aligned" in lib.lfamd_last_error()

    assert lib.lfamd_decay_attention(0, ctypes.byref(decay()), DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, NULL, 0, NULL) == 1
    assert b"last_state" in lib.lfamd_last_error()  # the first state's memory

    def b(d, g, dt=0, ws=DUMMY, n=1 << 40):
        return lib.lfamd_decay_attention_backward(dt, ctypes.byref(d), DUMMY, DUMMY, DUMMY, NULL, ctypes.byref(g) if g else None, ws, n, NULL)

    full = L.DecayGrads(grad_out=16, grad_q=16, grad_k=16, grad_v=16)
    assert b(decay(), None) == 1 and b(decay(), full, 3) == 2
    assert b(decay(), L.DecayGrads(grad_out=16, grad_k=16)) == 1 and b"together" in lib.lfamd_last_error()
    assert b(decay(), L.DecayGrads(grad_out=16, grad_state=16)) == 1 and b"grad_state" in lib.lfamd_last_error()
    assert b(decay(), L.DecayGrads(grad_q=16)) == 1
    assert b(decay(), L.DecayGrads(grad_out=16, grad_k=16, grad_v=16, grad_state=32, grad_last_state=32)) == 1
    assert b(decay(), full, ws=NULL) == 1 and b(decay(), full, ws=DUMMY, n=8) == 1  # shared heads: fp32 parts
    assert b(decay(), full, ws=ctypes.c_void_p(24)) == 1
    assert b(decay(), L.DecayGrads()) == 0 and b(decay(batch=0), full) == 0
    bsize = lib.lfamd_decay_attention_backward_workspace_size
    assert bsize(0, ctypes.byref(decay())) >= 4 * 8 * (16 + 24) * 4 and bsize(0, ctypes.byref(decay(kv_heads=4))) == 0
    strides = (ctypes.c_int64 * 2)(1536, 384)
    s = lambda d, q=DUMMY, st=DUMMY: lib.lfamd_decay_attention_step(0, ctypes.byref(d), q, DUMMY, DUMMY, DUMMY, st, strides, NULL)  # noqa: E731
    assert s(decay()) == 1 and b"one token" in lib.lfamd_last_error()
    assert s(decay(tokens=1), q=NULL) == 1 and s(decay(tokens=1), st=NULL) == 1 and s(decay(tokens=1, batch=0)) == 0


def test_gated_norm_refusals(lib):
    def f(d, dt=0, x=DUMMY, total=DUMMY):
        return lib.lfamd_gated_add_rms_norm(dt, ctypes.byref(d) if d else None, x, DUMMY, DUMMY, NULL, DUMMY, DUMMY, total, NULL, NULL, NULL)

    assert f(None) == 1 and f(norm(), 3) == 2 and f(norm(), 7) == 2 and f(norm(weight_dtype=2), 1) == 2 and f(norm(gate_dtype=1)) == 2
    assert f(norm(rows=-1)) == 1 and f(norm(gate_rows=-1)) == 1 and f(norm(gate_rows=5)) == 1 and f(norm(scale=float("inf"))) == 1
    assert f(norm(width=0)) == 3 and f(norm(width=8193)) == 3 and f(norm(rows=2 ** 30)) == 3
    assert f(norm(), x=NULL) == 1 and f(norm(), total=NULL) == 1 and f(norm(rows=0)) == 0

    def b(d, ws=DUMMY, n=1 << 40, gy=DUMMY, wp=DUMMY, rp=DUMMY, gate=DUMMY, dwp=DUMMY, dg=DUMMY):
        return lib.lfamd_gated_add_rms_norm_backward(0, ctypes.byref(d), gy, 8, NULL, 8, DUMMY, DUMMY, DUMMY, wp, gate, DUMMY, rp, DUMMY,
                                                     DUMMY, DUMMY, dwp, dg, ws, n, NULL)

    assert b(norm(), gy=NULL) == 1 and b(norm(), rp=NULL) == 1 and b(norm(), wp=NULL) == 1 and b(norm(), gate=NULL) == 1
    assert b(norm(), ws=NULL) == 1 and b(norm(), n=8) == 1 and b(norm(), ws=ctypes.c_void_p(18)) == 1 and b"aligned" in lib.lfamd_last_error()
    size = lib.lfamd_gated_add_rms_norm_backward_workspace_size
    assert size(0, ctypes.byref(norm())) >= 2 * 8 * 4 and size(0, ctypes.byref(norm(rows=0))) == 0 and size(0, ctypes.byref(norm(width=9000))) == 0


def test_cpu_tensors_raise():
    import laplacianformer_amd as lf

    q, lg = torch.zeros(1, 2, 3, 8), torch.zeros(2)
    for fn in (lambda: lf.decay_attention(q, q, q, lg), lambda: lf.decay_attention_step(q, q, q, lg, torch.zeros(1, 2, 8, 8)),
               lambda: lf.gated_add_rms_norm(q, torch.ones(8), q)):
        with pytest.raises(RuntimeError, match="GPU"):
            fn()
    with pytest.raises(RuntimeError, match="no gradient"):
        lf.decay_attention_step(q.requires_grad_(), q, q, lg, torch.zeros(1, 2, 8, 8))


# Scratch bytes per lane of the kernels that do not fit their registers (1024 threads have 128 each): (kernel, type, its integer arguments): the most that it may take.
SCRATCH = {
    ("gated_add_rms_norm_bwd_kernel", "f", (1024, 2, 0, 1)): 36, ("gated_add_rms_norm_bwd_kernel", "f", (1024, 2, 1, 1)): 108,
    ("gated_add_rms_norm_bwd_kernel", "f", (1024, 2, 1, 0)): 64, ("gated_add_rms_norm_bwd_kernel", "f", (1024, 2, 2, 1)): 24,
    ("gated_add_rms_norm_bwd_kernel", "f16s", (1024, 1, 1, 1)): 60, ("gated_add_rms_norm_bwd_kernel", "bf16s", (1024, 1, 1, 1)): 72,
    ("gated_add_rms_norm_bwd_kernel", "bf16s", (1024, 1, 1, 0)): 16,
}


def test_kernels_scratch(tmp_path):
    seen, over = set(), []
    for k in _kernels(tmp_path):
        m = re.search(r"\d(decay_[a-z_]*kernel|gated_[a-z_]*kernel)(?:I(f|NS_\d+(b?f16s)E)((?:L[ib]\d+E)*)E)?", k["name"])
        if not m:
            continue
        key = (m[1], m[3] or m[2], tuple(int(x) for x in re.findall(r"L[ib](\d+)E", m[4] or "")))
        seen.add(key)
        if int(k.get("private_segment_fixed_size", 0)) > SCRATCH.get(key, 0):
            over.append((key, k["private_segment_fixed_size"]))
    assert not over, over
    assert len(seen) >= 120 and set(SCRATCH) <= seen
