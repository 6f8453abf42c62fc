"""The transformer-block operators' checks that need no GPU: refusals of the C entries before any device
call, CPU tensors at the public entry points, and the ctypes layout of the call structs."""
import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL, DUMMY = ctypes.c_void_p(0), ctypes.c_void_p(16)


@pytest.fixture(scope="module")
def lib():
    import laplacianformer_amd as lf

    return lf.capi()


def desc(**kw):
    import laplacianformer_amd._lib as L

    d = L.Attention(batch=1, heads=4, kv_heads=2, q_len=8, k_len=9, head_dim=16, scale=0.25)
    for n, x in kw.items():
        setattr(d, n, x)
    return d


def test_struct_layout(tmp_path):
    """The ctypes structs have the C structs' sizes and offsets."""
    import laplacianformer_amd._lib as L

    src = ['#include <stddef.h>', '#include <stdio.h>', '#include "laplacianformer_amd.h"', "int main(void) {"]
    want = []
    for name, cls in (("lfamd_attention", L.Attention), ("lfamd_attention_grads", L.AttentionGrads)):
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


def test_attention_refusals(lib):
    f = lambda d, dt=0, q=DUMMY: lib.lfamd_softmax_attention(dt, ctypes.byref(d) if d else None, q, DUMMY, DUMMY, DUMMY, NULL, NULL, 0, NULL)
    assert f(desc(), 3) == 2 and b"dtype" in lib.lfamd_last_error()
    assert f(None) == 1
    assert f(desc(batch=-1)) == 1
    assert f(desc(head_dim=129)) == 3 and b"head size 129" in lib.lfamd_last_error()
    assert f(desc(head_dim=0)) == 3
    assert f(desc(kv_heads=3)) == 1 and f(desc(kv_heads=0)) == 1 and f(desc(heads=0)) == 1
    assert f(desc(scale=0.0)) == 1 and f(desc(scale=float("nan"))) == 1 and f(desc(scale=float("inf"))) == 1
    assert f(desc(mask_kind=5)) == 1 and f(desc(mask_kind=1)) == 1  # unknown; no mask pointer
    assert f(desc(k_len=2 ** 31)) == 3 and f(desc(q_len=2 ** 30)) == 3  # two heads share a key head
    assert f(desc(batch=2 ** 31)) == 3
    assert f(desc(), q=NULL) == 1 and b"null" in lib.lfamd_last_error()
    assert f(desc(batch=0)) == 0 and f(desc(q_len=0)) == 0 and f(desc(heads=0, kv_heads=0)) == 0
    b = lambda d, g, dt=0, ws=DUMMY, n=1 << 40: lib.lfamd_softmax_attention_backward(
        dt, ctypes.byref(d), DUMMY, DUMMY, DUMMY, DUMMY, DUMMY, ctypes.byref(g) if g else None, ws, n, NULL)
    import laplacianformer_amd._lib as L

    full = L.AttentionGrads(grad_out=16, grad_q=16, grad_k=16, grad_v=16)
    assert b(desc(), None) == 1
    assert b(desc(), L.AttentionGrads(grad_out=16, grad_k=16)) == 1 and b"together" in lib.lfamd_last_error()
    assert b(desc(), L.AttentionGrads(grad_q=16)) == 1
    assert b(desc(), full, 3) == 2
    assert b(desc(), full, 0, NULL) == 1 and b(desc(), full, 0, DUMMY, 4) == 1
    assert b(desc(), full, 0, ctypes.c_void_p(24)) == 1 and b"aligned" in lib.lfamd_last_error()
    assert b(desc(batch=0), full) == 0
    size = lib.lfamd_softmax_attention_backward_workspace_size
    assert size(0, ctypes.byref(desc())) >= 4 * 8 * 4
    assert size(1, ctypes.byref(desc())) > size(2, ctypes.byref(desc()))  # fp16: the gradients' bounds
    assert size(3, ctypes.byref(desc())) == 0 and size(0, ctypes.byref(desc(head_dim=200))) == 0
    fsize = lib.lfamd_softmax_attention_workspace_size
    assert fsize(2, ctypes.byref(desc())) == 0 and fsize(2, ctypes.byref(desc(q_len=1, k_len=100000))) > 0
    stats = lib.lfamd_softmax_attention_stats_size
    assert stats(0, ctypes.byref(desc())) == 4 * 8 * 4 and stats(2, ctypes.byref(desc())) == 4 * 8 * (4 + 2 * 16)
    assert stats(1, ctypes.byref(desc(mask_kind=2, head_dim=1, q_len=7))) == 4 * 7 * (8 + 2)
    assert stats(3, ctypes.byref(desc())) == 0
    long = desc(q_len=1, k_len=100000)
    assert f(long, 2) == 1 and b"workspace" in lib.lfamd_last_error()


def test_norm_refusals(lib):
    f = lambda dt=0, wt=0, x=DUMMY, res=NULL, s=NULL, rows=4, width=8: lib.lfamd_add_rms_norm(
        dt, x, width, res, width, wt, DUMMY, DUMMY, s, NULL, rows, width, 1e-6, NULL)
    assert f(3, 3) == 2 and f(1, 2) == 2 and f(7) == 2
    assert f(rows=-1) == 1 and f(width=0) == 3 and f(width=16385) == 3
    assert f(x=NULL) == 1 and f(res=DUMMY) == 1  # a residual without a place for the sum
    assert f(rows=0) == 0
    f8 = lambda scale: lib.lfamd_add_rms_norm_fp8(0, DUMMY, 8, NULL, 8, 0, DUMMY, DUMMY, scale, NULL, 4, 8, 1e-6, NULL)
    assert f8(NULL) == 1
    b = lambda ws=NULL, n=0, dw=DUMMY, gy=DUMMY: lib.lfamd_add_rms_norm_backward(
        0, gy, 8, NULL, 8, DUMMY, 8, NULL, 8, 0, DUMMY, DUMMY, DUMMY, dw, 4, 8, ws, n, NULL)
    assert b() == 1 and b"workspace" in lib.lfamd_last_error()
    assert b(ctypes.c_void_p(18), 1 << 20) == 1 and b"aligned" in lib.lfamd_last_error()
    assert b(gy=NULL) == 1
    size = lib.lfamd_add_rms_norm_backward_workspace_size
    assert size(0, 4, 8) >= 32 and size(0, 0, 8) == 0 and size(0, 4, 16385) == 0


def test_rotary_refusals(lib):
    s3 = (ctypes.c_int64 * 3)(64, 64, 16)

    def f(dt=0, B=1, N=4, d=16, sections=(4, 4), base=100.0, q=DUMMY, heads=1, axes=None):
        sec = (ctypes.c_int64 * max(len(sections), 1))(*sections)
        return lib.lfamd_rotary(dt, q, s3, DUMMY, s3, heads, NULL, NULL, NULL, NULL, 0, B, N, d, DUMMY, 0, s3,
                                len(sections) if axes is None else axes, sec, base, 0, 0, NULL)

    assert f(3) == 2 and f(B=-1) == 1
    assert f(sections=()) == 3 and f(axes=9, sections=(1,) * 9) == 3
    assert f(sections=(4, 5)) == 1 and b"room for 8" in lib.lfamd_last_error()
    assert f(sections=(0, 0)) == 1 and f(sections=(-1, 4)) == 1 and f(sections=(2 ** 40,)) == 1
    assert f(sections=(128, 1), d=1024) == 1 and f(d=1025) == 3
    assert f(base=0.0) == 1 and f(base=float("nan")) == 1
    assert f(q=NULL) == 1 and f(B=70000) == 3
    assert f(B=0) == 0 and f(N=0) == 0 and f(heads=0) == 0


def test_cpu_tensors_are_refused():
    import laplacianformer_amd as lf

    x, w = torch.randn(2, 8), torch.randn(8)
    q = torch.randn(1, 2, 4, 8)
    for fn in (lambda: lf.add_rms_norm(x, w), lambda: lf.add_rms_norm_fp8(x, w),
               lambda: lf.rotary(q, None, lf.grid_positions((2, 2)), [2, 2]), lambda: lf.softmax_attention(q, q, q),
               lambda: lf.AttentionBlock(8, 2)(torch.randn(1, 4, 8))):
        with pytest.raises(RuntimeError, match="must be on GPU"):
            fn()


def test_host_helpers():
    import laplacianformer_amd as lf

    p = lf.grid_positions((2, 3), start=(5, -1))
    assert p.dtype == torch.int32 and p.tolist() == [[5, 5, 5, 6, 6, 6], [-1, 0, 1, -1, 0, 1]]
    assert lf.rotary_sections(64, 2) == [16, 16] and lf.rotary_sections(128, 3) == [22, 21, 21]
    with pytest.raises(ValueError):
        lf.AttentionBlock(30, 4)


def test_forward_mode_is_refused():
    """A dual tensor without requires_grad takes no autograd node: its tangent must not be dropped silently."""
    import laplacianformer_amd as lf
    from torch.autograd import forward_ad

    r = lambda *s: torch.randn(*s)
    x, w, q, pos = r(2, 8), r(8), r(1, 2, 4, 8), lf.grid_positions((2, 2))
    mask = r(4, 4)
    with forward_ad.dual_level():
        d = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for fn in (lambda: lf.add_rms_norm(d(x), w), lambda: lf.add_rms_norm(x, d(w)), lambda: lf.add_rms_norm(x, w, d(x)),
                   lambda: lf.add_rms_norm_fp8(d(x), w), lambda: lf.add_rms_norm_fp8(x, w, d(x)),
                   lambda: lf.rotary(d(q), None, pos, [2, 2]), lambda: lf.rotary(q, d(q), pos, [2, 2]),
                   lambda: lf.softmax_attention(d(q), q, q), lambda: lf.softmax_attention(q, d(q), q),
                   lambda: lf.softmax_attention(q, q, d(q)), lambda: lf.softmax_attention(q, q, q, mask=d(mask))):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                fn()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                fn()


def test_block_infers_no_axes_from_a_token_count():
    """Tokens that are no square's and have neither grid nor positions raise, before any kernel; a causal block
    and a batch with lengths take one axis at any count, and a block without positions needs no grid."""
    import laplacianformer_amd as lf

    for n in (10, 63, 65):
        with pytest.raises(ValueError, match="no square"):
            lf.AttentionBlock(8, 2)(torch.randn(1, n, 8))
        with pytest.raises(ValueError, match="no square"):
            lf.AttentionBlock(8, 2, attention="laplacian", positions=False)(torch.randn(1, n, 8))
        x, k = torch.randn(1, n, 8), torch.ones(1, dtype=torch.int32)
        for fn in (lambda: lf.AttentionBlock(8, 2, causal=True)(x), lambda: lf.AttentionBlock(8, 2)(x, lengths=k),
                   lambda: lf.AttentionBlock(8, 2, positions=False)(x), lambda: lf.AttentionBlock(8, 2)(x, grid=(1, n)),
                   lambda: lf.AttentionBlock(8, 2)(x, positions=torch.zeros(1, n, dtype=torch.int32))):
            with pytest.raises(RuntimeError, match="must be on GPU"):
                fn()


def test_laplacian_block_refuses_grids_before_any_kernel():
    """The Laplacian attention pools two axes: other grids, and masks or lengths, raise by name."""
    import laplacianformer_amd as lf

    block = lf.AttentionBlock(8, 2, attention="laplacian", pool=2)
    x = torch.randn(1, 64, 8)
    for grid in ((64,), (4, 4, 4), (1, 64), (64, 1)):
        with pytest.raises(ValueError, match="two axes"):
            block(x, grid=grid)
    for kw in ({"mask": torch.ones(64, 64, dtype=torch.bool)}, {"lengths": torch.ones(1, dtype=torch.int32)}):
        with pytest.raises(ValueError, match="neither mask"):
            block(x, **kw)
    for kw in ({}, {"grid": (4, 16)}):
        with pytest.raises(RuntimeError, match="must be on GPU"):
            block(x, **kw)


def test_grid_positions_refuse_missing_starts():
    """A start per axis: with fewer, the axes behind them were dropped, and with them their tokens."""
    import laplacianformer_amd as lf

    for start in ((5,), (1, 2, 3), ()):
        with pytest.raises(ValueError, match="as many starts"):
            lf.grid_positions((2, 3), start=start)
    assert lf.grid_positions((2, 3), start=[0, 7])[1].tolist() == [7, 8, 9, 7, 8, 9]


def test_no_mask_is_planned_without_queries_or_keys(lib):
    """A call without queries, or without keys, may come with an empty mask, whose pointer is null, and strides of 0,
    which say that the mask is the same for every query: it is taken as a call without a mask throughout."""
    fwd, bwd, stats = (lib.lfamd_softmax_attention_workspace_size, lib.lfamd_softmax_attention_backward_workspace_size,
                       lib.lfamd_softmax_attention_stats_size)
    for sizes in ({"q_len": 0}, {"k_len": 0}, {"q_len": 0, "k_len": 0}):
        for kind in (1, 2, 3, 4):
            for dt in (0, 1, 2):
                for f in (fwd, bwd, stats):
                    assert f(dt, ctypes.byref(desc(mask_kind=kind, **sizes))) == f(dt, ctypes.byref(desc(**sizes)))
