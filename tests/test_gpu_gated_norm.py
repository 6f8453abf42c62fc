"""gated_add_rms_norm against its 64-bit form."""
import pytest
import torch

import blockcheck as bc
import decaycheck as dc
from lfcheck import TORCH_DT, gen

pytestmark = pytest.mark.gpu

WIDTHS = [1, 3, 8, 64, 100, 333, 512, 513, 1024, 2048, 2056, 4096, 4100, 8189, 8192]


def check(gpu, dtype, shape, gate, post, scale=1.0, w32=False, with_gs=True, seed=0, eps=1e-5):
    """Outputs and all gradients. gate: None or its shape; w32: weights and gate in float32."""
    import laplacianformer_amd as lf

    print(f"gated norm {dtype} {shape} gate {gate} post {post} scale {scale} {w32}", flush=True)
    W, wt = shape[-1], torch.float32 if w32 else TORCH_DT[dtype]
    x, res = gen(shape, seed + 1, dtype), gen(shape, seed + 2, dtype, 2.0)
    w, wp = ((1 + 0.2 * gen((W,), seed + 3 + i, "f32")).to(wt) for i in range(2))
    wp = wp if post else None
    g = None if gate is None else gen(gate, seed + 5, "f32", 0.5).to(wt)
    gy, gs = gen(shape, seed + 6, dtype), gen(shape, seed + 7, dtype) if with_gs else None
    ref = dc.gated_norm(x, w, res, wp, g, scale, eps, gy, gs)
    d = {n: t.to(gpu).requires_grad_() for n, t in (("x", x), ("w", w), ("res", res), ("wp", wp), ("gate", g)) if t is not None}
    call = lambda: lf.gated_add_rms_norm(d["x"], d["w"], d["res"], post_weight=d.get("wp"), gate=d.get("gate"), scale=scale,  # noqa: E731
                                         eps=eps)
    y, total = call()
    names = list(d)
    grads = torch.autograd.grad((y, total) if with_gs else y, [d[n] for n in names], (gy.to(gpu), gs.to(gpu)) if with_gs else gy.to(gpu))
    what = (dtype, shape, gate, post, scale)
    bc.assert_within(y, *ref["y"], (*what, "y"))
    bc.assert_within(total, *ref["sum"], (*what, "sum"))
    for n, t in zip(names, grads):
        assert t.dtype == d[n].dtype
        bc.assert_within(t, *ref["d" + n], (*what, "d" + n))
    with torch.no_grad():
        again = call()
        assert torch.equal(again[0], y) and torch.equal(again[1], total)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_widths(gpu, dtype, width):
    check(gpu, dtype, (3, 5, width), (width,), True, 0.5)
    check(gpu, dtype, (3, 5, width), (3, 1, width), True, w32=True)
    check(gpu, dtype, (3, 5, width), (3, 5, width), True, -1.5)
    check(gpu, dtype, (2, 1, width), None, False, 0.25, with_gs=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("post", [True, False])
def test_gates(gpu, dtype, post):
    """Each layout of the gate, with many rows for few gates and few rows for many."""
    for shape, gate in (((301, 96), (96,)), ((301, 96), (1, 96)), ((301, 96), (301, 96)), ((2, 1500, 40), (2, 1, 40)),
                        ((700, 2, 40), (700, 1, 40)), ((4, 9, 33, 64), (4, 1, 1, 64)), ((4, 9, 33, 64), (4, 9, 1, 64)),
                        ((1, 800, 520), (1, 1, 520)), ((3, 40, 1030), (3, 1, 1030)), ((40,), (40,)), ((5, 2600), None)):
        check(gpu, dtype, shape, gate, post, 0.7, w32=len(shape) == 3)
