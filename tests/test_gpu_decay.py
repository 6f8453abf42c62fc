"""decay_attention and decay_attention_step against their 64-bit forms."""
import math

import pytest
import torch

import blockcheck as bc
import decaycheck as dc
from lfcheck import TORCH_DT, gen

pytestmark = pytest.mark.gpu

DECAYS = {"slow": [math.log1p(-2.0 ** -5), math.log1p(-2.0 ** -9), math.log1p(-2.0 ** -12), -0.3],
          "fast": [-1.0, -0.25, -5.0, -40.0], "none": [0.0, 0.0, -0.0, 0.0], "edge": [float("-inf"), 0.0, -1e-7, -1e30]}


def decays(kind, H):
    return torch.tensor((DECAYS[kind] * H)[:H], dtype=torch.float32)


def leaf(t, gpu):
    return t.to(gpu).requires_grad_()


def check(gpu, dtype, B, H, Hk, N, d, e, kind="slow", state=True, lengths=None, scale=None, seed=0, size=1.0):
    """Forward, last state and every gradient of one call."""
    import laplacianformer_amd as lf

    print(f"decay {dtype} B{B} H{H}/{Hk} N{N} d{d} e{e} {kind} {lengths}", flush=True)
    q, k, v = gen((B, H, N, d), seed + 1, dtype, size), gen((B, Hk, N, d), seed + 2, dtype, size), gen((B, Hk, N, e), seed + 3, dtype, size)
    g, lg = gen((B, H, N, e), seed + 4, dtype), decays(kind, H)
    s0, gl = (gen((B, H, d, e), seed + 5, "f32", 2.0), gen((B, H, d, e), seed + 6, "f32")) if state else (None, None)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    sc = 1.0 / math.sqrt(d) if scale is None else scale
    ref = dc.decay(q, k, v, lg, sc, s0, n, g, gl)
    qd, kd, vd = (leaf(x, gpu) for x in (q, k, v))
    sd = leaf(s0, gpu) if state else None
    out, last = lf.decay_attention(qd, kd, vd, lg.to(gpu), state=sd, lengths=None if n is None else n.to(gpu), scale=scale,
                                   return_state=True)
    assert out.dtype == q.dtype and last.dtype == torch.float32
    what = (dtype, B, H, Hk, N, d, e, kind)
    bc.assert_within(out, *ref["out"], (*what, "out"))
    bc.assert_within(last, *ref["last"], (*what, "last"))
    leaves = [qd, kd, vd] + ([sd] if state else [])
    grads = torch.autograd.grad((out, last) if state else (out,), leaves, (g.to(gpu), gl.to(gpu)) if state else (g.to(gpu),))
    for name, x in zip(("dq", "dk", "dv", "dstate"), grads):
        bc.assert_within(x, *ref[name], (*what, name))
    return out


SIZES = [(1, 1, 1, 1, 1, 1), (2, 3, 1, 2, 3, 8), (1, 2, 2, 31, 16, 32), (2, 2, 1, 32, 32, 32), (1, 4, 2, 33, 33, 50), (1, 2, 2, 64, 64, 64),
         (2, 2, 2, 65, 80, 80), (1, 3, 3, 100, 96, 40), (1, 2, 1, 129, 128, 128), (2, 4, 4, 196, 32, 64), (1, 2, 2, 300, 64, 32),
         (1, 2, 2, 97, 100, 128), (1, 1, 1, 515, 128, 16), (3, 2, 2, 40, 8, 128)]


@pytest.mark.parametrize("shape", SIZES, ids=str)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sizes(gpu, dtype, shape):
    check(gpu, dtype, *shape)


@pytest.mark.parametrize("kind", ["fast", "none", "edge"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_decays(gpu, dtype, kind):
    check(gpu, dtype, 1, 4, 2, 150, 48, 64, kind)
    check(gpu, dtype, 2, 4, 4, 70, 64, 64, kind, state=False)
