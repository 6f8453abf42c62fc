"""decay_attention and decay_attention_step at values and lengths where the arithmetic, not the formula, could fail."""
import math

import pytest
import torch

import blockcheck as bc
import decaycheck as dc
from lfcheck import TORCH_DT, gen

pytestmark = pytest.mark.gpu


def run(gpu, q, k, v, lg, scale, g=None, state=None):
    """{name: tensor} of out and last, and with g of the gradients."""
    import laplacianformer_amd as lf

    leaves = [t.to(gpu).requires_grad_(g is not None) for t in (q, k, v)]
    out, last = lf.decay_attention(*leaves, lg.to(gpu), state=None if state is None else state.to(gpu), scale=scale, return_state=True)
    res = {"out": out, "last": last}
    if g is not None:
        res.update(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, g.to(gpu))))
    return res


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("first,second", [(3, 5), (12, 30), (8, 39)])
def test_scores_that_overflow_outside_the_triangle(gpu, dtype, first, second):
    """An early query of 1e20 and a later key of 1e20 meet in no output; nor do an early gradient and a later value."""
    B, H, N, d = 1, 2, 40, 16
    lg = torch.tensor([-0.01, -1.0])
    for big, late in (("q", "k"), ("g", "v")):
        print(f"decay overflow {dtype} {first} {second} {big}{late}", flush=True)
        x = {n: gen((B, H, N, d), 400 + i, dtype) for i, n in enumerate("qkvg")}
        x[big][:, :, first] = 1e20
        x[late][:, :, second] = 1e20
        ref = dc.decay(x["q"], x["k"], x["v"], lg, 0.25, None, None, x["g"])
        for name, got in run(gpu, x["q"], x["k"], x["v"], lg, 0.25, x["g"]).items():
            bc.assert_within(got, *ref[name], (dtype, first, second, big, name))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_values_that_are_not_finite(gpu, dtype):
    """A NaN or an infinity of a query stays with its token, of a key it reaches later ones; of a value it reaches the
    other tokens of its tile too, but none in front of that, and no other head or sequence."""
    B, H, N, d = 2, 2, 75, 32  # tiles of tokens 0-10, 11-42, 43-74
    lg, at = torch.tensor([-0.02, -0.5]), 60
    x = [gen((B, H, N, d), 410 + i, dtype) for i in range(3)]
    ref, bound = dc.decay(*x, lg, 0.2)["out"]
    for bad in (math.nan, math.inf):
        for i, name in enumerate("qkv"):
            print(f"decay {bad} in {name} {dtype}", flush=True)
            y = [t.clone() for t in x]
            y[i][1, 1, at, 5] = bad
            out = run(gpu, *y, lg, 0.2)["out"].cpu()
            ok = torch.ones(B, H, N, dtype=torch.bool)
            ok[1, 1, at:at + 1 if name == "q" else N] = False
            if name == "v":
                ok[1, 1, 43:] = False
            assert not bool(torch.isfinite(out[1, 1, at]).all())
            bc.assert_within(out[ok], ref[ok], bound[ok], (dtype, bad, name))
