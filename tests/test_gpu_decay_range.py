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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_steps(gpu, dtype):
    """4096 tokens one by one: no error of the decay adds up, and the prompt's form ends in the same state.

    With x = 1 - a about 2^-10 and random keys and values a state holds some 1 / (2 x) = 512 tokens' energy. Each token's two
    roundings are at most 2^-24 of the state and of what is added, rms 2^-24 / sqrt(3), and add up as their squares: sqrt(512) 2^-24 / sqrt(3)
    = 7.8e-7 of the state's norm, and 2^-24 from the second. A factor a - 1 off by 2^-23 of itself gives 0.7 2^-23. Sum 9.2e-7; a head's norm of
    256 elements keeps to a tenth of that, twice it is allowed. (A factor a off by half its unit, 2^-25, alone gives
    0.7 1024 2^-25 = 2.1e-5.)"""
    import laplacianformer_amd as lf

    print(f"decay many steps {dtype}", flush=True)
    H, T, d = 32, 4096, 16
    lg = torch.tensor([-(1.0 + h / 37.0) / 1024 for h in range(H)])
    K, V = (gen((T, 1, H, 1, d), 420 + i, dtype).to(gpu) for i in range(2))
    L, state = lg.to(gpu), torch.zeros(1, H, d, d, device=gpu)
    with torch.no_grad():
        for t in range(T):
            lf.decay_attention_step(K[t], K[t], V[t], L, state)
        k, v = (x[:, 0, :, 0].transpose(0, 1)[None] for x in (K, V))
        _, last = lf.decay_attention(k, k, v, L, return_state=True)
    left = torch.exp(lg.double()[:, None] * torch.arange(T - 1, -1, -1).double())
    k, v = k[0].cpu().double(), v[0].cpu().double()
    ref = (k * left[..., None]).transpose(-1, -2) @ v
    for got, name in ((state, "steps"), (last, "prompt")):
        err = (got[0].cpu().double() - ref).norm(dim=(1, 2)) / ref.norm(dim=(1, 2))
        assert err.max() <= 1.9e-6, (dtype, name, err.max().item())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_step_decays_around_the_border(gpu, dtype):
    """The step's two forms of the decay, on both sides of where they meet, and a decay of nothing and of all; bounds as
    in test_step, where fast heads' states vanish beside what is added to them and in front of them."""
    import laplacianformer_amd as lf

    lg = torch.tensor([0.0, -1e-7, -0.49, -0.5, -0.51, -3.0, -100.0, -math.inf])
    H, d, e = len(lg), 20, 36
    for size in (1e-3, 1.0, 1e6):
        q, k, v = gen((1, H, 1, d), 430, dtype), gen((1, H, 1, d), 431, dtype), gen((1, H, 1, e), 432, dtype)
        s0 = gen((1, H, d, e), 433, "f32", size)
        state = s0.to(gpu)
        out = lf.decay_attention_step(q.to(gpu), k.to(gpu), v.to(gpu), lg.to(gpu), state, scale=0.2)
        a, kv = torch.exp(lg.double()).view(1, H, 1, 1), k.double().transpose(-1, -2) * v.double()
        S, mag = a * s0.double() + kv, a * s0.double().abs() + kv.abs()
        bc.assert_within(state, S, 6 * bc.U32 * mag, (dtype, size, "state"))
        ref, m = 0.2 * (q.double() @ S), 0.2 * (q.double().abs() @ mag)
        c = (d + 16) * bc.U32
        # Outputs of 0.2 * 20 products with states of up to 4e6: fp16 ends at 65504, and what lies well beyond is an infinity.
        out, most = out.cpu(), torch.finfo(out.dtype).max
        fits = ref.abs() < 0.99 * most
        bound = c * m + bc.unit(TORCH_DT[dtype]) * (ref.abs() + c * m)
        bc.assert_within(out[fits], ref[fits], bound[fits], (dtype, size, "out"))
        assert bool(torch.isinf(out[ref.abs() > 1.01 * most]).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_very_slow_heads(gpu, dtype):
    """Decays of some 2^-15.6 a token over 32768 tokens, in heads enough that no sequence is cut: no error of a whole tile's factor
    adds up over the 1024 tiles.

    The state grows as the square root of the tokens. A tile goes into it in r = 16 accumulations (fp32; bf16: 2 of each of
    3 pieces, 6) and one rounding of its factor, each rms 2^-24 / sqrt(3) of the state then, which add up as their squares:
    sqrt((r + 1) 1024 / 2) 2^-24 / sqrt(3) = 3.2e-6 (2.1e-6) of the last state. One and a half times that is allowed. (A factor off by half
    its unit, 2^-25, alone gives 2^-25 1024 / sqrt(3) = 1.8e-5.)"""
    import ctypes

    import laplacianformer_amd as lf
    import laplacianformer_amd._lib as L

    print(f"decay very slow heads {dtype}", flush=True)
    H, B, N, d = 32, 128, 32768, 8
    lg = torch.tensor([-(1.0 + h / 37.0) * 2e-5 for h in range(H)])
    desc = L.Decay(batch=B, heads=H, kv_heads=H, tokens=N, key_dim=d, value_dim=d, log_decay=16, scale=1.0)
    assert lf.capi().lfamd_decay_attention_workspace_size(lf.dtype_code(TORCH_DT[dtype]), ctypes.byref(desc)) == 0
    k, v = (gen((1, H, N, d), 440 + i, dtype).to(gpu) for i in range(2))
    with torch.no_grad():
        _, last = lf.decay_attention(k.expand(B, -1, -1, -1), k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), lg.to(gpu), return_state=True)
    left = torch.exp(lg.double()[:, None] * torch.arange(N - 1, -1, -1).double())
    ref = (k[0].cpu().double() * left[..., None]).transpose(-1, -2) @ v[0].cpu().double()
    err = (last[B // 2].cpu().double() - ref).norm(dim=(1, 2)) / ref.norm(dim=(1, 2))
    assert err.max() <= (4.8e-6 if dtype == "f32" else 3.2e-6), (dtype, err.max().item())


def _tile_steps(k, v, lg, N):
    """sum over tiles of a^(tokens behind it) (sum over j of |k_j|) (largest a^(tile's end - j) |v_j|), [B, H, d, e]: what one
    step of the value operand's second piece, relative to the tile's largest value in the column, comes to in the state."""
    front = -N % 32
    K, V = (torch.cat((torch.zeros(*x.shape[:2], front, x.shape[3], dtype=torch.float64), x.double().abs()), 2) for x in (k, v))
    n = (N + front) // 32
    K, V = (x.view(*x.shape[:2], n, 32, x.shape[3]) for x in (K, V))
    inside = dc.powers(lg, 31 - torch.arange(32))[None, :, None, :, None]
    behind = dc.powers(lg, 32 * (n - 1 - torch.arange(n)))[None, :, :, None, None]
    return (behind * K.sum(3)[..., :, None] * (inside * V).amax(3)[..., None, :]).sum(2)


@pytest.mark.parametrize("N", [20, 32, 64, 75, 200, 2500])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_columns_of_very_different_sizes(gpu, dtype, N):
    """Value columns of 1 to 1e-5 and an outlier of 600 in the first tile beside them; the states' columns do not see one
    another, in any type. Bound: decaycheck's with, in fp16, half a step 2^-25 of the value operand's second piece over a largest
    value of 2^8 in the tile's column, 2^-33 of that."""
    import laplacianformer_amd as lf

    print(f"decay columns {dtype} {N}", flush=True)
    B, H, d, e = 1, 4, 24, 40
    lg = torch.tensor([-2.0 ** -12, -0.03, 0.0, -1.5])
    q, k, v, g = (gen((B, H, N, x), 450 + i, "f32") for i, x in enumerate((d, d, e, e)))
    size = torch.logspace(0, -5, 8)[torch.arange(e) % 8]
    v, g = v * size, g * size.flip(0)
    v[:, :, 3, 0], g[:, :, -2, 33] = 600.0, -300.0
    v[:, :, N // 2:, 9] = 0.0
    q, k, v, g = (x.to(TORCH_DT[dtype]) for x in (q, k, v, g))
    s0 = gen((B, H, d, e), 455, "f32") * size
    ref = dc.decay(q, k, v, lg, 0.2, s0, None, g)
    leaves = [x.to(gpu).requires_grad_() for x in (q, k, v, s0)]
    out, last = lf.decay_attention(*leaves[:3], lg.to(gpu), state=leaves[3], scale=0.2, return_state=True)
    grads = torch.autograd.grad(out, leaves, g.to(gpu))
    extra = {}
    if dtype == "f16":
        extra["last"] = 2.0 ** -33 * _tile_steps(k, v, lg, N)
        # Backwards: the same on the queries and the outputs' gradients, whose tiles begin where the sequence does.
        a = torch.exp(lg.double())[None, :, None, None]
        extra["dstate"] = 2.0 ** -33 * 0.2 * a * _tile_steps(q.flip(2), g.flip(2), lg, N)
    for name, x in zip(("out", "last", "dq", "dk", "dv", "dstate"), (out, last, *grads)):
        bc.assert_within(x, ref[name][0], ref[name][1] + extra.get(name, 0.0), (dtype, N, name))


def test_fp16_states_of_other_sizes_than_the_values(gpu):
    """fp16: large and small states beside small and large values, zero columns and tiles, and scales far from 1."""
    import laplacianformer_amd as lf

    lg = torch.tensor([-0.01, -1.0])
    for ss, vs, scale in ((1e12, 1e-6, 0.1), (1e-12, 3e4, 0.1), (0.0, 6e4, 1e4), (1.0, 1e-4, 1e-8), (1e-20, 1e-3, 1.0)):
        print("decay fp16 states", ss, vs, scale, flush=True)
        q, k, v, g = (gen((1, 2, 100, 32), 460 + i, "f32") for i in range(4))
        k[:, :, 40:80] = 0.0
        v[:, :, :, 5], v[:, :, 10:70, 6] = 0.0, 0.0
        q, k, v, g = q.half(), k.half(), (v * vs).clamp(-6e4, 6e4).half(), g.half()
        s0 = gen((1, 2, 32, 32), 465, "f32") * ss
        s0[..., 7] = 0.0
        ref = dc.decay(q, k, v, lg, scale, s0, None, g)
        leaves = [x.to(gpu).requires_grad_() for x in (q, k, v, s0)]
        out, last = lf.decay_attention(*leaves[:3], lg.to(gpu), state=leaves[3], scale=scale, return_state=True)
        grads = torch.autograd.grad(out, leaves, g.to(gpu))
        step = 2.0 ** -33 * _tile_steps(k, v, lg, 100)
        bc.assert_within(last, ref["last"][0], ref["last"][1] + step, (ss, vs, scale, "last"))
        for name, x in zip(("out", "dq", "dk", "dv", "dstate"), (out, *grads)):
            if ref[name][0].abs().max() < torch.finfo(x.dtype).max:
                a = torch.exp(lg.double())[None, :, None, None]
                step = 2.0 ** -33 * scale * a * _tile_steps(q.flip(2), g.flip(2), lg, 100) if name == "dstate" else 0.0
                bc.assert_within(x, ref[name][0], ref[name][1] + step, (ss, vs, scale, name))


def test_decays_that_require_a_gradient(gpu):
    """They have none, which is no reason to refuse a call that records none."""
    import laplacianformer_amd as lf

    q, lg = torch.randn(1, 2, 5, 8, device=gpu), torch.full((2,), -0.1, device=gpu)
    want, leaf = lf.decay_attention(q, q, q, lg), lg.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        lf.decay_attention(q, q, q, leaf)
    with torch.no_grad():
        assert torch.equal(lf.decay_attention(q, q, q, leaf), want)
        one = q[:, :, :1]
        lf.decay_attention_step(one, one, one, leaf, torch.zeros(1, 2, 8, 8, device=gpu))
    with torch.inference_mode():
        assert torch.equal(lf.decay_attention(q, q, q, leaf), want)


def _long(q, k, v, lg, first):
    """sum over j <= i of a^(i - j) (q_i . k_j) v_j + a^(i + 1) q_i first in 64 bits by chunks, the same of the terms'
    magnitudes, and the state behind the last token."""
    out, mag, step = torch.empty_like(v), torch.empty_like(v), 256
    S, M = first, first.abs()
    for n in range(0, q.shape[2], step):
        x, y, z = (t[:, :, n:n + step] for t in (q, k, v))
        i = torch.arange(x.shape[2])
        D, ahead = dc.powers(lg, i[:, None] - i)[None], dc.powers(lg, i + 1)[None, ..., None]
        out[:, :, n:n + step] = ((x @ y.transpose(-1, -2)) * D) @ z + ahead * (x @ S)
        mag[:, :, n:n + step] = ((x.abs() @ y.abs().transpose(-1, -2)) * D) @ z.abs() + ahead * (x.abs() @ M)
        y, whole = y * dc.powers(lg, len(i) - 1 - i)[None, ..., None], dc.powers(lg, torch.tensor(len(i)))[None, :, None, None]
        S, M = whole * S + y.transpose(-1, -2) @ z, whole * M + y.abs().transpose(-1, -2) @ z.abs()
    return out, mag, S


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [1, 24])
def test_long_gradients(gpu, dtype, heads):
    """20011 tokens, two query heads to each key head, keys narrower than values, a state and its gradient, in sequences cut into few
    segments and into many. Bound: test_long's count of additions for one run and the shared heads' one, and decaycheck's pieces; in fp16
    decaycheck's steps of the largest score and state. States, norm-relative: the slowest head's holds 64 tiles' energy of up to 17 roundings of rms
    2^-24 / sqrt(3) each, 1.1e-6; 2^-18 is allowed."""
    import laplacianformer_amd as lf

    H, N, d, e, scale = 2 * heads, 20011, 24, 40, 0.2
    print(f"decay long gradients {dtype} H{H}", flush=True)
    lg = torch.tensor(([-2.0 ** -12, -2.0 ** -6, -2.0 ** -9, -0.4] * heads)[:H])
    q, k, v, g = (gen((1, h, N, x), 470 + i, dtype) for i, (h, x) in enumerate(((H, d), (heads, d), (heads, e), (H, e))))
    s0, gl = gen((1, H, d, e), 475, "f32"), gen((1, H, d, e), 476, "f32")
    leaves = [x.to(gpu).requires_grad_() for x in (q, k, v, s0)]
    res = lf.decay_attention(*leaves[:3], lg.to(gpu), state=leaves[3], scale=scale, return_state=True)
    grads = torch.autograd.grad(res, leaves, (g.to(gpu), gl.to(gpu)))
    Q, G = q.double(), g.double()
    K, V = (x.double().repeat_interleave(2, 1) for x in (k, v))
    turn = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    back = lambda x: x.flip(2)  # noqa: E731
    R = gl.double() * torch.exp(-lg.double())[None, :, None, None] / scale  # a^(N - 1 - i) in place of a^(N - i)
    ref = {"out": _long(Q, K, V, lg, s0.double()), "dq": _long(G, V, K, lg, turn(s0.double())),
           "dk": _long(back(V), back(G), back(Q), lg, turn(R)), "dv": _long(back(K), back(Q), back(G), lg, R)}
    u = bc.unit(TORCH_DT[dtype])
    c = (64 + 3 * N / 32 + 64 + 2) * bc.U32 + (0.0 if dtype == "f32" else 2 * u * u + 2.0 ** -22)
    for name, got in zip(("out", "dq", "dk", "dv"), (res[0], *grads[:3])):
        want, mag, _ = (scale * x for x in ref[name])
        if name in ("dk", "dv"):
            want, mag = (back(x).reshape(1, heads, 2, N, -1).sum(2) for x in (want, mag))
        err = c * mag + (2.0 ** -38 * 64 * mag.amax() if dtype == "f16" else 0.0)
        bc.assert_within(got, want, err + u * (want.abs() + err), (dtype, H, name))
    for name, got in (("last", res[1]), ("dstate", grads[3])):
        want = ref["out"][2] if name == "last" else scale * torch.exp(lg.double())[None, :, None, None] * ref["dv"][2]
        assert (got.cpu().double() - want).norm() <= 2.0 ** -18 * want.norm(), (dtype, H, name)
