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


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strides_and_empty(gpu, dtype):
    import laplacianformer_amd as lf

    t = TORCH_DT[dtype]
    buf, res, gates = gen((6, 5, 80), 11, dtype), gen((5, 6, 48), 12, dtype), gen((5, 1, 60), 13, dtype)
    w, wp = gen((48,), 14, dtype), gen((48,), 15, dtype)
    for x in (buf.transpose(0, 1)[..., :48], buf.transpose(0, 1)[..., 7:55]):
        gate = gates[..., 5:53]
        ref = dc.gated_norm(x, w, res, wp, gate, 0.5, 1e-6, res, x)
        xd = buf.to(gpu).as_strided(x.shape, x.stride(), x.storage_offset()).requires_grad_()
        gd = gates.to(gpu)[..., 5:53].requires_grad_()
        rd, wd, pd = (y.to(gpu).requires_grad_() for y in (res, w, wp))
        y, total = lf.gated_add_rms_norm(xd, wd, rd, post_weight=pd, gate=gd, scale=0.5)
        grads = torch.autograd.grad((y, total), (xd, rd, wd, pd, gd), (res.to(gpu), x.to(gpu)))
        for name, got in zip(("y", "sum", "dx", "dres", "dw", "dwp", "dgate"), (y, total, *grads)):
            bc.assert_within(got, *ref[name], name)
        (only,) = torch.autograd.grad(lf.gated_add_rms_norm(xd, wd, rd, post_weight=pd, gate=gd, scale=0.5)[1], rd, res.to(gpu))
        assert torch.equal(only, res.to(gpu))
    for shape, gate in (((0, 48), (48,)), ((3, 0, 48), (3, 1, 48)), ((0, 2, 48), (0, 1, 48))):
        x = torch.empty(shape, dtype=t, device=gpu, requires_grad=True)
        g, wd = torch.ones(gate, dtype=t, device=gpu, requires_grad=True), w.to(gpu).requires_grad_()
        y, total = lf.gated_add_rms_norm(x, wd, x.detach(), post_weight=wd, gate=g)
        dx, dw, dg = torch.autograd.grad((y, total), (x, wd, g), (torch.empty_like(y), torch.empty_like(y)))
        assert dx.shape == x.shape and dg.shape == g.shape and bool((dw == 0).all()) and bool((dg == 0).all())
    zeros = torch.zeros(3, 48, dtype=t, device=gpu)
    y, total = lf.gated_add_rms_norm(zeros, w.to(gpu), zeros, post_weight=wp.to(gpu))
    assert bool((y == 0).all()) and bool((total == 0).all())


def test_many_rows_and_gates(gpu):
    """More rows than a grid has workgroups, and more gates than a grid's second axis: signs come out, and each
    gate's gradient is the sum of its two rows'."""
    import laplacianformer_amd as lf

    rows = 9_000_002
    x = torch.ones(rows // 2, 2, 2, dtype=torch.bfloat16, device=gpu)
    x[::3, 0, 0] = -4.0
    x[::3, 0, 1] = 4.0
    ones = torch.ones(2, dtype=torch.bfloat16, device=gpu)
    y, total = lf.gated_add_rms_norm(x, ones, torch.zeros_like(x), gate=torch.full((rows // 2, 1, 2), 2.0, dtype=torch.bfloat16, device=gpu))
    assert torch.equal(y, x.sign()) and torch.equal(total, 2 * x)
    x, gate = x[:100_000].clone(), torch.ones(100_000, 1, 2, dtype=torch.float32, device=gpu, requires_grad=True)
    _, total = lf.gated_add_rms_norm(x, ones, x, gate=gate)
    (dg,) = torch.autograd.grad(total, gate, torch.ones_like(total))
    assert torch.equal(dg, x.float().sum(1, keepdim=True))


def test_gradients_against_differences(gpu):
    import laplacianformer_amd as lf

    x, res, w, wp, gate = (gen(s, 31 + i, "f32") for i, s in enumerate(((3, 4, 50), (3, 4, 50), (50,), (50,), (3, 1, 50))))
    gy, gs = gen((3, 4, 50), 37, "f32"), gen((3, 4, 50), 38, "f32")
    d = [t.to(gpu).requires_grad_() for t in (x, res, w, wp, gate)]
    grads = torch.autograd.grad(lf.gated_add_rms_norm(d[0], d[2], d[1], post_weight=d[3], gate=d[4], scale=0.7), d, (gy.to(gpu), gs.to(gpu)))

    def loss(x, r, w, wp, gate):
        unit = lambda t: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
        s = r + 0.7 * gate * unit(x) * wp
        return ((unit(s) * w * gy.double()).sum() + (s * gs.double()).sum()).item()

    base = [t.double() for t in (x, res, w, wp, gate)]
    for i in range(5):
        way = gen(tuple(base[i].shape), 40 + i, "f32").double()
        p, m = list(base), list(base)
        p[i], m[i] = base[i] + 1e-6 * way, base[i] - 1e-6 * way
        want, got = (loss(*p) - loss(*m)) / 2e-6, (grads[i].cpu().double() * way).sum().item()
        size = (grads[i].cpu().double().abs() * way.abs()).sum().item()
        assert abs(got - want) <= 1e-4 * size, (i, got, want, size)


def test_graph_repeats_and_refusals(gpu):
    import laplacianformer_amd as lf
    from torch.autograd import forward_ad

    x, r = gen((4, 300, 520), 50, "bf16").to(gpu).requires_grad_(), gen((4, 300, 520), 51, "bf16").to(gpu)
    g, gate = gen((4, 300, 520), 52, "bf16").to(gpu), gen((4, 1, 520), 53, "bf16").to(gpu).requires_grad_()
    w = torch.ones(520, device=gpu, requires_grad=True)

    def fn(t, gt, wt):
        y, s = lf.gated_add_rms_norm(t, wt, r, post_weight=wt, gate=gt, scale=0.5)
        return y + s

    def eager():
        leaves = [t.detach().clone().requires_grad_() for t in (x, gate, w)]
        out = fn(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    want = eager()
    step = lf.GraphedStep(fn, [x, gate, w], g)
    for _ in range(3):
        step.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([step.out, *step.grads], want))
        assert all(torch.equal(a, b) for a, b in zip(eager(), want))
    f = lf.gated_add_rms_norm
    x, w = x.detach()[:, :7, :64].contiguous(), w.detach()[:64]
    bad = [lambda: f(x, w, x[:, :6]), lambda: f(x, w[:63], x), lambda: f(x, w, x.half()), lambda: f(x, w.half(), x), lambda: f(x, w, x, post_weight=w[:5]),
           lambda: f(x, w, x, gate=x[0]), lambda: f(x, w, x, gate=x[:, :, :1]), lambda: f(x, w, x, gate=x[:1]), lambda: f(x, w, x, gate=x[:, :3]),
           lambda: f(x, w, x, gate=x.half()), lambda: f(x, w, x, gate=x.cpu()), lambda: f(x, w, x, scale=float("inf")), lambda: f(x.double(), w, x.double()),
           lambda: f(x.cpu(), w.cpu(), x.cpu()), lambda: f(x, w, None), lambda: f(torch.zeros(2, 8193, device=gpu), torch.zeros(8193, device=gpu),
                                                                                 torch.zeros(2, 8193, device=gpu))]
    for i, fn in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError, AttributeError)):
            fn()
            raise AssertionError(f"call {i} was taken")
    t = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(f(t, w, x)[0], t, x, create_graph=True)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
        f(forward_ad.make_dual(x, x), w, x)


def _plain_block(block, x, res, gate, lengths, first):
    """An AttentionBlock with decay attention and post norm in 64 bits."""
    p = {n: t.detach().double().requires_grad_() for n, t in block.named_parameters()}
    unit = lambda t: t / (t.square().mean(-1, keepdim=True) + block.eps).sqrt()  # noqa: E731
    if first:
        total, y = x, unit(x) * p["weight"]
    else:
        total = res + block.residual_scale * gate * unit(x) * p["post_weight"]
        y = unit(total) * p["weight"]
    B, N, C = x.shape
    H, Hk = block.heads, block.kv_heads
    d = C // H
    qkv = (y @ p["qkv.weight"].T + p["qkv.bias"]).view(B, N, H + 2 * Hk, d).transpose(1, 2)
    q, k, v = qkv.split((H, Hk, Hk), 1)
    angle = torch.arange(N).double()[:, None] * block.base ** (-torch.arange(d // 2).double() / (d // 2))

    def turn(t):
        a, b = t.chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)

    live = (torch.arange(N) < lengths.view(B, 1))[:, None, :, None]
    q, k, v = turn(q), turn(k).repeat_interleave(H // Hk, 1) * live, v.repeat_interleave(H // Hk, 1)
    n = torch.arange(N)
    o = (q @ k.transpose(-1, -2) * dc.powers(block._log_decay.cpu(), n[:, None] - n)[None] @ v) * d ** -0.5 * live
    o = unit(o.transpose(1, 2).reshape(B, N, C)) * p["out_weight"]
    return o @ p["proj.weight"].T + p["proj.bias"], total, p


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_blocks_together(gpu, dtype):
    """Two AttentionBlocks with decay attention, post norms, gates, shared heads and lengths, run and differentiated together.
    Bound, norm-relative: per block and direction eleven roundings of the type in a row (norm, projection, rotary,
    attention, its norm, projection, the sum and their gradients), a condition of 4 for the norms' and attention's
    cancellations, two blocks: 2 * 44 u; fp32's products add sums of up to 96 terms: 2 * 400 u."""
    import laplacianformer_amd as lf

    print(f"decay blocks {dtype}", flush=True)
    torch.manual_seed(11)
    t = TORCH_DT[dtype]
    B, N, C = 2, 75, 96
    blocks = torch.nn.ModuleList([lf.AttentionBlock(C, 6, 2, attention="decay", post_norm=i == 1, residual_scale=0.5 if i else 1.0)
                                  for i in range(2)]).to(t)
    x, g, gs = (gen((B, N, C), 60 + i, dtype) for i in range(3))
    gate, lengths = gen((B, 1, C), 63, dtype), torch.tensor([N, N - 20], dtype=torch.int32)
    X, G = x.double().requires_grad_(), gate.double().requires_grad_()
    y0, s0, p0 = _plain_block(blocks[0], X, None, None, lengths, True)
    y1, s1, p1 = _plain_block(blocks[1], y0, s0, G, lengths, False)
    names = [f"{i}.{n}" for i, p in enumerate((p0, p1)) for n in p]
    want = [y1, s1, *torch.autograd.grad((y1, s1), [X, G, *p0.values(), *p1.values()], (g.double(), gs.double()))]
    blocks = blocks.to(gpu)
    xd, gd = x.to(gpu).requires_grad_(), gate.to(gpu).requires_grad_()
    n = lengths.to(gpu)
    y, s = blocks[0](xd, lengths=n)
    y, s = blocks[1](y, s, lengths=n, gate=gd)
    got = [y, s, *torch.autograd.grad((y, s), [xd, gd, *blocks.parameters()], (g.to(gpu), gs.to(gpu)))]
    assert [f"{n}" for n, _ in blocks.named_parameters()] == names
    u = bc.unit(t) * (800 if dtype == "f32" else 88)
    for name, a, b in zip(["out", "sum", "x", "gate", *names], got, want):
        err = (a.detach().cpu().double() - b).norm() / b.norm()
        assert err <= u, (name, err.item(), u)


def test_blocks_autocast_graph_and_refusals(gpu):
    """Blocks of all three attentions in a row with post norms under autocast, and captured; what a block refuses."""
    import laplacianformer_amd as lf

    torch.manual_seed(12)
    blocks = torch.nn.ModuleList([lf.AttentionBlock(64, 2, attention=a, pool=2, post_norm=True) for a in ("decay", "softmax", "laplacian")]).to(gpu)
    x, g = gen((2, 64, 64), 70, "f32").to(gpu).requires_grad_(), gen((2, 64, 64), 71, "f32").to(gpu)
    gate = gen((64,), 72, "bf16").to(gpu)

    def fn(t):
        y, s = t, None
        for b in blocks:
            y, s = b(y, s, grid=(8, 8), gate=gate if s is not None else None)
        return s

    want = fn(x)
    (wx,) = torch.autograd.grad(want, x, g)
    with torch.autocast("cuda", torch.bfloat16):
        y, s = blocks[0](x, grid=(8, 8))
        assert y.dtype == torch.bfloat16 and s.dtype == torch.float32
        got = fn(x)
        (gx,) = torch.autograd.grad(got, x, g)
    assert got.dtype == torch.float32
    tol = 6 * 44 * bc.unit(torch.bfloat16)
    for a, b in ((got, want), (gx, wx)):
        assert (a - b).norm() / b.norm() <= tol
    want, wx, got, gx = want.detach(), wx, None, None
    y = s = None
    step = lf.GraphedStep(fn, [x], g)
    for _ in range(3):
        step.replay()
        torch.cuda.synchronize()
        assert torch.equal(step.out, want) and torch.equal(step.grads[0], wx)
    for kw in ({"attention": "decay", "log_decay": [0.0]}, {"attention": "softmax", "log_decay": [0.0, 0.0]}):
        with pytest.raises(ValueError):
            lf.AttentionBlock(64, 2, **kw)
    for kw in ({"mask": torch.ones(64, 64, dtype=torch.bool, device=gpu)}, {"gate": gate}):
        with pytest.raises(ValueError):
            blocks[0](x, **kw)
    half = lf.AttentionBlock(64, 2, attention="decay").to(gpu).bfloat16()
    assert half(x.bfloat16())[0].dtype == torch.bfloat16 and half._log_decay.dtype == torch.float32
