"""add_rms_norm, add_rms_norm_fp8, rotary and AttentionBlock against their 64-bit forms."""
import math

import pytest
import torch

import blockcheck as bc
from lfcheck import TORCH_DT, gen

pytestmark = pytest.mark.gpu

WIDTHS = [1, 3, 8, 64, 100, 333, 512, 513, 1024, 2056, 4096, 4100, 8192, 16377, 16384]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_norm(gpu, dtype, width):
    import laplacianformer_amd as lf

    print(f"norm {dtype} {width}", flush=True)
    for rows, w32, with_res in ((1, False, True), (5, True, True), (301 if width < 5000 else 9, False, False)):
        x, res = gen((rows, width), 1, dtype), gen((rows, width), 2, dtype, 2.0) if with_res else None
        w = (1 + 0.2 * gen((width,), 3, "f32")).to(torch.float32 if w32 else TORCH_DT[dtype])
        gy, gs = gen((rows, width), 4, dtype), gen((rows, width), 5, dtype) if with_res else None
        ref = bc.rms_norm(x, w, res, 1e-5, gy, gs)
        xd, wd = x.to(gpu).requires_grad_(), w.to(gpu).requires_grad_()
        if with_res:
            rd = res.to(gpu).requires_grad_()
            y, total = lf.add_rms_norm(xd, wd, rd, eps=1e-5)
            dx, dr, dw = torch.autograd.grad((y, total), (xd, rd, wd), (gy.to(gpu), gs.to(gpu)))
            bc.assert_within(total, *ref["sum"], (dtype, width, rows, "sum"))
            assert torch.equal(dx, dr)
            # the sum alone, and the norm alone, reach the inputs too
            y, total = lf.add_rms_norm(xd, wd, rd, eps=1e-5)
            (only,) = torch.autograd.grad(total, xd, gs.to(gpu))
            assert torch.equal(only, gs.to(gpu))
        else:
            y = lf.add_rms_norm(xd, wd, eps=1e-5)
            dx, dw = torch.autograd.grad(y, (xd, wd), gy.to(gpu))
        for name, t in (("y", y), ("dx", dx), ("dw", dw)):
            bc.assert_within(t, *ref[name], (dtype, width, rows, name))
        assert dw.dtype == w.dtype
        with torch.no_grad():
            again = lf.add_rms_norm(xd, wd, rd if with_res else None, eps=1e-5)
            assert torch.equal(again[0] if with_res else again, y)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_norm_strides_and_shapes(gpu, dtype):
    """Rows of a wider buffer, transposed leading dimensions, odd offsets, one dimension, no rows."""
    import laplacianformer_amd as lf

    t = TORCH_DT[dtype]
    buf, res = gen((6, 5, 80), 11, dtype), gen((5, 6, 48), 12, dtype)
    w = gen((48,), 13, dtype)
    for x in (buf[..., 8:56], buf[..., 7:55], buf.transpose(0, 1)[..., :48]):
        r = res if x.shape == res.shape else gen(tuple(x.shape), 14, dtype)
        ref = bc.rms_norm(x, w, r, 1e-6, r, x)
        xd, rd, wd = (y.to(gpu) for y in (buf, r, w))
        off = x.storage_offset()
        xd = xd.as_strided(x.shape, x.stride(), off).requires_grad_()
        rd.requires_grad_(), wd.requires_grad_()
        y, total = lf.add_rms_norm(xd, wd, rd)
        dx, dr, dw = torch.autograd.grad((y, total), (xd, rd, wd), (r.to(gpu), x.to(gpu)))
        for name, got in (("y", y), ("sum", total), ("dx", dx), ("dx", dr), ("dw", dw)):
            bc.assert_within(got, *ref[name], name)
    one = gen((48,), 15, dtype)
    bc.assert_within(lf.add_rms_norm(one.to(gpu), w.to(gpu)), *bc.rms_norm(one, w, None, 1e-6)["y"], "1d")
    x0, w0 = torch.empty(0, 48, dtype=t, device=gpu, requires_grad=True), w.to(gpu).requires_grad_()
    y = lf.add_rms_norm(x0, w0)
    dx, dw = torch.autograd.grad(y, (x0, w0), torch.empty_like(y))
    assert y.shape == x0.shape and dx.shape == x0.shape and bool((dw == 0).all())
    zeros = torch.zeros(3, 48, dtype=t, device=gpu)
    assert bool((lf.add_rms_norm(zeros, w.to(gpu)) == 0).all())


@pytest.mark.parametrize("width", [1, 7, 64, 100, 512, 3000, 4096, 16384])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_norm_fp8(gpu, dtype, width):
    """y8 * scale is within half an e4m3 step (2^-4 relative, 2^-10 of the scale below 2^-6) of y."""
    import laplacianformer_amd as lf

    print(f"norm fp8 {dtype} {width}", flush=True)
    x, res, w = gen((9, width), 21, dtype), gen((9, width), 22, dtype), 1 + 0.1 * gen((width,), 23, "f32")
    x[4], res[4] = 0, 0
    w = w.to(TORCH_DT[dtype])
    y8, scale, total = lf.add_rms_norm_fp8(x.to(gpu), w.to(gpu), res.to(gpu))
    assert y8.dtype == torch.float8_e4m3fn and scale.shape == (9, 1) and scale.dtype == torch.float32
    y, _ = bc.rms_norm(x, w, res, 1e-6)["y"]
    c = 100 * bc.U32
    top = y.abs().amax(-1, keepdim=True)
    want = torch.where(top > 0, top / 448.0, 1.0)
    bc.assert_within(scale, want, c * want, "scale")
    bc.assert_within(total, *bc.rms_norm(x, w, res, 1e-6)["sum"], "sum")
    got = y8.cpu().double() * scale.cpu().double()
    bc.assert_within(got, y, (2.0 ** -4 + c) * y.abs() + 2.0 ** -10 * want, "y8")
    assert bool((y8.float().abs().amax(-1).cpu()[top[:, 0] > 0] == 448).all())
    # the rounding itself: to nearest, as torch rounds the same quotient
    y32 = lf.add_rms_norm(x.float().to(gpu) + res.float().to(gpu), w.float().to(gpu)) / scale
    near = (y32.to(torch.float8_e4m3fn).float() != y8.float()).float().mean().item()
    assert near <= 1e-3 or dtype == "f32" and near <= 1e-3, near
    with pytest.raises(RuntimeError, match="no gradient"):
        lf.add_rms_norm_fp8(x.to(gpu).requires_grad_(), w.to(gpu))
    y8b, _ = lf.add_rms_norm_fp8(total, w.to(gpu))
    assert y8b.shape == x.shape
    # a row far below eps: its scale would be subnormal, it becomes zeros
    if dtype != "f16":
        y8c, sc = lf.add_rms_norm_fp8(torch.full((2, width), 1e-38, dtype=TORCH_DT[dtype], device=gpu), w.to(gpu), eps=1.0)
        assert bool((y8c.float() == 0).all()) and bool((sc == 1).all())


def test_norm_many_rows(gpu):
    """More rows than a grid has workgroups: each sign of a two-element row comes out."""
    import laplacianformer_amd as lf

    rows = 9_000_001
    x = torch.ones(rows, 2, dtype=torch.bfloat16, device=gpu)
    x[::3, 0] = -4.0
    x[::3, 1] = 4.0
    y = lf.add_rms_norm(x, torch.ones(2, dtype=torch.bfloat16, device=gpu))
    assert torch.equal(y, x.sign())  # rstd = 1 / |x| (eps rounds away)


def test_norm_gradients_against_differences(gpu):
    import laplacianformer_amd as lf

    x, res, w = gen((7, 50), 31, "f32"), gen((7, 50), 32, "f32"), gen((50,), 33, "f32")
    gy, gs = gen((7, 50), 34, "f32"), gen((7, 50), 35, "f32")
    d = [t.to(gpu).requires_grad_() for t in (x, res, w)]
    grads = torch.autograd.grad(lf.add_rms_norm(d[0], d[2], d[1]), d, (gy.to(gpu), gs.to(gpu)))

    def loss(a, b, c):
        s = a + b
        y = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * c
        return ((y * gy.double()).sum() + (s * gs.double()).sum()).item()

    base = [t.double() for t in (x, res, w)]
    for i in range(3):
        dirn = gen(base[i].shape, 36 + i, "f32").double()
        p, m = list(base), list(base)
        p[i], m[i] = base[i] + 1e-5 * dirn, base[i] - 1e-5 * dirn
        num = (loss(*p) - loss(*m)) / 2e-5
        ana = (grads[i].cpu().double() * dirn).sum().item()
        assert abs(num - ana) <= 1e-5 * max(1.0, dirn.numel() ** 0.5), (i, num, ana)


def test_norm_refusals(gpu):
    import laplacianformer_amd as lf

    x, w = torch.randn(3, 8, device=gpu), torch.randn(8, device=gpu)
    for args, msg in (((x.double(), w.double()), "unsupported dtype"), ((x, w.half()), "input's dtype or fp32"),
                      ((x, w[:7]), "last size"), ((x, w, x[:2]), "same shape"), ((x, w, x.half()), "scalar type"),
                      ((x.cpu(), w), "must be on GPU"), ((x, w.cpu()), "same GPU"),
                      ((torch.randn(2, 16385, device=gpu), torch.randn(16385, device=gpu)), "width 16385")):
        with pytest.raises(RuntimeError, match=msg):
            lf.add_rms_norm(*args)
        with pytest.raises(RuntimeError, match=msg):
            lf.add_rms_norm_fp8(*args)


# (B, H, Hk, grid, d, sections)
ROTARY = [(1, 1, 1, (1,), 2, [1]), (2, 3, 1, (5, 7), 32, [8, 8]), (2, 2, 2, (3, 4, 5), 64, [8, 12, 12]),
          (1, 4, 2, (17, 3), 48, [4, 12]), (1, 2, 1, (4, 9), 50, [13, 12]), (2, 1, 1, (6, 6), 7, [1, 2]),
          (1, 3, 1, (33,), 128, [40]), (1, 1, 1, (40,), 256, [128]), (3, 8, 2, (1, 1), 80, [20, 20]), (1, 2, 2, (4, 4), 64, [0, 32])]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rotary(gpu, dtype, case, interleaved):
    import laplacianformer_amd as lf

    print(f"rotary {dtype} {case} {interleaved}", flush=True)
    B, H, Hk, grid, d, sections = case
    N = math.prod(grid)
    q, k = gen((B, H, N, d), 41, dtype), gen((B, N, Hk, d), 42, dtype).transpose(1, 2)
    gq, gk = gen((B, N, H, d), 43, dtype).transpose(1, 2), gen((B, Hk, N, d), 44, dtype)
    pos = lf.grid_positions(grid, start=[1000 * i - 3 for i in range(len(grid))])
    assert pos.shape == (len(grid), N)
    per_batch = torch.stack([pos + 100003 * b for b in range(B)], 1).long()
    for p in (pos, per_batch):
        qd, kd = q.to(gpu).requires_grad_(), k.to(gpu).requires_grad_()
        q2, k2 = lf.rotary(qd, kd, p.to(gpu), sections, base=500.0, interleaved=interleaved)
        dq, dk = torch.autograd.grad((q2, k2), (qd, kd), (gq.to(gpu), gk.to(gpu)))
        for x, y, inv in ((q, q2, False), (k, k2, False), (gq, dq, True), (gk, dk, True)):
            ref, tol = bc.rotary(x, p, sections, 500.0, interleaved, inv)
            bc.assert_within(y, ref, tol, (case, inv))
        (only,) = torch.autograd.grad(lf.rotary(qd, kd, p.to(gpu), sections, 500.0, interleaved)[1], kd, gk.to(gpu))
        assert torch.equal(only, dk)
    q3, none = lf.rotary(q.to(gpu), None, pos.to(gpu), sections, 500.0, interleaved)
    assert none is None
    ref, tol = bc.rotary(q, pos, sections, 500.0, interleaved)
    bc.assert_within(q3, ref, tol, "q alone")


def test_rotary_far_positions(gpu):
    """Positions up to 2^31 - 1 and below zero; the first pair's angle is the position in radians."""
    import laplacianformer_amd as lf

    pos = torch.tensor([[0, 1, -1, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32)
    x = gen((1, 1, 7, 64), 51, "f32")
    y, _ = lf.rotary(x.to(gpu), None, pos.to(gpu), [32])
    ref, _ = bc.rotary(x, pos, [32], 10000.0, False)
    size = torch.cat([x[..., :32].abs() + x[..., 32:].abs()] * 2, -1).double()
    # per position: 2^-50 of it (64-bit frequencies and products), else as blockcheck.rotary
    tol = size * (pos.double().abs().view(1, 1, 7, 1) * 2.0 ** -50 + 8 * bc.U32 + math.pi * 2.0 ** -24) + bc.U32 * ref.abs()
    bc.assert_within(y, ref, tol, "far")


def test_rotary_layouts_and_empty(gpu):
    """Views into one buffer, odd offsets, expanded heads, no tokens."""
    import laplacianformer_amd as lf

    qkv = gen((2, 12, 6, 16), 52, "bf16")
    pos = lf.grid_positions((3, 4))
    q, k, _ = qkv.to(gpu).transpose(1, 2).split(2, dim=1)
    q2, k2 = lf.rotary(q, k, pos.to(gpu), [4, 4])
    for x, y in ((qkv[:, :, :2], q2), (qkv[:, :, 2:4], k2)):
        bc.assert_within(y, *bc.rotary(x.transpose(1, 2), pos, [4, 4], 10000.0, False), "buffer")
    flat = torch.zeros(2 * 2 * 12 * 16 + 1, dtype=torch.bfloat16, device=gpu)
    odd = flat[1:].view(2, 2, 12, 16)
    odd.copy_(q)
    assert torch.equal(lf.rotary(odd, None, pos.to(gpu), [4, 4])[0], q2)
    wide = q[:, :1].expand(-1, 3, -1, -1)
    assert torch.equal(lf.rotary(wide, None, pos.to(gpu), [4, 4])[0], q2[:, :1].expand(-1, 3, -1, -1))
    e, _ = lf.rotary(q[:, :, :0], None, pos[:, :0].to(gpu), [4, 4])
    assert e.shape == (2, 2, 0, 16)


def test_rotary_refusals(gpu):
    import laplacianformer_amd as lf

    q, pos = torch.randn(2, 3, 4, 16, device=gpu), torch.zeros(2, 4, dtype=torch.int32, device=gpu)
    assert lf.rotary_sections(50, 3) == [9, 8, 8]
    for args, msg in (((q.double(), None, pos, [4, 4]), "unsupported dtype"), ((q, q[:, :, :3], pos, [4, 4]), "heads only"),
                      ((q, q.half(), pos, [4, 4]), "scalar type"), ((q, None, pos, [4, 5]), "room for 8"),
                      ((q, None, pos, [4]), "positions must be"), ((q, None, pos, [0, 0]), "0 pairs"),
                      ((q, None, pos.float(), [4, 4]), "int32 or int64"), ((q, None, pos.cpu(), [4, 4]), "same GPU"),
                      ((q, None, pos, [4, -1]), "section 1"), ((q[0], None, pos, [4, 4]), "q must be"),
                      ((q, None, pos, [4, 4], 0.0), "base must be"), ((q, None, pos, [4, 4], float("inf")), "base must be"),
                      ((q.cpu(), None, pos, [4, 4]), "must be on GPU"), ((q, None, pos[:, :3], [4, 4]), "positions must be")):
        with pytest.raises(RuntimeError, match=msg):
            lf.rotary(*args)


def _block_reference(block, x, res, grid, positions, lengths, g, gs):
    """The block in 64 bits on the CPU, with autograd: (out, sum, gradients of x, residual and parameters)."""
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in block.named_parameters()}
    x, res = x.double().requires_grad_(), res.double().requires_grad_()
    B, N, C = x.shape
    H, Hk, d = block.heads, block.kv_heads, C // block.heads
    s = x + res
    y = s / (s.square().mean(-1, keepdim=True) + block.eps).sqrt() * p["weight"]
    qkv = (y @ p["qkv.weight"].t() + p["qkv.bias"]).view(B, N, H + 2 * Hk, d).transpose(1, 2)
    q, k, v = qkv.split((H, Hk, Hk), dim=1)
    n = [len(r) for r in torch.arange(d // 2).tensor_split(len(grid))]

    def turn(t):
        angle = torch.cat([positions[a][:, None].double() * 10000.0 ** (-torch.arange(m).double() / m) for a, m in enumerate(n)], -1)
        a, b = t[..., :d // 2], t[..., d // 2:]
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1)

    q, k = turn(q), turn(k)
    k, v = k.repeat_interleave(H // Hk, 1), v.repeat_interleave(H // Hk, 1)
    z = q @ k.transpose(-1, -2) / math.sqrt(d)
    i = torch.arange(N)
    ok = (i.view(1, 1, 1, N) < lengths.view(B, 1, 1, 1)) & (i.view(1, 1, N, 1) < lengths.view(B, 1, 1, 1))
    if block.causal:
        ok = ok & (i.view(1, 1, 1, N) <= i.view(1, 1, N, 1))
    z = z.masked_fill(~ok, -1e300)
    a = torch.softmax(z, -1) * ok
    o = (a @ v).transpose(1, 2).reshape(B, N, C) @ p["proj.weight"].t() + p["proj.bias"]
    names = list(p)
    grads = torch.autograd.grad((o, s), [x, res] + [p[k] for k in names], (g.double(), gs.double()))
    return o.detach(), s.detach(), dict(zip(["x", "residual"] + names, grads))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attention_block(gpu, dtype, causal):
    """Norm, projections, rotary positions and softmax attention with shared heads and uneven lengths, run
    together and differentiated. Bound: norm-relative, with every stage's rounding (u of the type, nine
    of them in a row from the norm to the gradient of the weights) adding at most its unit times a
    condition of 4 for the softmax: 36 u; fp32's products add their sums of up to 96 terms: 400 u."""
    import laplacianformer_amd as lf

    print(f"attention block {dtype} causal={causal}", flush=True)
    torch.manual_seed(5)
    B, grid, dim, heads, kv = 2, (6, 9), 96, 6, 2
    N, t = math.prod(grid), TORCH_DT[dtype]
    block = lf.AttentionBlock(dim, heads, kv, causal=causal).to(t)
    x, res, g, gs = (gen((B, N, dim), 60 + i, dtype) for i in range(4))
    lengths = torch.tensor([N, N - 20], dtype=torch.int32)
    o, s, ref = _block_reference(block, x, res, grid, lf.grid_positions(grid), lengths, g, gs)
    block = block.to(gpu)
    xd, rd = x.to(gpu).requires_grad_(), res.to(gpu).requires_grad_()
    out, total = block(xd, rd, grid=grid, lengths=lengths.to(gpu))
    torch.autograd.backward((out, total), (g.to(gpu), gs.to(gpu)))
    got = {"x": xd.grad, "residual": rd.grad, **{n: p.grad for n, p in block.named_parameters()}}
    u = bc.unit(t) * (400 if dtype == "f32" else 36)
    for name, y, r in [("out", out, o), ("sum", total, s)] + [(n, got[n], ref[n]) for n in ref]:
        err = (y.detach().cpu().double() - r).norm() / r.norm()
        assert err <= u, (name, err.item(), u)


def test_attention_block_chain_and_graph(gpu):
    """Two blocks, softmax and laplacian, in a row: a captured step gives the eager one's bits, replay after
    replay with eager work between, and fresh values in its inputs."""
    import laplacianformer_amd as lf

    print("attention block graph", flush=True)
    torch.manual_seed(6)
    a = lf.AttentionBlock(64, 2).to(gpu).half()
    b = lf.AttentionBlock(64, 2, attention="laplacian", pool=2).to(gpu).half()
    x, g = gen((2, 64, 64), 70, "f16").to(gpu).requires_grad_(), gen((2, 64, 64), 71, "f16").to(gpu)

    def fn(t):
        y, s = a(t, grid=(8, 8))
        y, s = b(y, s, grid=(8, 8))
        return y + s

    def eager():
        t = x.detach().clone().requires_grad_()
        out = fn(t)
        (gx,) = torch.autograd.grad(out, t, g)
        return out.detach(), gx

    step = lf.GraphedStep(fn, [x], g)
    for rep in range(3):
        want = eager()
        step.replay()
        torch.cuda.synchronize()
        assert torch.equal(step.out, want[0]) and torch.equal(step.grads[0], want[1]), rep
        with torch.no_grad():
            x.copy_(gen((2, 64, 64), 72 + rep, "f16"))


def test_attention_block_refusals(gpu):
    import laplacianformer_amd as lf

    for args, kw in (((30, 4), {}), ((32, 4, 3), {}), ((32, 4), {"attention": "linear"}),
                     ((32, 4, 2), {"attention": "laplacian"}), ((32, 4), {"attention": "laplacian", "causal": True})):
        with pytest.raises(ValueError):
            lf.AttentionBlock(*args, **kw)
    with pytest.raises(ValueError, match="token grid"):
        lf.AttentionBlock(32, 4).to(gpu)(torch.randn(1, 10, 32, device=gpu), grid=(3, 3))
    with pytest.raises(ValueError, match="neither mask"):
        lf.AttentionBlock(32, 2, attention="laplacian").to(gpu)(
            torch.randn(1, 64, 32, device=gpu), lengths=torch.ones(1, dtype=torch.int32, device=gpu))


def test_norm_and_rotary_streams_and_graphs(gpu):
    import laplacianformer_amd as lf

    print("norm and rotary graphs", flush=True)
    pos = lf.grid_positions((10, 10), gpu)
    x = gen((4, 100, 2, 32), 80, "bf16").to(gpu).requires_grad_()
    r = gen((4, 100, 2, 32), 81, "bf16").to(gpu)
    w = torch.ones(32, dtype=torch.bfloat16, device=gpu)
    g = gen((4, 2, 100, 32), 82, "bf16").to(gpu)

    def fn(t):
        y, s = lf.add_rms_norm(t, w, r)
        q, k = lf.rotary(y.transpose(1, 2), s.transpose(1, 2), pos, [8, 8])
        return q + k

    def eager():
        t = x.detach().clone().requires_grad_()
        out = fn(t)
        return out.detach(), torch.autograd.grad(out, t, g)[0]

    want = eager()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(eager())
    torch.cuda.synchronize()
    step = lf.GraphedStep(fn, [x], g)
    for _ in range(3):
        step.replay()
        torch.cuda.synchronize()
        got.append((step.out.detach().clone(), step.grads[0].clone()))
        eager()
    for o, d in got:
        assert torch.equal(o, want[0]) and torch.equal(d, want[1])


def test_forward_mode_is_refused(gpu):
    """A tangent of an input, or of an output gradient, raises: none is dropped."""
    import laplacianformer_amd as lf
    from torch.autograd import forward_ad

    q = torch.randn(1, 2, 4, 8, device=gpu)
    w, pos = torch.ones(8, device=gpu), lf.grid_positions((2, 2), gpu)
    fns = (lambda t: lf.add_rms_norm(t, w), lambda t: lf.rotary(t, None, pos, [2, 2])[0],
           lambda t: lf.softmax_attention(t, q, q))
    with forward_ad.dual_level():
        for fn in fns:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                fn(forward_ad.make_dual(q, q))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                fn(forward_ad.make_dual(q.clone().requires_grad_(), q))
            x = q.clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(fn(x), x, forward_ad.make_dual(q, q))


@pytest.mark.parametrize("attention", ["softmax", "laplacian"])
@pytest.mark.parametrize("amp", ["bf16", "f16"])
def test_attention_blocks_under_autocast(gpu, amp, attention):
    """Three blocks in a row under autocast, as a pyramid's stage trains: each projection's 16-bit output meets the fp32
    residual stream. The sums stay fp32, and every gradient arrives in its leaf's type. Against the same blocks in
    fp32: per block and direction nine roundings of the type in a row (as in test_attention_block), each of at
    most u, through three blocks and back; a condition of 4 for the attention: 6 * 36 u of the norm."""
    import laplacianformer_amd as lf

    print(f"attention blocks autocast {amp} {attention}", flush=True)
    torch.manual_seed(7)
    blocks = torch.nn.ModuleList([lf.AttentionBlock(64, 2, attention=attention, pool=2) for _ in range(3)]).to(gpu)
    x = gen((2, 64, 64), 90, "f32").to(gpu).requires_grad_()
    g, gs = gen((2, 64, 64), 91, "f32").to(gpu), gen((2, 64, 64), 92, "f32").to(gpu)

    def step():
        y, s = x, None
        for b in blocks:
            y, s = b(y, s, grid=(8, 8))
        leaves = [x, *blocks.parameters()]
        return y, s, torch.autograd.grad((y, s), leaves, (g.to(y.dtype), gs), allow_unused=False)

    want = step()
    with torch.autocast("cuda", TORCH_DT[amp]):
        got = step()
    assert got[0].dtype == TORCH_DT[amp] and got[1].dtype == torch.float32
    tol = 6 * 36 * bc.unit(TORCH_DT[amp])
    for i, (a, w) in enumerate(zip([got[0], got[1], *got[2]], [want[0], want[1], *want[2]])):
        assert i == 0 or a.dtype == torch.float32
        err = (a.double() - w.double()).norm() / w.double().norm()
        assert err <= tol, (i, err.item(), tol)


def test_block_prefixes_across_square_counts(gpu):
    """Without a grid a causal block gives a prefix the outputs that it has in the longer sequence, and a padded batch
    those of any padding, whether or not a token count is a square's. Sums in another order only: fp32, and the
    products' bound of test_attention_block."""
    import laplacianformer_amd as lf

    torch.manual_seed(8)
    x = gen((2, 65, 48), 95, "f32").to(gpu)
    tol = 400 * bc.U32
    causal = lf.AttentionBlock(48, 3, causal=True).to(gpu)
    plain = lf.AttentionBlock(48, 3).to(gpu)
    lengths = torch.tensor([48, 31], dtype=torch.int32, device=gpu)
    with torch.no_grad():
        want, padded = causal(x)[0], plain(x, lengths=lengths)[0]
        for n in (48, 49, 50, 63, 64):
            print("prefix", n, flush=True)
            got = causal(x[:, :n])[0]
            assert (got - want[:, :n]).norm() <= tol * want[:, :n].norm(), n
            got = plain(x[:, :n], lengths=lengths)[0]
            for b, m in enumerate(lengths.tolist()):
                assert (got[b, :m] - padded[b, :m]).norm() <= tol * padded[b, :m].norm(), (n, b)
        square = plain(x[:, :64])[0]
        assert torch.equal(square, plain(x[:, :64], grid=(8, 8))[0])


@pytest.mark.parametrize("width", [5, 64, 333, 1024, 2056, 4096, 8192, 16381, 16384])
def test_norm_backward_of_fp32_addends(gpu, width):
    """The C entry's fp32 backward from both addends, which the autograd node leaves to the stored sum."""
    import ctypes

    import laplacianformer_amd as lf

    print(f"norm backward fp32 addends {width}", flush=True)
    lib, rows = lf.capi(), 37
    x, res, gy, gs = (gen((rows, width), 100 + i, "f32") for i in range(4))
    w = 1 + 0.2 * gen((width,), 104, "f32")
    ref = bc.rms_norm(x, w, res, 1e-5, gy, gs)
    t = [a.to(gpu) for a in (x, res, gy, gs, w)]
    y, total, dx, dw = (torch.empty_like(a) for a in (t[0], t[0], t[0], t[4]))
    rstd = torch.empty(rows, device=gpu)
    p = lambda a: ctypes.c_void_p(a.data_ptr())
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    lf.check(lib.lfamd_add_rms_norm(0, p(t[0]), width, p(t[1]), width, 0, p(t[4]), p(y), p(total), p(rstd), rows, width, 1e-5, st))
    n = lib.lfamd_add_rms_norm_backward_workspace_size(0, rows, width)
    ws = torch.empty(n, dtype=torch.uint8, device=gpu)
    lf.check(lib.lfamd_add_rms_norm_backward(0, p(t[2]), width, p(t[3]), width, p(t[0]), width, p(t[1]), width, 0, p(t[4]), p(rstd),
                                             p(dx), p(dw), rows, width, p(ws), n, st))
    torch.cuda.synchronize()
    for name, got in (("y", y), ("sum", total), ("dx", dx), ("dw", dw)):
        bc.assert_within(got, *ref[name], (width, name))
