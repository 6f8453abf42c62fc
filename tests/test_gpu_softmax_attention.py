"""softmax_attention, forward and backward, against its 64-bit form at the sizes, masks, layouts and
lengths where it can go wrong; the bounds are those of blockcheck.attention."""
import math

import pytest
import torch

import blockcheck as bc
from lfcheck import TORCH_DT, gen

pytestmark = pytest.mark.gpu

# (B, H, Hk, N, M, d)
SHAPES = [
    (1, 1, 1, 1, 1, 8), (2, 4, 2, 1, 1, 64), (1, 2, 2, 17, 19, 1), (1, 2, 1, 33, 65, 40), (2, 3, 3, 129, 127, 32),
    (1, 8, 2, 5, 300, 128), (1, 16, 2, 4, 33, 64), (1, 16, 2, 5, 129, 32), (2, 2, 2, 200, 200, 50), (1, 4, 1, 64, 1000, 64),
    (1, 1, 1, 700, 30, 16), (1, 2, 2, 257, 256, 97), (1, 6, 2, 140, 140, 80), (1, 1, 1, 31, 1, 128), (3, 5, 5, 1, 70, 24),
]
MODES = ["plain", "causal", "lengths", "causal_lengths", "bool", "bias", "key_mask"]


def make(shape, mode, dtype, seed):
    """CPU inputs and keyword arguments of one call."""
    B, H, Hk, N, M, d = shape
    q, k, v, g = gen((B, H, N, d), seed, dtype), gen((B, Hk, M, d), seed + 1, dtype), gen((B, Hk, M, d), seed + 2, dtype), \
        gen((B, H, N, d), seed + 3, dtype)
    r = torch.Generator().manual_seed(seed + 4)
    kw = {}
    if "causal" in mode:
        kw["causal"] = True
    if "lengths" in mode:
        kw["k_lengths"] = torch.randint(0, M + 2, (B,), generator=r, dtype=torch.int32)
        kw["q_lengths"] = torch.randint(0, N + 2, (B,), generator=r, dtype=torch.int32)
        kw["k_lengths"][0], kw["q_lengths"][0] = max(M - 3, 1), N + 5
        if mode == "causal_lengths":
            kw["q_starts"] = kw["k_lengths"] - N
    if mode == "bool":
        kw["mask"] = torch.rand(B, 1, N, M, generator=r) > 0.3
        kw["mask"][:, :, :: 7] = False
    elif mode == "bias":
        m = torch.randn(1, H, N, M, generator=r)
        m = torch.where(m > 1.5, bc.NEG, m)
        m[:, :, :: 5] = bc.NEG
        kw["mask"] = m.to(TORCH_DT[dtype])
    elif mode == "key_mask":
        kw["mask"] = torch.rand(B, 1, 1, M, generator=r) > 0.3
    return q, k, v, g, kw


def on(gpu, kw):
    return {n: x.to(gpu) if torch.is_tensor(x) else x for n, x in kw.items()}


def call(gpu, q, k, v, g, kw):
    import laplacianformer_amd as lf

    a, b, c = (t.to(gpu).requires_grad_() for t in (q, k, v))
    out = lf.softmax_attention(a, b, c, **on(gpu, kw))
    assert out.dtype == q.dtype and out.shape == q.shape
    grads = torch.autograd.grad(out, (a, b, c), g.to(gpu))
    return dict(zip(("out", "dq", "dk", "dv"), (out, *grads)))


def reference(q, k, v, g, kw, scale=None):
    kw = dict(kw)
    kw.pop("scale", None)
    ok, bias = bc.allowed(q.shape[0], q.shape[1], q.shape[2], k.shape[2], **kw)
    return bc.attention(q, k, v, g, ok, bias, scale or 1 / math.sqrt(q.shape[3]))


def check(got, ref, tag):
    for name, (y, tol) in ref.items():
        bc.assert_within(got[name], y, tol, (tag, name))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_forward_and_gradients(gpu, dtype, shape, mode):
    print(f"softmax attention {dtype} {shape} {mode}", flush=True)
    q, k, v, g, kw = make(shape, mode, dtype, 1000 + 7 * len(mode) + shape[3])
    check(call(gpu, q, k, v, g, kw), reference(q, k, v, g, kw), (dtype, shape, mode))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_layouts(gpu, dtype):
    """Token-major tensors, views into one buffer, odd offsets, and key heads broadcast by a stride of 0."""
    import laplacianformer_amd as lf

    print(f"softmax attention layouts {dtype}", flush=True)
    B, H, N, d = 2, 3, 70, 32
    t = TORCH_DT[dtype]
    qkv = gen((B, N, 3 * H, d), 5, dtype)
    g = gen((B, N, H, d), 6, dtype)
    x = qkv.to(gpu).requires_grad_()
    q, k, v = x.transpose(1, 2).split(H, dim=1)
    out = lf.softmax_attention(q, k, v, causal=True)
    (dx,) = torch.autograd.grad(out, x, g.to(gpu).transpose(1, 2))
    cq, ck, cv = qkv.transpose(1, 2).split(H, dim=1)
    ref = reference(cq, ck, cv, g.transpose(1, 2), {"causal": True})
    got = dict(zip(("dq", "dk", "dv"), dx.transpose(1, 2).split(H, dim=1)), out=out)
    check(got, ref, "buffer")
    # one element into a buffer: nothing is 16-byte aligned
    flat = torch.zeros(B * H * N * d + 1, dtype=t, device=gpu)
    odd = flat[1:].view(B, H, N, d)
    odd.copy_(cq)
    out2 = lf.softmax_attention(odd, ck.to(gpu), cv.to(gpu), causal=True)
    bc.assert_within(out2, *ref["out"], "odd offset")
    # rows a channel longer than the head
    wide = torch.zeros(B, H, N, d + 1, dtype=t, device=gpu)
    wide[..., :d] = ck.to(gpu)
    out3 = lf.softmax_attention(cq.to(gpu), wide[..., :d], cv.to(gpu), causal=True)
    bc.assert_within(out3, *ref["out"], "odd rows")
    # one key head expanded to all
    k1, v1 = ck[:, :1].to(gpu).requires_grad_(), cv[:, :1].to(gpu).requires_grad_()
    qd = cq.to(gpu).requires_grad_()
    o = lf.softmax_attention(qd, k1.expand(-1, H, -1, -1), v1.expand(-1, H, -1, -1))
    grads = torch.autograd.grad(o, (qd, k1, v1), g.to(gpu).transpose(1, 2))
    shared = reference(cq, ck[:, :1], cv[:, :1], g.transpose(1, 2), {})
    u = bc.unit(t)
    full = reference(cq, ck[:, :1].repeat(1, H, 1, 1), cv[:, :1].repeat(1, H, 1, 1), g.transpose(1, 2), {})
    for name, y in zip(("out", "dq", "dk", "dv"), (o, *grads)):
        tol = shared[name][1]
        if name in ("dk", "dv"):  # autograd adds the heads' gradients, each rounded, and rounds their sums
            tol = full[name][1].sum(1, keepdim=True) + H * u * full[name][0].abs().sum(1, keepdim=True)
        bc.assert_within(y, shared[name][0], tol, ("expanded", name))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N", [1, 3, 40])
def test_tokens_over_a_cache(gpu, dtype, N):
    """New tokens over caches filled to uneven lengths, whose rest holds NaN; a sequence without
    keys; enough keys that they are split over workgroups."""
    print(f"softmax attention cache {dtype} N={N}", flush=True)
    B, H, Hk, M, d = 4, 8, 2, 3000, 64
    lengths = torch.tensor([2999, 0, 37, 1500], dtype=torch.int32)
    q, k, v, g, _ = make((B, H, Hk, N, M, d), "plain", dtype, 40)
    kw = {"k_lengths": lengths, "causal": True, "q_starts": lengths - N}
    ref = reference(q, k, v, g, kw)
    behind = (torch.arange(M).view(1, 1, M, 1) >= lengths.view(B, 1, 1, 1))
    k2, v2 = (torch.where(behind, float("nan"), t) for t in (k, v))
    got = call(gpu, q, k2, v2, g, kw)
    check(got, ref, "cache")
    assert bool((got["out"][1] == 0).all()) and bool((got["dq"][1] == 0).all())


@pytest.mark.parametrize("d", [48, 50, 97])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_what_is_masked_may_hold_anything(gpu, dtype, d):
    """NaN and infinities in keys that a length or a mask over keys takes out, and in queries behind
    q_lengths, reach nothing; those keys' and queries' gradients are 0."""
    print(f"softmax attention non-finite {dtype} {d}", flush=True)
    B, H, Hk, N, M = 2, 4, 2, 70, 150
    q, k, v, g, _ = make((B, H, Hk, N, M, d), "plain", dtype, 60)
    for kind in ("bool", "bias"):
        keep = torch.rand(B, 1, 1, M, generator=torch.Generator().manual_seed(61)) > 0.4
        mask = keep if kind == "bool" else torch.where(keep, 0.25, bc.NEG)
        kw = {"mask": mask, "q_lengths": torch.tensor([N - 9, N], dtype=torch.int32),
              "k_lengths": torch.tensor([M, M - 50], dtype=torch.int32)}
        ref = reference(q, k, v, g, kw)
        dead = (~keep[:, :, 0, :, None]) | (torch.arange(M).view(1, 1, M, 1) >= kw["k_lengths"].view(B, 1, 1, 1))
        gone = torch.arange(N).view(1, 1, N, 1) >= kw["q_lengths"].view(B, 1, 1, 1)
        bad = torch.where(torch.arange(d) % 2 == 0, float("nan"), float("inf"))
        got = call(gpu, torch.where(gone, bad, q.float()).to(q.dtype), torch.where(dead, bad, k.float()).to(k.dtype),
                   torch.where(dead, -bad, v.float()).to(v.dtype), torch.where(gone, bad, g.float()).to(g.dtype), kw)
        check(got, ref, kind)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_lowest_value_masks(gpu, dtype):
    """Additive masks of the type's lowest value: next to other keys they remove a key; a row that
    holds nothing else spreads over all its keys (and -inf rows give 0)."""
    print(f"softmax attention lowest {dtype}", flush=True)
    B, H, N, M, d = 1, 2, 40, 90, 32
    t = TORCH_DT[dtype]
    q, k, v, g, _ = make((B, H, H, N, M, d), "plain", dtype, 70)
    low = torch.finfo(t).min
    mask = torch.where(torch.rand(1, 1, N, M, generator=torch.Generator().manual_seed(71)) > 0.5, low, 0.0).to(t)
    mask[..., 3, :] = low
    mask[..., 5, :] = bc.NEG
    mask[..., 6, :40] = bc.NEG
    mask[..., 6, 40:] = low
    kw = {"mask": mask}
    check(call(gpu, q, k, v, g, kw), reference(q, k, v, g, kw), "lowest")


@pytest.mark.parametrize("magnitude", [1e-6, 3e4])
def test_fp16_gradient_range(gpu, magnitude):
    """Output gradients far below and above 1 (a mean over many tokens, a scaled loss): dz leaves
    fp16's range on both sides, the results do not (v is small where g is large)."""
    print(f"softmax attention fp16 range {magnitude}", flush=True)
    shape = (1, 2, 2, 130, 600, 64)
    q, k, v, g, kw = make(shape, "plain", "f16", 80)
    g = (g.float() * magnitude).clamp(-6e4, 6e4).half()
    if magnitude > 1:
        k = (k.float() * 1e-2).half()  # dq = scale dz k stays below 65504
        q = (q.float() * 1e-2).half()
    check(call(gpu, q, k, v, g, kw), reference(q, k, v, g, kw), magnitude)


def test_growing_scores(gpu):
    """Scores that rise along the keys by far more than the slack of the running maximum, and fall."""
    print("softmax attention growing scores", flush=True)
    for sign in (1.0, -1.0):
        M, d = 900, 16
        q = torch.ones(1, 1, 40, d)
        k = (sign * torch.arange(M).view(1, 1, M, 1) / 8.0).expand(1, 1, M, d).contiguous()
        v, g = gen((1, 1, M, d), 91, "f32"), gen((1, 1, 40, d), 92, "f32")
        check(call(gpu, q, k, v, g, {}), reference(q, k, v, g, {}), sign)


@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_scale(gpu, scale):
    q, k, v, g, _ = make((1, 2, 2, 50, 60, 24), "plain", "f32", 95)
    check(call(gpu, q, k, v, g, {"scale": scale}), reference(q, k, v, g, {}, scale), scale)


def test_gradients_against_differences(gpu):
    """Directional derivatives of the 64-bit form by central differences against the kernels' gradients."""
    print("softmax attention differences", flush=True)
    q, k, v, g, kw = make((1, 4, 2, 37, 41, 24), "bias", "f32", 100)
    got = call(gpu, q, k, v, g, kw)
    ok, bias = bc.allowed(1, 4, 37, 41, **kw)

    def loss(a, b, c):
        return (bc.attention(a, b, c, None, ok, bias, 24 ** -0.5)["out"][0] * g.double()).sum().item()

    x = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        for seed in range(3):
            dirn = gen(x[i].shape, 110 + seed, "f32").double()
            h = 1e-5
            plus, minus = list(x), list(x)
            plus[i], minus[i] = x[i] + h * dirn, x[i] - h * dirn
            num = (loss(*plus) - loss(*minus)) / (2 * h)
            ana = (got[name].cpu().double() * dirn).sum().item()
            # differences: h^2 times third derivatives of order 10, and 1e-16 / h of the loss;
            # the kernels' part: the bound on every element
            tol = (reference(q, k, v, g, kw)[name][1] * dirn.abs()).sum().item() + 1e-6 * max(1.0, abs(num))
            assert abs(num - ana) <= tol, (name, seed, num, ana, tol)


def test_offsets_beyond_32_bits(gpu):
    """Keys whose rows are 2^16 elements apart, 40000 of them (offsets beyond 2^31 elements)."""
    import laplacianformer_amd as lf

    print("softmax attention long offsets", flush=True)
    M, d = 40000, 32
    q, k, v, g, _ = make((1, 1, 1, 3, M, d), "plain", "bf16", 120)
    big = torch.empty(M * 65536, dtype=torch.bfloat16, device=gpu)
    kd, vd = (big[o:].as_strided((1, 1, M, d), (0, 0, 65536, 1)) for o in (0, 64))
    kd.copy_(k), vd.copy_(v)
    kd, vd = kd.requires_grad_(), vd.requires_grad_()
    qd = q.to(gpu).requires_grad_()
    out = lf.softmax_attention(qd, kd, vd)
    grads = torch.autograd.grad(out, (qd, kd, vd), g.to(gpu))
    check(dict(zip(("out", "dq", "dk", "dv"), (out, *grads))), reference(q, k, v, g, {}), "offsets")


def test_empty(gpu):
    """No keys, no queries, no sequences."""
    import laplacianformer_amd as lf

    print("softmax attention empty", flush=True)
    for B, H, N, M in ((2, 2, 5, 0), (2, 2, 0, 7), (0, 2, 5, 7), (2, 2, 0, 0)):
        q = torch.randn(B, H, N, 16, device=gpu, requires_grad=True)
        k, v = (torch.randn(B, H, M, 16, device=gpu, requires_grad=True) for _ in range(2))
        out = lf.softmax_attention(q, k, v)
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        assert out.shape == q.shape and bool((out == 0).all())
        for t, x in zip(grads, (q, k, v)):
            assert t.shape == x.shape and bool((t == 0).all())


@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_some_gradients(gpu, which):
    """Only the gradients that are asked for, the same bits as all together."""
    import laplacianformer_amd as lf

    q, k, v, g, kw = make((2, 4, 2, 90, 100, 32), "bool", "bf16", 130)
    want = call(gpu, q, k, v, g, kw)
    x = [t.to(gpu).requires_grad_(w) for t, w in zip((q, k, v), which)]
    out = lf.softmax_attention(*x, **on(gpu, kw))
    out.backward(g.to(gpu))
    for t, name, w in zip(x, ("dq", "dk", "dv"), which):
        assert (t.grad is not None) == w
        if w:
            assert torch.equal(t.grad, want[name]), name


def test_repeats_streams_and_graphs(gpu):
    """The same bits again, on two streams at once, and from two graphs replayed in turn."""
    import laplacianformer_amd as lf

    print("softmax attention streams and graphs", flush=True)
    probs = [make((2, 8, 2, 3, 2500, 64), "lengths", "bf16", 140), make((1, 4, 4, 200, 1500, 32), "causal", "f16", 150)]
    want = [call(gpu, *p) for p in probs]
    for _ in range(3):
        for p, w in zip(probs, want):
            got = call(gpu, *p)
            assert all(torch.equal(got[n], w[n]) for n in w)
    streams = [torch.cuda.Stream() for _ in probs]
    torch.cuda.synchronize()
    got = []
    for s, p in zip(streams, probs):
        with torch.cuda.stream(s):
            got.append(call(gpu, *p))
    torch.cuda.synchronize()
    for a, w in zip(got, want):
        assert all(torch.equal(a[n], w[n]) for n in w)
    steps, held = [], []
    for q, k, v, g, kw in probs:
        x = [t.to(gpu).requires_grad_() for t in (q, k, v)]
        held.append((g.to(gpu), on(gpu, kw)))  # a replay reads them: they have to live as long as the step
        steps.append(lf.GraphedStep(lambda a, b, c, kw=held[-1][1]: lf.softmax_attention(a, b, c, **kw), x, held[-1][0]))
    for rep in range(3):
        for s in steps:
            s.out.detach().fill_(7.0)
            s.replay()
        torch.cuda.synchronize()
        for s, w, p in zip(steps, want, probs):
            assert torch.equal(s.out, w["out"]), rep
            for t, n in zip(s.grads, ("dq", "dk", "dv")):
                assert torch.equal(t, w[n]), (rep, n)
            call(gpu, *p)  # eager work between replays


def test_mask_broadcasts(gpu):
    """Masks of fewer dimensions, broadcast along every axis, transposed, and expanded."""
    import laplacianformer_amd as lf

    B, H, N, M, d = 2, 4, 37, 150, 32
    q, k, v, _, _ = make((B, H, 2, N, M, d), "plain", "f32", 160)
    r = torch.Generator().manual_seed(161)
    masks = [torch.rand(N, M, generator=r) > 0.3, torch.rand(M, generator=r) > 0.3, torch.rand(B, 1, N, 1, generator=r) > 0.3,
             torch.rand(H, 1, M, generator=r) > 0.3, (torch.rand(M, N, generator=r) > 0.3).t(),
             (torch.rand(1, 1, 1, M, generator=r) > 0.3).expand(B, H, N, M), torch.tensor(True), torch.tensor(False),
             torch.randn(H, N, 1, generator=r), torch.randn(M, N, generator=r).t(), torch.randn(B, 1, 1, M, generator=r)]
    for i, m in enumerate(masks):
        print("mask", i, tuple(m.shape), flush=True)
        out = lf.softmax_attention(q.to(gpu), k.to(gpu), v.to(gpu), mask=m.to(gpu))
        ref = reference(q, k, v, None, {"mask": torch.broadcast_to(m, (B, H, N, M))})
        bc.assert_within(out, *ref["out"], i)


def test_no_second_derivative(gpu):
    import laplacianformer_amd as lf

    q = torch.randn(1, 2, 4, 8, device=gpu, requires_grad=True)
    w = torch.ones(8, device=gpu)
    pos = torch.zeros(1, 4, dtype=torch.int32, device=gpu)
    for out in (lf.softmax_attention(q, q, q), lf.add_rms_norm(q, w), lf.rotary(q, None, pos, [4])[0]):
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(out.sum(), q, create_graph=True)


def test_refusals(gpu):
    import laplacianformer_amd as lf

    r = lambda *s, **k: torch.randn(*s, device=gpu, **k)
    q, k = r(2, 4, 5, 16), r(2, 2, 7, 16)
    ok = lf.softmax_attention(q, k, k)
    assert ok.shape == q.shape
    bad = [
        (dict(q=q.double(), k=k.double(), v=k.double()), "unsupported dtype"),
        (dict(q=q, k=k.half(), v=k), "scalar type"),
        (dict(q=q, k=k, v=k[:, :, :6]), "same shape"),
        (dict(q=q, k=r(2, 3, 7, 16), v=r(2, 3, 7, 16)), "do not share"),
        (dict(q=r(2, 4, 5, 129), k=r(2, 4, 5, 129), v=r(2, 4, 5, 129)), "head size 129"),
        (dict(q=q, k=r(1, 2, 7, 16), v=r(1, 2, 7, 16)), "batch or channels"),
        (dict(q=q[0], k=k[0], v=k[0]), "must be \\[batch"),
        (dict(q=q, k=k, v=k, scale=0.0), "positive and finite"),
        (dict(q=q, k=k, v=k, scale=float("nan")), "positive and finite"),
        (dict(q=q, k=k, v=k, scale=-1.0), "positive and finite"),
        (dict(q=q, k=k, v=k, mask=torch.ones(2, 4, 5, 6, dtype=torch.bool, device=gpu)), "broadcast"),
        (dict(q=q, k=k, v=k, mask=torch.ones(1, 2, 4, 5, 7, dtype=torch.bool, device=gpu)), "broadcast"),
        (dict(q=q, k=k, v=k, mask=torch.ones(5, 7, dtype=torch.int32, device=gpu)), "mask must be bool"),
        (dict(q=q, k=k, v=k, mask=torch.ones(5, 7, dtype=torch.bool)), "mask must be on the same GPU"),
        (dict(q=q, k=k, v=k, mask=r(5, 7).requires_grad_()), "no gradient"),
        (dict(q=q, k=k, v=k, k_lengths=torch.ones(2, dtype=torch.int64, device=gpu)), "k_lengths must be"),
        (dict(q=q, k=k, v=k, q_starts=torch.ones(3, dtype=torch.int32, device=gpu)), "q_starts must be"),
        (dict(q=q, k=k, v=k, q_lengths=torch.ones(2, dtype=torch.int32)), "q_lengths must be on the same GPU"),
        (dict(q=q, k=k.cpu(), v=k), "must be on GPU"),
    ]
    for kw, msg in bad:
        with pytest.raises(RuntimeError, match=msg):
            lf.softmax_attention(**kw)


@pytest.mark.parametrize("d", [20, 64])
def test_windows_into_one_row(gpu, d):
    """Tokens that are windows one element apart into a row, fewer than channels: tokens and channels have the same
    stride. Outputs and gradients have places of their own, and the bits of a copy's."""
    import laplacianformer_amd as lf

    print(f"softmax attention windows {d}", flush=True)
    N = d // 2 + 1
    rows = [gen((2, 3, N + d - 1), 170 + i, "bf16").to(gpu) for i in range(4)]
    q, k, v, g = (r.unfold(-1, d, 1) for r in rows)
    assert q.shape == (2, 3, N, d) and q.stride()[2:] == (1, 1) and torch.empty_like(q).stride(3) != 1
    pos = torch.arange(N, dtype=torch.int32, device=gpu)[None]

    def step(q, k, v, g):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        a, b = lf.rotary(q, k, pos, [d // 2])
        out = lf.softmax_attention(q, k, v, causal=True)
        return [a, b, out, *torch.autograd.grad(out, (q, k, v), g), *torch.autograd.grad((a, b), (q, k), (g, g))]

    for x, y in zip(step(q, k, v, g), step(*(t.contiguous() for t in (q, k, v, g)))):
        assert x.stride(3) == 1 and torch.equal(x, y)


def _splits_keys(q, k, kw):
    """Whether the forward of this call splits its keys: its workspace holds more than a mask's bits."""
    import ctypes

    import laplacianformer_amd as lf
    import laplacianformer_amd._lib as L

    assert "mask" not in kw or kw["mask"].dtype != torch.bool
    kind = {None: 0, torch.float32: 2, torch.float16: 3, torch.bfloat16: 4}[kw["mask"].dtype if "mask" in kw else None]
    B, H, N, d = q.shape
    desc = L.Attention(batch=B, heads=H, kv_heads=k.shape[1], q_len=N, k_len=k.shape[2], head_dim=d, scale=1.0, mask_kind=kind)
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[q.dtype]
    return lf.capi().lfamd_softmax_attention_workspace_size(code, ctypes.byref(desc)) > 0


@pytest.mark.parametrize("mode", ["plain", "bias", "lengths", "causal_lengths"])
@pytest.mark.parametrize("d", [24, 64, 80, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_split_keys_of_many_rows(gpu, dtype, d, mode):
    """More rows than eight workgroups per CU join, each with a few of a workgroup's threads, over keys that are split;
    lengths leave some splits, and a whole sequence, without keys."""
    print(f"softmax attention split rows {dtype} {d} {mode}", flush=True)
    shape = (4, 4, 4, 160, 1000, d)
    q, k, v, g, kw = make(shape, mode, dtype, 180)
    if "lengths" in mode:
        kw["k_lengths"] = torch.tensor([1000, 37, 0, 500], dtype=torch.int32)
        kw["q_lengths"] = torch.tensor([160, 160, 160, 90], dtype=torch.int32)
        if mode == "causal_lengths":
            kw["q_starts"] = kw["k_lengths"] - 160
    assert 4 * 4 * 160 > 8 * torch.cuda.get_device_properties(gpu).multi_processor_count and _splits_keys(q, k, kw)
    check(call(gpu, q, k, v, g, kw), reference(q, k, v, g, kw), (dtype, d, mode))


@pytest.mark.parametrize("d", [16, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_empty_masks(gpu, dtype, d):
    """No queries or no keys, with masks expanded to that: empty tensors of strides 0. The others' gradients are 0."""
    import laplacianformer_amd as lf

    print(f"softmax attention empty masks {dtype} {d}", flush=True)
    t = TORCH_DT[dtype]
    for N, M in ((0, 150), (5, 0), (0, 0)):
        ones = torch.ones(2, 1, 1, min(M, 1) * M, device=gpu)
        for mask in (ones.bool(), ones, ones.to(t)):
            mask = mask.expand(2, 4, N, M)
            assert mask.numel() == 0
            q = torch.randn(2, 4, N, d, dtype=t, device=gpu, requires_grad=True)
            k, v = (torch.randn(2, 2, M, d, dtype=t, device=gpu, requires_grad=True) for _ in range(2))
            out = lf.softmax_attention(q, k, v, mask=mask, k_lengths=torch.tensor([M, 3], dtype=torch.int32, device=gpu))
            grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
            torch.cuda.synchronize()
            assert bool((out == 0).all()) and all(bool((x == 0).all()) for x in grads)
