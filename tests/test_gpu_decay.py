"""decay_attention and decay_attention_step against their 64-bit forms."""
import ctypes
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


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_joined_segments(gpu, dtype):
    """Sequences long enough for segments in launches of their own (a workspace says so), with every result checked."""
    import laplacianformer_amd as lf
    import laplacianformer_amd._lib as L

    for N, d, e, H, Hk in ((2500, 64, 64, 2, 1), (2333, 32, 80, 1, 1)):
        desc = L.Decay(batch=1, heads=H, kv_heads=Hk, tokens=N, key_dim=d, value_dim=e, log_decay=16, scale=1.0)
        assert lf.capi().lfamd_decay_attention_workspace_size(lf.dtype_code(TORCH_DT[dtype]), ctypes.byref(desc)) > 0
        check(gpu, dtype, 1, H, Hk, N, d, e, "slow", lengths=None if H == 1 else [N - 700])
        check(gpu, dtype, 1, H, Hk, N, d, e, "fast", state=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long(gpu, dtype):
    """33001 tokens against the recurrence itself. Bound: decaycheck's count with the tokens' additions within tiles and
    from tile to tile, 64 + N / 32 of them at one time, on magnitudes that the recurrence sums beside the values."""
    import laplacianformer_amd as lf

    print(f"decay long {dtype}", flush=True)
    N, d = 33001, 16
    q, k, v = (gen((1, 1, N, d), 300 + i, dtype) for i in range(3))
    lg = decays("slow", 3)[2:]
    out, last = lf.decay_attention(q.to(gpu), k.to(gpu), v.to(gpu), lg.to(gpu), return_state=True)
    a = math.exp(lg.double().item())
    Q, K, V = (x[0, 0].double().numpy() for x in (q, k, v))
    S, M = K[0][:, None] * V[0] * 0, K[0][:, None] * V[0] * 0
    ref, mag = V * 0, V * 0
    for t in range(N):
        S = a * S + K[t][:, None] * V[t]
        M = a * M + abs(K[t])[:, None] * abs(V[t])
        ref[t], mag[t] = Q[t] @ S / 4, abs(Q[t]) @ M / 4
    c = (64 + 3 * N / 32 + 64) * bc.U32 + (0.0 if dtype == "f32" else 2.0 ** -16 + 2.0 ** -16)
    u = bc.unit(TORCH_DT[dtype])
    ref, mag = torch.from_numpy(ref)[None, None], torch.from_numpy(mag)[None, None]
    bc.assert_within(out, ref, c * mag + u * (ref.abs() + c * mag), "out")
    S, M = torch.from_numpy(S)[None, None], torch.from_numpy(M)[None, None]
    bc.assert_within(last, S, ((64 + 3 * N / 32 + 64) * bc.U32 + 2.0 ** -22) * M, "last")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strides(gpu, dtype):
    """Tokens in front of heads, slices of one packed projection at even and odd places, broadcast batches and heads."""
    import laplacianformer_amd as lf

    B, H, N, d = 2, 3, 70, 32
    lg = decays("slow", H)
    packed = gen((B, N, H * 3 * d + 3), 40, dtype)
    wide = gen((B, H, N, 2 * d + 8), 41, dtype)
    one = gen((1, 1, N, d), 42, dtype)
    cases = []
    for off in (0, 1, 2):
        x = packed[..., off:off + 3 * H * d].view(B, N, 3, H, d).permute(2, 0, 3, 1, 4) if off == 0 else \
            packed.as_strided((3, B, H, N, d), (H * d, N * (H * 3 * d + 3), d, H * 3 * d + 3, 1), off)
        cases.append(tuple(x))
    cases.append((wide[..., :d], wide[..., 8:d + 8], wide[..., d:2 * d]))
    cases.append((one.expand(B, H, N, d), wide[..., :d], one.expand(B, H, N, d)))
    for q, k, v in cases:
        ref = dc.decay(q, k, v, lg, d ** -0.5, g=(g := gen((B, H, N, d), 43, dtype)))
        base = {id(t): t for t in (packed, wide, one)}
        dev = []
        for t in (q, k, v):
            src = next(b for b in base.values() if b.untyped_storage().data_ptr() == t.untyped_storage().data_ptr())
            dev.append(src.to(gpu).as_strided(t.shape, t.stride(), t.storage_offset()).requires_grad_())
            assert dev[-1].stride() == t.stride()
        out = lf.decay_attention(*dev, lg.to(gpu))
        grads = torch.autograd.grad(out, dev, g.to(gpu).transpose(1, 2).contiguous().transpose(1, 2))
        bc.assert_within(out, *ref["out"], "out")
        for name, x in zip(("dq", "dk", "dv"), grads):
            bc.assert_within(x, *ref[name], name)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_lengths(gpu, dtype):
    """What lies behind a length is not read, gives zeros and takes no gradient; lengths are clamped."""
    import laplacianformer_amd as lf

    B, H, Hk, N, d = 6, 4, 2, 101, 48
    lengths = [0, 1, 32, 77, 101, 300]
    check(gpu, dtype, B, H, Hk, N, d, d, lengths=lengths)
    q, k, v, g = (gen((B, h, N, d), 50 + i, dtype) for i, h in enumerate((H, Hk, Hk, H)))
    lg, s0 = decays("slow", H), gen((B, H, d, d), 55, "f32")
    n = torch.tensor(lengths[:-1] + [-5], dtype=torch.int32)
    ref = dc.decay(q, k, v, lg, d ** -0.5, s0, n, g)
    dev = [t.to(gpu) for t in (q, k, v, g)]
    for b, m in enumerate(n.tolist()):
        for t in dev:
            t[b, :, max(m, 0):] = float("nan")
    leaves = [t.requires_grad_() for t in dev[:3]] + [s0.to(gpu).requires_grad_()]
    out, last = lf.decay_attention(*leaves[:3], lg.to(gpu), state=leaves[3], lengths=n.to(gpu), return_state=True)
    grads = torch.autograd.grad(out, leaves, dev[3])
    bc.assert_within(out, *ref["out"], "out")
    bc.assert_within(last, *ref["last"], "last")
    for name, x in zip(("dq", "dk", "dv", "dstate"), grads):
        bc.assert_within(x, *ref[name], name)
    assert torch.equal(last[0], leaves[3][0]) and bool((out[0] == 0).all()) and bool((grads[1][-1] == 0).all())


def test_ranges(gpu):
    """fp16: scores beyond the type's range beside small values, values near its smallest, and a state that decays
    to nothing; bf16 with wide ranges; states far above the type's range."""
    import laplacianformer_amd as lf

    lg = decays("slow", 2)
    for qs, vs, ss, dtype in ((40.0, 1e-3, 1.0, "f16"), (1.0, 3e-5, 0.0, "f16"), (1e-3, 1.0, 1e5, "f16"), (1e-12, 1e15, 1.0, "bf16")):
        print("range", qs, vs, ss, dtype, flush=True)
        q, k, v = gen((1, 2, 130, 64), 60, dtype, qs), gen((1, 2, 130, 64), 61, dtype, qs), gen((1, 2, 130, 64), 62, dtype, vs)
        s0, g = gen((1, 2, 64, 64), 63, "f32", ss), gen((1, 2, 130, 64), 64, dtype)
        ref = dc.decay(q, k, v, lg, 0.125, s0, None, g)
        leaves = [leaf(t, gpu) for t in (q, k, v, s0)]
        out, last = lf.decay_attention(*leaves[:3], lg.to(gpu), state=leaves[3], return_state=True)
        bc.assert_within(last, *ref["last"], "last")
        grads = dict(zip(("dq", "dk", "dv", "dstate"), torch.autograd.grad(out, leaves, g.to(gpu))))
        for name, x in {"out": out, **grads}.items():
            if ref[name][0].abs().max() < torch.finfo(x.dtype).max:
                bc.assert_within(x, *ref[name], (qs, vs, ss, dtype, name))
    for dtype in ("f16", "bf16", "f32"):
        q, z = gen((1, 2, 700, 32), 65, dtype).to(gpu), torch.zeros(1, 2, 700, 32, dtype=TORCH_DT[dtype], device=gpu)
        out, last = lf.decay_attention(q, z, z, torch.tensor([-1.0, -0.2], device=gpu), state=torch.ones(1, 2, 32, 32, device=gpu),
                                       return_state=True)
        assert bool((last < 1e-30).all()) and bool(torch.isfinite(out).all()) and bool((out[:, :, 690:].float().abs() < 1e-20).all())  # which fp16 itself holds as 0


def test_gradients_against_differences(gpu):
    import laplacianformer_amd as lf

    B, H, Hk, N, d, e = 1, 2, 1, 45, 8, 12
    x = [gen(s, 70 + i, "f32") for i, s in enumerate(((B, H, N, d), (B, Hk, N, d), (B, Hk, N, e), (B, H, d, e)))]
    lg, g, gl = decays("fast", H), gen((B, H, N, e), 75, "f32"), gen((B, H, d, e), 76, "f32")
    leaves = [leaf(t, gpu) for t in x]
    res = lf.decay_attention(*leaves[:3], lg.to(gpu), state=leaves[3], return_state=True)
    grads = torch.autograd.grad(res, leaves, (g.to(gpu), gl.to(gpu)))

    def loss(q, k, v, s0):
        S, total, a = s0.clone(), 0.0, torch.exp(lg.double())[None, :, None, None]
        for t in range(N):
            S = a * S + k[:, :, t, :, None].repeat_interleave(H // Hk, 1) * v[:, :, t, None, :].repeat_interleave(H // Hk, 1)
            total = total + ((q[:, :, t, None, :] @ S)[:, :, 0] * d ** -0.5 * g[:, :, t].double()).sum()
        return total + (S * gl.double()).sum()

    base = [t.double() for t in x]
    for i in range(4):
        way = gen(tuple(base[i].shape), 80 + i, "f32").double()
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * way, base[i] - 1e-5 * way
        want = ((loss(*up) - loss(*down)) / 2e-5).item()
        got = (grads[i].cpu().double() * way).sum().item()
        size = (grads[i].cpu().double().abs() * way.abs()).sum().item()
        # differences of a polynomial: 1e-10 of the loss's terms over 2e-5; the gradient's fp32 sums
        assert abs(got - want) <= 1e-4 * size, (i, got, want, size)


def test_only_some_gradients(gpu):
    import laplacianformer_amd as lf

    q, k, v = (gen((1, 2, 40, 16), 90 + i, "bf16").to(gpu) for i in range(3))
    lg, s0, g = decays("slow", 2).to(gpu), gen((1, 2, 16, 16), 94, "f32").to(gpu), gen((1, 2, 40, 16), 93, "bf16").to(gpu)
    full = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    want = torch.autograd.grad(lf.decay_attention(*full[:3], lg, state=full[3]), full, g)
    for i in range(4):
        x = [t.clone() for t in (q, k, v, s0)]
        x[i].requires_grad_()
        out, last = lf.decay_attention(*x[:3], lg, state=x[3], return_state=True)
        assert torch.equal(torch.autograd.grad(out, x[i], g)[0], want[i])
    # through the last state alone
    x = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    _, last = lf.decay_attention(*x[:3], lg, state=x[3], return_state=True)
    dq, dk, dv, ds = torch.autograd.grad(last, x, torch.ones_like(last), allow_unused=True)
    ref = dc.decay(*(t.cpu() for t in (q, k, v)), lg.cpu(), 0.25, s0.cpu(), None, torch.zeros(1, 2, 40, 16).bfloat16(), torch.ones(1, 2, 16, 16))
    assert bool((dq == 0).all())
    for name, y in (("dk", dk), ("dv", dv), ("dstate", ds)):
        bc.assert_within(y, *ref[name], name)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_step(gpu, dtype):
    """One token on a state, odd sizes and shared heads; the state in a larger buffer; against the recurrence: out is a
    sum of d products with a state of two roundings, the state one fma."""
    import laplacianformer_amd as lf

    for B, H, Hk, d, e in ((1, 1, 1, 1, 1), (3, 4, 2, 32, 32), (2, 6, 3, 50, 80), (2, 2, 1, 128, 128), (1, 3, 3, 33, 5), (2, 2, 2, 100, 127)):
        print("step", dtype, B, H, Hk, d, e, flush=True)
        q, k, v = gen((B, H, 1, d), 100, dtype), gen((B, Hk, 1, d), 101, dtype), gen((B, Hk, 1, e), 102, dtype)
        lg, pool = decays("edge", H), gen((B, 2, H + 1, d, e), 103, "f32", 2.0)
        dev = pool.to(gpu)
        state = dev[:, 1, 1:]
        before = dev._version
        out = lf.decay_attention_step(q.to(gpu), k.to(gpu), v.to(gpu), lg.to(gpu), state)
        assert dev._version > before
        a = torch.exp(lg.double()).view(1, H, 1, 1)
        K, V = k.double().repeat_interleave(H // Hk, 1), v.double().repeat_interleave(H // Hk, 1)
        S0 = pool[:, 1, 1:].double()
        S = a * S0 + K.transpose(-1, -2) * V
        mag = a * S0.abs() + K.abs().transpose(-1, -2) * V.abs()
        bc.assert_within(state, S, 6 * bc.U32 * mag, "state")  # the exponential to two of 2^-23
        ref, m = d ** -0.5 * (q.double() @ S), d ** -0.5 * (q.double().abs() @ mag)
        c = (d + 16) * bc.U32
        bc.assert_within(out, ref, c * m + bc.unit(TORCH_DT[dtype]) * (ref.abs() + c * m), "out")
        rest = torch.ones(pool.shape, dtype=torch.bool)
        rest[:, 1, 1:] = False
        assert torch.equal(dev.cpu()[rest], pool[rest])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prompt_pieces_and_steps(gpu, dtype):
    """A prompt in pieces whose states go on, then tokens one by one, as a server runs them: rows of the
    whole sequence's outputs, and its last state (the bounds of both added)."""
    import laplacianformer_amd as lf

    B, H, Hk, N, d = 2, 4, 2, 150, 64
    q, k, v = (gen((B, h, N, d), 110 + i, dtype) for i, h in enumerate((H, Hk, Hk)))
    lg = decays("slow", H)
    ref = dc.decay(q, k, v, lg, d ** -0.5)
    Q, K, V, L = (t.to(gpu) for t in (q, k, v, lg))
    outs, state = [], None
    with torch.no_grad():
        for a, b in ((0, 1), (1, 65), (65, 140)):
            o, state = lf.decay_attention(Q[:, :, a:b], K[:, :, a:b], V[:, :, a:b], L, state=state, return_state=True)
            outs.append(o)
        for t in range(140, N):
            outs.append(lf.decay_attention_step(Q[:, :, t:t + 1], K[:, :, t:t + 1], V[:, :, t:t + 1], L, state))
    bc.assert_within(torch.cat(outs, 2), ref["out"][0], 2 * ref["out"][1], "out")
    bc.assert_within(state, ref["last"][0], 2 * ref["last"][1], "last")


def test_empty(gpu):
    import laplacianformer_amd as lf

    lg = torch.zeros(2, device=gpu)
    s0 = torch.randn(1, 2, 8, 8, device=gpu, requires_grad=True)
    e = torch.empty(1, 2, 0, 8, device=gpu, requires_grad=True)
    out, last = lf.decay_attention(e, e, e, lg, state=s0, return_state=True)
    assert out.shape == (1, 2, 0, 8) and torch.equal(last, s0)
    de, ds = torch.autograd.grad((out, last), (e, s0), (torch.empty_like(out), torch.ones_like(last)))
    assert de.shape == e.shape and bool((ds == 1).all())
    none = torch.empty(0, 2, 5, 8, device=gpu)
    out, last = lf.decay_attention(none, none, none, lg, return_state=True)
    assert out.shape == none.shape and last.shape == (0, 2, 8, 8)
    assert lf.decay_attention_step(none[:, :, :1], none[:, :, :1], none[:, :, :1], lg, torch.empty(0, 2, 8, 8, device=gpu)).shape == (0, 2, 1, 8)
    _, last = lf.decay_attention(e.detach(), e.detach(), e.detach(), lg, return_state=True)
    assert bool((last == 0).all())


def test_streams_graphs_and_repeats(gpu):
    """Training on two streams at once and as a captured step, in both plans; a prompt and in-place steps captured as
    two graphs that are replayed in turn with eager work between: the same bits each time."""
    import laplacianformer_amd as lf

    for N, H, d in ((200, 2, 64), (2400, 2, 32)):
        lg = decays("slow", H).to(gpu)
        x, g = gen((1, H, N, d), 120, "bf16").to(gpu).requires_grad_(), gen((1, H, N, d), 121, "bf16").to(gpu)

        def eager():
            t = x.detach().clone().requires_grad_()
            out = lf.decay_attention(t, t, t, lg)
            return out.detach(), torch.autograd.grad(out, t, g)[0]

        want = eager()
        torch.cuda.synchronize()
        got = []
        for s in [torch.cuda.Stream() for _ in range(2)]:
            with torch.cuda.stream(s):
                got.append(eager())
        torch.cuda.synchronize()
        step = lf.GraphedStep(lambda t: lf.decay_attention(t, t, t, lg), [x], g)
        for _ in range(3):
            step.replay()
            torch.cuda.synchronize()
            got.append((step.out.detach().clone(), step.grads[0].clone()))
            eager()
        for o, dx in got:
            assert torch.equal(o, want[0]) and torch.equal(dx, want[1])

    lg = decays("slow", 2).to(gpu)
    q = gen((3, 2, 90, 32), 130, "f16").to(gpu)
    tok = gen((3, 2, 1, 32), 131, "f16").to(gpu)
    state = torch.zeros(3, 2, 32, 32, device=gpu)

    def prompt():
        out, last = lf.decay_attention(q, q, q, lg, return_state=True)
        state.copy_(last)
        return out

    def token():
        return lf.decay_attention_step(tok, tok, tok, lg, state)

    with torch.no_grad():
        want = [prompt().clone()] + [token().clone() for _ in range(3)]
        end = state.clone()
        graphs = []
        for fn in (prompt, token):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                fn()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = fn()
            graphs.append((gr, out))
        for _ in range(3):
            got = []
            for gr, out in [graphs[0]] + [graphs[1]] * 3:
                gr.replay()
                torch.cuda.synchronize()
                got.append(out.clone())
                lf.decay_attention(q, q, q, lg)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(state, end)


def test_refusals(gpu):
    import laplacianformer_amd as lf
    from torch.autograd import forward_ad

    q = torch.randn(1, 4, 5, 8, device=gpu)
    lg, s0 = torch.zeros(4, device=gpu), torch.zeros(1, 4, 8, 8, device=gpu)
    f = lf.decay_attention
    bad = [lambda: f(q.double(), q.double(), q.double(), lg), lambda: f(q, q.half(), q, lg), lambda: f(q, q[:, :3], q[:, :3], lg),
           lambda: f(q, q[:, :, :4], q, lg), lambda: f(q, q, q[:, :2], lg), lambda: f(q[0], q[0], q[0], lg), lambda: f(q, q[..., :4], q, lg),
           lambda: f(q, q, q, lg.double()), lambda: f(q, q, q, lg[:3]), lambda: f(q, q, q, lg.cpu()), lambda: f(q, q, q, lg, scale=0.0),
           lambda: f(q, q, q, lg, state=s0.half()), lambda: f(q, q, q, lg, state=s0[:, :3]), lambda: f(q, q, q, lg, state=s0.cpu()),
           lambda: f(q, q, q, lg, lengths=torch.ones(1, device=gpu)), lambda: f(q, q, q, lg, lengths=torch.ones(2, dtype=torch.int32, device=gpu)),
           lambda: f(q, q, torch.randn(1, 4, 5, 129, device=gpu), lg), lambda: f(q.cpu(), q.cpu(), q.cpu(), lg.cpu()),
           lambda: f(q, q, q, lg.clone().requires_grad_())]
    one = q[:, :, :1]
    step = lf.decay_attention_step
    bad += [lambda: step(q, q, q, lg, s0), lambda: step(one, one, one, lg, s0.half()), lambda: step(one, one, one, lg, s0.transpose(-1, -2)),
            lambda: step(one, one, one, lg, s0[:, :1].expand(1, 4, 8, 8)), lambda: step(one, one, one, lg, s0[..., :4]),
            lambda: step(one, one, one, lg, s0.clone().requires_grad_()),
            lambda: step(one.expand(2, 4, 1, 8), one.expand(2, 4, 1, 8), one.expand(2, 4, 1, 8), lg, s0.as_strided((2, 4, 8, 8), (32, 64, 8, 1)))]
    for i, fn in enumerate(bad):
        with pytest.raises(RuntimeError):
            fn()
            raise AssertionError(f"call {i} was taken")
    x = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(f(x, q, q, lg), x, q, create_graph=True)
    with forward_ad.dual_level():
        for fn in (lambda t: f(t, q, q, lg), lambda t: f(q, q, q, lg, state=forward_ad.make_dual(s0, s0)),
                   lambda t: step(t[:, :, :1], one, one, lg, s0)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                fn(forward_ad.make_dual(q, q))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(f(x, q, q, lg), x, forward_ad.make_dual(q, q))


def test_state_saved_for_backward_is_watched(gpu):
    """A state that a recorded call has kept and a step changes: its backward raises."""
    import laplacianformer_amd as lf

    q, lg = torch.randn(1, 2, 6, 8, device=gpu, requires_grad=True), torch.zeros(2, device=gpu)
    s0 = torch.zeros(1, 2, 8, 8, device=gpu)
    out = lf.decay_attention(q, q, q, lg, state=s0)
    with torch.no_grad():
        t = torch.randn(1, 2, 1, 8, device=gpu)
        lf.decay_attention_step(t, t, t, lg, s0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
