"""Performance cases of the transformer-block operators on one GPU.

Three operators that surround and replace the Laplacian-kernel attention in a block:
  norm    add_rms_norm: the residual's addition and the root-mean-square norm (training: with
          the gradients), and add_rms_norm_fp8, whose output is e4m3 with one scale per row;
  rotary  rotary positions of q and k over the axes of an image or a video;
  attn    softmax_attention, forward and with the gradients of q, k and v.

Where ``own`` is false, ``run`` computes them from elementary tensor operations in 32 bits
(the angles of rotary positions in 64); where it is true it calls the framework.

fp64 is left out: the operators refuse it.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
BASE = 10000.0
F8_MAX = 448.0


def _lf():
    import laplacianformer_amd as lf
    return lf


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

def _norm(name, rows, width, dtype, mode):
    """mode: "infer" (sum and norm), "fp8" (sum and 8-bit norm), "train" (with the gradients)."""
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "dtype": dtype, "mode": mode}


def _rotary(name, B, H, Hk, grid, d, dtype, interleaved, train, far=0, layout="bhnd"):
    """grid: "t x h x w" or "h x w" as text; far: the first position on every axis."""
    return {"name": name, "kind": "rotary", "B": B, "H": H, "Hk": Hk, "grid": grid, "d": d, "dtype": dtype,
            "interleaved": interleaved, "train": train, "far": far, "layout": layout}


def _attn(name, B, H, Hk, N, M, d, dtype, train, causal=False, lengths=False, mask="none", layout="bhnd"):
    """layout: the order of the tensors in memory ("bnhd" is what a projection's output gives)."""
    return {"name": name, "kind": "attn", "B": B, "H": H, "Hk": Hk, "N": N, "M": M, "d": d, "dtype": dtype,
            "train": train, "causal": causal, "lengths": lengths, "mask": mask, "layout": layout}


def listed():
    return [
        # The norm of a single token of a small model: a launch and its latency.
        _norm("norm_token_bf16", 1, 512, "bf16", "infer"),
        # The norms before the projections of 14 x 14 x 64 tokens, trained; a width that is no multiple of a vector.
        _norm("norm_stage3_odd_f32", 12544, 333, "f32", "train"),
        # A long batch's norm whose output goes into an 8-bit product.
        _norm("norm_long_fp8_bf16", 16384, 4096, "bf16", "fp8"),
        # New tokens of eight sequences at far positions of a long video.
        _rotary("rotary_tokens_f32", 8, 8, 2, "1x1x1", 64, "f32", True, False, far=1000000),
        # q and k of 28 x 28 tokens, trained in mixed precision.
        _rotary("rotary_stage2_f16", 64, 2, 2, "28x28", 64, "f16", False, True),
        # A video of 16 frames of 32 x 32 tokens, as the projections lay it out.
        _rotary("rotary_video_bf16", 4, 16, 4, "16x32x32", 128, "bf16", False, False, layout="bnhd"),
        # One new token for each of 16 sequences, over caches filled to different lengths.
        _attn("attn_token_bf16", 16, 32, 8, 1, 8192, 128, "bf16", False, lengths=True),
        # A whole small attention in the default type.
        _attn("attn_tiny_f32", 2, 2, 2, 196, 196, 32, "f32", True),
        # A late stage, 14 x 14 tokens and four heads of 32 channels, in mixed precision.
        _attn("attn_stage3_f16", 64, 4, 4, 196, 196, 32, "f16", True),
        # Shared heads of 80 channels, sequences of uneven lengths, keys that a mask takes out.
        _attn("attn_ragged_bf16", 6, 6, 2, 1003, 1003, 80, "bf16", True, causal=True, lengths=True, mask="bool",
              layout="bnhd"),
        # Many tokens, all to all: the largest training step.
        _attn("attn_stress_bf16", 8, 8, 8, 4096, 4096, 64, "bf16", True),
        # A long prompt with shared heads.
        _attn("attn_prompt_bf16", 1, 32, 8, 8192, 8192, 128, "bf16", False, causal=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "rotary", "attn", "attn"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "norm":
        width = rng.choice([_log_int(rng, 8, 8192), 8 * _log_int(rng, 8, 1024)])
        rows = _log_int(rng, 1, max(2, min(65536, (1 << 24) // width)))
        mode = rng.choice(["infer", "train", "train", "fp8"])
        c = _norm("", rows, width, dtype, mode)
    elif kind == "rotary":
        d = rng.choice([16, 32, 48, 64, 64, 80, 96, 128])
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 4])
        if rng.random() < 0.5:
            sizes = [_log_int(rng, 1, 64), _log_int(rng, 1, 64)]
        else:
            sizes = [_log_int(rng, 1, 16), _log_int(rng, 1, 32), _log_int(rng, 1, 32)]
        most = max(1, int(4.0e7 // (math.prod(sizes) * H * d)))
        c = _rotary("", _log_int(rng, 1, min(64, most)), H, Hk, "x".join(map(str, sizes)), d, dtype,
                    rng.random() < 0.5, rng.random() < 0.5, far=rng.choice([0, 0, _log_int(rng, 1, 1000000)]),
                    layout=rng.choice(["bhnd", "bnhd"]))
    else:
        d = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 50])
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 2, 4, 5])
        shape = rng.choice(["self", "self", "cross", "token"])
        M = _log_int(rng, 1, 16384) if shape == "token" else _log_int(rng, 16, 4096)
        N = M if shape == "self" else rng.choice([1, 1, 2, 5]) if shape == "token" else _log_int(rng, 1, 2048)
        train = shape != "token" and rng.random() < 0.6
        # fp32 products run at a sixteenth of the 16-bit rate; what is left is shared by the batch.
        most = (1.0e11 if dtype == "f32" else 4.0e11) / (14.0 * H * N * M * d)
        if most < 1:
            M = max(16, int(M * math.sqrt(most)))
            N = M if shape == "self" else max(1, int(N * math.sqrt(most)))
        most = min(64.0, max(1.0, most), 2.0e8 / (Hk * M * d), 1.0e9 / (H * N * M))
        c = _attn("", _log_int(rng, 1, max(1.0, most)), H, Hk, N, M, d, dtype, train,
                  causal=shape != "cross" and rng.random() < 0.5, lengths=rng.random() < 0.4,
                  mask=rng.choice(["none", "none", "none", "bool", "bias"]), layout=rng.choice(["bhnd", "bnhd"]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _heads(gen, case, H, N, dtype):
    """[B, H, N, d] in the case's memory order."""
    B, d = case["B"], case["d"]
    if case["layout"] == "bnhd":
        return _randn(gen, (B, N, H, d), dtype).transpose(1, 2)
    return _randn(gen, (B, H, N, d), dtype)


def _sections(d, axes):
    """The rotated pairs of each axis: d / 2 pairs dealt out evenly, the first axis takes what is left over."""
    n = d // 2 // axes
    return [d // 2 - n * (axes - 1)] + [n] * (axes - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "norm":
        shape = (case["rows"], case["width"])
        s["x"], s["residual"] = _randn(gen, shape, t), _randn(gen, shape, t, 2.0)
        s["weight"] = (1.0 + 0.1 * torch.randn(case["width"], generator=gen, device="cuda")).to(t)
        leaves = ("x", "residual", "weight")
        if case["mode"] == "train":
            s["gy"], s["gs"] = _randn(gen, shape, t), _randn(gen, shape, t)
    elif case["kind"] == "rotary":
        sizes = [int(x) for x in case["grid"].split("x")]
        N = math.prod(sizes)
        s["q"], s["k"] = _heads(gen, case, case["H"], N, t), _heads(gen, case, case["Hk"], N, t)
        axes = torch.meshgrid(*[torch.arange(n, device="cuda", dtype=torch.int32) for n in sizes], indexing="ij")
        s["positions"] = torch.stack([a.reshape(-1) for a in axes]) + case["far"]
        s["sections"] = _sections(case["d"], len(sizes))
        leaves = ("q", "k")
        if case["train"]:
            s["gq"], s["gk"] = _heads(gen, case, case["H"], N, t), _heads(gen, case, case["Hk"], N, t)
    else:
        B, N, M = case["B"], case["N"], case["M"]
        s["q"] = _heads(gen, case, case["H"], N, t)
        s["k"], s["v"] = _heads(gen, case, case["Hk"], M, t), _heads(gen, case, case["Hk"], M, t)
        leaves = ("q", "k", "v")
        if case["train"]:
            s["g"] = _heads(gen, case, case["H"], N, t)
        s["k_lengths"] = s["q_starts"] = s["mask"] = None
        if case["lengths"]:  # between half full and full, a sequence at least one long
            n = torch.rand(B, generator=gen, device="cuda") * 0.5 + 0.5
            s["k_lengths"] = (n * M).ceil().clamp(min=1).to(torch.int32)
            if case["causal"] and N != M:  # the queries are the last tokens of each sequence
                s["q_starts"] = s["k_lengths"] - N
        if case["mask"] == "bool":  # whole keys taken out, the same for every head, and a few rows with nothing left
            u = torch.rand(B, 1, N, M, generator=gen, device="cuda")
            s["mask"] = (u[:, :, :1] > 0.2) & (u > 0.05)
            s["mask"][:, :, :: 97] &= u[:, :, :: 97, :1] > 0.5
        elif case["mask"] == "bias":  # a bias by head, with -inf in places
            u = torch.randn(1, case["H"], N, M, generator=gen, device="cuda")
            s["mask"] = torch.where(u > 2.0, float("-inf"), u)
    if case.get("train") or case.get("mode") == "train":
        for x in leaves:
            s[x].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------

def _plain_norm(s):
    case, t = s["case"], s["x"].dtype
    x = s["x"].detach().float() + s["residual"].detach().float()
    w = s["weight"].detach().float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    y = n * w
    if case["mode"] == "infer":
        return y.to(t), x.to(t)
    if case["mode"] == "fp8":
        scale = y.abs().amax(-1, keepdim=True) / F8_MAX
        scale = torch.where(scale > 0, scale, 1.0)
        return (y / scale).to(torch.float8_e4m3fn), scale, x.to(t)
    gy, gs = s["gy"].float(), s["gs"].float()
    gn = gy * w
    dx = (r * (gn - n * (gn * n).mean(-1, keepdim=True)) + gs).to(t)
    return y.to(t), x.to(t), dx, dx, (gy * n).sum(0).to(t)


def _angles(positions, sections):
    """[N, pairs] in 64 bits: on each axis, pair j of n turns by position * BASE^(-j / n)."""
    out = []
    for p, n in zip(positions, sections):
        f = BASE ** (-torch.arange(n, device=p.device, dtype=torch.float64) / n)
        out.append(p.double()[:, None] * f)
    return torch.cat(out, -1)


def _turn(x, cos, sin, interleaved):
    x = x.detach().float()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    u, v = a * cos - b * sin, a * sin + b * cos
    return torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)


def _plain_rotary(s):
    case, t = s["case"], s["q"].dtype
    a = _angles(s["positions"], s["sections"])
    cos, sin, i = a.cos().float(), a.sin().float(), case["interleaved"]
    out = (_turn(s["q"], cos, sin, i).to(t), _turn(s["k"], cos, sin, i).to(t))
    if case["train"]:
        out += (_turn(s["gq"], cos, -sin, i).to(t), _turn(s["gk"], cos, -sin, i).to(t))
    return out


def _allowed(s):
    """What may be attended to, as truth values that broadcast to [B, H, N, M], or None for everything."""
    case = s["case"]
    N, M, dev = case["N"], case["M"], s["q"].device
    j = torch.arange(M, device=dev)
    ok = None
    if case["causal"]:
        first = M - N if s["q_starts"] is None else s["q_starts"].reshape(-1, 1, 1, 1)
        ok = j <= torch.arange(N, device=dev)[:, None] + first
    if s["k_lengths"] is not None:
        inside = j < s["k_lengths"].reshape(-1, 1, 1, 1)
        ok = inside if ok is None else ok & inside
    if case["mask"] == "bool":
        ok = s["mask"] if ok is None else ok & s["mask"]
    return ok


def _plain_attn(s):
    case, t = s["case"], s["q"].dtype
    B, H, Hk, N, M, d = (case[x] for x in ("B", "H", "Hk", "N", "M", "d"))
    G, scale = H // Hk, 1.0 / math.sqrt(d)
    q = s["q"].detach().float().reshape(B, Hk, G * N, d)
    k, v = s["k"].detach().float().contiguous(), s["v"].detach().float().contiguous()
    z = (q @ k.transpose(-1, -2).contiguous()).mul_(scale).view(B, H, N, M)
    if case["mask"] == "bias":
        z += s["mask"]
    ok = _allowed(s)
    if ok is not None:
        z.masked_fill_(~ok, float("-inf"))
    top = z.amax(-1, keepdim=True)
    p = z.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    p = p.view(B, Hk, G * N, M)
    o = p @ v
    out = o.view(B, H, N, d).to(t)
    if not case["train"]:
        return (out,)
    g = s["g"].float().reshape(B, Hk, G * N, d)
    dv = p.transpose(-1, -2).contiguous() @ g
    dz = (g @ v.transpose(-1, -2).contiguous()).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = dz @ k
    dk = dz.transpose(-1, -2).contiguous() @ q
    return out, dq.view(B, H, N, d).to(t), dk.to(t), dv.to(t)


def run(s):
    case = s["case"]
    if not own:
        return {"norm": _plain_norm, "rotary": _plain_rotary, "attn": _plain_attn}[case["kind"]](s)
    lf = _lf()
    if case["kind"] == "norm":
        x, residual, weight = s["x"], s["residual"], s["weight"]
        if case["mode"] == "infer":
            return lf.add_rms_norm(x, weight, residual, eps=EPS)
        if case["mode"] == "fp8":
            return lf.add_rms_norm_fp8(x, weight, residual, eps=EPS)
        y, total = lf.add_rms_norm(x, weight, residual, eps=EPS)
        grads = torch.autograd.grad((y, total), (x, residual, weight), (s["gy"], s["gs"]))
        return (y.detach(), total.detach(), *grads)
    if case["kind"] == "rotary":
        q, k = lf.rotary(s["q"], s["k"], s["positions"], s["sections"], base=BASE, interleaved=case["interleaved"])
        if not case["train"]:
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"])))
    out = lf.softmax_attention(s["q"], s["k"], s["v"], mask=s["mask"], causal=case["causal"],
                               k_lengths=s["k_lengths"], q_starts=s["q_starts"])
    if not case["train"]:
        return (out,)
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["g"]))


# ---------------------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        R, W = case["rows"], case["width"]
        if case["mode"] == "infer":
            return {"bytes": (4 * R + 1) * W * e, "flops": 5 * R * W}
        if case["mode"] == "fp8":
            return {"bytes": (3 * R + 1) * W * e + R * W + 4 * R, "flops": 8 * R * W}
        # x, residual, gy, gs in; y, the sum and its gradient out (one tensor is the gradient of both addends).
        return {"bytes": (7 * R + 2) * W * e, "flops": 16 * R * W}
    if case["kind"] == "rotary":
        N = math.prod(int(x) for x in case["grid"].split("x"))
        n = case["B"] * (case["H"] + case["Hk"]) * N * case["d"] * (2 if case["train"] else 1)
        return {"bytes": 2 * e * n, "flops": 3 * n}
    B, H, Hk, N, M, d = (case[x] for x in ("B", "H", "Hk", "N", "M", "d"))
    fill = 0.75 if case["lengths"] else 1.0  # the mean of what prepare draws
    # The pairs that a causal mask leaves: the last min(N, M) queries see one key less each, backwards.
    n = min(N, M)
    pairs = N * M - (n * (n - 1) // 2 + (N - n) * M if case["causal"] else 0)
    if case["causal"] and N == M:  # the queries behind a sequence's end see all of it
        pairs = N * M * (fill - fill * fill / 2) + N * fill / 2
    else:
        pairs = pairs * fill
    kv = 2 * B * Hk * M * d * e * fill
    q = 2 * B * H * N * d * e
    m = {"none": 0, "bool": B * N * M, "bias": 4 * H * N * M}[case["mask"]]
    if not case["train"]:
        return {"bytes": q + kv + m, "flops": 4 * B * H * pairs * d}
    # Two products forward; backward the scores again, and the gradients of p, v, q and k.
    return {"bytes": 2 * q + 2 * kv + m, "flops": 14 * B * H * pairs * d}


# ---------------------------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------------------------

def _exact_norm(s):
    case = s["case"]
    total = (s["x"].detach().double() + s["residual"].detach().double()).requires_grad_()
    w = s["weight"].detach().double().requires_grad_()
    y = w * total / (total.square().sum(-1, keepdim=True) / total.shape[-1] + EPS).sqrt()
    if case["mode"] == "infer":
        return y.detach(), total.detach()
    if case["mode"] == "fp8":
        y = y.detach()
        largest = y.abs().max(-1, keepdim=True).values
        scale = torch.where(largest == 0, torch.ones_like(largest), largest / F8_MAX)
        return y / scale, scale, total.detach()
    grads = torch.autograd.grad((y, total), (total, w), (s["gy"].double(), s["gs"].double()))
    return y.detach(), total.detach(), grads[0], grads[0], grads[1]


def _exact_rotary(s):
    case = s["case"]
    freq, axis = [], []
    for a, n in enumerate(s["sections"]):
        freq += [math.exp(-math.log(BASE) * j / n) for j in range(n)]
        axis += [a] * n
    freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
    where = s["positions"].double().t()[:, axis]
    turn = torch.polar(torch.ones_like(where), where * freq)

    def go(x, turn):
        x = x.detach().double()
        h = x.shape[-1] // 2
        if case["interleaved"]:
            z = torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) * turn
            return torch.view_as_real(z).reshape(x.shape)
        z = torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous()) * turn
        return torch.cat((z.real, z.imag), -1)

    out = (go(s["q"], turn), go(s["k"], turn))
    if case["train"]:
        out += (go(s["gq"], turn.conj()), go(s["gk"], turn.conj()))
    return out


def _exact_attn(s):
    """One sequence and head at a time, the gradients by the softmax's Jacobian."""
    case = s["case"]
    B, H, Hk, N, M, d = (case[x] for x in ("B", "H", "Hk", "N", "M", "d"))
    dev, f = s["q"].device, torch.float64
    out = torch.zeros(B, H, N, d, dtype=f, device=dev)
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(B, Hk, M, d, dtype=f, device=dev) for _ in range(2))
    rows, cols = torch.arange(N, device=dev).view(N, 1), torch.arange(M, device=dev).view(1, M)
    for b in range(B):
        for h in range(H):
            q, k, v = s["q"][b, h].detach().double(), s["k"][b, h * Hk // H].detach().double(), \
                s["v"][b, h * Hk // H].detach().double()
            z = torch.matmul(q, k.t()) / math.sqrt(d)
            gone = torch.zeros(N, M, dtype=torch.bool, device=dev)
            if case["causal"]:
                gone |= cols - rows > (M - N if s["q_starts"] is None else s["q_starts"][b])
            if s["k_lengths"] is not None:
                gone |= cols >= s["k_lengths"][b]
            if case["mask"] == "bool":
                gone |= ~s["mask"][b, 0]
            elif case["mask"] == "bias":
                z = z + s["mask"][0, h].double()
            z = torch.where(gone, -math.inf, z)
            lse = torch.logsumexp(z, -1, keepdim=True)
            p = torch.where(lse == -math.inf, 0.0, torch.exp(z - torch.where(lse == -math.inf, 0.0, lse)))
            out[b, h] = p @ v
            if case["train"]:
                g = s["g"][b, h].double()
                dp = g @ v.t()
                dz = p * dp - p * (p * dp).sum(-1, keepdim=True)
                dq[b, h] = dz @ k / math.sqrt(d)
                dk[b, h * Hk // H] += dz.t() @ q / math.sqrt(d)
                dv[b, h * Hk // H] += p.t() @ g
    return (out, dq, dk, dv) if case["train"] else (out,)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attn": _exact_attn}[case["kind"]](s)
