"""Performance cases of the decaying linear attention and the gated double norm on one GPU.

Three operators that stand beside softmax_attention and add_rms_norm in a block:
  decay   decay_attention: causal linear attention whose memory decays by a factor of each head,
            S_t = exp(log_decay) S_(t-1) + k_t v_t^T,   out_t = scale S_t^T q_t,
          over whole sequences (training: with the gradients of q, k and v, and of the state);
  step    decay_attention_step: the same for one new token, on a state that it updates in place;
  norm    gated_add_rms_norm: a block's output through its own norm, a gate and a residual scale
          onto the residual, and the next block's norm of that sum,
            sum = residual + scale gate norm(x) post_weight,   y = norm(sum) weight
          (training: with the gradients of all five).

Where ``own`` is false, ``run`` computes them from elementary tensor operations in 32 bits
(the decays' powers in 64), the attention in chunks whose states are joined by one product;
where it is true it calls the framework.

fp64 is left out: the operators refuse it.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
CHUNK = 128  # tokens of a chunk of the plain form


def _lf():
    import laplacianformer_amd as lf
    return lf


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------

def _decay(name, B, H, Hk, N, d, dv, dtype, train, decay="slow", lengths=False, state=False, layout="bhnd"):
    """decay: "slow" (1 - 2^-5 to 1 - 2^-12 by head), "fast" (e^-1 to e^-1/128), "none"; state: one is
    given and the last one returned; layout: the order of the tensors in memory ("bnhd" is what a
    projection's output gives)."""
    return {"name": name, "kind": "decay", "B": B, "H": H, "Hk": Hk, "N": N, "d": d, "dv": dv, "dtype": dtype,
            "train": train, "decay": decay, "lengths": lengths, "state": state, "layout": layout}


def _step(name, B, H, Hk, d, dv, dtype, decay="slow"):
    return {"name": name, "kind": "step", "B": B, "H": H, "Hk": Hk, "d": d, "dv": dv, "dtype": dtype, "decay": decay}


def _norm(name, B, N, width, dtype, train, gate, post=True, scale=1.0):
    """gate: "none", "channel" (one for all), "sequence" (one per sequence), "token"; post: with a norm of x."""
    return {"name": name, "kind": "norm", "B": B, "N": N, "width": width, "dtype": dtype, "train": train, "gate": gate,
            "post": post, "scale": scale}


def listed():
    return [
        # A whole small attention in the default type.
        _decay("decay_tiny_f32", 2, 2, 2, 196, 32, 32, "f32", True),
        # A late stage, 14 x 14 tokens and four heads of 32 channels, in mixed precision.
        _decay("decay_stage3_f16", 64, 4, 4, 196, 32, 32, "f16", True),
        # The next piece of a prompt, from the state that the pieces before it left, in the default type.
        _decay("decay_piece_f32", 4, 8, 8, 515, 64, 64, "f32", False, state=True),
        # Shared heads of 80 channels, sequences of uneven lengths, trained through their states.
        _decay("decay_ragged_bf16", 6, 6, 2, 1003, 80, 80, "bf16", True, decay="fast", lengths=True, state=True,
               layout="bnhd"),
        # Many tokens: the largest training step.
        _decay("decay_stress_bf16", 8, 8, 8, 16384, 64, 64, "bf16", True),
        # A long prompt with shared heads, whose state the tokens behind it go on from.
        _decay("decay_prompt_bf16", 1, 32, 8, 32768, 128, 128, "bf16", False, state=True, layout="bnhd"),
        # A new token of one sequence of a small model: a launch and its latency.
        _step("step_token_f32", 1, 4, 4, 32, 32, "f32"),
        # New tokens of a few sequences, odd sizes, values wider than keys.
        _step("step_odd_f16", 7, 6, 2, 50, 80, "f16", decay="fast"),
        # New tokens of many sequences.
        _step("step_batch_bf16", 64, 32, 8, 128, 128, "bf16"),
        # The norms around a single token of a small model.
        _norm("norm_token_bf16", 1, 1, 512, "bf16", False, "channel"),
        # The norms between blocks of 14 x 14 tokens, trained, with a gate for each channel.
        _norm("norm_stage3_odd_f32", 64, 196, 333, "f32", True, "channel", scale=0.5),
        # A long batch, trained, with gates that a condition gives for each sequence.
        _norm("norm_long_bf16", 8, 2048, 4096, "bf16", True, "sequence"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decay", "decay", "decay", "step", "norm", "norm"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind == "norm":
        width = rng.choice([_log_int(rng, 8, 8192), 8 * _log_int(rng, 8, 1024)])
        rows = _log_int(rng, 1, max(2, min(65536, (1 << 24) // width)))
        B = _log_int(rng, 1, min(rows, 64))
        c = _norm("", B, max(1, rows // B), width, dtype, rng.random() < 0.6,
                  rng.choice(["none", "channel", "channel", "sequence", "sequence", "token"]), post=rng.random() < 0.7,
                  scale=rng.choice([1.0, 1.0, 0.5, 0.1]))
    else:
        d = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 50])
        dv = rng.choice([d, d, d, 32, 64, 128, 72])
        Hk = rng.choice([1, 2, 3, 4, 8])
        H = Hk * rng.choice([1, 1, 1, 2, 4])
        decay = rng.choice(["slow", "slow", "slow", "fast", "none"])
        if kind == "step":
            c = _step("", _log_int(rng, 1, max(1, int(3.0e7 // (H * d * dv)))), H, Hk, d, dv, dtype, decay)
        else:
            N = _log_int(rng, 1, 32768)
            train = rng.random() < 0.6
            most = int((2.5e7 if train else 1.0e8) // (H * N * max(d, dv)))
            if most < 1:
                N = max(1, int(N * (2.5e7 if train else 1.0e8) / (H * N * max(d, dv))))
            c = _decay("", _log_int(rng, 1, min(64, max(1, most))), H, Hk, N, d, dv, dtype, train, decay=decay,
                       lengths=rng.random() < 0.3, state=rng.random() < 0.4, layout=rng.choice(["bhnd", "bnhd"]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------

def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _heads(gen, case, H, d, dtype):
    """[B, H, N, d] in the case's memory order."""
    B, N = case["B"], case.get("N", 1)
    if case.get("layout") == "bnhd":
        return _randn(gen, (B, N, H, d), dtype).transpose(1, 2)
    return _randn(gen, (B, H, N, d), dtype)


def _log_decay(case):
    """fp32 [H]."""
    h = torch.arange(case["H"], dtype=torch.float64) % 8
    if case["decay"] == "none":
        x = torch.zeros_like(h)
    elif case["decay"] == "fast":
        x = -torch.exp2(-h)
    else:
        x = torch.log1p(-torch.exp2(-5 - h))
    return x.float().cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    s = {"case": case}
    B = case["B"]
    if case["kind"] == "norm":
        N, W = case["N"], case["width"]
        s["x"], s["residual"] = _randn(gen, (B, N, W), t), _randn(gen, (B, N, W), t, 2.0)
        s["weight"], s["post_weight"] = ((1.0 + 0.1 * torch.randn(W, generator=gen, device="cuda")).to(t) for _ in range(2))
        shape = {"none": None, "channel": (W,), "sequence": (B, 1, W), "token": (B, N, W)}[case["gate"]]
        s["gate"] = None if shape is None else _randn(gen, shape, t, 0.5)
        if not case["post"]:
            s["post_weight"] = None
        leaves = ("x", "residual", "weight", "post_weight", "gate")
        if case["train"]:
            s["gy"], s["gs"] = _randn(gen, (B, N, W), t), _randn(gen, (B, N, W), t)
    else:
        H, Hk, d, dv = (case[x] for x in ("H", "Hk", "d", "dv"))
        s["q"], s["k"], s["v"] = _heads(gen, case, H, d, t), _heads(gen, case, Hk, d, t), _heads(gen, case, Hk, dv, t)
        s["log_decay"] = _log_decay(case)
        s["state"] = s["lengths"] = None
        if case["kind"] == "step" or case["state"]:
            s["state"] = _randn(gen, (B, H, d, dv), torch.float32, 4.0)
        leaves = ("q", "k", "v", "state")
        if case["kind"] == "decay":
            if case["lengths"]:  # between half full and full, a sequence at least one long
                n = torch.rand(B, generator=gen, device="cuda") * 0.5 + 0.5
                s["lengths"] = (n * case["N"]).ceil().clamp(min=1).to(torch.int32)
            if case["train"]:
                s["g"] = _heads(gen, case, H, dv, t)
                if case["state"]:
                    s["g_state"] = _randn(gen, (B, H, d, dv), torch.float32, 0.25)
    if case.get("train"):
        for x in leaves:
            if s[x] is not None:
                s[x].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------

def _pow(log_decay, n):
    """exp(log_decay * n) for whole n >= 0, [H] + n's shape, 0 where n < 0; formed in 64 bits."""
    x = torch.exp(log_decay.double().view((-1,) + (1,) * n.dim()) * n.clamp(min=0))
    return torch.where(n < 0, 0.0, x).float()


def _chunked(q, k, v, log_decay, first):
    """out_t = sum over j <= t of decay^(t - j) (q_t . k_j) v_j + decay^(t + 1) q_t . first, for fp32 [B, H, N, .]."""
    B, H, N, d = q.shape
    n = -(-N // CHUNK)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, n * CHUNK - N)).view(B, H, n, CHUNK, -1) for x in (q, k, v))
    i = torch.arange(CHUNK, device=q.device)
    inside = (q @ k.transpose(-1, -2).contiguous()) * _pow(log_decay, i[:, None] - i)[:, None]
    out = inside @ v
    del inside
    add = (k * _pow(log_decay, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2).contiguous() @ v
    m = torch.arange(n, device=q.device)
    # The state in front of every chunk, from all chunks before it.
    before = _pow(log_decay, CHUNK * (m[:, None] - 1 - m)) @ add.view(B, H, n, -1)
    if first is not None:
        before = before + _pow(log_decay, CHUNK * m)[..., None] * first.reshape(B, H, 1, -1)
    out += (q * _pow(log_decay, i + 1)[:, None, :, None]) @ before.view(B, H, n, d, -1)
    return out.view(B, H, n * CHUNK, -1)[:, :, :N]


def _plain_decay(s):
    case, t = s["case"], s["q"].dtype
    B, H, Hk, N = (case[x] for x in ("B", "H", "Hk", "N"))
    G, scale = H // Hk, 1.0 / math.sqrt(case["d"])
    lg, dev = s["log_decay"], s["q"].device
    pos = torch.arange(N, device=dev)
    length = torch.full((B,), N, device=dev) if s["lengths"] is None else s["lengths"].long()
    live = (pos < length[:, None])[:, None, :, None]
    q = s["q"].detach().float() * live
    k, v = (s[x].detach().float().repeat_interleave(G, 1) * live for x in ("k", "v"))
    first = None if s["state"] is None else s["state"].detach()
    out = ((_chunked(q, k, v, lg, first) * scale) * live).to(t)
    # How far each token is in front of its sequence's end, as a power of the decay: [B, H, N, 1].
    left = _pow(lg, length[:, None] - 1 - pos).transpose(0, 1)[..., None]
    res = (out,)
    if case["state"]:
        whole = _pow(lg, length).t()[..., None, None]
        res += ((k * left).transpose(-1, -2).contiguous() @ v + whole * first,)
    if not case["train"]:
        return res
    g = s["g"].float() * live
    dq = _chunked(g, v, k, lg, None if first is None else first.transpose(-1, -2).contiguous()) * scale * live
    # The other two run against the sequence, from its end.
    qr, kr, vr, gr = (x.flip(2) for x in (q, k, v, g))
    dk = _chunked(vr, gr, qr, lg, None).flip(2) * scale
    dv = _chunked(kr, qr, gr, lg, None).flip(2) * scale
    if case["state"]:
        gs = s["g_state"]
        dk += left * (v @ gs.transpose(-1, -2).contiguous())
        dv += left * (k @ gs)
        dstate = whole * gs + scale * ((q * _pow(lg, pos + 1)[None, ..., None]).transpose(-1, -2).contiguous() @ g)
    dk, dv = ((x * live).view(B, Hk, G, N, -1).sum(2).to(t) for x in (dk, dv))
    return res + (dq.to(t), dk, dv) + ((dstate,) if case["state"] else ())


def _plain_step(s):
    G, state = s["case"]["H"] // s["case"]["Hk"], s["state"]
    k, v = (s[x].float().repeat_interleave(G, 1) for x in ("k", "v"))
    state.mul_(s["log_decay"].exp()[:, None, None]).add_(k.transpose(-1, -2) * v)
    out = (s["q"].float().transpose(-1, -2) * state).sum(-2, keepdim=True) * (1.0 / math.sqrt(s["case"]["d"]))
    return out.to(s["q"].dtype), state


def _plain_norm(s):
    case, t = s["case"], s["x"].dtype
    scale = case["scale"]
    x, r, w = (s[n].detach().float() for n in ("x", "residual", "weight"))
    wp = s["post_weight"].detach().float() if case["post"] else None
    gate = s["gate"].detach().float() if s["gate"] is not None else torch.ones((), device=x.device)
    if case["post"]:
        rp = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        m = x * rp
        z = m * wp
    else:
        z = x
    total = r + scale * gate * z
    rs = torch.rsqrt((total * total).mean(-1, keepdim=True) + EPS)
    n = total * rs
    y = (n * w).to(t)
    if not case["train"]:
        return y, total.to(t)
    gy, gs = s["gy"].float(), s["gs"].float()
    gn = gy * w
    ds = gs + rs * (gn - n * (gn * n).mean(-1, keepdim=True))
    dz = scale * gate * ds
    res = (y, total.to(t))
    if case["post"]:
        gm = dz * wp
        res += ((rp * (gm - m * (gm * m).mean(-1, keepdim=True))).to(t),)
    else:
        res += (dz.to(t),)
    res += (ds.to(t), (gy * n).sum((0, 1)).to(t))
    if case["post"]:
        res += ((dz * m).sum((0, 1)).to(t),)
    if case["gate"] != "none":
        dg = scale * ds * z
        dg = dg.sum((0, 1)) if case["gate"] == "channel" else dg.sum(1, keepdim=True) if case["gate"] == "sequence" else dg
        res += (dg.to(t),)
    return res


def run(s):
    case = s["case"]
    if not own:
        return {"norm": _plain_norm, "decay": _plain_decay, "step": _plain_step}[case["kind"]](s)
    lf = _lf()
    if case["kind"] == "step":
        return lf.decay_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"]), s["state"]
    if case["kind"] == "decay":
        res = lf.decay_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], lengths=s["lengths"],
                                 return_state=case["state"])
        res = res if case["state"] else (res,)
        if not case["train"]:
            return res
        leaves = [s[x] for x in ("q", "k", "v", "state") if s[x] is not None]
        grads = torch.autograd.grad(res, leaves, [s["g"]] + ([s["g_state"]] if case["state"] else []))
        return (*(x.detach() for x in res), *grads)
    y, total = lf.gated_add_rms_norm(s["x"], s["weight"], s["residual"], post_weight=s["post_weight"], gate=s["gate"],
                                     scale=case["scale"], eps=EPS)
    if not case["train"]:
        return y, total
    leaves = [s[x] for x in ("x", "residual", "weight", "post_weight", "gate") if s[x] is not None]
    return (y.detach(), total.detach(), *torch.autograd.grad((y, total), leaves, (s["gy"], s["gs"])))


# ---------------------------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        n, W = case["B"] * case["N"], case["width"]
        g = {"none": 0, "channel": W, "sequence": case["B"] * W, "token": n * W}[case["gate"]]
        params = (2 if case["post"] else 1) * W + g
        if not case["train"]:
            return {"bytes": (4 * n * W + params) * e, "flops": (12 if case["post"] else 7) * n * W}
        # x, residual, gy, gs in; y, the sum and the gradients of x and the residual out.
        return {"bytes": (8 * n * W + 2 * params) * e, "flops": (36 if case["post"] else 22) * n * W}
    B, H, Hk, d, dv = (case[x] for x in ("B", "H", "Hk", "d", "dv"))
    if case["kind"] == "step":
        return {"bytes": 8 * B * H * d * dv + B * (H + Hk) * (d + dv) * e, "flops": 5 * B * H * d * dv}
    fill = 0.75 if case["lengths"] else 1.0  # the mean of what prepare draws
    n = B * case["N"]
    # q, k, v in and out written (zeros behind a length too); with gradients, g in and three out.
    qk, vo = n * (H + Hk) * d, n * (H + Hk) * dv
    size = fill * (qk + n * Hk * dv) + n * H * dv
    state = 2 * 4 * B * H * d * dv if case["state"] else 0
    # By token and head: k v^T onto the state and the state times q; backward the state again, the
    # gradient's state, and three products with them.
    flops = 4 * fill * n * H * d * dv
    if case["train"]:
        size += fill * n * H * dv + qk + n * Hk * dv
        state *= 2
        flops += 10 * fill * n * H * d * dv
    return {"bytes": size * e + state, "flops": flops}


# ---------------------------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------------------------

def _exact_decay(s):
    """The recurrences themselves, token by token."""
    case = s["case"]
    B, H, Hk, d, dv = (case[x] for x in ("B", "H", "Hk", "d", "dv"))
    N = case.get("N", 1)
    scale = case["d"] ** -0.5
    head = torch.arange(H, device="cuda") // (H // Hk)
    rows = lambda x: x.detach().double().permute(2, 0, 1, 3).reshape(x.shape[2], -1, x.shape[3]).contiguous()  # noqa: E731
    q, k, v = rows(s["q"]), rows(s["k"][:, head]), rows(s["v"][:, head])
    gamma = torch.exp(s["log_decay"].double()).repeat(B).view(-1, 1, 1)
    first = torch.zeros(B * H, d, dv, dtype=torch.float64, device="cuda")
    if s["state"] is not None:
        first = s["state"].detach().double().reshape(B * H, d, dv).clone()
    length = [N] * B if s["lengths"] is None else s["lengths"].tolist()
    ends = torch.tensor(length, device="cuda").repeat_interleave(H).view(-1, 1, 1)
    # A sequence that has ended keeps its state: its token adds nothing and decays nothing.
    live = [(ends > t).double() for t in range(N)] if min(length) < N else None
    out, dq = torch.zeros(N, B * H, dv, dtype=torch.float64, device="cuda"), torch.zeros_like(q)
    g = rows(s["g"]) if case.get("train") else None
    S = first.clone()
    for t in range(N):
        if live is None:
            S.mul_(gamma).addcmul_(k[t][:, :, None], v[t][:, None, :])
            out[t] = torch.bmm(q[t][:, None], S)[:, 0]
        else:
            S = torch.where(live[t] > 0, S * gamma + k[t][:, :, None] * v[t][:, None, :], S)
            out[t] = (torch.bmm(q[t][:, None], S) * live[t])[:, 0]
        if g is not None:
            dq[t] = torch.bmm(S, g[t][:, :, None])[:, :, 0]
            if live is not None:
                dq[t] *= live[t][:, 0]
    back = lambda x: x.view(N, B, H, -1).permute(1, 2, 0, 3)  # noqa: E731
    res = (scale * back(out),)
    if case["kind"] == "step" or case["state"]:
        res += (S.view(B, H, d, dv),)
    if g is None:
        return res
    dk, dv_ = torch.zeros_like(k), torch.zeros_like(v)
    # R: the gradient of the state behind token t.
    R = s["g_state"].double().reshape(B * H, d, dv).clone() if case["state"] else torch.zeros_like(first)
    for t in reversed(range(N)):
        if live is None:
            R.addcmul_(q[t][:, :, None], g[t][:, None, :], value=scale)
            dk[t], dv_[t] = torch.bmm(R, v[t][:, :, None])[:, :, 0], torch.bmm(k[t][:, None], R)[:, 0]
            R.mul_(gamma)
        else:
            P = R + scale * q[t][:, :, None] * g[t][:, None, :]
            dk[t] = torch.bmm(P, v[t][:, :, None])[:, :, 0] * live[t][:, 0]
            dv_[t] = torch.bmm(k[t][:, None], P)[:, 0] * live[t][:, 0]
            R = torch.where(live[t] > 0, P * gamma, R)
    share = lambda x: back(x).reshape(B, Hk, H // Hk, N, -1).sum(2)  # noqa: E731
    res += (scale * back(dq), share(dk), share(dv_))
    return res + ((R.view(B, H, d, dv),) if case["state"] else ())


def _exact_norm(s):
    """The formula, and its gradients by automatic differentiation."""
    case = s["case"]
    names = [n for n in ("x", "residual", "weight", "post_weight", "gate") if s[n] is not None]
    p = {n: s[n].detach().double().requires_grad_() for n in names}
    unit = lambda a: a / torch.sqrt(a.square().sum(-1, keepdim=True) / a.shape[-1] + EPS)  # noqa: E731
    z = unit(p["x"]) * p["post_weight"] if case["post"] else p["x"]
    if s["gate"] is not None:
        z = p["gate"] * z
    total = p["residual"] + case["scale"] * z
    y = unit(total) * p["weight"]
    if not case["train"]:
        return y.detach(), total.detach()
    grads = torch.autograd.grad((y, total), [p[n] for n in names], (s["gy"].double(), s["gs"].double()))
    return (y.detach(), total.detach(), *grads)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if case["kind"] == "norm" else _exact_decay(s)
