"""Plain 64-bit forms of the transformer-block operators on the CPU, with the bounds their tests hold them to.

Every bound is a sum of roundings, each at most u |value| (u = finfo.eps / 2 of the type, 2^-24 in
fp32 arithmetic), carried through the formula. U32 counts fp32 steps: a sum of n terms
is off by at most n U32 times the sum of their magnitudes."""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
NEG = float("-inf")


def unit(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def assert_within(got, ref, tol, what):
    """|got - ref| <= tol everywhere, with finite results.

    The bounds count a rounding as u |value|; below the type's smallest normal number values are
    whole multiples of smallest_normal * eps, and a rounding is off by up to half of that (fp16:
    2^-14 * 2^-10 / 2 = 2^-25), whatever the value."""
    info = torch.finfo(got.dtype)
    tol = tol + info.smallest_normal * info.eps / 2
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if not ref.numel():
        return
    assert bool(torch.isfinite(got).all()), (what, "not finite", int((~torch.isfinite(got)).sum()))
    over = ((got - ref).abs() - tol).max().item()
    assert over <= 0, (what, "over the bound by", over, "largest bound", tol.max().item())


def allowed(B, H, N, M, causal=False, k_lengths=None, q_lengths=None, q_starts=None, mask=None):
    """[B, H, N, M] truth values, and the additive part of the mask (or None)."""
    i, j = torch.arange(N).view(N, 1), torch.arange(M).view(1, M)
    ok = torch.ones(B, H, N, M, dtype=torch.bool)
    if causal:
        first = torch.full((B,), M - N) if q_starts is None else q_starts.cpu().long()
        ok &= j <= i + first.view(B, 1, 1, 1)
    if k_lengths is not None:
        ok &= j < k_lengths.cpu().long().clamp(0, M).view(B, 1, 1, 1)
    if q_lengths is not None:
        ok &= i < q_lengths.cpu().long().clamp(0, N).view(B, 1, 1, 1)
    bias = None
    if mask is not None:
        m = mask.cpu()
        if m.dtype == torch.bool:
            ok &= m
        else:
            bias = torch.broadcast_to(m.double(), (B, H, N, M))
            ok &= bias != NEG
            bias = torch.where(ok, bias, 0.0)
    return ok, bias


def attention(q, k, v, g, ok, bias, scale):
    """{name: (reference, bound)} for out, and dq, dk, dv if g is given. q, k, v, g: CPU tensors
    of one type, their masked rows finite."""
    u, t = unit(q.dtype), q.dtype
    B, H, N, d = q.shape
    Hk, M = k.shape[1], k.shape[2]
    G = H // Hk
    Q, K, V = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    s = scale * (Q @ K.transpose(-1, -2))
    x = s + bias if bias is not None else s
    x = torch.where(ok, x, NEG)
    top = x.amax(-1, keepdim=True) if M else x.new_full((B, H, N, 1), NEG)
    top = torch.where(top == NEG, 0.0, top)
    e = torch.exp(x - top)
    l = e.sum(-1, keepdim=True)
    p = e / torch.where(l > 0, l, 1.0)
    out = p @ V
    # A score: d products summed, the scale and the bias added, the maximum subtracted and
    # log2(e) multiplied in, each a rounding of at most the values so far; 2^-22 for exp2 and
    # log2 themselves (both good to 2 of 2^-23).
    mag = scale * (Q.abs() @ K.abs().transpose(-1, -2))
    size = torch.where(ok, mag + s.abs() + (bias.abs() if bias is not None else 0.0), 0.0)
    worst = size.amax(-1, keepdim=True) if M else size.sum(-1, keepdim=True)
    ds = U32 * ((d + 4) * mag + 4 * (size + worst)) + 2.0 ** -22
    # relative error of p: its own score's, and the sum's (its largest score error, and M terms)
    rp = ds + (ds.amax(-1, keepdim=True) if M else 0.0) + (M + 4) * U32
    # a p that is subnormal in fp16, next to a sum of at least 1; the matrix cores and the exponential take
    # results below fp32's smallest normal number, 2^-126, for 0
    flush = 2.0 ** -126
    tiny = 2.0 ** -25 if t == torch.float16 else flush
    pv = p @ V.abs()
    err_o = (p * rp) @ V.abs() + (u + M * U32) * pv + tiny * (ok.double() @ V.abs())
    res = {"out": (out, err_o + u * (out.abs() + err_o))}
    if g is None:
        return res
    Gd = g.double()
    dp = Gd @ V.transpose(-1, -2)
    delta = (Gd * out).sum(-1, keepdim=True)
    dz = p * (dp - delta)
    gv = Gd.abs() @ V.abs().transpose(-1, -2)
    err_delta = (Gd.abs() * res["out"][1]).sum(-1, keepdim=True) + d * U32 * (Gd.abs() * out.abs()).sum(-1, keepdim=True)
    size_z = p * (dp.abs() + delta.abs())
    # fp16: dz times f is rounded, f bound <= 2^14 with f bound > 2^12: subnormal steps of 2^-25 / f
    low = 2.0 ** -25 * 2.0 ** -12 * (Gd.norm(dim=-1).amax() * V.norm(dim=-1).amax() + delta.abs().amax()) if t == torch.float16 else 0.0
    err_z = p * (d * U32 * gv + err_delta) + (rp + 4 * U32) * size_z + u * dz.abs() + (low + flush * (1 + dp.abs() + delta.abs())) * ok.double()
    group = lambda y: y.view(B, Hk, G, M, d).sum(2)
    n = N * G
    dq = scale * (dz @ K)
    tq = scale * (err_z @ K.abs() + M * U32 * (dz.abs() @ K.abs()))
    dk = scale * group(dz.transpose(-1, -2) @ Q)
    tk = scale * group(err_z.transpose(-1, -2) @ Q.abs() + n * U32 * (dz.abs().transpose(-1, -2) @ Q.abs()))
    pt = p.transpose(-1, -2)
    dv = group(pt @ Gd)
    tiny = 2.0 ** -40 if t == torch.float16 else flush
    tv = group((p * (rp + u + n * U32)).transpose(-1, -2) @ Gd.abs() + tiny * ok.double().transpose(-1, -2) @ Gd.abs())
    for name, y, e_ in (("dq", dq, tq), ("dk", dk, tk), ("dv", dv, tv)):
        res[name] = (y, e_ * (1 + u) + u * y.abs() + 4 * U32 * y.abs())
    return res


def rms_norm(x, weight, residual, eps, gy=None, gs=None):
    """{name: (reference, bound)} for y, sum and, if gy is given, dx and dw."""
    u, W = unit(x.dtype), x.shape[-1]
    s = x.double() + (residual.double() if residual is not None else 0.0)
    w = weight.double()
    r = 1.0 / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    n = s * r
    y = n * w
    # 64 terms per thread at most, and a tree of ten; the sum's own rounding twice
    c = 96 * U32
    res = {"y": (y, c * y.abs() + u * y.abs() * (1 + c)), "sum": (s, (u + U32) * s.abs())}
    if gy is None:
        return res
    g = gy.double()
    us = U32 if residual is not None else 0.0  # the fp32 sum, or in fp32 the stored one
    gn = g * w
    dot = (gn * n).mean(-1, keepdim=True)
    err_n = (us + c) * n.abs()
    err_dot = (gn.abs() * err_n).mean(-1, keepdim=True) + c * (gn * n).abs().mean(-1, keepdim=True)
    core = r * (gn - n * dot)
    dx = core + (gs.double() if gs is not None else 0.0)
    err = r * (err_n * dot.abs() + n.abs() * err_dot + c * (gn.abs() + (n * dot).abs()))
    rows = x.numel() // W if W else 0
    flat = lambda t: t.reshape(-1, W)
    dw = flat(g * n).sum(0)
    err_w = flat(g.abs() * err_n).sum(0) + rows * U32 * flat((g * n).abs()).sum(0)
    uw = unit(weight.dtype)
    res["dx"] = (dx, err + (u + 2 * U32) * (dx.abs() + err))
    res["dw"] = (dw, err_w + uw * (dw.abs() + err_w))
    return res


def rotary(x, positions, sections, base, interleaved, inverse=False):
    """(reference, bound); positions [A, N] or [A, B, N]."""
    u, P = unit(x.dtype), sum(sections)
    pos = positions.cpu().double()
    if pos.dim() == 2:
        pos = pos[:, None].expand(-1, x.shape[0], -1)
    angle = torch.cat([pos[a][..., None] * torch.tensor([base ** (-j / n) for j in range(n)], dtype=torch.float64)
                       for a, n in enumerate(sections)], -1)[:, None]  # [B, 1, N, P]
    if inverse:
        angle = -angle
    X = x.double()
    a, b = (X[..., 0:2 * P:2], X[..., 1:2 * P:2]) if interleaved else (X[..., :P], X[..., P:2 * P])
    y0, y1 = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    ref = X.clone()
    if interleaved:
        ref[..., 0:2 * P:2], ref[..., 1:2 * P:2] = y0, y1
    else:
        ref[..., :P], ref[..., P:2 * P] = y0, y1
    # The angle: 64-bit frequency and product on both sides (2^-51 of the position), 2^-32 turns
    # of truncation, and 2^-25 half turns of rounding; sine and cosine to 4 of 2^-24, and the sum.
    da = pos.abs().amax() * 2.0 ** -50 + 2 * math.pi * 2.0 ** -32 + math.pi * 2.0 ** -25 if pos.numel() else 0.0
    tol = torch.zeros_like(X)
    size = (a.abs() + b.abs()) * (da + 8 * U32)
    if interleaved:
        tol[..., 0:2 * P:2] = tol[..., 1:2 * P:2] = size
    else:
        tol[..., :P] = tol[..., P:2 * P] = size
    return ref, tol + u * (ref.abs() + tol)
