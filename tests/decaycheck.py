"""Plain 64-bit forms of decay_attention and gated_add_rms_norm on the CPU, with the bounds their tests hold them to.

The attention's bounds: every result is a sum of terms (decay power) x (three operand values), and ``mag`` is
the same sum of the terms' magnitudes. A term carries, relative to its magnitude,
  U32 = 2^-24 for each addition that its partial sums go through: at most d (the score, or the state times the
      query), the tokens N (within tiles and from tile to tile), 2 roundings a tile (the state's decay) and 64 more
      (scales, the shared heads, the segments' join);
  the powers: an exponent |log_decay| n of at most 32 tokens is rounded once and the exponential is good to two
      of 2^-23, 16 U32 with the factors; n tokens further away take n / 32 factors of half a step each;
  the pieces: a value of a type of unit u is carried in two (bf16's state operand in three) pieces, off by at most
      u^2 (u^3): 2 u^2 for the scores and the state of one term.
In fp16 the pieces are whole multiples of 2^-24 of values scaled to a largest of at least 2^14: 2^-39 of the
largest value each, which is not relative to the term: ``tiny``."""
from __future__ import annotations

import torch

from blockcheck import U32, unit


def powers(log_decay, n):
    """exp(log_decay n), [H] + n's shape; 0 where n < 0."""
    lg = log_decay.double().view((-1,) + (1,) * n.dim())
    x = torch.where(n == 0, 1.0, torch.exp(lg * n.clamp(min=1)))
    return torch.where(n < 0, 0.0, x)


def _run(q, k, v, D):
    """sum_j D_ij (q_i . k_j) v_j and the sum of its magnitudes."""
    kt = k.transpose(-1, -2)
    return ((q @ kt) * D) @ v, ((q.abs() @ kt.abs()) * D) @ v.abs()


def decay(q, k, v, log_decay, scale, state=None, lengths=None, g=None, g_last=None):
    """{name: (reference, bound)}: out, last and, if g is given, dq, dk, dv and dstate."""
    t = q.dtype
    u = unit(t)
    B, H, N, d = q.shape
    Hk, e = k.shape[1], v.shape[3]
    G = H // Hk
    L = torch.full((B,), N) if lengths is None else lengths.cpu().long().clamp(0, N)
    pos = torch.arange(N)
    live = (pos < L.view(B, 1))[:, None, :, None]
    clean = lambda x: torch.where(live, x.double(), 0.0)  # noqa: E731
    Q, K, V = clean(q), clean(k).repeat_interleave(G, 1), clean(v).repeat_interleave(G, 1)
    S0 = torch.zeros(B, H, d, e, dtype=torch.float64) if state is None else state.double()
    lg = log_decay.cpu()
    D = powers(lg, pos[:, None] - pos)[None]                          # [1, H, N, N]
    ahead = powers(lg, pos + 1)[None, :, :, None]                     # from the state in front
    left = powers(lg, L.view(B, 1) - 1 - pos).transpose(0, 1)[..., None]  # to the sequence's end
    whole = powers(lg, L).t()[..., None, None]
    T = lambda x: x.transpose(-1, -2)  # noqa: E731
    worst = lg.double().clamp(min=-200.0).abs().amax().item() if H else 0.0
    pieces = 0.0 if t == torch.float32 else 2 * u * u + 2.0 ** -22
    c = (max(d, e) + N + N / 16 + 64 + 16 + 32 * min(worst, 4.0)) * U32 + pieces

    def tiny(x, y, z, first):
        """fp16: the pieces' absolute steps in one run of the operator on (x, y, z)."""
        if t != torch.float16 or not N:
            return 0.0
        p = (x.abs() @ T(y.abs())).amax().item() * scale
        s = max(((T(y.abs()) * 1.0) @ z.abs()).amax().item(), first.abs().amax().item())
        return 2.0 ** -38 * (p * z.abs().amax().item() * 32 + s * x.abs().sum(-1).amax().item())

    def rounded(ref, mag, extra=0.0, unit_=u):
        err = c * mag + extra
        return ref, err + unit_ * (ref.abs() + err)

    a, m = _run(Q, K, V, D)
    out = scale * (a + ahead * (Q @ S0)) * live
    mag = scale * (m + ahead * (Q.abs() @ S0.abs()))
    res = {"out": rounded(out, mag, tiny(Q, K, V, S0))}
    last = whole * S0 + T(K * left) @ V
    res["last"] = rounded(last, whole * S0.abs() + T(K.abs() * left) @ V.abs(), 0.0, U32)
    if g is None:
        return res
    g = clean(g)
    R = torch.zeros_like(S0) if g_last is None else g_last.double()
    a, m = _run(g, V, K, D)
    dq = scale * (a + ahead * (g @ T(S0))) * live
    mq = scale * (m + ahead * (g.abs() @ T(S0.abs())))
    Db = T(D)
    a, m = _run(V, g, Q, Db)
    dk, mk = (scale * a + left * (V @ T(R))) * live, scale * m + left * (V.abs() @ T(R.abs()))
    a, m = _run(K, Q, g, Db)
    dv, mv = (scale * a + left * (K @ R)) * live, scale * m + left * (K.abs() @ R.abs())
    share = lambda x: x.reshape(B, Hk, G, N, x.shape[-1]).sum(2)  # noqa: E731
    res["dq"] = rounded(dq, mq, tiny(g, V, K, S0))
    res["dk"] = rounded(share(dk), share(mk), G * tiny(V, g, Q, R))
    res["dv"] = rounded(share(dv), share(mv), G * tiny(K, Q, g, R))
    ds = whole * R + scale * T(Q * ahead) @ g
    res["dstate"] = rounded(ds, whole * R.abs() + scale * T(Q.abs() * ahead) @ g.abs(), 0.0, U32)
    return res


def gated_norm(x, weight, residual, post_weight, gate, scale, eps, gy=None, gs=None):
    """{name: (reference, bound)}: y, sum and, if gy is given, dx, dres, dw, dwp and dgate.

    First-order error propagation through the formula: a mean over a row is off by c = 96 U32 of its terms'
    magnitudes (at most 64 terms in a thread and a tree of ten, and the root's), a product by U32."""
    u, W = unit(x.dtype), x.shape[-1]
    c = 96 * U32
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    X, r, w = x.double(), residual.double(), weight.double()
    if post_weight is not None:
        rx = 1.0 / (mean(X.square()) + eps).sqrt()
        m, wp = X * rx, post_weight.double()
        err_m = c * m.abs()
    else:
        rx, m, wp, err_m = torch.ones(()).double(), X, torch.ones(W).double(), 0.0 * X
    g = gate.double() if gate is not None else torch.ones(W).double()
    z = m * wp
    err_z = err_m * wp.abs() + U32 * z.abs()
    s = r + scale * g * z
    err_s = abs(scale) * g.abs() * (err_z + 3 * U32 * z.abs()) + U32 * s.abs()
    ms = mean(s.square()) + eps
    rs = 1.0 / ms.sqrt()
    rel = mean(s.abs() * err_s) / ms + c
    n = s * rs
    err_n = rs * err_s + (rel + U32) * n.abs()
    y = n * w
    err_y = err_n * w.abs() + U32 * y.abs()
    res = {"y": (y, err_y + u * (y.abs() + err_y)), "sum": (s, err_s + u * (s.abs() + err_s))}
    if gy is None:
        return res
    G = gy.double()
    gn = G * w
    dot = mean(gn * n)
    err_dot = mean(gn.abs() * err_n) + (c + 2 * U32) * mean((gn * n).abs())
    core = rs * (gn - n * dot)
    err_ds = rs * (err_n * dot.abs() + n.abs() * err_dot) + (rel + 4 * U32) * rs * (gn.abs() + (n * dot).abs())
    ds = core + (gs.double() if gs is not None else 0.0)
    err_ds = err_ds + U32 * ds.abs()
    rows = max(1, x.numel() // W)
    flat = lambda t: t.expand_as(X).reshape(-1, W)  # noqa: E731

    def summed(terms, err, like):
        """Over the dimensions that `like` has once."""
        if like.dim() == 1:
            total, e, size = flat(terms).sum(0), flat(err).sum(0), flat(terms.abs()).sum(0)
        else:
            dims = [i for i in range(like.dim()) if like.shape[i] == 1 and terms.shape[i] != 1]
            pick = lambda t: t.sum(dims, keepdim=True) if dims else t  # noqa: E731
            total, e, size = pick(terms), pick(err), pick(terms.abs())
        e = e + (rows + 8) * U32 * size
        return total, e + unit(like.dtype) * (total.abs() + e)

    dm = scale * g * wp * ds
    err_dm = (scale * g * wp).abs() * err_ds + 4 * U32 * dm.abs()
    if post_weight is not None:
        back = mean(dm * m)
        err_back = mean(err_dm * m.abs() + dm.abs() * err_m) + (c + 2 * U32) * mean((dm * m).abs())
        dx = rx * (dm - m * back)
        err_x = rx * (err_dm + err_m * back.abs() + m.abs() * err_back) + (c + 4 * U32) * rx * (dm.abs() + (m * back).abs())
        res["dwp"] = summed(scale * g * ds * m, abs(scale) * g.abs() * (err_ds * m.abs() + ds.abs() * err_m), post_weight)
    else:
        dx, err_x = dm, err_dm
    res["dx"] = (dx, err_x + u * (dx.abs() + err_x))
    res["dres"] = (ds, err_ds + u * (ds.abs() + err_ds))
    res["dw"] = summed(G * n, G.abs() * err_n, weight)
    if gate is not None:
        res["dgate"] = summed(scale * ds * z, abs(scale) * (err_ds * z.abs() + ds.abs() * err_z), gate)
    return res
