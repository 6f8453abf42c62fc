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
