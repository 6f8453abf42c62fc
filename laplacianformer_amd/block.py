"""Operators of a transformer block around the attention (no counterpart in the
reference, which ships its two operators only): the norm with the residual's
addition, rotary positions on the token grid, exact softmax attention, and
``AttentionBlock``, which joins them with either attention.

All run on hand-written HIP kernels in float32, float16 and bfloat16 (float64 and CPU
tensors are refused), take strided inputs where the last dimension's elements are
adjacent, and record into a HIP graph. Results do not depend on the launch: the same
call gives the same bits. Gradients are of first order (no create_graph); forward-mode tangents are refused.
"""
from __future__ import annotations

import math
from typing import Sequence

import torch

from ._lib import ext
from .attention import laplacian_attention


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """Root-mean-square norm over the last dimension, with the residual's addition.

    ``sum = x + residual``, ``y = sum / sqrt(mean(sum^2) + eps) * weight`` (statistics of the
    float32 sum). Returns ``(y, sum)`` in x's type, which is the residual's too, or ``y`` alone without a residual.
    ``weight`` has x's type or float32; the last dimension is at most 16384. With autograd, which keeps x (and
    in 16-bit types the residual, for the unrounded sum; in float32 the sum in their place) for the backward.
    """
    out = ext().AddRmsNorm(x, weight, residual, eps)
    return out[0] if residual is None else tuple(out)


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """add_rms_norm with y in 8 bits for a scaled matrix product, without gradients.

    Returns ``(y8, scale)`` or ``(y8, scale, sum)``: y8 is float8_e4m3fn, scale float32
    ``[..., 1]`` with ``y = y8 * scale`` and ``scale = max|y| / 448`` over each row (1 for a
    row of zeros or of values below 2^-117, which become zeros).
    """
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    y, scale, total = ext().AddRmsNorm_fp8(x, weight, residual, eps)
    return (y, scale) if residual is None else (y, scale, total)


def rotary_sections(head_dim: int, axes: int) -> list[int]:
    """head_dim // 2 channel pairs dealt evenly to the axes; the first takes the remainder."""
    n = head_dim // 2 // axes
    return [head_dim // 2 - n * (axes - 1)] + [n] * (axes - 1)


def grid_positions(grid: Sequence[int], device=None, start: Sequence[int] | None = None) -> torch.Tensor:
    """int32 ``[axes, tokens]``: the coordinates of a row-major token grid (height x width,
    time x height x width, ...), axis a counted from ``start[a]`` (default 0)."""
    if start is not None and len(start) != len(grid):
        raise ValueError(f"a grid of {len(grid)} axes takes as many starts, not {len(start)}")
    axes = [torch.arange(s, s + n, dtype=torch.int32, device=device)
            for n, s in zip(grid, start if start is not None else [0] * len(grid))]
    return torch.stack([a.reshape(-1) for a in torch.meshgrid(*axes, indexing="ij")])


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, sections: Sequence[int],
           base: float = 10000.0, interleaved: bool = False):
    """Rotary positions over several axes, for q ``[B, H, N, d]`` and k ``[B, Hk, N, d]`` (or None).

    ``positions`` is int32 or int64, ``[axes, N]`` or ``[axes, B, N]``; ``sections[a]`` channel
    pairs belong to axis a, in order, and pair j of axis a turns by ``position_a * base **
    (-j / sections[a])``, with the angle in fp32 accuracy at any position (base >= 1; below, where
    ``|position| / base`` is at most 2^78). Pair p is channels ``(p, p + pairs)``, or
    ``(2 p, 2 p + 1)`` if ``interleaved``; channels behind the pairs are copied. At most 128
    pairs. Returns ``(q', k')``. With autograd.
    """
    return tuple(ext().Rotary(q, k, positions, sections, base, interleaved))


def softmax_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: torch.Tensor | None = None,
                      causal: bool = False, k_lengths: torch.Tensor | None = None,
                      q_lengths: torch.Tensor | None = None, q_starts: torch.Tensor | None = None,
                      scale: float | None = None) -> torch.Tensor:
    """Exact softmax attention of q ``[B, H, N, d]`` over k, v ``[B, Hk, M, d]`` -> ``[B, H, N, d]``.

    H is a multiple of Hk: query head h reads key head ``h // (H // Hk)``. d is at most 128.
    ``mask`` broadcasts to ``[B, H, N, M]``: bool (True attends) or an additive float32, float16
    or bfloat16 tensor (-inf removes the key), without a gradient. ``k_lengths``, ``q_lengths``
    and ``q_starts`` are int32 ``[B]``: keys from ``k_lengths[b]`` on take no part and are not
    read, queries from ``q_lengths[b]`` on are not read and give 0. ``causal``: query n sees the
    keys up to ``q_starts[b] + n`` (default: ``M - N``, the queries are the last tokens); for new
    tokens over a cache filled to uneven lengths, ``q_starts = k_lengths - N``. ``scale``
    (positive) defaults to ``1 / sqrt(d)``.

    A query that nothing is left for gives 0. Keys that ``k_lengths``, or a mask that is broadcast
    over heads and queries, takes out may hold anything, as may queries from ``q_lengths[b]`` on;
    elsewhere masked keys and values (and queries and output gradients) have to be finite, as a probability of
    0 is multiplied by them. 16-bit types round the
    probabilities to that type in front of the product with v. With autograd, which keeps, beside the
    inputs, the output and a number per row (two with an additive mask), in 16-bit types what the
    output's rounding took off: a second tensor of its size.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.shape[-1] else 1.0
    return ext().SoftmaxAttention(q, k, v, mask, causal, k_lengths, q_lengths, q_starts, scale)


class AttentionBlock(torch.nn.Module):
    """The attention half of a pre-norm transformer block on a token grid.

    ``forward(x, residual)`` adds and norms (add_rms_norm), projects to q, k and v, turns q
    and k by their tokens' grid positions (rotary), attends, and projects back. It returns
    ``(out, sum)``: the next block's ``(x, residual)``, also under autocast, where out is of 16 bits and the
    sum stays float32 (x and residual of different types are widened to the wider one). ``attention`` is "softmax"
    (softmax_attention, ``kv_heads`` key heads shared by ``heads`` query heads) or
    "laplacian" (laplacian_attention with ``pool`` and ``iters``, one key head per query head, a grid of two
    axes). Caches of keys and the 8-bit norm are for callers of the functions: the block takes neither.
    """

    def __init__(self, dim: int, heads: int, kv_heads: int | None = None, attention: str = "softmax",
                 positions: bool = True, base: float = 10000.0, causal: bool = False, pool: int = 4, iters: int = 10,
                 eps: float = 1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if dim % heads or heads % kv_heads:
            raise ValueError("dim must be divisible by heads, and heads by kv_heads")
        if attention not in ("softmax", "laplacian"):
            raise ValueError("attention must be 'softmax' or 'laplacian'")
        if attention == "laplacian" and (causal or kv_heads != heads):
            raise ValueError("laplacian attention is not causal and shares no key heads")
        self.heads, self.kv_heads, self.attention, self.causal = heads, kv_heads, attention, causal
        self.positions, self.base, self.pool, self.iters, self.eps = positions, base, pool, iters, eps
        d = dim // heads
        self.weight = torch.nn.Parameter(torch.ones(dim))
        self.qkv = torch.nn.Linear(dim, (heads + 2 * kv_heads) * d)
        self.proj = torch.nn.Linear(dim, dim)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, grid: Sequence[int] | None = None,
                positions: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None):
        """x, residual [B, N, dim]. ``grid``: the token grid, ``positions`` [axes, N] or [axes, B, N] in its
        place. With neither, the tokens of a causal block, or of a batch with ``lengths``, are sequences: one axis,
        whatever N is, so that a prefix has the same positions; else N has to be a square's.
        ``mask`` and ``lengths`` (int32 [B], the tokens that each sequence has) go to softmax_attention."""
        B, N, C = x.shape
        d = C // self.heads
        if self.attention == "laplacian" and (mask is not None or lengths is not None):
            raise ValueError("laplacian attention takes neither mask nor lengths")
        if grid is None and (self.attention == "laplacian" or self.positions and positions is None):
            side = math.isqrt(N)
            if self.causal or lengths is not None:
                grid = (N,)
            elif side * side == N:
                grid = (side, side)
            else:
                raise ValueError(f"N={N} tokens are no square: their grid is missing")
        if grid is not None and math.prod(grid) != N:
            raise ValueError(f"token grid {tuple(grid)} does not match N={N}")
        if self.attention == "laplacian" and (len(grid) != 2 or any(n % self.pool for n in grid)):
            raise ValueError(f"laplacian attention pools a grid of two axes by {self.pool}, not {tuple(grid)}")
        if residual is None:
            y, total = add_rms_norm(x, self.weight, eps=self.eps), x
        else:
            if x.dtype != residual.dtype:  # under autocast: a 16-bit projection beside the fp32 stream, which stays fp32
                wide = torch.promote_types(x.dtype, residual.dtype)
                x, residual = x.to(wide), residual.to(wide)
            y, total = add_rms_norm(x, self.weight, residual, eps=self.eps)
        qkv = self.qkv(y).view(B, N, self.heads + 2 * self.kv_heads, d).transpose(1, 2)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        if self.positions:
            if positions is None:
                positions = grid_positions(grid, x.device)
            q, k = rotary(q, k, positions, rotary_sections(d, positions.shape[0]), self.base)
        if self.attention == "softmax":
            o = softmax_attention(q, k, v, mask=mask, causal=self.causal, k_lengths=lengths, q_lengths=lengths)
        else:
            o = laplacian_attention(q.contiguous(), k.contiguous(), v.contiguous(), grid=tuple(grid), pool=self.pool,
                                    iters=self.iters)
        return self.proj(o.transpose(1, 2).reshape(B, N, C)), total
