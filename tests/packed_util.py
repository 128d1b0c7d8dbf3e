"""Attention of packed prompts restated plainly (torch, CPU, 64 bits), with the error bound that follows from a
kernel's roundings."""

from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24  # half a step of f32, relative
U_BF16 = torch.finfo(torch.bfloat16).eps / 2


def packed_reference(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens, window: int) -> tuple[torch.Tensor, torch.Tensor]:
    """q ``[T, H, R, D]``, k / v ``[T, H, D]`` of sequences of ``lens`` tokens: the attention in 64 bits and how far a
    right kernel's bf16 result may be off."""

    T, H, R, D = q.shape
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros((T, H, R, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    a = 0
    for n in lens:
        i = torch.arange(n)
        hidden = i[None, :] > i[:, None]
        if window:
            hidden |= i[None, :] <= i[:, None] - window
        for h in range(H):
            for r in range(R if n else 0):
                s = (q[a:a + n, h, r] @ k[a:a + n, h].T).masked_fill(hidden, -math.inf)
                size = (q[a:a + n, h, r].abs() @ k[a:a + n, h].abs().T).masked_fill(hidden, 0.0)
                top = s.amax(dim=-1, keepdim=True)
                w = torch.softmax(s, dim=-1)
                out[a:a + n, h, r] = w @ v[a:a + n, h]
                mass = w @ v[a:a + n, h].abs()
                # |ds| <= (D + 2) u sum |q k|; exp2's argument s log2(e) - m log2(e) is rounded relative to |s| and |m|
                # and its result by 2 u, 4 u (1 + |s| + |m|) in all; the weights' relative error is twice the worst of them
                # (numerator and denominator) and (n + 16) u of the sums
                ds = (D + 2) * U32 * size + 4 * U32 * (1 + s.masked_fill(hidden, 0.0).abs() + top.abs())
                rel = 2 * ds.amax(dim=-1, keepdim=True) + (2 * n + 16) * U32
                bound[a:a + n, h, r] = (U_BF16 + rel) * mass * (1 + U_BF16) + U_BF16 * out[a:a + n, h, r].abs() + 1e-37
        a += n
    return out, bound
