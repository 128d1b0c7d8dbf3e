"""The paged cache restated plainly (torch, CPU, 64 bits) for its tests: packing, quantising, append,
attention and the error bounds that follow from the roundings."""

from __future__ import annotations

import math

import torch

from gemma4_posttrain_jax_amd import _lib
from gemma4_posttrain_jax_amd.kvcache import PagedLayerCache, new_paged_layer

U32 = 2.0 ** -24  # half a step of f32, relative
U_BF16 = torch.finfo(torch.bfloat16).eps / 2
U_E4M3 = torch.finfo(torch.float8_e4m3fn).eps / 2
ALL_FLAGS = (_lib.G4_APPEND_NORM_Q | _lib.G4_APPEND_ROPE_Q | _lib.G4_APPEND_NORM_K | _lib.G4_APPEND_ROPE_K
             | _lib.G4_APPEND_NORM_V)


def to_e4m3(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Vectors ``[..., D]`` -> (f64 e4m3 values before the scale, integer exponents ``[...]``)."""

    x = x.double()
    top = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(dim=-1)
    frac, exp = torch.frexp(top)
    e = torch.where(frac <= 0.875, exp - 9, exp - 8)
    e = torch.where(top > 0, e, torch.full_like(e, -100)).clamp(-100, 120)
    y = x * torch.exp2(-e.double())[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    y = torch.where(x.isfinite(), torch.round(y / step) * step, torch.full_like(y, math.nan))
    return y, e


def dequantised(x: torch.Tensor) -> torch.Tensor:
    y, e = to_e4m3(x)
    return y * torch.exp2(e.double())[..., None]


def slots_of(layer: PagedLayerCache) -> tuple[torch.Tensor, torch.Tensor]:
    """f64 keys and values ``[P, H, page, D]`` of a device cache, element by element from the layout's formula."""

    P, H, ps, D, f8 = layer.num_pages, layer.kv_heads, layer.page_size, layer.head_dim, layer.e4m3
    kr = 64 if f8 else 32
    s, d = torch.arange(ps)[:, None], torch.arange(D)[None, :]
    r = s % 32
    kidx = (((s // 32 * (D // kr) + d // kr) * 2 + r // 4 % 2) * 16 + r // 8 * 4 + r % 4) * kr + d % kr
    vidx = (s // 8 * D + d) * 8 + s % 8
    out = []
    for t, idx, scale in ((layer.key, kidx, layer.key_scale), (layer.value, vidx, layer.value_scale)):
        x = t.cpu().double().reshape(P, H, -1)[:, :, idx.reshape(-1)].view(P, H, ps, D)
        if f8:
            x = x * torch.exp2(scale.cpu().view(torch.uint8).double() - 127)[..., None]
        out.append(x)
    return out[0], out[1]


def filled(P: int, H: int, D: int, ps: int, e4m3: bool, k: torch.Tensor, v: torch.Tensor, device) -> PagedLayerCache:
    """A device cache holding slot-major ``k`` / ``v [P, H, ps, D]`` (quantised where e4m3)."""

    layer = new_paged_layer(P, H, D, ps, e4m3=e4m3, device=device)
    kr = 64 if e4m3 else 32
    parts = []
    for x in (k, v):
        if e4m3:
            y, e = to_e4m3(x)
            parts.append((y.float().to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)))
        else:
            parts.append((x.to(torch.bfloat16), None))
    kt = parts[0][0].view(P, H, ps // 32, 4, 2, 4, D // kr, kr).permute(0, 1, 2, 6, 4, 3, 5, 7).reshape(layer.key.shape)
    vt = parts[1][0].view(P, H, ps // 8, 8, D).transpose(3, 4).reshape(layer.value.shape)
    raw = (lambda t: t.view(torch.uint8)) if e4m3 else (lambda t: t)
    raw(layer.key).copy_(kt)
    raw(layer.value).copy_(vt)
    if e4m3:
        layer.key_scale.view(torch.uint8).copy_(parts[0][1])
        layer.value_scale.view(torch.uint8).copy_(parts[1][1])
    return layer


def attention(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths, q: torch.Tensor,
              window: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The attention of slot-major f64 pages in 64 bits, and how far a right kernel's bf16 result may be off
    ``[B, H, R, D]``: the scores' and sums' f32 errors, half a bf16 step of each probability and of the result."""

    P, H, ps, D = k.shape
    B, R = q.shape[0], q.shape[2]
    out = torch.zeros((B, H, R, D), dtype=torch.float64)
    bound = torch.zeros_like(out)
    q = q.cpu().double()
    for b in range(B):
        n = min(int(lengths[b]), table.shape[1] * ps)
        pos = [p for p in range(max(0, n - window) if window else 0, n) if 0 <= int(table[b, p // ps]) < P]
        if not pos:
            continue
        page = torch.tensor([int(table[b, p // ps]) for p in pos])
        slot = torch.tensor([p % ps for p in pos])
        kk, vv = k[page, :, slot], v[page, :, slot]  # [n, H, D]
        for h in range(H):
            s = q[b, h] @ kk[:, h].T
            top = s.amax(dim=-1, keepdim=True)
            w = torch.exp(s - top)
            w = w / w.sum(dim=-1, keepdim=True)
            out[b, h] = w @ vv[:, h]
            mass = w @ vv[:, h].abs()
            # |ds| <= (D + 2) u sum |q k| (products, sums and the scale), exp's argument and result 4 u (1 + |s - max|);
            # the weights' relative error is twice the worst of them (numerator and denominator), and n u of the sum
            ds = (D + 2) * U32 * (q[b, h].abs() @ kk[:, h].abs().T) + 4 * U32 * (1 + (s - top).abs().clamp(max=100))
            rel = 2 * ds.amax(dim=-1, keepdim=True) + (2 * len(pos) + 16) * U32
            bound[b, h] = (U_BF16 + rel) * mass * (1 + U_BF16) + U_BF16 * out[b, h].abs() + 1e-37
    return out, bound


def prepared(x: torch.Tensor, w: torch.Tensor | None, norm: bool, rope, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm and rotation of ``x [..., D]`` in 64 bits and the f32 error a right kernel may have before its
    rounding: D / 64 + 12 roundings of the norm (the sum of squares counts half, it goes through a root) and 3
    of the rotation, each relative to the terms."""

    x = x.double()
    D = x.shape[-1]
    if norm:
        x = x / (x.square().mean(dim=-1, keepdim=True) + eps).sqrt()
        if w is not None:
            x = x * w.double()
    size = x.abs()
    if rope is not None:
        cos, sin = (t.double() for t in rope)
        half = D // 2
        x = x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin
        size = size * cos.abs() + torch.cat([size[..., half:], size[..., :half]], dim=-1) * sin.abs()
    return x, (D // 64 + 15) * U32 * size * (1.0 if norm or rope is not None else 0.0)
