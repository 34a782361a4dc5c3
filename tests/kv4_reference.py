"""The 4-bit cache and its operators from their definitions, in 64 bits, for the tests."""
import math

import torch


def pack(codes: torch.Tensor, is_key: bool) -> torch.Tensor:
    """Codes [..., D] in [-8, 7] as bytes [..., D / 2], dim by dim."""
    dim = codes.shape[-1]
    out = torch.zeros(*codes.shape[:-1], dim // 2, dtype=torch.int64, device=codes.device)
    for d in range(dim):
        if is_key:
            byte, low = d % 32 // 8 * (dim // 8) + d // 32 * 4 + d % 8 // 2, d % 2 == 0
        else:
            byte, low = d % 32 // 4 * (dim // 16) + d // 32 * 2 + d % 4 // 2, d % 2 == 0
        out[..., byte] += (codes[..., d].long() + 8) * (1 if low else 16)
    return out.to(torch.uint8)


def unpack(rows: torch.Tensor, is_key: bool) -> torch.Tensor:
    """Bytes [..., D / 2] as codes [..., D]."""
    dim = 2 * rows.shape[-1]
    out = torch.empty(*rows.shape[:-1], dim, dtype=torch.float64, device=rows.device)
    for d in range(dim):
        if is_key:
            byte = d % 32 // 8 * (dim // 8) + d // 32 * 4 + d % 8 // 2
        else:
            byte = d % 32 // 4 * (dim // 16) + d // 32 * 2 + d % 4 // 2
        nibble = rows[..., byte].long()
        out[..., d] = (nibble // 16 if d % 2 else nibble % 16).double() - 8
    return out


def quantise(x: torch.Tensor):
    """bf16 rows [..., D] -> codes [..., D] and scales [..., D / 32] (bf16)."""
    groups = x.double().unflatten(-1, (-1, 32))
    largest = groups.abs().amax(-1)
    finite = groups.isfinite().all(-1)
    scale = (largest / 7).to(torch.bfloat16)
    scale = torch.where(largest < 2.0 ** -100, torch.zeros_like(scale), scale)
    quotient = groups.abs() / scale.double().unsqueeze(-1)
    code = torch.ceil(quotient - 0.5).clamp(0, 7) * groups.sign()
    dead = (~finite | (scale == 0)).unsqueeze(-1)
    code = torch.where(dead, torch.zeros_like(code), code)
    scale = torch.where(finite, scale, torch.full_like(scale, float("nan")))
    return code.flatten(-2), scale


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return (codes.unflatten(-1, (-1, 32)) * scales.double().unsqueeze(-1)).flatten(-2)


def axis_of_pair(sections, interleaved):
    if not interleaved:
        return [a for a, share in enumerate(sections) for _ in range(share)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def rope_axes(x: torch.Tensor, n_heads, dim, positions, sections, theta, interleaved=False, inverse=False):
    out = x.double().clone()
    pos = positions.double().reshape(len(sections), -1)
    heads = out[:, :n_heads * dim].clone().reshape(x.shape[0], n_heads, dim)
    for i, a in enumerate(axis_of_pair(sections, interleaved)):
        angle = pos[a] * theta ** (-2.0 * i / dim) * (-1 if inverse else 1)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        u, v = heads[:, :, i].clone(), heads[:, :, i + dim // 2].clone()
        heads[:, :, i] = u * c - v * s
        heads[:, :, i + dim // 2] = v * c + u * s
    out[:, :n_heads * dim] = heads.reshape(x.shape[0], -1)
    return out


def attend(q, k, v):
    """q [g, D], k, v [n, D] in 64 bits -> (out [g, D], p [g, n], sum_k p |v| [g, D], largest sum_d |q k| / sqrt(D))."""
    scale = 1 / math.sqrt(q.shape[1])
    p = torch.softmax(q @ k.t() * scale, dim=-1)
    return p @ v, p, p @ v.abs(), float((q.abs() @ k.abs().t()).max() * scale)


def evict_order(weights, n, keep, recent):
    """Slots that stay of one head's `n`, ascending."""
    if n <= keep:
        return list(range(n))
    old = n - recent
    w = [math.inf if math.isnan(x) else x for x in weights[:old].tolist()]
    heavy = sorted(range(old), key=lambda i: (-w[i], i))[:keep - recent]
    return sorted(heavy) + list(range(old, n))
