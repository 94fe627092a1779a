"""Plain restatement of the 4-bit KV cache (include/chatnet_cuda.h) in torch, 64 bits where it computes."""
from __future__ import annotations

import torch

X_MAX = 524032.0  # 8 * 65504


def positions_of(hd: int):
    """For value e of a row: (byte, shift) of its nibble."""
    nb = hd // 32
    e = torch.arange(hd)
    b, i, g = e // 32, (e % 32) // 8, e % 8
    return g * 2 * nb + 2 * b + i // 2, 4 * (i % 2)


def quantize(x):
    """fp32 [..., hd] -> levels uint8 [..., hd], scales fp16 [..., nb]."""
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-X_MAX, X_MAX)
    xb = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = xb.amin(-1), xb.amax(-1)
    d = (torch.where(-lo >= hi, lo, hi) * -0.125).half()
    f = d.double()[..., None]
    q = torch.where(f == 0, torch.full_like(f, 8.0), (xb.double() / f + 8.5).floor().clamp(0, 15))
    return q.to(torch.uint8).reshape(x.shape), d


def pack(levels):
    """levels [..., hd] -> bytes [..., hd / 2]."""
    hd = levels.shape[-1]
    byte, shift = positions_of(hd)
    out = torch.zeros(*levels.shape[:-1], hd // 2, dtype=torch.int32, device=levels.device)
    for s in (0, 4):
        at = (shift == s).nonzero()[:, 0]
        out[..., byte[at]] |= levels[..., at].int() << s
    return out.to(torch.uint8)


def unpack(quants):
    hd = quants.shape[-1] * 2
    byte, shift = positions_of(hd)
    return (quants[..., byte.to(quants.device)].int() >> shift.to(quants.device)) & 15


def values(quants, scales, dtype=torch.float64):
    lv = unpack(quants).to(dtype) - 8
    return (lv.reshape(*lv.shape[:-1], -1, 32) * scales.to(dtype)[..., None]).flatten(-2)


def rope_table(ctx_len: int, hd: int, base: float = 10000.0):
    inv = base ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    a = torch.arange(ctx_len, dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def rotate(x, table_rows, neox: bool):
    """x [n, heads, hd] by table rows [n, hd / 2, 2], in x's type, one rounding per product and sum."""
    c, s = table_rows[:, None, :, 0].to(x.dtype), table_rows[:, None, :, 1].to(x.dtype)
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if neox else (x[..., 0::2], x[..., 1::2])
    r0, r1 = a * c - b * s, a * s + b * c
    return torch.cat([r0, r1], -1) if neox else torch.stack([r0, r1], -1).flatten(-2)


def attend(q, k, v, pos: int, scale: float):
    """q [n, heads, hd], k / v [kv, ctx, hd] in 64 bits; token i sees positions 0..pos + i.
    Returns out [n, heads, hd] and, per (token, head), the largest |score| bound scale * sum |q k|."""
    n, heads, hd = q.shape
    mul = heads // k.shape[0]
    out = torch.empty_like(q)
    size = torch.empty(n, heads, dtype=q.dtype, device=q.device)
    seen = pos + n
    mask = torch.arange(seen, device=q.device)[None] > pos + torch.arange(n, device=q.device)[:, None]
    for h in range(heads):
        kk, vv = k[h // mul, :seen], v[h // mul, :seen]
        s = (q[:, h] @ kk.T * scale).masked_fill(mask, -torch.inf)
        out[:, h] = torch.softmax(s, -1) @ vv
        size[:, h] = (q[:, h].abs() @ kk.abs().T * scale).masked_fill(mask, 0).amax(-1)
    return out, size
