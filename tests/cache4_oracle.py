"""Plain 64-bit form of the 4-bit rows' layout and rounding (tests only)."""
import math

import numpy as np
import torch

F64 = torch.float64
GROUP = 32
LARGEST = {torch.bfloat16: 3.3895313892515355e38, torch.float16: 65504.0}


def row_bytes(dim):
    return -(-(dim // 2 + dim // 8) // 16) * 16


def nearest(x, dtype):
    """fp64 values in the 16-bit type, rounded once (the type's own conversion goes by fp32): ties to even."""
    first = x.to(dtype)
    bits = first.view(torch.int16)
    best, err = first.clone(), (first.to(F64) - x).abs()
    for step in (-1, 1):
        near = (bits + step).view(dtype)
        far = (near.to(F64) - x).abs()
        better = (far < err) | ((far == err) & (near.view(torch.int16) & 1 == 0) & (best.view(torch.int16) & 1 == 1))
        better &= near.isfinite() & x.isfinite()
        best, err = torch.where(better, near, best), torch.where(better, far, err)
    return best


def quantise(x):
    """16-bit rows [..., D] on the CPU -> codes [..., groups, 32] int, scale and low [..., groups] in their type."""
    dtype = x.dtype
    groups = x.unflatten(-1, (-1, GROUP))
    wide = groups.to(F64)
    low, high = wide.amin(-1), wide.amax(-1)
    bad = ~wide.isfinite().all(-1)
    # The range in halves, and its part of 7.5, each rounded to fp32 as the format says.
    half = (0.5 * high.float() - 0.5 * low.float()).to(F64)
    scale = nearest((half / 7.5).float().to(F64), dtype)
    over = (15 * scale.to(F64) + low).float() > LARGEST[dtype]
    scale = torch.where(over, (scale.view(torch.int16) - 1).view(dtype), scale)
    scale = torch.where(scale.to(F64) < 2.0 ** -126, torch.zeros_like(scale), scale)
    away = (0.5 * wide - 0.5 * low[..., None]).float().to(F64) * 2
    step = scale.to(F64)[..., None]
    quotient = np.asarray(torch.where(step > 0, away / torch.where(step > 0, step, 1.0), 0.0))
    codes = torch.from_numpy(np.rint(np.nan_to_num(quotient, nan=0.0, posinf=0.0, neginf=0.0))).clamp(0, 15).long()
    # A quotient that fp64 rounded onto a border: compare exactly.
    for c in (-1, 0):
        border = (codes + c).to(F64) + 0.5
        at = away == border * step
        codes = torch.where(at & (step > 0), (codes + c) + (codes + c) % 2, codes).clamp(0, 15)
    nan = torch.full_like(scale, math.nan)
    codes = torch.where(bad[..., None], 0, codes)
    return codes, torch.where(bad, nan, scale), torch.where(bad, nan, low.to(dtype))


def values(codes, scale, low):
    dtype = scale.dtype
    return nearest(codes.to(F64) * scale.to(F64)[..., None] + low.to(F64)[..., None], dtype).flatten(-2)


def pack(codes, scale, low):
    """Cache rows uint8 [..., bytes] (what fills them up: zeros)."""
    dim = codes.shape[-2] * GROUP
    out = np.zeros((*codes.shape[:-2], row_bytes(dim)), np.uint8)
    flat = codes.flatten(-2).numpy()
    for d in range(dim):
        w, r = divmod(d, 8)
        bit = 16 * (r % 2) + 4 * (r // 2)
        out[..., 4 * w + bit // 8] |= (flat[..., d] << (bit % 8)).astype(np.uint8)
    pairs = torch.stack([scale, low], -1).flatten(-2).view(torch.int16).numpy().view(np.uint8)
    out[..., dim // 2:dim // 2 + dim // 8] = pairs
    return torch.from_numpy(out)


def unpack(rows, dim, dtype):
    """16-bit rows [..., D] of cache rows (uint8 on the CPU)."""
    raw = rows.numpy()
    codes = np.zeros((*rows.shape[:-1], dim), np.int64)
    for d in range(dim):
        w, r = divmod(d, 8)
        bit = 16 * (r % 2) + 4 * (r // 2)
        codes[..., d] = raw[..., 4 * w + bit // 8] >> (bit % 8) & 15
    pairs = torch.from_numpy(np.ascontiguousarray(raw[..., dim // 2:dim // 2 + dim // 8])).view(dtype).unflatten(-1, (-1, 2))
    return values(torch.from_numpy(codes).unflatten(-1, (-1, GROUP)), pairs[..., 0].clone(), pairs[..., 1].clone())


def same(a, b):
    """Equal values, NaN where the other has NaN (the sign of zero aside)."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())
