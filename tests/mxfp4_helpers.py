"""4-bit microscaled rows by their definition, in 64 bits on the CPU."""
from __future__ import annotations

import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantise(x):
    """(codes int64 [M, 32 blocks], scale bytes int64 [M, blocks]) of rows x."""
    x = x.detach().cpu().double()
    M, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % 32)).view(M, -1, 32)
    top = b.abs().amax(-1)
    bad = ~b.isfinite().all(-1)
    # the exponent bits of a float64 are the whole part of its logarithm (float32's smallest values are normal there)
    e = torch.where(top > 0, (top.view(torch.int64) >> 52) - 1023 - 2, -127).clamp(min=-127)
    e = torch.where(bad, 0, e)
    a = torch.where(bad[..., None], 0.0, b.abs()) / torch.exp2(e.double())[..., None]
    d = (a[..., None] - GRID).abs()
    near = d.amin(-1, keepdim=True)
    # of two codes as near, the even one
    code = torch.where(d == near, torch.arange(8) + 8 * (torch.arange(8) % 2), 99).amin(-1) % 8
    code = torch.where(a > 6, 7, code)
    code = torch.where(bad[..., None], 0, code + 8 * torch.signbit(b).long())
    return code.view(M, -1), torch.where(bad, 255, e + 127)


def pack(codes):
    """uint8 [M, 16 blocks]."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8)


def values(codes, scales, K):
    """float64 [M, K] that they stand for."""
    v = torch.where(codes >= 8, -GRID[codes % 8], GRID[codes % 8])
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    return (v.view(v.shape[0], -1, 32) * s[..., None]).reshape(v.shape[0], -1)[:, :K]


def random_rows(M, K, seed, lo=110, hi=135):
    """(codes, scale bytes) with every code, and scales of wide range; padding columns 0."""
    g = torch.Generator().manual_seed(seed)
    blocks = -(-K // 32)
    codes = torch.randint(0, 16, (M, 32 * blocks), generator=g)
    codes[:, K:] = 0
    return codes, torch.randint(lo, hi + 1, (M, blocks), generator=g)


def on_device(codes, scales, K):
    from llm_accelerator_b200 import mxfp4
    return mxfp4.Mxfp4.from_tensors(pack(codes).cuda(), scales.to(torch.uint8).cuda(), K)
