"""4-bit weights from the definition, in 64 bits: the oracle of ops.functional's mx4 ops."""
from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(w):
    """(codes [N, K/2], scales [N, K/32]) of w: the nearest grid point by comparing distances, ties to the even code."""
    n, k = w.shape
    x = w.double().cpu().view(n, k // 32, 32)
    a = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    frac, e = torch.frexp(torch.where(bad, torch.ones_like(a), a))  # a = frac 2^e, 0.5 <= frac < 1
    byte = (e - 1 - 2 + (frac > 0.875).int() + 127).clamp(2, 252)
    byte = torch.where(a == 0, torch.full_like(byte, 2), byte)
    mag = (x * torch.pow(torch.tensor(2.0, dtype=torch.float64), (127 - byte).double()).unsqueeze(-1)).abs().clamp(max=6.0)
    d = (mag.unsqueeze(-1) - GRID).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best                                  # one grid point, or two at a tie: the even code of them
    codes = torch.arange(8)
    pick = torch.where(near, torch.where(codes % 2 == 0, codes, codes + 100), 1000).amin(-1)
    pick = torch.where(pick >= 100, pick - 100, pick)
    code = (pick + 8 * torch.signbit(x).int()).to(torch.uint8)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).view(n, k)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    return (code[:, 0::2] | (code[:, 1::2] << 4)), byte.to(torch.uint8)


def values(codes, scales):
    """float64 [N, K]"""
    n = codes.shape[0]
    c = torch.stack((codes & 15, codes >> 4), -1).view(n, -1).cpu().long()
    v = GRID[c % 8] * (1.0 - 2.0 * (c // 8))
    byte = scales.cpu().long()
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), (byte - 127).double())
    s = torch.where(byte == 255, torch.full_like(s, float("nan")), s)
    return v * s.repeat_interleave(32, 1)
