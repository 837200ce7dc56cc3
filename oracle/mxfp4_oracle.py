"""Plain 64-bit restatement of the microscaled 4-bit operators and of rotary positions, in
torch so that it runs where its inputs are.  Test infrastructure only."""
from __future__ import annotations

import torch

BLOCK = 32
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exponent(x: torch.Tensor) -> torch.Tensor:
    """floor(log2 |x|) of float64 values (FP32 subnormals are float64 normals)."""
    return ((x.view(torch.int64) >> 52) & 2047) - 1023


def quantise(x: torch.Tensor):
    """(codes uint8 (rows, 16 * blocks), scales uint8 (rows, blocks)) of a 2-D tensor."""
    rows, n = x.shape
    blocks = -(-n // BLOCK)
    d = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=x.device)
    d[:, :n] = x.double()
    d = d.view(rows, blocks, BLOCK)
    top = d.abs().amax(-1)
    fine = torch.isfinite(d).all(-1)
    e = (_exponent(torch.where(fine, top, torch.ones_like(top))) - 2).clamp(-127, 127)
    y = torch.where(fine[..., None], d, torch.zeros_like(d)) * torch.exp2(-e.double())[..., None]
    # nearest value; of two equally near ones that with the even code
    a = y.abs().clamp(max=6.0)
    grid = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    dist = (a[..., None] - grid).abs()
    best = dist.amin(-1, keepdim=True)
    code = torch.arange(8, device=x.device)
    cost = torch.where(dist == best, code % 2, torch.full_like(code, 2))
    code = cost.argmin(-1)
    code = code + 8 * torch.signbit(y).long()
    code = torch.where(fine[..., None], code, torch.zeros_like(code)).view(rows, -1).to(torch.uint8)
    scales = torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def dequantise(codes: torch.Tensor, scales: torch.Tensor, n: int) -> torch.Tensor:
    """float64 values (rows, n); scale byte 255 is NaN."""
    rows = codes.shape[0]
    grid = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(rows, -1, BLOCK).long()
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (grid[c] * s[..., None]).reshape(rows, -1)[:, :n]


def rotate(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, layout: str, scale: float = 1.0):
    """float64 (tokens, heads, dim), the rotation written element by element."""
    y = x.double().clone()
    half = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = torch.cos(angle), torch.sin(angle)
    for i in range(half):
        a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a] = scale * (xa * c[:, None, i] - xb * s[:, None, i])
        y[..., b] = scale * (xa * s[:, None, i] + xb * c[:, None, i])
    return y
