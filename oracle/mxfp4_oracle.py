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


def digits(v: torch.Tensor, count: int) -> list[torch.Tensor]:
    """The rows of ``v`` as ``count`` packed rows each, whose sum they are but for what is left: every
    one is the quantised remainder of those before it.  float64 values, the first digits first."""
    left, found = v.double(), []
    for _ in range(count):
        found.append(dequantise(*quantise(left), v.shape[1]))
        left = left - found[-1]
    return found


def digit_bound(v):
    """Error of single elements that were taken apart into 12 packed rows and added up in FP32.  A row leaves at most a quarter of
    the block's largest remainder (between 4 and 8 scales: rounding leaves up to 1, saturation up to 2 of 8), so after
    12 of them 2^-24 of the block's largest element T; the sum from the smallest row on rounds its partial sums, which are
    at most T/4^d plus what is left, and at last the element: 2^-24 (|v| + T/3).  2^-20 of slack for products of these.
    Rows end at the smallest scale's half code: 2^-129."""
    blocks = -(-v.shape[1] // 32)
    top = torch.nn.functional.pad(v.abs(), (0, blocks * 32 - v.shape[1])).view(v.shape[0], blocks, 32).amax(-1)
    top = top.repeat_interleave(32, 1)[:, :v.shape[1]]
    return (2.0 ** -24 * top + 2.0 ** -24 * (v.abs() + top / 3)) * (1 + 2.0 ** -20) + 2.0 ** -129


def digit_cases(rows, n, device="cpu"):
    """Vectors that take many digits: normal ones of very different sizes, all ones in the mantissa (every row saturates and
    leaves a quarter), those beside small elements, one element far below its block's largest."""
    gen = torch.Generator(device=device).manual_seed(rows * n)
    v = torch.randn(rows, n, generator=gen, device=device) * torch.exp2(torch.randint(-30, 30, (rows, n), generator=gen, device=device).float())
    ones = 1 - 2.0 ** -24
    v[0] = ones * torch.exp2((torch.arange(n, device=device) // 32 % 7 - 3).float())
    v[-1] = torch.randn(n, generator=gen, device=device)
    v[-1, ::2] = -ones
    v[1, 5::32], v[1, 6::32] = ones, 1.25 * 2.0 ** -20
    return v


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
