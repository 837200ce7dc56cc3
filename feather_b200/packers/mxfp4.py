"""Microscaled 4-bit packers: 32 consecutive elements of the last dimension share a
power-of-two scale, each element is an E2M1 code (0, .5, 1, 1.5, 2, 3, 4, 6 and
their negatives).  No counterpart in the reference, whose packers stop at 8 bits
(feather/packers/fp8.py).

A row of ``n`` elements is ``ceil(n / 32)`` blocks: 16 bytes of codes (the even
element in the low half of its byte; a short last block is filled up with zero
codes) and one scale byte ``2 ** (byte - 127)`` each, 255 standing for NaN.  This is
the layout of the OCP microscaling formats.
"""
from __future__ import annotations

import torch

from .. import _lib
from .fp8 import _require_cuda

__all__ = ["pack_mxfp4_tensor", "unpack_mxfp4_tensor"]

BLOCK = 32
BLOCK_BYTES = 16
DTYPE_IDS = {torch.float16: _lib.SRC_F16, torch.float32: _lib.SRC_F32, torch.bfloat16: _lib.SRC_BF16}
# bytes, and torch's own names for them where it has them
_CODE_DTYPES = tuple(d for d in (torch.uint8, getattr(torch, "float4_e2m1fn_x2", None)) if d is not None)
_SCALE_DTYPES = tuple(d for d in (torch.uint8, getattr(torch, "float8_e8m0fnu", None)) if d is not None)


def blocks_of(n: int) -> int:
    return -(-n // BLOCK)


def dtype_id(dtype: torch.dtype, name: str) -> int:
    found = DTYPE_IDS.get(dtype)
    if found is None:
        raise TypeError(f"{name} must be float16, bfloat16 or float32, got {dtype}")
    return found


def as_packed(codes: torch.Tensor, scales: torch.Tensor, rows: int, n: int, name: str) -> int:
    """Validate a packed operand of ``rows`` rows of ``n`` elements -- CUDA, contiguous, bytes,
    one device, long enough, rows of the right length -- and return its device's index.  (The library checks that codes
    are 16-byte aligned.)"""
    blocks = (n + BLOCK - 1) // BLOCK
    if isinstance(codes, torch.Tensor) and isinstance(scales, torch.Tensor):
        idx = codes.get_device()
        if (idx >= 0 and scales.get_device() == idx
                and codes.dtype in _CODE_DTYPES and scales.dtype in _SCALE_DTYPES
                and codes.is_contiguous() and scales.is_contiguous()
                and codes.numel() >= rows * blocks * BLOCK_BYTES and scales.numel() >= rows * blocks
                and (blocks == 0 or not (codes.shape[-1] % (blocks * BLOCK_BYTES) or scales.shape[-1] % blocks))):
            return idx
    for t, kind, dtypes, need in ((codes, "codes", _CODE_DTYPES, rows * blocks * BLOCK_BYTES),
                                  (scales, "scales", _SCALE_DTYPES, rows * blocks)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}_{kind} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name}_{kind} must be a CUDA tensor: feather_b200 has no CPU path")
        if t.dtype not in dtypes:
            raise ValueError(f"{name}_{kind} must hold packed bytes (uint8), got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name}_{kind} must be contiguous")
        if t.numel() < need:
            raise ValueError(f"{name}_{kind} holds {t.numel()} bytes, {rows}x{n} needs {need}")
        if blocks and t.shape[-1] % (need // rows if rows else 1):
            raise ValueError(f"{name}_{kind} of shape {tuple(t.shape)} does not have rows of {need // rows} bytes (n={n})")
    raise ValueError(f"{name}_codes and {name}_scales must be on the same device")


# The calls below launch on the current stream of their operands' device; with another device
# current they make it current and start over, so that the usual case pays one comparison.
current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _lib.current_stream_ptr)


def pack_mxfp4_tensor(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantise a float16/bfloat16/float32 tensor of shape ``(..., n)`` along its last dimension.

    Returns ``(codes, scales)``, uint8 of shapes ``(..., 16 * ceil(n / 32))`` and
    ``(..., ceil(n / 32))``, on ``x``'s device (a CPU tensor is packed on the current CUDA
    device, as by ``pack_fp8_tensor``).  The scale of a block is ``2 ** (floor(log2 max|x|) - 2)``,
    codes are rounded to nearest even and saturate at 6 scales; a block with an infinity or a
    NaN decodes to NaN throughout."""
    if not isinstance(x, torch.Tensor):
        raise TypeError("pack_mxfp4_tensor expects a torch.Tensor")
    src = dtype_id(x.dtype, "x")
    if x.dim() == 0:
        raise ValueError("x needs a last dimension to be packed along")
    if not x.is_cuda:
        _require_cuda()
        codes, scales = pack_mxfp4_tensor(x.cuda())
        return codes.cpu(), scales.cpu()
    lib = _lib.load()
    device = x.device
    idx = device.index
    if current_device() != idx:
        with torch.cuda.device(idx):
            return pack_mxfp4_tensor(x)
    if not x.is_contiguous():
        x = x.contiguous()
    *lead, n = x.shape
    blocks = (n + BLOCK - 1) // BLOCK
    codes = torch.empty(*lead, blocks * BLOCK_BYTES, dtype=torch.uint8, device=device)
    scales = torch.empty(*lead, blocks, dtype=torch.uint8, device=device)
    total = x.numel()
    if total:
        status = lib.feather_encode_mxfp4(x.data_ptr(), src, codes.data_ptr(), scales.data_ptr(), total // n, n,
                                          current_stream(idx))
        if status:
            _lib.check(status)
    return codes, scales


def unpack_mxfp4_tensor(codes: torch.Tensor, scales: torch.Tensor, n: int | None = None,
                        dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of packed rows, shape ``(..., n)``; ``n`` defaults to the whole blocks.

    One rounding to ``dtype``: float32 and bfloat16 hold every value (below bfloat16's
    subnormals aside), float16 rounds and overflows to infinity like any conversion."""
    dst = dtype_id(dtype, "dtype")
    if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor):
        raise TypeError("codes and scales must be torch.Tensors")
    *lead, blocks = scales.shape or (-1,)
    if codes.shape != (*lead, BLOCK_BYTES * blocks):
        raise ValueError(f"codes (..., 16 * blocks) and scales (..., blocks) do not match: "
                         f"{tuple(codes.shape)}, {tuple(scales.shape)}")
    n = blocks * BLOCK if n is None else int(n)
    if n < 0 or (n + BLOCK - 1) // BLOCK != blocks:
        raise ValueError(f"n={n} does not have {blocks} blocks of {BLOCK}")
    rows = scales.numel() // blocks if blocks else 0
    idx = as_packed(codes, scales, rows, n, "m")
    if current_device() != idx:
        with torch.cuda.device(idx):
            return unpack_mxfp4_tensor(codes, scales, n, dtype)
    out = torch.empty(*lead, n, dtype=dtype, device=codes.device)
    if rows:
        status = _lib.load().feather_decode_mxfp4(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), dst, rows, n,
                                                  current_stream(idx))
        if status:
            _lib.check(status)
    return out
