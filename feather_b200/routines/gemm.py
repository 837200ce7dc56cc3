"""Products with microscaled 4-bit matrices (``feather_b200.packers.mxfp4``).

``gemv_mxfp4_acc_fp32_gpu`` multiplies a packed matrix with one or a few vectors, dense or
packed, and is bound by the matrix's bytes; ``gemm_mxfp4_acc_fp32_gpu`` multiplies two packed
matrices on the tensor cores' microscaled kind.  No counterpart in the reference, whose GEMV
multiplies packed FP8 (feather/routines/gemv.py).
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from ..packers.mxfp4 import BLOCK_BYTES, as_packed, blocks_of, current_device, current_stream, dtype_id

__all__ = ["gemv_mxfp4_acc_fp32_gpu", "gemm_mxfp4_acc_fp32_gpu"]

MAX_VECTORS = 64


def _shape(m_shape) -> tuple[int, int]:
    if len(m_shape) != 2:
        raise ValueError("m_shape must be the unpacked (M, N) of the matrix")
    M, N = int(m_shape[0]), int(m_shape[1])
    if M < 0 or N < 0:
        raise ValueError("m_shape must not be negative")
    return M, N


def _check_out(out, n, dtype, device):
    if out.dtype != dtype or out.numel() != n or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {dtype} tensor of {n} elements on the operands' device")


def gemv_mxfp4_acc_fp32_gpu(m_codes: torch.Tensor, m_scales: torch.Tensor, v: torch.Tensor, m_shape,
                            v_scales: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[b, r] = sum_j value(m[r, j]) * v[b, j]`` with FP32 accumulation
    (``feather_gemv_mxfp4``), float32 of shape ``(M,)`` or ``(batch, M)``.

    ``m_codes``, ``m_scales``: what ``pack_mxfp4_tensor`` returns for an ``(M, N)`` matrix.
    ``v``: a contiguous float16, bfloat16 or float32 tensor of shape ``(N,)`` or ``(batch, N)``, or
    packed codes together with ``v_scales``.  Up to eight vectors go through one pass over the
    matrix (four float32 ones where it is small); at most 64.

    What a vector's elements are used with: packed ones exactly; one or two vectors, or more on small
    matrices, to ``2 ** -23`` of the element (float32; float16 and bfloat16 exactly) or ``2 ** -39`` of the largest in its
    32-element block; more on large matrices (three 16-bit or two float32 ones, from ``columns * M * N = 80 * 2 ** 20`` on,
    a float32 vector counting as two columns) to ``2 ** -24`` of the largest in the block or ``2 ** -129``."""
    M, N = _shape(m_shape)
    idx = as_packed(m_codes, m_scales, M, N, "m")
    if not isinstance(v, torch.Tensor):
        raise TypeError("v must be a torch.Tensor")
    dims = v.dim()
    if dims != 1 and dims != 2:
        raise ValueError("v must be one vector or a (batch, N) tensor of them")
    shape = v.shape
    batch = 1 if dims == 1 else shape[0]
    if v_scales is None:
        v_dtype = dtype_id(v.dtype, "v (without v_scales)")
        if shape[-1] != N:
            raise ValueError(f"v has {shape[-1]} elements per vector, the matrix has N={N}")
        if not v.is_contiguous():
            raise ValueError("v must be contiguous")
        scales_ptr = None
    else:
        as_packed(v, v_scales, batch, N, "v")
        if shape[-1] != blocks_of(N) * BLOCK_BYTES:
            raise ValueError(f"packed vectors of N={N} have {blocks_of(N) * BLOCK_BYTES} bytes each, got {shape[-1]}")
        v_dtype, scales_ptr = _lib.SRC_MXFP4, v_scales.data_ptr()
    if v.get_device() != idx:
        raise ValueError("v must be a CUDA tensor on the matrix's device")
    if batch > MAX_VECTORS:
        raise ValueError(f"at most {MAX_VECTORS} vectors: pack them and use gemm_mxfp4_acc_fp32_gpu")
    if current_device() != idx:
        with torch.cuda.device(idx):
            return gemv_mxfp4_acc_fp32_gpu(m_codes, m_scales, v, m_shape, v_scales, out)
    if out is not None:
        _check_out(out, batch * M, torch.float32, v.device)
    elif dims == 1:
        out = torch.empty(M, dtype=torch.float32, device=v.device)
    else:
        out = torch.empty(batch, M, dtype=torch.float32, device=v.device)
    if M and batch:
        lib = _lib.load()
        # one FP32 or two 16-bit vectors never need one
        need = 0 if batch == 1 or scales_ptr is not None else lib.feather_gemv_mxfp4_workspace_bytes(M, N, batch, v_dtype)
        ws = torch.empty(need, dtype=torch.uint8, device=v.device) if need else None
        status = lib.feather_gemv_mxfp4(m_codes.data_ptr(), m_scales.data_ptr(), v.data_ptr(), v_dtype, scales_ptr,
                                        out.data_ptr(), ws.data_ptr() if need else None, M, N, batch, current_stream(idx))
        if status:
            _lib.check(status)
    return out


def gemm_mxfp4_acc_fp32_gpu(m_codes: torch.Tensor, m_scales: torch.Tensor, x_codes: torch.Tensor, x_scales: torch.Tensor,
                            m_shape, out_dtype: torch.dtype = torch.float32,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[b, r] = sum_j value(m[r, j]) * value(x[b, j])``, both operands packed, FP32
    accumulation, one rounding to ``out_dtype`` (float32, bfloat16, float16); shape
    ``(batch, M)`` (``feather_gemm_mxfp4``).

    ``x_codes``, ``x_scales``: what ``pack_mxfp4_tensor`` returns for a ``(batch, N)`` tensor (or
    ``(..., N)``: the leading dimensions are rows)."""
    M, N = _shape(m_shape)
    dst = dtype_id(out_dtype, "out_dtype")
    idx = as_packed(m_codes, m_scales, M, N, "m")
    if not isinstance(x_codes, torch.Tensor) or not isinstance(x_scales, torch.Tensor):
        raise TypeError("x_codes and x_scales must be torch.Tensors")
    *lead, row_bytes = x_codes.shape or (-1,)
    if row_bytes != blocks_of(N) * BLOCK_BYTES:
        raise ValueError(f"packed rows of N={N} have {blocks_of(N) * BLOCK_BYTES} bytes each, got {tuple(x_codes.shape)}")
    batch = math.prod(lead)
    if as_packed(x_codes, x_scales, batch, N, "x") != idx:
        raise ValueError("m and x must be on the same device")
    if current_device() != idx:
        with torch.cuda.device(idx):
            return gemm_mxfp4_acc_fp32_gpu(m_codes, m_scales, x_codes, x_scales, m_shape, out_dtype, out)
    if out is not None:
        _check_out(out, batch * M, out_dtype, x_codes.device)
    else:
        out = torch.empty(*lead, M, dtype=out_dtype, device=x_codes.device)
    if M and batch:
        status = _lib.load().feather_gemm_mxfp4(m_codes.data_ptr(), m_scales.data_ptr(), x_codes.data_ptr(),
                                                x_scales.data_ptr(), out.data_ptr(), dst, M, N, batch, current_stream(idx))
        if status:
            _lib.check(status)
    return out
