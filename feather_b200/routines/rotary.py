"""Rotary positions between a projection and the packed attention: the first elements of every
head are pairs that are turned by an angle growing with the token's position.  No counterpart
in the reference.

``rotary_frequencies`` makes the 64-bit inverse frequencies a program keeps,
``rotary_gpu`` turns queries or keys and, with ``mode``, packs them to FP8 words head by head,
which is what ``flash_attention_fp8_e5m2_acc_fp32_gpu`` takes.
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from ..packers.fp8 import _tag, as_words
from ..packers.mxfp4 import current_device, current_stream, dtype_id

__all__ = ["rotary_frequencies", "rotary_gpu"]

LAYOUTS = {"half": 0, "interleaved": 1}
MAX_ROTATED = 1024


def rotary_frequencies(rotated: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, low: float | None = None, high: float | None = None,
                       device="cuda") -> torch.Tensor:
    """``rotated / 2`` inverse frequencies ``base ** (-2 i / rotated)`` as float64 on ``device``.

    ``scaling`` stretches them to contexts ``factor`` times longer:

    * ``"linear"``: every frequency is divided by ``factor``;
    * ``"base"``: the base grows by ``factor ** (rotated / (rotated - 2))``, so that the lowest
      frequency is divided by ``factor`` and the highest stays;
    * ``"ramp"``: by the number of turns a pair makes over ``original_length`` positions: above
      ``high`` (default 32) unchanged, below ``low`` (default 1) divided by ``factor``, in between a
      straight line over the pairs' index.  Usually used with ``scale = 0.1 ln(factor) + 1`` in
      ``rotary_gpu``;
    * ``"bands"``: by the wavelength against ``original_length``: shorter than ``original_length /
      high`` (default 4) unchanged, longer than ``original_length / low`` (default 1) divided by
      ``factor``, in between a straight line in the number of turns.
    """
    rotated = int(rotated)
    if rotated < 2 or rotated % 2 or rotated > MAX_ROTATED:
        raise ValueError(f"rotated must be even and between 2 and {MAX_ROTATED}, got {rotated}")
    if not (base > 1.0 and math.isfinite(base)) or not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling not in (None, "linear", "base", "ramp", "bands"):
        raise NotImplementedError(f"scaling {scaling!r} not supported")
    if scaling in ("ramp", "bands") and (original_length is None or original_length < 1):
        raise ValueError(f"scaling {scaling!r} needs original_length")
    i = torch.arange(0, rotated, 2, dtype=torch.float64)
    if scaling == "base" and rotated > 2:
        base = base * factor ** (rotated / (rotated - 2))
    freq = torch.pow(torch.tensor(base, dtype=torch.float64), -i / rotated)
    if scaling == "linear":
        freq = freq / factor
    elif scaling in ("ramp", "bands"):
        low = 1.0 if low is None else float(low)
        high = (32.0 if scaling == "ramp" else 4.0) if high is None else float(high)
        if not 0.0 < low < high:
            raise ValueError("low must be above 0 and below high")
        if scaling == "ramp":
            def index(turns: float) -> float:   # the pair that makes so many turns over the original length
                return rotated * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
            first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), rotated - 1)
            keep = 1.0 - ((i / 2 - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        else:
            turns = original_length * freq / (2 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq / factor * (1.0 - keep) + freq * keep
    return freq.to(device)


def rotary_gpu(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, layout: str = "half",
               mode: str | None = None, scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Turn the heads of ``x`` (``feather_rotary``).

    ``x``: ``(tokens, heads, dim)`` float16, bfloat16 or float32, ``dim`` contiguous, any token and
    head strides.  ``positions``: ``(tokens,)`` int64 or int32.  ``inv_freq``: float64, one per pair
    (``rotary_frequencies``); the first ``2 * len(inv_freq)`` elements of a head turn, the others
    pass through.  ``layout``: pairs ``(i, i + rotated / 2)`` for "half", ``(2 i, 2 i + 1)`` for
    "interleaved".  ``scale`` multiplies the turned elements.

    Returns ``(tokens, heads, dim)`` of ``x``'s type (``out`` may be ``x`` itself where it is
    contiguous), or with ``mode`` "E5M2" / "E4M3" the FP8 words ``(heads, tokens, dim / 4)``: one
    head's ``result[h]`` is a packed (tokens, dim) matrix.  Words written to ``out`` come back
    tagged with ``mode`` too, and an ``out`` that carries a tag has it changed.

    The angles are computed in 64 bits, ``|angle| * 2 ** -51`` off at most before the FP32 sine and
    cosine of what is left of a turn: position ``2 ** 26`` loses nothing, ``2 ** 31`` up to a
    millionth of a radian."""
    if not (isinstance(x, torch.Tensor) and isinstance(positions, torch.Tensor) and isinstance(inv_freq, torch.Tensor)):
        raise TypeError("x, positions and inv_freq must be torch.Tensors")
    if layout not in LAYOUTS:
        raise NotImplementedError(f"layout {layout!r} not supported")
    out_mode = -1 if mode is None else _lib.mode_id(mode)
    dtype = dtype_id(x.dtype, "x")
    idx = x.get_device()
    if idx < 0 or positions.get_device() != idx or inv_freq.get_device() != idx:
        raise ValueError("x, positions and inv_freq must be CUDA tensors on one device: feather_b200 has no CPU path")
    if x.dim() != 3:
        raise ValueError("x must be (tokens, heads, dim)")
    tokens, heads, dim = x.shape
    wide = positions.dtype is torch.int64
    if (not wide and positions.dtype is not torch.int32) or positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int64 or int32 tensor, one per token")
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 vector")
    rotated = 2 * inv_freq.numel()
    if rotated < 2 or rotated > dim or rotated > MAX_ROTATED:
        raise ValueError(f"inv_freq turns {rotated} elements of heads of {dim} (at least 2, at most {MAX_ROTATED})")
    if mode is not None and dim % 4:
        raise ValueError("packed heads are whole words: dim must be a multiple of 4")
    token_stride, head_stride, last = x.stride()
    total = tokens * heads * dim
    if last != 1 and total:
        raise ValueError("the last dimension of x must be contiguous")
    if current_device() != idx:
        with torch.cuda.device(idx):
            return rotary_gpu(x, positions, inv_freq, layout, mode, scale, out)
    if mode is None:
        if out is None:
            out = torch.empty(tokens, heads, dim, dtype=x.dtype, device=x.device)
        elif out.dtype != x.dtype or out.numel() != total or out.device != x.device or not out.is_contiguous():
            raise ValueError("out must be a contiguous tensor of x's type and size on its device")
    elif out is None:
        out = torch.empty(heads, tokens, dim // 4, dtype=torch.uint32, device=x.device)
    else:
        out = as_words(out, "out")
        if out.numel() != total // 4 or out.device != x.device:
            raise ValueError("out must hold heads * tokens * dim / 4 packed words on x's device")
    if total:
        status = _lib.load().feather_rotary(x.data_ptr(), dtype, token_stride, head_stride, positions.data_ptr(),
                                            1 if wide else 0, inv_freq.data_ptr(), out.data_ptr(), out_mode, tokens, heads,
                                            dim, rotated, LAYOUTS[layout], scale, current_stream(idx))
        if status:
            _lib.check(status)
    return out if mode is None else _tag(out, mode)
