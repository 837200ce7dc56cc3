"""Microscaled 4-bit operators and rotary positions, host side: the oracle against the formats'
definition, refusals of the C ABI and of the Python surface, the frequency tables.  No GPU."""
import math
import os
import subprocess
import sys

import pytest
import torch

import feather_b200 as fb
from oracle import mxfp4_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from feather_b200.csrc import build
    build.build()
    from feather_b200 import _lib
    return _lib.load()


def test_oracle_rounds_to_the_nearest_even_code():
    # ties between neighbours, the saturating end, signs; a 4 in the block makes the scale 1
    x = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.9, -0.25, -0.0, -0.26, -5.1]
    codes, scales = O.quantise(torch.tensor([x]))
    assert scales.tolist() == [[127]]
    got = O.dequantise(codes, scales, len(x))[0].tolist()
    assert got == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, 0.0, 0.0, -0.5, -6.0]
    assert codes[0, 5] >> 4 == 8 and codes[0, 5] & 15 == 8     # elements 10 and 11: -0.25 and -0.0 keep their sign


def test_oracle_scale_edges():
    x = torch.zeros(6, 32)
    x[1, 3] = 2.0 ** -149                       # FP32's smallest
    x[2, 0] = torch.finfo(torch.float32).max
    x[3, 31] = float("inf")
    x[4, 1] = float("nan")
    x[5, 7] = -8.0
    codes, scales = O.quantise(x)
    assert scales.flatten().tolist() == [0, 0, 252, 255, 255, 128]
    assert int(codes[3].sum()) == 0 and int(codes[4].sum()) == 0
    assert O.dequantise(codes, scales, 32)[3].isnan().all()
    assert O.dequantise(codes, scales, 32)[5, 7] == -8.0


def test_c_entry_points_refuse_before_any_device_call(lib):
    p, odd = 4096, 4097
    enc, dec, gemv, gemm, rot = (lib.feather_encode_mxfp4, lib.feather_decode_mxfp4, lib.feather_gemv_mxfp4,
                                 lib.feather_gemm_mxfp4, lib.feather_rotary)
    assert enc(None, 0, None, None, 0, 5, None) == 0 and dec(None, None, None, 0, 5, 0, None) == 0
    assert enc(p, 0, p, p, -1, 5, None) == -1 and dec(p, p, p, 0, 1, -5, None) == -1
    assert enc(p, 3, p, p, 1, 5, None) == -3 and dec(p, p, p, 3, 1, 5, None) == -3
    assert enc(None, 0, p, p, 1, 5, None) == -1 and dec(p, None, p, 0, 1, 5, None) == -1
    assert enc(odd, 0, p, p, 1, 5, None) == -2 and enc(p, 0, p + 8, p, 1, 5, None) == -2
    assert dec(p, p, p + 2, 1, 1, 5, None) == -2 and dec(p + 1, p, p, 1, 1, 5, None) == -2
    assert enc(p, 0, p, p, 1, 1 << 31, None) == -8
    assert gemv(p, p, p, 0, None, p, None, 0, 8, 1, None) == 0 and gemv(p, p, p, 0, None, p, None, 8, 8, 0, None) == 0
    assert gemv(p, p, p, 4, None, p, None, 8, 8, 1, None) == -3 and gemv(p, p, p, 0, None, p, None, 8, -8, 1, None) == -1
    assert gemv(p, p, p, 3, None, p, None, 8, 8, 1, None) == -1            # a packed vector without its scales
    assert gemv(p, p, p, 0, None, p, None, 8, 8, 65, None) == -8
    assert gemv(p + 1, p, p, 0, None, p, None, 8, 8, 1, None) == -2 and gemv(p, p, p + 2, 3, p, p, None, 8, 8, 1, None) == -2
    assert gemm(p, p, p, p, p, 3, 8, 8, 8, None) == -3 and gemm(p, p, p, p, None, 0, 8, 8, 8, None) == -1
    assert gemm(p, p, p, p, p, 0, 0, 8, 8, None) == 0 and gemm(p, None, p, p, p, 0, 8, 8, 8, None) == -1
    assert gemm(p, p, p + 8, p, p, 0, 8, 8, 8, None) == -2 and gemm(p, p, p, p, odd, 0, 8, 8, 8, None) == -2
    args = dict(x=p, dtype=1, ts=64, hs=64, pos=p, wide=1, inv=p, out=p, mode=-1, tokens=2, heads=1, dim=64, rotated=64, layout=0)

    def rotary(**kw):
        a = {**args, **kw}
        return rot(a["x"], a["dtype"], a["ts"], a["hs"], a["pos"], a["wide"], a["inv"], a["out"], a["mode"], a["tokens"],
                   a["heads"], a["dim"], a["rotated"], a["layout"], 1.0, None)
    assert rotary(rotated=63) == -1 and rotary(rotated=66) == -1 and rotary(rotated=0) == -1 and rotary(tokens=-1) == -1
    assert rotary(dtype=3) == -3 and rotary(mode=2) == -3 and rotary(layout=2) == -3
    assert rotary(tokens=0) == 0 and rotary(heads=0) == 0
    assert rotary(dim=66, mode=0) == -1 and rotary(pos=None) == -1
    assert rotary(inv=p + 4) == -2 and rotary(pos=p + 4) == -2 and rotary(x=odd) == -2 and rotary(mode=0, out=p + 2) == -2
    assert rotary(dim=2048, rotated=2048) == -8


def test_python_surface_refuses_on_the_host():
    codes, scales = torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8)
    x = torch.zeros(2, 32)
    with pytest.raises(TypeError):
        fb.pack_mxfp4_tensor(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(TypeError):
        fb.pack_mxfp4_tensor([1.0])
    with pytest.raises(ValueError):
        fb.pack_mxfp4_tensor(torch.tensor(1.0))
    with pytest.raises(TypeError):
        fb.unpack_mxfp4_tensor(codes, scales, 32, torch.int32)
    with pytest.raises(ValueError):
        fb.unpack_mxfp4_tensor(codes, scales[:1], 32)               # shapes that do not match
    for n in (0, 33, -1):
        with pytest.raises(ValueError):
            fb.unpack_mxfp4_tensor(codes, scales, n)                # not one block's worth
    with pytest.raises(ValueError):
        fb.unpack_mxfp4_tensor(codes, scales, 32)                   # not on a GPU
    with pytest.raises(ValueError):
        fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x[0], (2, 32))
    with pytest.raises(ValueError):
        fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x[0], (2,))
    with pytest.raises(ValueError):
        fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, codes, scales, (2, 32))
    with pytest.raises(TypeError):
        fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, codes, scales, (2, 32), out_dtype=torch.float64)
    with pytest.raises(NotImplementedError):
        fb.rotary_gpu(x[:, None], torch.arange(2), torch.ones(4, dtype=torch.float64), layout="quarter")
    with pytest.raises(NotImplementedError):
        fb.rotary_gpu(x[:, None], torch.arange(2), torch.ones(4, dtype=torch.float64), mode="E3M4")
    with pytest.raises(ValueError):
        fb.rotary_gpu(x[:, None], torch.arange(2), torch.ones(4, dtype=torch.float64))
    assert {"pack_mxfp4_tensor", "gemm_mxfp4_acc_fp32_gpu", "rotary_gpu"} <= set(__import__("feather").__all__)


def test_rotary_frequencies():
    f = fb.rotary_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,)
    for i in (0, 1, 17, 31):
        assert f[i].item() == pytest.approx(10000.0 ** (-2 * i / 64), rel=1e-14)
    assert torch.equal(fb.rotary_frequencies(64, 10000.0, "linear", 4.0, device="cpu"), f / 4)
    b = fb.rotary_frequencies(64, 10000.0, "base", 4.0, device="cpu")
    assert b[0] == 1.0 and b[31].item() == pytest.approx(f[31].item() / 4, rel=1e-13)
    for kind, high in (("ramp", 32.0), ("bands", 4.0)):
        s = fb.rotary_frequencies(128, 10000.0, kind, 8.0, original_length=4096, device="cpu")
        g = fb.rotary_frequencies(128, 10000.0, device="cpu")
        ratio = s / g
        turns = 4096 * g / (2 * math.pi)
        assert torch.equal(ratio[turns > high * 1.2], torch.ones_like(ratio[turns > high * 1.2]))
        assert torch.allclose(ratio[turns < 0.8], torch.full_like(ratio[turns < 0.8], 1 / 8), rtol=1e-14, atol=0)
        assert bool((ratio[1:] <= ratio[:-1] + 1e-12).all()) and bool(((ratio > 0.126) & (ratio < 0.999)).any())
    # one turn count inside the bands by hand: keep = (turns - 1) / 3
    s, g = fb.rotary_frequencies(128, 10000.0, "bands", 8.0, original_length=4096, device="cpu"), fb.rotary_frequencies(128, device="cpu")
    i = int(((4096 * g / (2 * math.pi) - 2.5).abs()).argmin())
    keep = (4096 * g[i].item() / (2 * math.pi) - 1) / 3
    assert s[i].item() == pytest.approx(g[i].item() * (keep + (1 - keep) / 8), rel=1e-13)
    for bad in (dict(rotated=63), dict(rotated=0), dict(rotated=2048), dict(rotated=64, base=1.0), dict(rotated=64, factor=0.5),
                dict(rotated=64, scaling="ramp"), dict(rotated=64, scaling="bands", original_length=10, low=4.0, high=2.0)):
        with pytest.raises(ValueError):
            fb.rotary_frequencies(**{"device": "cpu", **bad})
    with pytest.raises(NotImplementedError):
        fb.rotary_frequencies(64, scaling="other", device="cpu")


def test_angle_reduction_is_good_to_a_tenth_of_a_millionth():
    # the kernel's angle, restated in numpy precision: turns in 64 bits, the fraction in FP32
    p = torch.tensor([0, 1, 4095, 100003, 2 ** 20 + 1, 2 ** 31 - 1], dtype=torch.float64)[:, None]
    f = fb.rotary_frequencies(64, device="cpu")
    turns = p * f * 0.15915494309189533577
    part = (turns - torch.round(turns)).float()
    got = torch.sin((2 * math.pi) * part.double())
    # angle error: |p f| 2^-52 from the 64-bit products, half an ulp of a fraction below 1/2 (2^-26) times 2 pi
    bound = (p * f) * 2.0 ** -51 + 2 * math.pi * 2.0 ** -26
    assert bool(((got - torch.sin(p * f)).abs() <= bound).all())


def test_sizes_at_the_end_of_their_range(lib):
    p, big = 4096, 1 << 31
    assert lib.feather_gemv_mxfp4(p, p, p, 0, None, p, None, big - 127, 8, 1, None) == -8      # rows are counted in 32 bits
    assert lib.feather_gemv_mxfp4(p, p, p, 3, p, p, None, big, 8, 2, None) == -8
    # digits from columns x M x N = 80 M on, without passing 64 bits on the way; FP32 vectors are two columns each
    need = lib.feather_gemv_mxfp4_workspace_bytes
    assert need((1 << 62) + 1, 1 << 30, 64, 1) == need(1 << 20, 1 << 30, 8, 1) == 8 * 12 * (1 << 25) * 17
    for vectors, dtype in ((3, 0), (2, 1), (64, 2)):
        cols = vectors * (2 if dtype == 1 else 1)
        for n in (1, 33, 4096):
            m = -(-(80 << 20) // (cols * n))
            assert need(m, n, vectors, dtype) > 0 and need(m - 1, n, vectors, dtype) == 0
    assert need(100, 0, 64, 1) == 0 and need(1 << 40, 4096, 2, 0) == 0


@pytest.mark.parametrize("gone", ["torch.float8_e8m0fnu", "torch.float4_e2m1fn_x2", "torch._C._cuda_getDevice", "torch._C._cuda_getCurrentRawStream"])
def test_import_without_what_not_every_torch_has(gone):
    # a type or a private accessor that another torch lacks: the package imports, with the public calls in its place
    code = f"""
import torch
if hasattr({gone.rpartition('.')[0]}, {gone.rpartition('.')[2]!r}):
    del {gone}
import feather_b200 as fb, feather_b200._lib as lib, feather_b200.packers.mxfp4 as mx
assert fb.pack_fp8_tensor and torch.uint8 in mx._CODE_DTYPES and torch.uint8 in mx._SCALE_DTYPES
if {gone!r}.endswith("getDevice"):
    assert mx.current_device is torch.cuda.current_device
if {gone!r}.endswith("RawStream"):
    assert mx.current_stream is lib.current_stream_ptr
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert done.returncode == 0, done.stderr


def added_up(found):
    """The rows' sum in FP32, the smallest first."""
    total = found[-1].float()
    for d in found[-2::-1]:
        total = total + d.float()
    return total.double()


def test_twelve_digits_are_what_it_takes():
    v = O.digit_cases(4, 700)
    wide = v.double()
    ok = [bool(((added_up(O.digits(v, count)) - wide).abs() <= O.digit_bound(wide)).all()) for count in (10, 11, 12)]
    assert ok == [False, False, True]
    found = O.digits(v, 12)
    found[11] = torch.zeros_like(found[11])                       # a row that is lost, or has its neighbour's scale
    assert not bool(((added_up(found) - wide).abs() <= O.digit_bound(wide)).all())
    for lost in (0, 5, 10):
        found = O.digits(v, 12)
        found[lost] = 2 * found[lost]
        assert not bool(((added_up(found) - wide).abs() <= O.digit_bound(wide)).all())
