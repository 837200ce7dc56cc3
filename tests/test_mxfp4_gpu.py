"""Microscaled 4-bit operators and rotary positions on the GPU against the 64-bit oracle."""
import math

import pytest
import torch

import feather_b200 as fb
from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def values(rows, n, seed, dtype=torch.float32, spread=3.0):
    """Normal values whose blocks and columns differ in size by powers of two."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, n, generator=gen, device="cuda")
    return (x * torch.exp2(spread * torch.randn(n, generator=gen, device="cuda")).clamp(2.0 ** -9, 2.0 ** 9)).to(dtype)


def packed(rows, n, seed, spread=3.0):
    return O.quantise(values(rows, n, seed, spread=spread))


def same_bits(a, b):
    return a.shape == b.shape and torch.equal(a, b)


# ---------------------------------------------------------------- quantise --
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (1, 2048), (7, 160), (129, 1000), (64, 4096), (1001, 96)])
def test_pack_is_bit_exact(rows, n, dtype):
    x = values(rows, n, 11 * rows + n, DTYPES[dtype])
    codes, scales = fb.pack_mxfp4_tensor(x)
    want_codes, want_scales = O.quantise(x)
    assert codes.dtype == scales.dtype == torch.uint8 and codes.device == x.device
    assert same_bits(scales, want_scales) and same_bits(codes, want_codes)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [64, 63])
def test_pack_edges(dtype, n):
    t = DTYPES[dtype]
    info = torch.finfo(t)
    x = torch.zeros(12, n, dtype=t, device="cuda")
    x[1] = -0.0
    x[2, 5] = info.smallest_normal * info.eps      # the type's smallest
    x[3, :] = info.max
    x[4, 40] = float("inf")
    x[5, 2] = float("nan")
    x[6, 3] = -float("inf")
    x[7, :8] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=t)
    x[8, :8] = torch.tensor([-4.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0], dtype=t)
    x[9, 33:37] = torch.tensor([7.9, 6.0, 6.1, -7.9], dtype=t)
    x[10, 1] = info.tiny
    x[11, 0], x[11, 1] = info.max, info.tiny       # the far ends in one block
    codes, scales = fb.pack_mxfp4_tensor(x)
    want_codes, want_scales = O.quantise(x)
    assert same_bits(scales, want_scales) and same_bits(codes, want_codes)
    back = fb.unpack_mxfp4_tensor(codes, scales, n)
    want = O.dequantise(want_codes, want_scales, n).float()
    assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back.nan_to_num(7.0), want.nan_to_num(7.0))
    assert back[4, 32:].isnan().all() and not back[4, :32].isnan().any()


def test_pack_shapes_views_and_cpu_input():
    x = values(6, 64, 5)
    whole = fb.pack_mxfp4_tensor(x)
    lead = fb.pack_mxfp4_tensor(x.view(2, 3, 64))
    assert lead[0].shape == (2, 3, 32) and lead[1].shape == (2, 3, 2)
    assert same_bits(lead[0].view(6, 32), whole[0]) and same_bits(lead[1].view(6, 2), whole[1])
    one = fb.pack_mxfp4_tensor(x[2])
    assert same_bits(one[0], whole[0][2]) and same_bits(one[1], whole[1][2])
    t = values(64, 6, 6)
    assert all(same_bits(a, b) for a, b in zip(fb.pack_mxfp4_tensor(t.T), fb.pack_mxfp4_tensor(t.T.contiguous())))
    odd = torch.empty(1 + 6 * 64, device="cuda")[1:].view(6, 64).copy_(x)       # a start off the 16-byte grid
    assert odd.data_ptr() % 16 and all(same_bits(a, b) for a, b in zip(fb.pack_mxfp4_tensor(odd), whole))
    host = fb.pack_mxfp4_tensor(x.cpu())
    assert not host[0].is_cuda and same_bits(host[0].cuda(), whole[0]) and same_bits(host[1].cuda(), whole[1])
    for shape in ((0, 64), (3, 0), (0,)):
        c, s = fb.pack_mxfp4_tensor(torch.empty(shape, device="cuda"))
        assert c.numel() == 0 and s.numel() == 0
        assert fb.unpack_mxfp4_tensor(c, s, shape[-1]).shape == shape


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 32), (3, 31), (9, 257), (5, 96), (130, 1024), (2, 5000)])
def test_unpack_every_byte_and_scale(rows, n, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows + n)
    blocks = -(-n // 32)
    codes = torch.randint(0, 256, (rows, 16 * blocks), generator=gen, device="cuda").to(torch.uint8)
    scales = torch.randint(0, 256, (rows, blocks), generator=gen, device="cuda").to(torch.uint8)
    got = fb.unpack_mxfp4_tensor(codes, scales, n, DTYPES[dtype])
    # the exact value, once through FP32 (exact but for what overflows there as well) and rounded
    want = O.dequantise(codes, scales, n).float().to(DTYPES[dtype])
    assert got.dtype == DTYPES[dtype] and got.shape == (rows, n)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(torch.where(got.isnan(), 0, got), torch.where(want.isnan(), 0, want))


# -------------------------------------------------------------------- gemv --
def gemv_bound(m, v, split):
    """Per element: a block's 32 products are added by the tensor core, whose FP32 sum may lose 2^-22 of the products' size
    per instruction (two have products of the block); two scalings round (2^-24 each); a warp adds
    its blocks, four lanes, at most 16 warps and the chunks in FP32 (2^-24 per addition); an FP32 vector is split with an error of
    2^-24 per element."""
    blocks = -(-m.shape[1] // 32)
    steps = math.ceil(blocks / 4) + 2 + 16 + 2 + (1 if split else 0) + math.ceil(blocks / 192)
    return (v.abs() @ m.abs().T) * (2 * 2.0 ** -22 + steps * 2.0 ** -24) + 1e-44


@pytest.mark.parametrize("vector", ["fp16", "bf16", "fp32", "mxfp4"])
@pytest.mark.parametrize("M,N,batch", [(1, 1, 1), (1, 32, 1), (17, 33, 1), (16, 128, 2), (3, 4000, 1), (256, 2048, 1), (250, 2080, 3),
                                       (2400, 256, 1), (2500, 100, 5), (4800, 4096, 1), (40, 30000, 2), (100, 1024, 8), (33, 640, 11),
                                       (100, 8192, 8), (21400, 20000, 2)])
def test_gemv(M, N, batch, vector):
    codes, scales = packed(M, N, M + N)
    m = O.dequantise(codes, scales, N)
    if vector == "mxfp4":
        v, v_scales = packed(batch, N, 7 * M + N)
        wide = O.dequantise(v, v_scales, N)
    else:
        v, v_scales = values(batch, N, 7 * M + N, DTYPES[vector], spread=2.0), None
        wide = v.double()
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N), v_scales=v_scales)
    assert got.dtype == torch.float32 and got.shape == (batch, M)
    want = wide @ m.T
    err = (got.double() - want).abs()
    assert bool((err <= gemv_bound(m, wide, vector == "fp32")).all()), (err / gemv_bound(m, wide, vector == "fp32")).max()
    one = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v[0], (M, N), v_scales=None if v_scales is None else v_scales[0])
    assert one.shape == (M,) and torch.equal(one, fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v[:1], (M, N),
                                             v_scales=None if v_scales is None else v_scales[:1])[0])
    assert torch.equal(got, fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N), v_scales=v_scales))   # the same bits again


def digits_bound(m, v):
    """Several dense vectors on a large matrix go to the tensor cores as a sum of 12 packed rows: what is left of an
    element is at most 2^-24 of its block's largest; N / 64 products in a row add into one FP32 sum per row and lose 2^-22 of the
    products' size each; the rows' sums are at most 4/3 of the first, 11 additions and up to 3 of a cluster's parts round."""
    blocks = -(-m.shape[1] // 32)
    top = torch.nn.functional.pad(v.abs(), (0, blocks * 32 - v.shape[1])).view(v.shape[0], blocks, 32).amax(-1)
    top = top.repeat_interleave(32, 1)[:, :v.shape[1]]
    steps = math.ceil(m.shape[1] / 64) + 1
    return top @ m.abs().T * 2.0 ** -24 + (v.abs() @ m.abs().T) * 2 * (steps * 2.0 ** -22 + 14 * 2.0 ** -24) + 1e-44


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,N,batch", [(9000, 4096, 3), (4100, 5000, 5), (2050, 5632, 8), (16400, 1024, 6), (3000, 3000, 11), (5000, 8192, 2)])
def test_gemv_several_vectors_on_large_matrices(M, N, batch, dtype):
    codes, scales = packed(M, N, M + N)
    m = O.dequantise(codes, scales, N)
    v = values(batch, N, M, DTYPES[dtype], spread=2.0)
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N))
    err, bound = (got.double() - v.double() @ m.T).abs(), digits_bound(m, v.double())
    assert bool((err <= bound).all()), (err / bound).max()
    assert torch.equal(got, fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N)))
    # not finite: the vectors that hold it, with the signs that arithmetic gives; the others keep their bits
    v = v.clone()
    v[0, N - 1], v[1, 7], v[1, N // 2] = float("inf"), -float("inf"), float("nan")
    if batch > 2:
        v[2, 3], v[2, 4], v[2, N - 40] = float("inf"), float("inf"), -float("inf")
    again = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N))
    want = v.double() @ m.T
    assert torch.equal(again.isnan(), want.isnan()) and torch.equal(again[want.isinf()].double(), want[want.isinf()])
    assert torch.equal(again[3:], got[3:])


def test_digits_of_numbers_just_below_powers_of_two():
    # the slowest expansion: every digit saturates and leaves a quarter
    M, N = 9000, 4096
    codes, scales = packed(M, N, 5, spread=0.0)
    m = O.dequantise(codes, scales, N)
    v = torch.full((3, N), 1 - 2.0 ** -24, device="cuda") * torch.exp2(torch.arange(N, device="cuda") // 32 % 5.0)
    v[1] *= -1
    v[2, ::2] = 2.0 ** -20
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N))
    assert bool(((got.double() - v.double() @ m.T).abs() <= digits_bound(m, v.double())).all())


def single_codes(M, N, seed):
    """A packed matrix with one code that is not zero per row: (codes, scales, its column, its value)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    row = torch.arange(M, device="cuda")
    k = (row * 37 + torch.div(row, N, rounding_mode="floor")) % N
    code = torch.randint(1, 8, (M,), generator=gen, device="cuda") + 8 * torch.randint(0, 2, (M,), generator=gen, device="cuda")
    codes = torch.zeros(M, -(-N // 32) * 16, dtype=torch.uint8, device="cuda")
    codes[row, k // 2] = (code << (4 * (k % 2))).to(torch.uint8)
    scales = torch.randint(120, 135, (M, -(-N // 32)), generator=gen, device="cuda").to(torch.uint8)
    grid = torch.tensor(O.VALUES + [-x for x in O.VALUES], dtype=torch.float64, device="cuda")
    return codes, scales, k, grid[code] * torch.exp2(scales[row, k // 32].double() - 127)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,N,batch", [(600, 512, 1), (600, 520, 1), (600, 512, 2), (600, 520, 2), (600, 512, 4), (600, 520, 8)])
def test_gemv_holds_every_element(M, N, batch, dtype):
    # every result one product.  A block's largest element is brought to [2^14, 2^15) and rounded to FP16, whose smallest step
    # is 2^-24: 2^-39 of the largest element at most, 16-bit vectors lose nothing else.  An FP32 element is the sum of two FP16
    # numbers of 11 bits: of an element from 2^e on the first leaves at most 2^(e - 11), and rounding that to 11 bits at most
    # 2^(e - 23) (1 + 2^-12 + 2^-23 loses that).  Then one FP32 rounding, of the two parts' sum.
    codes, scales, k, m = single_codes(M, N, M + batch)
    v = O.digit_cases(max(batch, 2), N, "cuda")[:batch]
    v[0, 64:96] = 1 + 2.0 ** -12 + 2.0 ** -23
    v = v.to(DTYPES[dtype])
    if dtype == "fp16":
        v = v.clamp(-60000, 60000)
    wide = v.double()
    blocks = -(-N // 32)
    top = torch.nn.functional.pad(wide.abs(), (0, blocks * 32 - N)).view(batch, blocks, 32).amax(-1).repeat_interleave(32, 1)[:, :N]
    bound = 2.0 ** -39 * top + (wide.abs() * (2.0 ** -23 + 2.0 ** -24) if dtype == "fp32" else 0)
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N)).double()
    err = (got - wide[:, k] * m).abs()
    assert bool((err <= bound[:, k] * m.abs()).all()), (err / (bound[:, k] * m.abs())).max()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,N,batch", [(9000, 4096, 3), (9000, 4096, 8), (9000, 4096, 9), (2500, 5000, 17), (2050, 16384, 4), (57001, 512, 3),
                                       (57001, 512, 9)])
def test_digits_hold_every_element(M, N, batch, dtype):
    # every result one product, so that no other element's error hides a row that is missing.  Matrices in one tile per
    # cluster and in more than three tiles per SM; batches whose last pass has one vector
    codes, scales, k, m = single_codes(M, N, M + batch)
    v = O.digit_cases(batch, N, "cuda").to(DTYPES[dtype])
    if dtype == "fp16":
        v = v.clamp(-60000, 60000)
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N)).double()
    err, bound = (got - v.double()[:, k] * m).abs(), O.digit_bound(v.double())[:, k] * m.abs()
    assert bool((err <= bound).all()), (err / bound).max()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("batch", [3, 9])
def test_digits_of_more_tiles_than_sms(batch, dtype):
    # three and more tiles per SM, the vectors that are not finite repaired in each
    M, N = 57001, 512
    codes, scales = random_packed(M, N, batch)
    scales[33333, 3] = 255
    m = O.dequantise(codes, scales, N)
    v = values(batch, N, 4, DTYPES[dtype], spread=2.0)
    fine = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N))
    v[batch - 1, 70], v[1, 5], v[1, 300] = float("inf"), -float("inf"), float("inf")
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N))
    want = v.double() @ m.T
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want.isinf()].double(), want[want.isinf()])
    keep = [b for b in range(batch) if b not in (1, batch - 1)]
    assert torch.equal(got[keep].nan_to_num(7.0), fine[keep].nan_to_num(7.0))
    err, bound = (got.double() - want)[keep].abs(), digits_bound(m.nan_to_num(0.0), v.double()[keep])
    assert bool((err <= bound)[want[keep].isfinite()].all())


def test_gemv_large():
    M, N = 9000, 16384
    codes, scales = packed(M, N, 3)
    m = O.dequantise(codes, scales, N)
    for dtype in DTYPES:
        v = values(1, N, 4, DTYPES[dtype], spread=2.0)
        got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N))
        assert bool(((got.double() - v.double() @ m.T).abs() <= gemv_bound(m, v.double(), dtype == "fp32")).all())


@pytest.mark.parametrize("M,batch", [(148 * 16 * 260 + 5, 1), (230001, 8)])
def test_gemv_more_rows_than_partial_sums_fit(M, batch):
    # one column tile, so that every warp takes rows; more 16-row groups per CTA than one round of partial sums
    N = 32
    gen = torch.Generator(device="cuda").manual_seed(8)
    codes = torch.randint(0, 256, (M, 16), generator=gen, device="cuda").to(torch.uint8)
    scales = torch.randint(120, 130, (M, 1), generator=gen, device="cuda").to(torch.uint8)
    v = values(batch, N, 4, torch.bfloat16)
    m = O.dequantise(codes, scales, N)
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N))
    assert bool(((got.double() - v.double() @ m.T).abs() <= gemv_bound(m, v.double(), False)).all())


@pytest.mark.parametrize("N", [2048, 5000, 2050])
def test_products_of_operands_off_the_grid(N):
    # scales that start on odd bytes and end where their buffer ends, vectors that start off the 16-byte grid
    M, batch = 300, 70
    codes, scales = packed(M, N, 1, spread=1.0)
    x, x_scales = packed(batch, N, 2, spread=1.0)

    def odd(t):
        buf = torch.full((t.numel() + 3,), 255, dtype=torch.uint8, device="cuda")     # NaN scales on either side
        out = buf[3:].view(t.shape)
        out.copy_(t)
        return out
    want = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N))
    assert bool(want.isfinite().all())
    assert torch.equal(fb.gemm_mxfp4_acc_fp32_gpu(codes, odd(scales), x, odd(x_scales), (M, N)), want)
    v = values(1, N, 3, torch.float16)
    w = torch.empty(N + 1, dtype=torch.float16, device="cuda")[1:].copy_(v[0])
    assert w.data_ptr() % 16
    assert torch.equal(fb.gemv_mxfp4_acc_fp32_gpu(codes, odd(scales), w, (M, N)), fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v[0], (M, N)))
    assert torch.equal(fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x[0], (M, N), v_scales=odd(x_scales)[0]),
                       fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x[0], (M, N), v_scales=x_scales[0]))
    out = torch.full((batch * M + 1,), 7.0, device="cuda", dtype=torch.bfloat16)      # a result off the grid, and what is behind it
    got = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N), out_dtype=torch.bfloat16, out=out[1:])
    assert torch.equal(got.view(batch, M), want.to(torch.bfloat16)) and out[0] == 7.0


def test_products_leave_what_is_behind_their_result():
    for M, batch in ((130, 33), (128, 40), (500, 129), (40, 1)):
        codes, scales = packed(M, 320, 1)
        x, x_scales = packed(batch, 320, 2)
        out = torch.full((batch + 3, M), 7.0, device="cuda")
        fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, 320), out=out[:batch])
        assert bool((out[batch:] == 7.0).all()) and bool((out[:batch] != 7.0).any())
        out.fill_(7.0)
        fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, torch.randn(320, device="cuda"), (M, 320), out=out[0])
        assert bool((out[1:] == 7.0).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_gemv_values_that_are_not_finite_and_far_scales(dtype):
    M, N = 40, 256
    codes, scales = packed(M, N, 1)
    scales = scales.clone()
    scales[3, 2] = 255                                # a NaN block: its row only
    m = O.dequantise(codes, scales, N)
    v = values(4, N, 2, DTYPES[dtype], spread=1.0)
    v[1, 70] = float("inf")
    v[2, 200] = float("nan")
    v[3] = 0
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N)).double()
    want = v.double() @ m.T
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want.isinf()], want[want.isinf()])
    fine = want.isfinite()
    bound = gemv_bound(m.nan_to_num(0.0), v.double().nan_to_num(0.0, 0.0, 0.0), dtype == "fp32")
    assert bool(((got - want).abs()[fine] <= bound[fine]).all())
    # blocks that differ by 2^40 in both operands, and far from one
    far = torch.exp2(torch.tensor([-20.0, 20.0, -4.0, 4.0], device="cuda").repeat_interleave(64)) if dtype != "fp16" else \
        torch.exp2(torch.tensor([-10.0, 10.0, -4.0, 4.0], device="cuda").repeat_interleave(64))
    v2 = (torch.randn(1, N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * far).to(DTYPES[dtype])
    codes, scales = O.quantise(values(M, N, 9, spread=0.0) / far.double().flip(0))
    m = O.dequantise(codes, scales, N)
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v2, (M, N)).double()
    assert bool(((got - v2.double() @ m.T).abs() <= gemv_bound(m, v2.double(), dtype == "fp32")).all())


@pytest.mark.parametrize("vector", ["bf16", "fp32", "mxfp4"])
@pytest.mark.parametrize("M,N,batch", [(40, 256, 1), (40, 300, 1), (40, 256, 2), (40, 256, 5), (9000, 4096, 3)])
@pytest.mark.parametrize("up", [126, -120])
def test_gemv_large_values_times_small_scales_and_the_reverse(M, N, batch, vector, up):
    # sums over unscaled codes leave FP32's range, the results (around 2^60 or 2^-20) do not
    kind = DTYPES.get(vector, torch.float32)
    v = (values(batch, N, 2, torch.float32, spread=0.0).clamp(-2, 2) * 2.0 ** up).double()
    codes, scales = O.quantise(values(M, N, 3, spread=0.0).double() * 2.0 ** (-60 if up > 0 else 100))
    if vector == "mxfp4":
        v, v_scales = O.quantise(v)
        wide = O.dequantise(v, v_scales, N)
    else:
        v, v_scales = v.to(kind), None
        wide = v.double()
    m = O.dequantise(codes, scales, N)
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N), v_scales=v_scales).double()
    if vector == "mxfp4" and batch > 1:
        bound = gemm_bound(m, wide, torch.float32)
    else:
        # digits end at the smallest scale's half code: what is left of an element may also be 2^-129
        bound = gemv_bound(m, wide, vector == "fp32") if M < 9000 else \
            digits_bound(m, wide) + 2.0 ** -129 * m.abs().sum(1)
    assert bool(((got - wide @ m.T).abs() <= bound).all())


@pytest.mark.parametrize("vector,up", [("bf16", -130), ("fp32", -130), ("fp32", -140), ("fp32", -148)])
@pytest.mark.parametrize("M,N,batch", [(40, 256, 1), (40, 300, 1), (300, 30000, 1), (40, 256, 2), (40, 300, 5), (40, 256, 8)])
def test_gemv_subnormal_vectors_times_large_scales(M, N, batch, vector, up):
    # blocks of subnormal elements (steps of 2^-133 and 2^-149), against a matrix that makes ordinary numbers of them.  Such a
    # block is taken to FP16 without a rounding where its largest element is below 2^-127: the factor is 2^126, so the
    # elements are multiples of 2^-23 below 1/2, which two FP16 hold (BF16: multiples of 2^-7, one does)
    v = (values(batch, N, 2, torch.float32, spread=0.0).clamp(-2, 2).double() * 2.0 ** up).to(DTYPES[vector])
    assert bool((v != 0).any())
    codes, scales = O.quantise(values(M, N, 3, spread=0.0).double() * 2.0 ** 120)
    m, wide = O.dequantise(codes, scales, N), v.double()
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N)).double()
    assert bool(((got - wide @ m.T).abs() <= gemv_bound(m, wide, False)).all())


@pytest.mark.parametrize("batch", [1, 2, 5])
def test_gemv_one_element_at_the_far_ends(batch):
    # every row one code, every result one product: both factors' order must lose nothing that the result could hold
    N = 96
    exponents = [-149, -140, -126, -113, -112, -60, 0, 60, 113, 127]
    v = torch.zeros(len(exponents) * batch, N, device="cuda", dtype=torch.float64)
    for i, e in enumerate(exponents):
        v[i * batch:(i + 1) * batch, 40] = 2.0 ** e
        v[i * batch:(i + 1) * batch, 5] = 2.0 ** -e if e not in (-149, -140) else 1.0   # the far end in another block
    v = v.float()
    codes = torch.zeros(255, N // 2, dtype=torch.uint8, device="cuda")
    codes[:, 20] = 1                                   # 0.5 at column 40
    scales = torch.full((255, N // 32), 127, dtype=torch.uint8, device="cuda")
    scales[:, 1] = torch.arange(255, device="cuda").to(torch.uint8)
    want = v.double() @ O.dequantise(codes, scales, N).T
    for i in range(len(exponents)):
        got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v[i * batch:(i + 1) * batch], (255, N))
        assert torch.equal(got, want[i * batch:(i + 1) * batch].float())        # powers of two, rounded once at FP32's ends


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_several_vectors_infinite_where_the_matrix_is_nan_elsewhere(dtype):
    M, N = 9000, 4096
    codes, scales = packed(M, N, 1)
    scales = scales.clone()
    scales[5, 7] = 255                                # a NaN block the infinity does not meet
    scales[77, 2] = 255                               # one that it does
    v = values(3, N, 2, DTYPES[dtype], spread=1.0)
    v[1, 70] = float("inf")
    got = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, v, (M, N)).double()
    want = v.double() @ O.dequantise(codes, scales, N).T
    assert torch.equal(got.isnan(), want.isnan()) and bool(want[1, 5].isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])


# -------------------------------------------------------------------- gemm --
def gemm_bound(m, x, dtype):
    """Per element: N / 64 products in a row add into one FP32 sum, each may lose 2^-22 of the products' size so far (the
    tensor core does not round to nearest); one rounding to the output type."""
    steps = math.ceil(m.shape[1] / 64) + 1
    size = x.abs() @ m.abs().T
    return size * steps * 2.0 ** -22 + (x @ m.T).abs() * torch.finfo(dtype).eps / 2 * 1.001 + torch.finfo(dtype).tiny


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,N,batch", [(1, 1, 1), (128, 256, 32), (128, 64, 1), (130, 33, 7), (200, 1000, 40), (77, 2080, 64),
                                       (1000, 288, 100), (300, 5000, 129), (2048, 512, 225), (513, 1536, 449), (5000, 160, 300)])
def test_gemm(M, N, batch, dtype):
    codes, scales = packed(M, N, M + N, spread=1.0)
    x, x_scales = packed(batch, N, 5 * M + N, spread=1.0)
    got = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N), out_dtype=DTYPES[dtype])
    assert got.dtype == DTYPES[dtype] and got.shape == (batch, M)
    m, w = O.dequantise(codes, scales, N), O.dequantise(x, x_scales, N)
    bound = gemm_bound(m, w, DTYPES[dtype])
    err = (got.double() - w @ m.T).abs()
    assert bool((err <= bound).all()), (err / bound).max()
    assert torch.equal(got, fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N), out_dtype=DTYPES[dtype]))


def random_packed(rows, n, seed):
    """Codes and scales of whole blocks, drawn directly."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(0, 256, (rows, n // 2), generator=gen, device="cuda").to(torch.uint8),
            torch.randint(120, 134, (rows, n // 32), generator=gen, device="cuda").to(torch.uint8))


@pytest.mark.parametrize("M,N,batch", [(57001, 96, 16), (57000, 2080, 5), (57000, 96, 20), (57001, 96, 64), (57000, 2080, 40),
                                       (57000, 96, 100), (57001, 1056, 128), (20000, 2080, 384), (20001, 2080, 384), (20000, 2080, 672),
                                       (20001, 2080, 672), (20000, 1056, 672), (19980, 96, 700), (20004, 2080, 700)])
def test_gemm_several_tiles_per_cta(M, N, batch):
    # more than three tiles of 128 rows for each of 148 SMs, for every width of tile (16, 32, 64, 128 and 224 rows of x): the
    # rings, the scale groups (an odd number of them where N is 2080), the two accumulators and the pieces of the result go
    # on from tile to tile; rows of the result on and off the 16-byte grid; the last tiles ragged both ways
    codes, scales = random_packed(M, N, M + N)
    x, x_scales = random_packed(batch, N, 5 * M + N)
    m, w = O.dequantise(codes, scales, N), O.dequantise(x, x_scales, N)
    want, size = w @ m.T, w.abs() @ m.abs().T
    del m
    for dtype in DTYPES.values():
        out = torch.full((batch + 1, M), 7.0, dtype=dtype, device="cuda")
        got = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N), out_dtype=dtype, out=out[:batch])
        bound = size * (math.ceil(N / 64) + 1) * 2.0 ** -22 + want.abs() * torch.finfo(dtype).eps / 2 * 1.001 + torch.finfo(dtype).tiny
        top = torch.finfo(dtype).max                   # FP16 overflows where the value does
        err = (got.double().clamp(-top, top) - want.clamp(-top, top)).abs()
        assert bool((err <= bound).all()), (err / bound).max()
        assert bool((out[batch] == 7.0).all())
        assert torch.equal(got, fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N), out_dtype=dtype))


def test_gemm_every_place_and_scale_is_its_own():
    # one element and one scale at a time: a row or a scale in the wrong place shows as a wrong number
    M, N, batch = 256, 512, 256
    codes = torch.zeros(M, N // 2, dtype=torch.uint8, device="cuda")
    x = torch.full((batch, N // 2), 0x22, dtype=torch.uint8, device="cuda")       # ones
    k = (torch.arange(M, device="cuda") * 37) % N
    codes[torch.arange(M, device="cuda"), k // 2] = torch.where(k % 2 == 0, 2, 32).to(torch.uint8)   # a one at column k of each row
    gen = torch.Generator(device="cuda").manual_seed(2)
    scales = torch.randint(117, 138, (M, N // 32), generator=gen, device="cuda").to(torch.uint8)
    x_scales = torch.randint(117, 138, (batch, N // 32), generator=gen, device="cuda").to(torch.uint8)
    got = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N))
    e = scales[torch.arange(M, device="cuda"), k // 32].int()[None, :] + x_scales.int()[:, k // 32]
    assert torch.equal(got, torch.exp2((e - 254).float()))


def test_gemm_scales_of_the_whole_range():
    # one element per row, scales from 2^-127 to 2^127: sums inside FP32's normal range are exact, larger ones infinite,
    # smaller ones at most the smallest normal number off
    M, N, batch = 256, 256, 160
    codes = torch.zeros(M, N // 2, dtype=torch.uint8, device="cuda")
    k = (torch.arange(M, device="cuda") * 37) % N
    codes[torch.arange(M, device="cuda"), k // 2] = torch.where(k % 2 == 0, 2, 32).to(torch.uint8)
    x = torch.full((batch, N // 2), 0x22, dtype=torch.uint8, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    scales = torch.randint(0, 255, (M, N // 32), generator=gen, device="cuda").to(torch.uint8)
    x_scales = torch.randint(0, 255, (batch, N // 32), generator=gen, device="cuda").to(torch.uint8)
    got = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N))
    want = O.dequantise(x, x_scales, N) @ O.dequantise(codes, scales, N).T
    normal = (want >= 2.0 ** -126) & (want < 2.0 ** 128)
    assert torch.equal(got[normal].double(), want[normal]) and bool(got[want >= 2.0 ** 128].isinf().all())
    assert bool((got[want < 2.0 ** -126].double() <= 2.0 ** -126).all())


def test_gemm_nan_scales_stay_in_their_row():
    M, N, batch = 150, 320, 50
    codes, scales = packed(M, N, 1, spread=1.0)
    x, x_scales = packed(batch, N, 2, spread=1.0)
    scales, x_scales = scales.clone(), x_scales.clone()
    scales[7, 9], x_scales[31, 0] = 255, 255
    got = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, x, x_scales, (M, N))
    want = O.dequantise(x, x_scales, N) @ O.dequantise(codes, scales, N).T
    assert torch.equal(got.isnan(), want.isnan())


# ------------------------------------------------------------------ rotary --
def rotary_bound(x, positions, inv_freq, layout, scale, dtype):
    """Angle: |p f| 2^-51 and 2 pi 2^-26; sine and cosine 2^-23; two products and a sum; the output's rounding."""
    angle = positions.double().abs().max() * inv_freq.max() * 2.0 ** -51 + 2 * math.pi * 2.0 ** -26 + 2.0 ** -23 + 3 * 2.0 ** -24
    half = inv_freq.numel()
    size = torch.zeros_like(x, dtype=torch.float64)
    for i in range(half):
        a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
        size[..., a] = size[..., b] = scale * (x[..., a].double().abs() + x[..., b].double().abs())
    return size * angle + O.rotate(x, positions, inv_freq, layout, scale).abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,heads,dim,rotated,start", [(1, 1, 2, 2, 0), (1, 36, 64, 64, 100003), (5, 3, 80, 40, 7), (3, 2, 96, 34, 2 ** 20),
                                                            (130, 4, 128, 64, 2 ** 31 - 131), (17, 1, 1024, 1024, 50), (2, 5, 33, 6, 9),
                                                            (1300, 7, 80, 40, 3), (40, 2, 88, 24, 3)])
def test_rotary(tokens, heads, dim, rotated, start, dtype, layout):
    gen = torch.Generator(device="cuda").manual_seed(tokens + dim)
    x = torch.randn(tokens, heads, dim, generator=gen, device="cuda").to(DTYPES[dtype])
    inv = fb.rotary_frequencies(rotated)
    for kind in (torch.int64, torch.int32):
        pos = torch.arange(start, start + tokens, device="cuda").to(kind)
        got = fb.rotary_gpu(x, pos, inv, layout, scale=1.25)
        bound = rotary_bound(x, pos, inv, layout, 1.25, DTYPES[dtype])
        assert got.dtype == x.dtype and bool(((got.double() - O.rotate(x, pos, inv, layout, 1.25)).abs() <= bound).all())
        assert torch.equal(got[..., rotated:], x[..., rotated:])
    again = x.clone()
    assert fb.rotary_gpu(again, pos, inv, layout, scale=1.25, out=again) is again and torch.equal(again, got)


@pytest.mark.parametrize("mode,kind,half_step,tiny", [("E5M2", torch.float8_e5m2, 2.0 ** -3, 2.0 ** -17), ("E4M3", torch.float8_e4m3fn, 2.0 ** -4, 2.0 ** -10)])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,heads,dim,rotated,layout", [(1, 4, 64, 64, "half"), (33, 3, 128, 64, "interleaved"), (7, 2, 20, 6, "half"),
                                                              (50, 3, 80, 40, "interleaved"), (9, 1, 88, 24, "half")])
def test_rotary_packed(tokens, heads, dim, rotated, layout, dtype, mode, kind, half_step, tiny):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(tokens, heads, dim, generator=gen, device="cuda").to(DTYPES[dtype])
    pos, inv = torch.randint(0, 5000, (tokens,), generator=gen, device="cuda"), fb.rotary_frequencies(rotated)
    words = fb.rotary_gpu(x, pos, inv, layout, mode=mode)
    assert words.dtype == torch.uint32 and words.shape == (heads, tokens, dim // 4) and words.feather_mode == mode
    got = words.as_subclass(torch.Tensor).view(kind).double().transpose(0, 1)
    want = O.rotate(x, pos, inv, layout)
    slack = rotary_bound(x, pos, inv, layout, 1.0, torch.float32)
    assert bool(((got - want).abs() <= want.abs() * half_step + tiny + 2 * slack).all())
    # away from the borders the words are the packer's of the same values
    dense = fb.rotary_gpu(x.float(), pos, inv, layout).transpose(0, 1).contiguous()
    assert torch.equal(words.as_subclass(torch.Tensor).flatten().view(torch.int32), fb.pack_fp8_tensor(dense, mode).as_subclass(torch.Tensor).view(torch.int32))


@pytest.mark.parametrize("mode", ["E5M2", "E4M3"])
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_rotary_packs_every_pattern_like_the_packer(dtype, mode):
    # position 0 turns nothing and the second elements are zero, so the first ones are packed as they are: all 65536
    # FP16 patterns, as FP16 and widened, and in FP32 the neighbours of each
    x = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.float16)
    if dtype == "fp32":
        w = x.float().view(torch.int32)
        x = torch.cat((w, w + 1, w - 1)).view(torch.float32)
    heads = torch.zeros(1, x.numel() // 32, 64, dtype=x.dtype, device="cuda")
    heads[0, :, :32] = x.view(-1, 32)
    words = fb.rotary_gpu(heads, torch.zeros(1, dtype=torch.int64, device="cuda"), fb.rotary_frequencies(64), mode=mode)
    got = words.as_subclass(torch.Tensor).view(torch.uint8).view(-1, 64)[:, :32].flatten()
    want = fb.pack_fp8_tensor(x, mode).as_subclass(torch.Tensor).view(torch.uint8)
    nan = x.isnan()                                    # the sign of a NaN is not kept by arithmetic
    assert torch.equal(got[~nan], want[~nan]) and torch.equal(got[nan] & 127, want[nan] & 127)


def test_rotary_words_in_a_buffer_carry_their_mode():
    # one buffer for both modes, tagged, untagged and typed otherwise: the calls that go by the tag decode what it holds now
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(6, 2, 64, generator=gen, device="cuda")
    pos, inv = torch.arange(6, device="cuda"), fb.rotary_frequencies(64)
    ones = {m: fb.pack_fp8_tensor(torch.ones(64, device="cuda"), m) for m in ("E5M2", "E4M3")}
    tagged = fb.rotary_gpu(x, pos, inv, mode="E5M2")
    for buffer in (tagged, torch.empty(2, 6, 16, dtype=torch.uint32, device="cuda"), torch.empty(2 * 6 * 16, dtype=torch.int32, device="cuda")):
        for mode in ("E4M3", "E5M2", "E4M3"):
            fresh = fb.rotary_gpu(x, pos, inv, mode=mode)
            got = fb.rotary_gpu(x, pos, inv, mode=mode, out=buffer)
            assert got.data_ptr() == buffer.data_ptr() and got.feather_mode == mode
            assert torch.equal(got.as_subclass(torch.Tensor).flatten().view(torch.int32), fresh.as_subclass(torch.Tensor).flatten().view(torch.int32))
            words = got.view(2, 96)[0]
            assert torch.equal(fb.gemv(words, ones[mode].as_subclass(torch.Tensor), (6, 64)), fb.gemv(fresh[0], ones[mode], (6, 64)))
            if buffer is tagged:
                assert got is buffer and tagged.feather_mode == mode


def test_rotary_strides_and_padding_rows_left_alone():
    gen = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(9, 3, 4, 64, generator=gen, device="cuda", dtype=torch.float16)
    inv, pos = fb.rotary_frequencies(64), torch.arange(9, device="cuda")
    k = qkv[:, 1]                                             # a slice of a fused projection: strided tokens
    assert not k.is_contiguous() and torch.equal(fb.rotary_gpu(k, pos, inv), fb.rotary_gpu(k.contiguous(), pos, inv))
    heads_first = qkv[:, 0].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(fb.rotary_gpu(heads_first, pos, inv), fb.rotary_gpu(qkv[:, 0].contiguous(), pos, inv))
    odd = torch.empty(1 + 9 * 4 * 64, device="cuda", dtype=torch.float16)[1:].view(9, 4, 64).copy_(k)
    assert torch.equal(fb.rotary_gpu(odd, pos, inv), fb.rotary_gpu(k, pos, inv))
    out = torch.full((10, 4, 64), 7.0, device="cuda", dtype=torch.float16)
    fb.rotary_gpu(k, pos, inv, out=out[:9])
    assert bool((out[9] == 7.0).all())
    assert fb.rotary_gpu(qkv[:0, 0], pos[:0], inv).shape == (0, 4, 64)


# ---------------------------------------------------------------- together --
def test_projections_rotation_and_attention_together():
    """Weights packed to 4 bits, a prompt projected, queries and keys rotated and packed, attended, packed again and
    projected back: each step against the oracle on the step's own inputs, and one token's GEMV against the prompt's GEMM."""
    hidden, heads, dim, tokens = 512, 4, 64, 96
    gen = torch.Generator(device="cuda").manual_seed(0)
    w = [fb.pack_mxfp4_tensor(0.05 * torch.randn(heads * dim, hidden, generator=gen, device="cuda")) for _ in range(3)]
    wo = fb.pack_mxfp4_tensor(0.05 * torch.randn(hidden, heads * dim, generator=gen, device="cuda"))
    x = torch.randn(tokens, hidden, generator=gen, device="cuda").to(torch.bfloat16)
    xc, xs = fb.pack_mxfp4_tensor(x)
    q, k, v = (fb.gemm_mxfp4_acc_fp32_gpu(*m, xc, xs, (heads * dim, hidden)) for m in w)
    for m, y in zip(w, (q, k, v)):
        m64, x64 = O.dequantise(*m, hidden), O.dequantise(xc, xs, hidden)
        assert bool(((y.double() - x64 @ m64.T).abs() <= gemm_bound(m64, x64, torch.float32)).all())
        one = fb.gemv_mxfp4_acc_fp32_gpu(*m, xc[5], (heads * dim, hidden), v_scales=xs[5])
        size = (x64[5:6].abs() @ m64.abs().T)[0]
        assert bool(((one - y[5]).abs() <= size * 2.0 ** -18).all())
    inv, pos = fb.rotary_frequencies(dim), torch.arange(1000, 1000 + tokens, device="cuda")
    qp, kp = (fb.rotary_gpu(t.view(tokens, heads, dim), pos, inv, mode="E5M2") for t in (q, k))
    outs = []
    from feather_b200.routines.attention import flash_attention_fp8_e5m2_acc_fp32_gpu
    for h in range(heads):
        vh = fb.pack_fp8_tensor(v.view(tokens, heads, dim)[:, h].contiguous(), "E5M2")
        o = flash_attention_fp8_e5m2_acc_fp32_gpu(qp[h], kp[h], vh, tokens, dim // 4)
        f = [fb.unpack_fp8_tensor(t.contiguous(), "E5M2").view(tokens, dim).double() for t in (qp[h], kp[h], vh)]
        s = torch.zeros(tokens, 128, dtype=torch.float64, device="cuda")      # the last key tile is filled with zero scores
        s[:, :tokens] = f[0] @ f[1].T / dim ** 0.5
        want = torch.softmax(s, -1)[:, :tokens] @ f[2]
        assert bool(((o.double() - want).abs() <= 5e-4 * f[2].abs().max()).all())
        outs.append(o)
    oc, os_ = fb.pack_mxfp4_tensor(torch.cat(outs, -1))
    y = fb.gemm_mxfp4_acc_fp32_gpu(*wo, oc, os_, (hidden, heads * dim), out_dtype=torch.bfloat16)
    m64, x64 = O.dequantise(*wo, heads * dim), O.dequantise(oc, os_, heads * dim)
    assert bool(((y.double() - x64 @ m64.T).abs() <= gemm_bound(m64, x64, torch.bfloat16)).all())


def test_captured_and_replayed_on_another_stream():
    M, N = 300, 512
    w, large = packed(M, N, 1), packed(3000, 8 * N, 2)
    x = torch.randn(4, N, device="cuda")
    inv, pos = fb.rotary_frequencies(60), torch.arange(4, device="cuda")
    stream = torch.cuda.Stream()

    def chain():
        c, s = fb.pack_mxfp4_tensor(x)
        a = fb.gemm_mxfp4_acc_fp32_gpu(*w, c, s, (M, N))
        b = fb.gemv_mxfp4_acc_fp32_gpu(*w, x, (M, N))
        r = fb.rotary_gpu(a.view(4, 5, 60), pos, inv)
        d = fb.gemv_mxfp4_acc_fp32_gpu(*large, x.repeat(1, 8), (3000, 8 * N))      # the digits' workspace is the graph's
        return c, s, a, b, r, fb.unpack_mxfp4_tensor(c, s), d
    with torch.cuda.stream(stream):
        chain()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = chain()
    for seed in (1, 2):
        x.copy_(torch.randn(4, N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        pos += 3
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, chain()))


def test_two_streams_at_once():
    M, N = 3000, 4096
    w = packed(M, N, 1)
    jobs = []
    for i in range(2):
        x = torch.randn(6, N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i))
        want = [fb.gemv_mxfp4_acc_fp32_gpu(*w, x, (M, N)), fb.gemm_mxfp4_acc_fp32_gpu(*w, *fb.pack_mxfp4_tensor(x), (M, N))]
        jobs.append((torch.cuda.Stream(), x, want))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (stream, x, _) in enumerate(jobs):
            with torch.cuda.stream(stream):
                got[i] += [fb.gemv_mxfp4_acc_fp32_gpu(*w, x, (M, N)), fb.gemm_mxfp4_acc_fp32_gpu(*w, *fb.pack_mxfp4_tensor(x), (M, N))]
    torch.cuda.synchronize()
    for (_, _, want), ys in zip(jobs, got):
        assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(ys))


def test_packed_right_before_it_is_multiplied():
    # operands written by the call just before, several times over in the same buffers of the allocator
    M, N = 5000, 4096
    x = torch.randn(4, N, device="cuda")
    for seed in range(4):
        a = torch.randn(M, N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        torch.cuda.synchronize()
        codes, scales = fb.pack_mxfp4_tensor(a)
        y = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x, (M, N))
        z = fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, *fb.pack_mxfp4_tensor(x), (M, N))
        one = fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x[0], (M, N))
        torch.cuda.synchronize()
        assert torch.equal(y, fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x, (M, N)))
        assert torch.equal(z, fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, *fb.pack_mxfp4_tensor(x), (M, N)))
        assert torch.equal(one, fb.gemv_mxfp4_acc_fp32_gpu(codes, scales, x[0], (M, N)))


def test_refusals_on_the_gpu():
    codes, scales = packed(8, 64, 1)
    x = torch.randn(64, device="cuda")
    ok = dict(m_codes=codes, m_scales=scales, v=x, m_shape=(8, 64))
    fb.gemv_mxfp4_acc_fp32_gpu(**ok)
    for bad in (dict(v=x[:63]), dict(v=torch.randn(1, 2, 64, device="cuda")), dict(v=torch.randn(128, device="cuda")[::2]),
                dict(m_shape=(9, 64)), dict(m_shape=(8, 65)), dict(m_scales=scales[:4]), dict(m_codes=codes[:, ::2]),
                dict(out=torch.empty(9, device="cuda")), dict(out=torch.empty(8, device="cuda", dtype=torch.float16)),
                dict(v=torch.randn(65, 64, device="cuda")), dict(v_scales=scales[0]), dict(v=x.cpu()),
                dict(m_scales=torch.zeros(8, 3, dtype=torch.uint8, device="cuda")), dict(m_codes=torch.zeros(8, 33, dtype=torch.uint8, device="cuda")),
                dict(m_codes=torch.zeros(8 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(8, 32))):
        with pytest.raises(ValueError):
            fb.gemv_mxfp4_acc_fp32_gpu(**{**ok, **bad})
    with pytest.raises(TypeError):
        fb.gemv_mxfp4_acc_fp32_gpu(**{**ok, "v": x.double()})
    with pytest.raises(ValueError):
        fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, codes[:, :16].contiguous(), scales, (8, 64))
    with pytest.raises(ValueError):
        fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, codes, scales[:7], (8, 64))
    h, inv, pos = torch.randn(4, 2, 64, device="cuda"), fb.rotary_frequencies(64), torch.arange(4, device="cuda")
    for bad in (dict(x=h[0]), dict(positions=pos[:3]), dict(positions=pos.float()), dict(inv_freq=inv.float()), dict(inv_freq=inv.repeat(2)),
                dict(inv_freq=inv[:0]), dict(x=h.transpose(1, 2)), dict(out=torch.empty(4, 2, 64, device="cuda", dtype=torch.float16)),
                dict(x=h[..., :62], inv_freq=inv[:31], mode="E5M2")):
        with pytest.raises(ValueError):
            fb.rotary_gpu(**{**dict(x=h, positions=pos, inv_freq=inv), **bad})
    assert bool((fb.gemv_mxfp4_acc_fp32_gpu(codes[:, :0].contiguous(), scales[:, :0].contiguous(), x[:0], (8, 0)) == 0).all())
    assert fb.gemv_mxfp4_acc_fp32_gpu(codes[:0], scales[:0], x, (0, 64)).shape == (0,)
    assert fb.gemm_mxfp4_acc_fp32_gpu(codes, scales, codes[:0], scales[:0], (8, 64)).shape == (0, 8)
