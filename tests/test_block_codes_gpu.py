"""8-bit operands with a scale for each block of 128: codes, values and the product."""
import pytest
import torch

import vcsr_b200 as V
from test_layers_gpu import BF16, E4M3, F16, F32, U, act_ref, busy, close, d, randn
from vcsr_b200 import layers as L

gpu = pytest.mark.gpu
B = 128


def spread(scale, rows, dim, block_rows):
    full = scale.repeat_interleave(block_rows, 0)[:rows]
    return full.repeat_interleave(B, 1)[:, :dim]


def codes_ref(x, block_rows):
    """Codes and scales in FP32 torch operations, which round as the kernel has to."""
    rows, dim = x.shape
    down, across = -(-rows // block_rows), -(-dim // B)
    padded = torch.zeros(down * block_rows, across * B, device=x.device)
    padded[:rows, :dim] = x.float()
    scale = padded.view(down, block_rows, across, B).abs().amax((1, 3)) * torch.tensor(1 / 448, device=x.device)
    divisor = torch.where(scale > 0, scale, torch.ones_like(scale))
    # a scale that underflows to few bits may be below max / 448: codes stop at 448
    return (x.float() / spread(divisor, rows, dim, block_rows)).clamp(-448, 448).to(E4M3), scale


def same(a, b):  # zeros' signs apart
    return torch.equal(a.float(), b.float())


SHAPES = [(1, 1), (1, 128), (3, 127), (5, 129), (17, 8), (128, 128), (129, 257), (64, 1000), (300, 384), (1, 4096),
          (1000, 136), (260, 2500)]


@gpu
@pytest.mark.parametrize("rows,dim", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1), (16, 16)])
def test_codes_bit_for_bit(rows, dim, dtype, block_rows, pad, offset):
    x = randn(rows, dim, dtype=dtype, seed=1, pad=pad, offset=offset)
    x[rows // 2] *= 100
    x[0, :B] = 0
    got = L.block_quantize(x, block_rows)
    codes, scale = codes_ref(x, block_rows)
    assert got.scale.shape == scale.shape and same(got.scale, scale) and same(got.codes, codes)
    values = d(codes.float()) * d(spread(scale, rows, dim, block_rows))
    for out in (F32, BF16, F16):
        close(L.block_dequantize(got.codes, got.scale, block_rows, out), values, 2 * U * values.abs())


@gpu
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("size", [1e-42, 1e-36, 1e-30, 1e-3, 1e30, 3e38])
def test_codes_of_tiny_and_huge_blocks(block_rows, size):
    x = randn(130, 260, seed=1).clamp(-1, 1) * size
    got = L.block_quantize(x, block_rows)
    codes, scale = codes_ref(x, block_rows)
    assert same(got.scale, scale) and same(got.codes, codes)


@gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_codes_of_ties(block_rows):
    """Scales that are powers of two leave exact ties, which go to the even code."""
    x = (torch.arange(0, 449 * 32, 7, device="cuda") / 32).view(1, -1)[:, :2048].repeat(3, 1)
    x[:, ::B] = 448.0
    got = L.block_quantize(x, block_rows)
    codes, scale = codes_ref(x, block_rows)
    assert bool((scale[0, :2] == 1).all()) and same(got.codes, codes) and same(got.scale, scale)


@gpu
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_not_finite_stays_in_its_block(block_rows, bad):
    x = randn(200, 400, seed=1)
    want = L.block_quantize(x, block_rows)
    x[130, 200] = bad
    got = L.block_quantize(x, block_rows)
    hit = torch.zeros_like(got.scale, dtype=torch.bool)
    hit[130 // block_rows, 1] = True
    assert torch.equal(~got.scale.isfinite(), hit) and got.scale[hit].isnan().item() == (bad != bad)
    assert torch.equal(got.scale[~hit], want.scale[~hit])
    inside = spread(hit, 200, 400, block_rows)
    assert torch.equal(got.codes.float()[~inside], want.codes.float()[~inside])
    assert bool(L.block_dequantize(got.codes, got.scale, block_rows)[inside].isnan().all())


@gpu
def test_codes_of_nothing():
    for rows, dim in ((0, 5), (5, 0)):
        for block_rows in (1, 128):
            q = L.block_quantize(randn(rows, dim), block_rows)
            assert q.codes.shape == (rows, dim) and q.scale.numel() == 0
            assert L.block_dequantize(q.codes, q.scale, block_rows).shape == (rows, dim)


def operands(M, N, K, pads=(0, 0, 0, 0), offset=0):
    """Codes over the whole range with scales from 1e-3 to 10 in size."""
    def codes(rows, pad, seed):
        v = torch.zeros(rows * (K + pad) + offset, device="cuda").to(E4M3)[offset:].view(rows, K + pad)[:, :K]
        v.copy_(randn(rows, K, seed=seed, scale=60.0).clamp(-448, 448))
        return v

    def scales(rows, pad, seed):
        return randn(rows, -(-K // B), seed=seed, pad=pad).exp_().mul_(0.01)

    return codes(M, pads[0], 1), codes(N, pads[1], 2), scales(M, pads[2], 3), scales(-(-N // B), pads[3], 4)


def check_product(M, N, K, out_dtype=BF16, act=None, bias=False, residual=False, pads=(0, 0, 0, 0), offset=0, out_pad=0):
    x, w, xs, ws = operands(M, N, K, pads, offset)
    b = randn(N, dtype=out_dtype, seed=5) if bias else None
    r = randn(M, N, dtype=out_dtype, seed=6, pad=out_pad) if residual else None
    y = randn(M, N, dtype=out_dtype, seed=7, pad=out_pad, offset=offset)
    got = L.block_linear(x, w, xs, ws, bias=b, residual=r, act=act, out=y)
    assert got is y
    xd = d(x.float()) * d(spread(xs, M, K, 1))
    wd = d(w.float()) * d(spread(ws, N, K, B))
    z = xd @ wd.t()
    # a block's 128 products in the tensor core, then a scale (rounded once), a product and
    # an addition per block
    slack = (2 * B + 2 * (K // B) + 12) * U * (xd.abs() @ wd.abs().t()) + (2 * U * d(b).abs() if bias else 0)
    if bias:
        z = z + d(b)
    a = act_ref(z, act)
    fast = 2.0 ** -13 if out_dtype != F32 and act in ("gelu", "silu") else 0
    ref = a + (d(r) if residual else 0)
    close(got, ref, 1.13 * slack + 8 * U * (z.abs() + ref.abs()) + fast * a.abs())
    if out_pad and M > 1:
        gaps = y.as_strided((M - 1, out_pad), (N + out_pad, 1), y.storage_offset() + N)
        assert bool((gaps.float() == 77.0).all())
    L.check()


SIZES = [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 129, 72), (3, 128, 128), (5, 257, 129), (8, 256, 512), (15, 40, 16),
         (16, 128, 1280), (17, 512, 640), (31, 200, 136), (33, 384, 264), (63, 127, 64), (64, 128, 1024), (65, 130, 200),
         (100, 96, 2048), (127, 255, 65), (128, 128, 256), (129, 1, 33), (200, 777, 150), (255, 256, 384), (257, 300, 88),
         (513, 128, 128), (1001, 63, 100), (2048, 640, 320), (1, 8192, 8192), (4, 130, 40000)]


@gpu
@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_product_sizes(M, N, K, out_dtype):
    check_product(M, N, K, out_dtype, bias=N % 2 == 0, residual=M % 2 == 1)


@gpu
@pytest.mark.parametrize("M,N,K", [(2600, 1000, 1111), (4000, 4096, 512), (9000, 260, 130), (3000, 3000, 3000)])
def test_product_many_tiles(M, N, K):
    check_product(M, N, K, act="gelu", bias=True, residual=True)


@gpu
@pytest.mark.parametrize("M", [5, 300, 4100])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
def test_product_epilogues(M, out_dtype, act):
    check_product(M, 600, 300, out_dtype, act, bias=True, residual=True)


@gpu
@pytest.mark.parametrize("M", [6, 130, 4100])
@pytest.mark.parametrize("pads,offset,out_pad", [((1, 0, 0, 3), 0, 3), ((16, 16, 5, 2), 16, 16), ((0, 3, 1, 0), 1, 1), ((0, 0, 0, 0), 0, 4)])
def test_product_strided(M, pads, offset, out_pad):
    check_product(M, 520, 272, pads=pads, offset=offset, out_pad=out_pad, residual=True)


@gpu
def test_product_residual_in_place():
    for M in (3, 5000):
        x, w, xs, ws = operands(M, 520, 384)
        r = randn(M, 520, dtype=BF16, seed=6)
        want = L.block_linear(x, w, xs, ws, residual=r)
        assert L.block_linear(x, w, xs, ws, residual=r, out=r) is r and torch.equal(r, want)


@gpu
def test_product_over_nothing():
    for M, N, K in ((3, 20, 0), (0, 20, 16), (3, 0, 16)):
        x, w, xs, ws = operands(M, N, K)
        b, r = randn(N, dtype=BF16, seed=5), randn(M, N, dtype=BF16, seed=6)
        close(L.block_linear(x, w, xs, ws, bias=b, residual=r), d(b) + d(r), 2 * U * (d(b).abs() + d(r).abs()))


@gpu
@pytest.mark.parametrize("M", [3, 300, 5000])
def test_product_not_finite(M):
    """A NaN code, and scales that are not finite, reach the outputs that read them."""
    N, K = 300, 400
    x, w, xs, ws = operands(M, N, K)
    want = d(L.block_linear(x, w, xs, ws, out_dtype=F32))
    x[1, 300], xs[0, 2], ws[1, 0] = float("nan"), float("nan"), float("nan")
    got = d(L.block_linear(x, w, xs, ws, out_dtype=F32))
    hit = torch.zeros(M, N, dtype=torch.bool)
    hit[:2], hit[:, 128:256] = True, True
    assert torch.equal(got.isnan(), hit) and torch.equal(got[~hit], want[~hit])


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 8192, 4096), (130, 512, 1024), (4096, 4096, 640)])
def test_product_repeats_bit_for_bit(M, N, K):
    x, w, xs, ws = operands(M, N, K)
    first = L.block_linear(x, w, xs, ws)
    for _ in range(5):
        assert torch.equal(L.block_linear(x, w, xs, ws), first)


@gpu
@pytest.mark.parametrize("M,N,K", [(4, 256, 1024), (33, 200, 4096), (300, 128, 64), (4096, 4096, 1024), (4096, 2048, 128)])
def test_a_wait_that_runs_out_is_reported(M, N, K):
    x, w, xs, ws = operands(M, N, K)
    want = L.block_linear(x, w, xs, ws)
    L.check()
    L.test_withhold_signal()
    L.block_linear(x, w, xs, ws)
    with pytest.raises(V.VcsrError) as e:
        L.check()
    assert e.value.status == 7 and "accumulator-full" in e.value.msg
    L.check()
    assert torch.equal(L.block_linear(x, w, xs, ws), want)
    L.check()


@gpu
@pytest.mark.parametrize("raw", [False, True])
def test_blocks_on_the_given_stream(raw):
    side = torch.cuda.Stream()
    x, w = randn(640, 512, dtype=BF16, seed=1), randn(256, 512, seed=2)

    def chain(x, **kw):
        q, k = L.block_quantize(x, **kw), L.block_quantize(w, 128, **kw)
        return L.block_linear(q.codes, k.codes, q.scale, k.scale, **kw), L.block_dequantize(q.codes, q.scale, **kw)

    busy(side)
    want = chain(x)
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    busy(side)
    with torch.cuda.stream(side):
        late.copy_(x)
    got = chain(late, stream=side.cuda_stream if raw else side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_block_refusals():
    x, w = randn(4, 200), randn(130, 200)
    q, k = L.block_quantize(x), L.block_quantize(w, 128)

    def refused(status, fn, *args, **kw):
        with pytest.raises(V.VcsrError) as e:
            fn(*args, **kw)
        assert e.value.status == status, e.value

    refused(1, L.block_quantize, x.cpu())
    refused(1, L.block_quantize, x[0])
    refused(5, L.block_quantize, x.double())
    refused(5, L.block_quantize, q.codes)
    refused(5, L.block_quantize, x, 64)
    refused(5, L.block_quantize, x, None)
    refused(1, L.block_dequantize, q.codes, q.scale[:3])
    refused(1, L.block_dequantize, q.codes, q.scale, 128)
    refused(5, L.block_dequantize, x, q.scale)
    refused(5, L.block_dequantize, q.codes, q.scale, out_dtype=E4M3)
    refused(1, L.block_linear, q.codes, k.codes, q.scale, k.scale[:1])
    refused(1, L.block_linear, q.codes, k.codes, q.scale[:, :1], k.scale)
    refused(1, L.block_linear, q.codes, k.codes, None, k.scale)
    refused(1, L.block_linear, q.codes, k.codes[:, :199], q.scale, k.scale)
    refused(5, L.block_linear, x, w, q.scale, k.scale)
    refused(5, L.block_linear, q.codes, k.codes, q.scale, k.scale.half())
    refused(5, L.block_linear, q.codes, k.codes, q.scale, k.scale, out_dtype=E4M3)
    refused(5, L.block_linear, q.codes, k.codes, q.scale, k.scale, act="tanh")
    refused(1, L.block_linear, q.codes, k.codes, q.scale, k.scale, bias=randn(129, dtype=BF16))
    refused(5, L.block_linear, q.codes, k.codes, q.scale, k.scale, residual=randn(4, 130))
    refused(1, L.block_linear, q.codes, k.codes, q.scale, k.scale, out=randn(130, 4, dtype=BF16).t())
