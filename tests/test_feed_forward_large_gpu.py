"""Layer norm, the gated product and the block-scaled operators on matrices of more than 2^31
values: the rows around the 2^31st value and at both ends against the formulas in 64 bits."""
import gc

import pytest
import torch

from test_block_codes_gpu import codes_ref, same, spread
from test_gated_gpu import act_ref, slope_ref
from test_layernorm_gpu import check_grad, ref
from test_layers_gpu import BF16, E4M3, F16, F32, HALF_TINY, HALF_ULP, U, close, d, randn
from vcsr_b200 import layers as L

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def freed():
    yield
    gc.collect()
    torch.cuda.empty_cache()


def looked_at(rows, pitch):
    mid = 2 ** 31 // pitch
    assert mid + 2 < rows - 1
    return [0, 1, mid - 1, mid, mid + 1, rows - 2, rows - 1]


def big(rows, cols, dtype, seed=0, scale=1.0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.empty(rows, cols + pad, device="cuda", dtype=dtype)
    for part in t.split(1 << 15):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
    return t[:, :cols]


def only(t, rows):
    """t with zeros in all rows but these."""
    keep = t[rows].clone()
    t.zero_()
    t[rows] = keep
    return t


@gpu
@pytest.mark.parametrize("rows,dim,dtype,pad", [(270000, 8000, BF16, 0), (270000, 8001, F16, 0), (540000, 4001, F32, 0),
                                                (270000, 8000, BF16, 1), (54000, 40000, BF16, 0), (90000001, 24, BF16, 0)])
def test_layernorm(rows, dim, dtype, pad):
    look = looked_at(rows, dim)
    x, w, b = big(rows, dim, dtype, 1, pad=pad), randn(dim, dtype=dtype, seed=3), randn(dim, dtype=dtype, seed=4)
    out = L.layernorm(x, w, b, residual=x, eps=1e-5, save_stats=True)
    s, mean, rstd, y, off_mean, off_rstd, off_y = ref(x[look], w, b, x[look], 1e-5)
    close(out.mean[look], mean, off_mean)
    close(out.rstd[look], rstd, off_rstd)
    close(out.y[look], y, off_y)
    close(out.sum[look], s, U * s.abs())
    s, dy = out.sum, only(out.y, look)
    del x
    g = L.layernorm_backward(dy, s, w, out.mean, out.rstd, dsum=s)
    check_grad(dy[look], s[look], w, out.mean[look], out.rstd[look], s[look], g._replace(dx=g.dx[look]))


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32, E4M3])
def test_gated_outputs(dtype):
    M, N, K = 270000, 4000, 16
    look = looked_at(M, 2 * N)
    x, w = big(M, K, dtype, 1), randn(2 * N, K, dtype=dtype, seed=2)
    scales = dict(x_scale=torch.ones(M, device="cuda"), w_scale=torch.ones(2 * N, device="cuda")) if dtype == E4M3 else {}
    out = L.gated_linear(x, w, act="relu", save_pre=True, **scales)
    xd, wd = d(x[look].float()), d(w.float())
    z, slack = xd @ wd.t(), (2 * K + 8) * U * (xd.abs() @ wd.abs().t())
    close(out.pre[look], z, slack)
    a, u = z[:, :N].clamp_min(0), z[:, N:]
    close(out.y[look], a * u, slack[:, :N] * (u.abs() + slack[:, N:]) + (a + slack[:, :N]) * slack[:, N:] + 4 * U * (a * u).abs())
    L.check()


@gpu
@pytest.mark.parametrize("dtype,act", [(BF16, "silu"), (F32, "relu")])
@pytest.mark.parametrize("N", [4000, 4001])
def test_gated_backward(dtype, act, N):
    M, K = 270000, 16
    look = looked_at(M, 2 * N)
    dy, pre = only(big(M, N, dtype, 1), look), big(M, 2 * N, dtype, 2)
    x, w = big(M, K, dtype, 3), randn(2 * N, K, dtype=dtype, seed=4)
    got = L.gated_linear_backward(dy, x, w, pre, act=act)
    L.check()
    e, g, u = d(dy[look]), d(pre[look])[:, :N], d(pre[look])[:, N:]
    dz = torch.cat([e * u * slope_ref(g, act), e * act_ref(g, act)], 1)
    unit = 16 * U + (2.0 ** -12 if dtype != F32 else 0)
    off = unit * torch.cat([(e * u).abs() * (1 + g.abs()), e.abs() * g.abs()], 1)
    rounded = off + (HALF_ULP[dtype] * dz.abs() + HALF_TINY[dtype] if dtype != F32 else 0)
    close(got.dx[look], dz @ d(w), (rounded + (4 * N + 4) * U * dz.abs()) @ d(w).abs())
    # all other rows add zeros
    close(got.dw, dz.t() @ d(x[look]), (rounded + 20 * U * dz.abs()).t() @ d(x[look]).abs())
    close(got.db, dz.sum(0), (off + 20 * U * dz.abs()).sum(0))
    rest = torch.ones(M, dtype=torch.bool, device="cuda")
    rest[look] = False
    assert not got.dx[rest].any()


@gpu
@pytest.mark.parametrize("K", [16000, 16001])
@pytest.mark.parametrize("which", ["x", "w"])
@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_gated_operands(K, which, dtype):
    """Operands of more than 2^31 values, read as they are and as aligned copies."""
    M, N = (140000, 8) if which == "x" else (8, 70000)
    look = looked_at(max(M, 2 * N), K)
    x, w = big(M, K, dtype, 1), big(2 * N, K, dtype, 2, scale=0.01 if dtype == BF16 else 1.0)
    scales = dict(x_scale=torch.ones(M, device="cuda"), w_scale=torch.full((2 * N,), 0.01, device="cuda")) if dtype == E4M3 else {}
    pre = L.gated_linear(x, w, act="relu", save_pre=True, **scales).pre
    L.check()
    if which == "x":
        x, pre = x[look], pre[look]
    else:
        w, pre = w[look], pre[:, look]
    xd, wd = d(x.float()), d(w.float()) * (0.01 if dtype == E4M3 else 1)
    close(pre, xd @ wd.t(), (2 * K + 8) * U * (xd.abs() @ wd.abs().t()))


@gpu
@pytest.mark.parametrize("rows,dim,dtype", [(270000, 8000, BF16), (270000, 8001, F32)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_block_codes(rows, dim, dtype, block_rows):
    x = big(rows, dim, dtype, 1)
    q = L.block_quantize(x, block_rows)
    values = L.block_dequantize(q.codes, q.scale, block_rows, BF16)
    for first in (0, 2 ** 31 // dim // 128 * 128, (rows - 1) // 128 * 128):
        at = slice(first, min(first + 128, rows))
        codes, scale = codes_ref(x[at], block_rows)
        down = slice(first // block_rows, first // block_rows + len(scale))
        assert same(q.scale[down], scale) and same(q.codes[at], codes)
        v = d(codes.float()) * d(spread(scale, len(codes), dim, block_rows))
        close(values[at], v, 2 * U * v.abs())


@gpu
@pytest.mark.parametrize("M,N,K", [(270000, 8000, 128), (140000, 8, 16000), (140000, 8, 16001), (8, 140000, 16000)])
def test_block_product(M, N, K):
    look = looked_at(max(M, N), N if K == 128 else K)
    x, w = (big(r, K, E4M3, i, scale=60.0) for i, r in enumerate((M, N)))
    xs, ws = (big(-(-r // b), -(-K // 128), F32, i + 2).exp_().mul_(0.01) for i, (r, b) in enumerate(((M, 1), (N, 128))))
    r = big(M, N, BF16, 5) if K == 128 else None
    y = L.block_linear(x, w, xs, ws, residual=r)
    L.check()
    wd_scale = ws.repeat_interleave(128, 0)[:N]
    if M > N:
        x, xs, y = x[look], xs[look], y[look]
        r = r[look] if r is not None else None
    else:
        w, wd_scale, y = w[look], wd_scale[look], y[:, look]
    xd = d(x.float()) * d(spread(xs, len(x), K, 1))
    wd = d(w.float()) * d(wd_scale.repeat_interleave(128, 1)[:, :K])
    z = xd @ wd.t() + (d(r) if r is not None else 0)
    close(y, z, (2 * 128 + 2 * (K // 128) + 12) * U * (xd.abs() @ wd.abs().t()) + 8 * U * z.abs())
