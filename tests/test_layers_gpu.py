"""The dense layer operators against their formulas in 64 bits.

Tolerances are bounds, not fits.  u = 2^-24 is FP32's unit roundoff; a result
stored in 16 bits adds half a unit in its last place (half of finfo.eps of its
value, 2^-8 for bfloat16 and 2^-11 for float16, and half the spacing of its
subnormals).  A sum of
K products in FP32, in any order, is off by at most K u sum|terms| (2 K u where
the accumulator truncates, as a tensor core's may)."""
import math

import pytest
import torch

import vcsr_b200 as V
from vcsr_b200 import layers as L

gpu = pytest.mark.gpu
F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
U = 2.0 ** -24
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
HALF_TINY = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}


def randn(*shape, dtype=F32, seed=0, scale=1.0, pad=0, offset=0):
    """A (rows, cols) tensor whose rows are `pad` values apart and which starts
    `offset` values into its storage."""
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(*shape, generator=g) * scale).to(dtype)
    if len(shape) == 1:
        buf = torch.zeros(shape[0] + offset, dtype=dtype, device="cuda")
        buf[offset:] = t.cuda()
        return buf[offset:]
    rows, cols = shape
    buf = torch.full((rows * (cols + pad) + offset,), 77.0, device="cuda").to(dtype)
    v = buf[offset:].view(rows, cols + pad)[:, :cols] if rows else buf[offset:].view(0, cols + pad)[:, :cols]
    v.copy_(t.cuda())
    return v


def d(t):
    return None if t is None else t.detach().double().cpu()


def close(got, ref, slack, dtype=None):
    """|got - ref| <= slack + one rounding to dtype, elementwise."""
    dtype = dtype or got.dtype
    got = d(got)
    assert got.shape == ref.shape
    bound = slack + HALF_ULP[dtype] * (ref.abs() + slack) + HALF_TINY[dtype]
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((got - ref).abs() - bound)[bad].max()))


# ----------------------------------------------------------------------- norm

def norm_ref(x, w, r, eps):
    s = d(x) + (d(r) if r is not None else 0)
    rstd = 1 / torch.sqrt((s * s).mean(1) + eps)
    return s, rstd, s * rstd[:, None] * d(w)


# from one value to rows that need a block's registers (8192, 16384) or passes
# (16500 single values, 40000); odd lengths take single-value access
NORM_SIZES = [(1, 1), (3, 7), (5, 16), (2, 32), (129, 33), (1000, 128), (7, 100), (33, 1000), (4, 1024),
              (1, 4096), (300, 4104), (9, 8192), (5, 8193), (3, 16384), (2, 16500), (3, 32768), (2, 40000)]


@gpu
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32), (F16, F16)])
def test_rmsnorm(rows, dim, x_dtype, y_dtype):
    x, r = randn(rows, dim, dtype=x_dtype, seed=1), randn(rows, dim, dtype=x_dtype, seed=2)
    w = randn(dim, dtype=F32 if dim % 2 else x_dtype, seed=3)
    for res in (None, r):
        out = L.rmsnorm(x, w, residual=res, eps=1e-5, out_dtype=y_dtype, save_rstd=True)
        s, rstd, y = norm_ref(x, w, res, 1e-5)
        # the mean is off by at most (dim + 2) u of itself, its root by half of
        # that; in practice far less: 64 partial sums of at most dim / 32 terms
        rel = (dim / 32 + 40) * U
        close(out.rstd, rstd, rel * rstd)
        close(out.y, y, (rel + 4 * U) * y.abs())
        if res is None:
            assert out.sum is x
        else:
            close(out.sum, s, U * s.abs())


# rows shorter than a 16-byte access, and enough odd ones to start everywhere in it
@gpu
@pytest.mark.parametrize("rows,dim", [(20, 1), (9, 3), (31, 5), (700, 17), (33, 1001), (9, 2051), (17, 6003)])
@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, BF16), (BF16, F32), (F16, F16), (BF16, E4M3)])
@pytest.mark.parametrize("pad", [0, 2])
def test_rmsnorm_odd_rows(rows, dim, x_dtype, y_dtype, pad):
    x, r = randn(rows, dim, dtype=x_dtype, seed=1, pad=pad), randn(rows, dim, dtype=x_dtype, seed=2, pad=pad)
    w, y = randn(dim, seed=3, offset=1), randn(rows, dim, dtype=BF16, pad=pad).to(y_dtype)
    if pad:
        y = torch.zeros(rows, dim + pad, device="cuda").to(y_dtype)[:, :dim]
    sums = randn(rows, dim, dtype=x_dtype, pad=pad)
    out = L.rmsnorm(x, w, residual=r, out=y, sum_out=sums, save_rstd=True)
    s, rstd, ref = norm_ref(x, w, r, 1e-6)
    close(sums, s, U * s.abs())
    rel = (dim / 32 + 48) * U
    if y_dtype == E4M3:
        top = ref.abs().amax(1)
        step = torch.maximum(ref.abs() * 2.0 ** -4, (top / 448 * 2.0 ** -10)[:, None]) * (1 + 2.0 ** -10)
        assert bool(((d(y.float()) * d(out.scale)[:, None] - ref).abs() <= step + rel * ref.abs()).all())
    else:
        close(y, ref, rel * ref.abs())
        dy, ds = randn(rows, dim, dtype=y_dtype, seed=5, pad=pad), randn(rows, dim, dtype=x_dtype, seed=6, pad=pad)
        dx, dw = L.rmsnorm_backward(dy, sums, w, out.rstd, dsum=ds)
        rx, rw, h, g = norm_grad_ref(dy, sums, w, out.rstd, ds)
        terms = (g * h).abs().mean(1, keepdim=True)
        mag = d(out.rstd)[:, None] * (g.abs() + h.abs() * terms * (dim / 32 + 40)) + d(ds).abs()
        close(dx, rx, 8 * U * mag)
        close(dw, rw, (rows + 4) * U * (d(dy) * h).abs().sum(0))
    if pad and rows > 1:  # what lies between the rows is untouched
        gaps = sums.as_strided((rows - 1, pad), (dim + pad, 1), sums.storage_offset() + dim)
        assert bool((gaps == 77.0).all())


@gpu
@pytest.mark.parametrize("x_dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", [(1, 0), (8, 0), (0, 1), (8, 4), (3, 5)])
def test_rmsnorm_strided(x_dtype, pad, offset):
    rows, dim = 37, 256
    x = randn(rows, dim, dtype=x_dtype, seed=1, pad=pad, offset=offset)
    r = randn(rows, dim, dtype=x_dtype, seed=2, pad=pad)
    w = randn(dim, dtype=x_dtype, seed=3, offset=offset)
    y = randn(rows, dim, dtype=BF16, pad=pad, offset=offset)
    keep = y.clone()
    sums = randn(rows, dim, dtype=x_dtype, pad=pad)
    got = L.rmsnorm(x, w, residual=r, out=y, sum_out=sums, eps=0.0)
    s, rstd, ref = norm_ref(x, w, r, 0.0)
    assert got.y is y and got.sum is sums and not torch.equal(keep, y)
    close(y, ref, 60 * U * ref.abs())
    close(sums, s, U * s.abs())
    if pad:  # what lies between the rows is untouched
        gaps = y.as_strided((rows - 1, pad), (dim + pad, 1), y.storage_offset() + dim)
        assert bool((gaps == torch.tensor(77.0).to(BF16).item()).all())


@gpu
@pytest.mark.parametrize("dim", [64, 1000, 1001, 40000])
@pytest.mark.parametrize("which", ["x", "residual"])
def test_rmsnorm_sum_in_place(dim, which):
    x, r, w = randn(11, dim, seed=1), randn(11, dim, seed=2), randn(dim, seed=3)
    s, rstd, ref = norm_ref(x, w, r, 1e-6)
    out = L.rmsnorm(x, w, residual=r, sum_out=x if which == "x" else r)
    close(out.y, ref, (dim / 32 + 44) * U * ref.abs())
    close(x if which == "x" else r, s, U * s.abs())


@gpu
@pytest.mark.parametrize("rows,dim", [(1, 16), (5, 128), (40, 1000), (3, 1001), (17, 4096), (2, 40000)])
@pytest.mark.parametrize("x_dtype", [F32, BF16, F16])
def test_rmsnorm_codes(rows, dim, x_dtype):
    x, r, w = randn(rows, dim, dtype=x_dtype, seed=1), randn(rows, dim, dtype=x_dtype, seed=2), randn(dim, seed=3)
    x[0] = 0
    r[0] = 0  # a row of zeros has scale 0
    out = L.rmsnorm(x, w, residual=r, out_dtype=E4M3)
    _, _, y = norm_ref(x, w, r, 1e-6)
    rel = (dim / 32 + 48) * U
    top = y.abs().amax(1)
    close(out.scale, top / 448, rel * top / 448)
    assert out.scale[0] == 0 and bool((out.y[0].float() == 0).all())
    # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale near zero)
    step = torch.maximum(y.abs() * 2.0 ** -4, (top / 448 * 2.0 ** -10)[:, None]) * (1 + 2.0 ** -10) + rel * y.abs()
    values = d(out.y.float()) * d(out.scale)[:, None]
    assert bool(((values - y).abs() <= step).all())
    for dtype in (F32, BF16, F16):
        for squared in (False, True):
            ref = values ** 2 if squared else values
            close(L.dequantize(out.y, out.scale, dtype, squared=squared), ref, 3 * U * ref.abs())


@gpu
def test_rmsnorm_codes_of_tiny_and_huge_rows():
    w = torch.ones(64, device="cuda") * 1e-37
    x = randn(4, 64, seed=1)
    out = L.rmsnorm(x, w, out_dtype=E4M3)
    _, _, y = norm_ref(x, w, None, 1e-6)
    values = d(out.y.float()) * d(out.scale)[:, None]
    # the scale (about 5e-40) is a subnormal: its spacing 2^-149 adds 2^-150 / 5e-40 = 2^-19
    step = torch.maximum(y.abs() * 2.0 ** -4, y.abs().amax(1, keepdim=True) / 448 * 2.0 ** -10)
    assert bool(((values - y).abs() <= step * (1 + 2.0 ** -8)).all())


@gpu
@pytest.mark.parametrize("y_dtype", [F32, BF16, E4M3])
def test_rmsnorm_not_finite_rows_stay_alone(y_dtype):
    x, w = randn(6, 200, seed=1), randn(200, seed=2)
    want = L.rmsnorm(x, w, out_dtype=y_dtype)
    y = want.y.float()
    x[1, 3], x[4, 7] = float("nan"), float("inf")
    got = L.rmsnorm(x, w, out_dtype=y_dtype).y.float()
    assert bool(got[1].isnan().all())
    assert bool(got[4, 7].isnan()) and bool((got[4, :7] == 0).all())
    for i in (0, 2, 3, 5):
        assert torch.equal(got[i], y[i])


@gpu
@pytest.mark.parametrize("dim", [200, 1001, 40000])
def test_rmsnorm_scales_show_what_is_not_finite(dim):
    """Rows in registers and rows in passes alike: NaN scales where a y is NaN, by its
    row or by the weight, and no other row is touched."""
    x, w = randn(5, dim, seed=1), randn(dim, seed=2)
    want = L.rmsnorm(x, w, out_dtype=E4M3)
    x[1, 3], x[3, dim - 1] = float("nan"), float("inf")
    got = L.rmsnorm(x, w, out_dtype=E4M3)
    assert got.scale.isnan().tolist() == [False, True, False, True, False]
    for i in (0, 2, 4):
        assert torch.equal(got.y[i].float(), want.y[i].float()) and got.scale[i] == want.scale[i]
    w[5] = float("nan")
    assert bool(L.rmsnorm(x, w, out_dtype=E4M3).scale.isnan().all())


@gpu
def test_rmsnorm_of_rows_without_values():
    x, w = randn(500, 0), randn(0)
    for _ in range(2):  # in memory that held something else
        torch.full((1000,), 5.0, device="cuda")
        out = L.rmsnorm(x, w, out_dtype=E4M3, save_rstd=True)
        assert out.y.shape == (500, 0) and bool(out.rstd.isnan().all()) and bool((out.scale == 0).all())
    dx, dw = L.rmsnorm_backward(x, x, w, out.rstd)
    assert dx.shape == (500, 0) and dw.shape == (0,)


def norm_grad_ref(dy, s, w, rstd, ds):
    h, g = d(s) * d(rstd)[:, None], d(dy) * d(w)
    dx = d(rstd)[:, None] * (g - h * (g * h).mean(1, keepdim=True))
    return dx + (d(ds) if ds is not None else 0), (d(dy) * h).sum(0), h, g


@gpu
@pytest.mark.parametrize("rows,dim", NORM_SIZES + [(5000, 128), (3001, 1000)])
@pytest.mark.parametrize("x_dtype,dy_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32)])
def test_rmsnorm_backward(rows, dim, x_dtype, dy_dtype):
    s = randn(rows, dim, dtype=x_dtype, seed=1)
    dy = randn(rows, dim, dtype=dy_dtype, seed=2)
    w = randn(dim, dtype=F32 if dim % 3 else x_dtype, seed=3)
    ds = randn(rows, dim, dtype=x_dtype, seed=4)
    rstd = (1 / torch.sqrt(s.float().square().mean(1) + 1e-5))
    for dsum in (None, ds):
        dx, dw = L.rmsnorm_backward(dy, s, w, rstd, dsum=dsum)
        rx, rw, h, g = norm_grad_ref(dy, s, w, rstd, dsum)
        terms = (g * h).abs().mean(1, keepdim=True)
        mag = d(rstd)[:, None] * (g.abs() + h.abs() * terms * (dim / 32 + 40)) + (d(ds).abs() if dsum is not None else 0)
        close(dx, rx, 8 * U * mag)
        close(dw, rw, (rows + 4) * U * (d(dy) * h).abs().sum(0))
        assert dw.dtype == w.dtype and dx.dtype == x_dtype
    again = L.rmsnorm_backward(dy, s, w, rstd, dsum=ds)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    assert L.rmsnorm_backward(dy, s, w, rstd, need_dweight=False)[1] is None


@gpu
def test_rmsnorm_backward_by_differences():
    """The gradient of sum(c y) + sum(e s) against central differences of the
    forward formula in 64 bits: with steps of 1e-4 these are off by about 1e-8,
    and the gradient by a few u of its terms."""
    x, r, w = randn(5, 24, seed=1), randn(5, 24, seed=2), randn(24, seed=3)
    c, e = randn(5, 24, seed=4), randn(5, 24, seed=5)
    out = L.rmsnorm(x, w, residual=r, eps=1e-5, save_rstd=True)
    dx, dw = L.rmsnorm_backward(c, out.sum, w, out.rstd, dsum=e)

    def loss(xx, ww):
        s = xx + d(r)
        y = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-5) * ww
        return float((d(c) * y).sum() + (d(e) * s).sum())

    for i in range(5):
        for j in range(24):
            a = d(x)
            a[i, j] += 1e-4
            b = d(x)
            b[i, j] -= 1e-4
            assert abs((loss(a, d(w)) - loss(b, d(w))) / 2e-4 - float(dx[i, j])) < 2e-5
    for j in range(24):
        a, b = d(w), d(w)
        a[j] += 1e-4
        b[j] -= 1e-4
        assert abs((loss(d(x), a) - loss(d(x), b)) / 2e-4 - float(dw[j])) < 2e-5


# --------------------------------------------------------------------- linear

def act_ref(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    return z * torch.sigmoid(z) if act == "silu" else z


def slope_ref(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def check_linear(M, N, K, dtype, act=None, bias=False, residual=False, pre=False, pads=(0, 0, 0),
                 offset=0, out_dtype=None):
    x = randn(M, K, dtype=F32, seed=1)
    w = randn(N, K, dtype=F32, seed=2, scale=max(K, 1) ** -0.5)
    xs = ws = None
    if dtype == E4M3:
        xs = x.abs().amax(1).clamp_min(1e-3) / 448 if K else torch.ones(M, device="cuda")
        ws = w.abs().amax(1).clamp_min(1e-3) / 448 if K else torch.ones(N, device="cuda")
        x, w = x / xs[:, None], w / ws[:, None]
        out_dtype = out_dtype or BF16
    else:
        out_dtype = dtype

    def laid(t, pad):
        v = torch.zeros(t.shape[0] * (t.shape[1] + pad) + offset, device="cuda").to(dtype)
        v = v[offset:].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
        v.copy_(t)
        return v

    x, w = laid(x, pads[0]), laid(w, pads[1])
    b = randn(N, dtype=out_dtype, seed=3) if bias else None
    r = randn(M, N, dtype=out_dtype, seed=4, pad=pads[2], offset=offset) if residual else None
    y = randn(M, N, dtype=out_dtype, seed=5, pad=pads[2], offset=offset)
    got = L.linear(x, w, bias=b, residual=r, act=act, x_scale=xs, w_scale=ws, out=y, save_pre=pre)
    xd, wd = d(x.float()), d(w.float())
    if xs is not None:
        xd, wd = xd * d(xs)[:, None], wd * d(ws)[:, None]
    z = xd @ wd.t()
    slack = (2 * K + 8) * U * (xd.abs() @ wd.abs().t() + (d(b).abs() if bias else 0))
    if bias:
        z = z + d(b)
    ref = act_ref(z, act)
    if residual:
        ref = ref + d(r)
    # the activations' slopes are below 1.13; FP32 erf and exp are within 4 u of 1
    close(got.y, ref, 1.13 * slack + 8 * U * (z.abs() + ref.abs()))
    if pre:
        close(got.pre, z, slack)
    else:
        assert got.pre is None
    if pads[2] and M > 1:
        gaps = y.as_strided((M - 1, pads[2]), (N + pads[2], 1), y.storage_offset() + N)
        assert bool((gaps.float() == 77.0 if out_dtype != E4M3 else gaps).all())
    return x, w, got


# from one token to many, sizes around the tiles' edges (16, 32, 64, 128, 256), odd ones
LINEAR_SIZES = [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 129, 72), (3, 128, 8), (5, 257, 63), (8, 256, 512),
                (15, 40, 16), (16, 128, 128), (17, 512, 640), (31, 200, 136), (33, 384, 264), (63, 127, 64),
                (64, 128, 1024), (65, 130, 200), (100, 96, 2048), (127, 255, 65), (128, 128, 64), (129, 1, 33),
                (200, 777, 150), (255, 256, 192), (257, 300, 88), (513, 128, 128), (1001, 63, 100), (2048, 640, 320)]


@gpu
@pytest.mark.parametrize("M,N,K", LINEAR_SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32, E4M3])
def test_linear_sizes(M, N, K, dtype):
    check_linear(M, N, K, dtype)
    check_linear(M, N, K, dtype, act="silu", bias=True, residual=True, pre=True)


# outputs of many tiles: more than one per pair of SMs, ragged at both edges
@gpu
@pytest.mark.parametrize("M,N,K", [(2500, 1300, 200), (5001, 2000, 64), (4096, 4096, 1024), (257, 9000, 72)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32, E4M3])
def test_linear_many_tiles(M, N, K, dtype):
    check_linear(M, N, K, dtype, act="gelu", bias=True, residual=True, pre=True)
    L.check()


# k long enough to be split, over and under the number of parts
@gpu
@pytest.mark.parametrize("M,N,K", [(1, 128, 8192), (5, 129, 4097), (16, 1024, 16384), (40, 256, 5000), (130, 300, 9000)])
@pytest.mark.parametrize("dtype", [BF16, F32, E4M3])
def test_linear_long_sums(M, N, K, dtype):
    check_linear(M, N, K, dtype, bias=True, residual=True)
    L.check()


@gpu
@pytest.mark.parametrize("dtype", [F32, F16])
def test_linear_longest_sum(dtype):
    """The longest k there may be, 2^31 - 1 (8.6 GB of FP32): values at its ends and
    between are all summed."""
    K = 2 ** 31 - 1
    x = torch.zeros(1, K, device="cuda", dtype=dtype)
    x[0, 0], x[0, 2 ** 30 + 5], x[0, K - 40], x[0, K - 1] = 1.0, 2.0, 3.0, 4.0
    b = torch.full((1,), 0.5, device="cuda", dtype=dtype)
    assert float(L.linear(x, x, bias=b).y) == 1 + 4 + 9 + 16 + 0.5
    L.check()


@gpu
@pytest.mark.parametrize("M", [1, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F32, E4M3])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias,residual,pre", [(True, False, False), (False, True, False), (False, False, True), (True, True, True)])
def test_linear_epilogues(M, dtype, act, bias, residual, pre):
    check_linear(M, 200, 96, dtype, act=act, bias=bias, residual=residual, pre=pre)


@gpu
@pytest.mark.parametrize("M", [1, 33, 260])
@pytest.mark.parametrize("dtype", [BF16, F32, E4M3])
@pytest.mark.parametrize("pads,offset", [((1, 0, 0), 0), ((0, 1, 3), 0), ((8, 16, 8), 0), ((16, 8, 1), 1), ((0, 0, 0), 3)])
def test_linear_strided(M, dtype, pads, offset):
    check_linear(M, 136, 80, dtype, act="relu", bias=True, residual=True, pads=pads, offset=offset)


@gpu
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M", [4, 200])
def test_linear_codes_out(out_dtype, M):
    check_linear(M, 96, 256, E4M3, bias=True, residual=True, pre=True, out_dtype=out_dtype)


def every(dtype, limit):
    """Every value of a 16-bit type up to `limit` in magnitude."""
    z = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    return z[z.float().abs() <= limit].cuda()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_linear_activations_keep_their_tails(dtype, act):
    """16-bit activations of every z to 12.5 are off by 2^-13 of themselves before they
    are rounded (FP32's exp of -z^2 / 2 is off by up to 79 * 1.5 u = 2^-17 of itself)."""
    z = every(dtype, 12.5)
    x, w = torch.zeros(len(z), 8, device="cuda", dtype=dtype), torch.zeros(8, 8, device="cuda", dtype=dtype)
    x[:, 0], w[:, 0] = z, 1.0
    ref = act_ref(d(z), act)
    for y in L.linear(x, w, act=act).y.unbind(1):
        close(y, ref, 2.0 ** -13 * ref.abs())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_linear_slopes_keep_their_tails(dtype, act):
    """Slopes of the same z, by dbias of one row: their terms (Phi and z phi; s and
    z s (1 - s)) are off by 2^-13 and 2^-16 of themselves, and sums with 1 by 4 u (1 + |z|)."""
    z = every(dtype, 12.5)
    n = len(z)
    g = L.linear_backward(torch.ones(1, n, device="cuda", dtype=dtype), torch.zeros(1, 8, device="cuda", dtype=dtype),
                          torch.zeros(n, 8, device="cuda", dtype=dtype), pre=z[None], act=act, need_dx=False, need_dw=False)
    t = d(z)
    s = torch.sigmoid(t)
    slack = {"relu": 0 * t,
             "gelu": (2.0 ** -13 * 0.5 * torch.special.erfc(t.abs() / math.sqrt(2))
                      + 2.0 ** -16 * t.abs() * torch.exp(-t * t / 2) * 0.4 + 4 * U * (t > 0)),
             "silu": 2.0 ** -16 * s * (1 + t.abs() * (1 - s)) + 4 * U * (1 + t.abs()) * s}[act]
    close(g.db, slope_ref(t, act), slack)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_empty(dtype):
    w, b = randn(7, 5, dtype=dtype), randn(7, dtype=dtype)
    assert L.linear(randn(0, 5, dtype=dtype), w, bias=b).y.shape == (0, 7)
    assert L.linear(randn(3, 5, dtype=dtype), w[:0]).y.shape == (3, 0)
    none = L.linear(randn(3, 0, dtype=dtype), w[:, :0].contiguous(), bias=b, act="relu").y
    assert torch.equal(none, b.clamp_min(0).expand(3, 7))
    g = L.linear_backward(randn(0, 7, dtype=dtype), randn(0, 5, dtype=dtype), w)
    assert g.dx.shape == (0, 5) and bool((g.dw == 0).all()) and bool((g.db == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [3, 150])
def test_linear_residual_in_place(dtype, M):
    x, w, r = randn(M, 64, dtype=dtype, seed=1), randn(48, 64, dtype=dtype, seed=2), randn(M, 48, dtype=dtype, seed=3)
    want = L.linear(x, w, residual=r, act="gelu").y
    got = L.linear(x, w, residual=r, act="gelu", out=r)
    assert got.y is r and torch.equal(r, want)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M", [2, 20, 140])
@pytest.mark.parametrize("place", ["x", "w"])
def test_linear_not_finite(dtype, M, place):
    """A NaN or infinity in x or w gives what the 64-bit sums give, in every
    output that reads it and in no other."""
    x, w = randn(M, 80, dtype=dtype, seed=1), randn(70, 80, dtype=dtype, seed=2)
    t = x if place == "x" else w
    t[0, 3], t[1, 79] = float("inf"), float("nan")
    t[1, 5] = float("-inf")
    x[:, 7] = 2.0  # exact in every type
    w[:, 7] = 0.0
    y, ref = d(L.linear(x, w).y), d(x) @ d(w).t()
    assert torch.equal(y.isnan(), ref.isnan())
    assert torch.equal(torch.where(y.isinf(), y, torch.zeros_like(y)), torch.where(ref.isinf(), ref, torch.zeros_like(ref)))


@gpu
def test_linear_not_finite_long_sums():
    """Infinities in every output of a long FP32 sum, with more tiles than SMs: the waits
    of the tile that follows last while they are summed again (a second here; the waits
    that knew nothing of it lasted 16 s, and gave up from K of about 2^19 on)."""
    M, N, K = 1280, 2048, 1 << 15
    x = torch.zeros(M, K, device="cuda")
    w = torch.full((N, K), 0.5, device="cuda")
    x[:, 1] = float("inf")
    x[5, K - 1] = float("-inf")
    x[:, 77] = 2.0
    r, b = randn(M, N, seed=1), randn(N, seed=2)
    y = L.linear(x, w, bias=b, residual=r, act="relu").y
    L.check()
    want = torch.full((M, N), float("inf"), device="cuda")
    want[5] = float("nan")
    assert torch.equal(y.nan_to_num(7.0, posinf=8.0, neginf=9.0), want.nan_to_num(7.0, posinf=8.0, neginf=9.0))
    x[:, 1], x[5, K - 1] = 0.0, 0.0
    assert torch.equal(L.linear(x, w).y, torch.ones(M, N, device="cuda"))


@gpu
def test_linear_float32_extremes():
    """FP32 values from 1e-30 to 1e30: the sums keep FP32 accuracy relative to their
    largest terms."""
    x, w = randn(40, 96, seed=1), randn(50, 96, seed=2)
    x[:, ::2] *= 1e30
    w[:, ::2] *= 1e-30
    x[:, 1::2] *= 1e-12
    w[:, 1::2] *= 1e12
    ref = d(x) @ d(w).t()
    close(L.linear(x, w).y, ref, 200 * U * (d(x).abs() @ d(w).abs().t()))


def check_linear_backward(M, N, K, dtype, act, pads=(0, 0, 0, 0)):
    dy, x = randn(M, N, dtype=dtype, seed=1, pad=pads[0]), randn(M, K, dtype=dtype, seed=2, pad=pads[1])
    w, pre = randn(N, K, dtype=dtype, seed=3, pad=pads[2]), randn(M, N, dtype=dtype, seed=4, pad=pads[3])
    g = L.linear_backward(dy, x, w, pre=pre if act else None, act=act)
    dz = d(dy) * slope_ref(d(pre), act)
    # dz: a few u of its factors' magnitude, and its rounding to the type
    off = 16 * U * d(dy).abs() * (1 + d(pre).abs())
    rounded = off + (HALF_ULP[dtype] * dz.abs() + HALF_TINY[dtype] if act and dtype != F32 else 0)
    close(g.dx, dz @ d(w), (rounded + (2 * N + 4) * U * dz.abs()) @ d(w).abs())
    close(g.dw, dz.t() @ d(x), (rounded + (2 * M + 4) * U * dz.abs()).t() @ d(x).abs())
    close(g.db, dz.sum(0), (off + (M + 4) * U * dz.abs()).sum(0))
    again = L.linear_backward(dy, x, w, pre=pre if act else None, act=act)
    for a, b in zip(g, again):
        assert torch.equal(a, b)
    part = L.linear_backward(dy, x, w, pre=pre if act else None, act=act, need_dw=False, need_db=False)
    assert part.dw is None and part.db is None and torch.equal(part.dx, g.dx)


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 64, 48), (3, 33, 65), (16, 128, 64), (65, 100, 72), (128, 256, 128),
                                   (200, 63, 190), (1000, 136, 264), (2047, 64, 40), (40, 1024, 600), (5000, 24, 16)])
@pytest.mark.parametrize("dtype,act", [(BF16, "gelu"), (F16, "silu"), (F32, "gelu"), (F32, None), (BF16, None), (F16, "relu")])
def test_linear_backward(M, N, K, dtype, act):
    check_linear_backward(M, N, K, dtype, act)


@gpu
@pytest.mark.parametrize("M,N,K", [(2600, 1000, 1111), (3000, 2048, 2304), (9000, 40, 2000)])
@pytest.mark.parametrize("dtype,act", [(BF16, "gelu"), (F16, None), (F32, "silu")])
def test_linear_backward_many_tiles(M, N, K, dtype, act):
    check_linear_backward(M, N, K, dtype, act)
    L.check()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("pads", [(1, 0, 0, 3), (8, 8, 8, 8), (0, 3, 1, 0)])
def test_linear_backward_strided(dtype, act, pads):
    check_linear_backward(130, 72, 96, dtype, act, pads)


# small (both products fit one round of the GPU), ragged, and large
@gpu
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (64, 64, 64), (33, 65, 5), (512, 1024, 1024), (1001, 777, 1501), (3000, 2048, 2304)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear_backward_of_chosen_outputs(M, N, K, dtype, act):
    """Every subset of the three gradients is what the full call gives, bit for bit."""
    dy, x, w, pre = (randn(*s, dtype=dtype, seed=i) for i, s in enumerate([(M, N), (M, K), (N, K), (M, N)]))
    full = L.linear_backward(dy, x, w, pre=pre, act=act)
    for wanted in range(8):
        need = dict(need_dx=bool(wanted & 1), need_dw=bool(wanted & 2), need_db=bool(wanted & 4))
        part = L.linear_backward(dy, x, w, pre=pre, act=act, **need)
        for name, want in need.items():
            got, ref = getattr(part, name[5:]), getattr(full, name[5:])
            assert got is None if not want else torch.equal(got, ref), (need, name)
    L.check()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_linear_grad_of_the_bias_takes_no_operands(dtype):
    """dbias alone through the C entry point, with x, w, dx and dw NULL."""
    dy = randn(40, 24, dtype=dtype, seed=1)
    db = torch.empty(24, device="cuda", dtype=dtype)
    a = V._LinearGradArgs(M=40, N=24, K=16, dy=dy.data_ptr(), lddy=24, dbias=db.data_ptr(),
                          dtype=L._TYPE[dtype])
    n = V.lib().vcsr_linear_grad_workspace(a)
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    assert V.lib().vcsr_linear_grad(a, torch.cuda.current_stream().cuda_stream) == 0
    close(db, d(dy).sum(0), 44 * U * d(dy).abs().sum(0))


@gpu
def test_linear_backward_takes_expanded_gradients():
    x, w = randn(30, 40, seed=1), randn(20, 40, seed=2)
    one = torch.ones((), device="cuda").expand(30, 20)
    g = L.linear_backward(one, x, w)
    close(g.dx, d(w).sum(0).expand(30, 40), 24 * U * d(w).abs().sum(0))


@gpu
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
def test_linear_backward_by_differences(act):
    """The gradient of sum(c y) against central differences of the forward formula
    in 64 bits (off by about 1e-8 with steps of 1e-4)."""
    x, w, b, c = randn(4, 6, seed=1), randn(5, 6, seed=2), randn(5, seed=3), randn(4, 5, seed=4)
    out = L.linear(x, w, bias=b, act=act, save_pre=True)
    g = L.linear_backward(c, x, w, pre=out.pre, act=act)
    base = {"dx": d(x), "dw": d(w), "db": d(b)}

    def loss(v):
        return float((d(c) * act_ref(v["dx"] @ v["dw"].t() + v["db"], act)).sum())

    for name, t in base.items():
        got = d(getattr(g, name)).flatten()
        for i in range(t.numel()):
            up = {k: v.clone() for k, v in base.items()}
            down = {k: v.clone() for k, v in base.items()}
            up[name].view(-1)[i] += 1e-4
            down[name].view(-1)[i] -= 1e-4
            assert abs((loss(up) - loss(down)) / 2e-4 - float(got[i])) < 2e-5


# ---------------------------------------------------------------------- AdamW

SIZES = [1, 255, 256, 257, 1000, 4096, 7, 0, 3001]


def adamw_ref(p, g, m, v, t, lr, b1, b2, eps, wd):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * wd) - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p, m, v


def tensors(dtype, seed, scale, offset=0):
    return [randn(n, dtype=dtype, seed=seed + i, scale=scale, offset=offset) for i, n in enumerate(SIZES)]


@gpu
@pytest.mark.parametrize("p_dtype,g_dtype,offset", [(F32, F32, 0), (F32, BF16, 1), (BF16, BF16, 3), (F16, F32, 0)])
def test_adamw_32(p_dtype, g_dtype, offset):
    params = tensors(p_dtype, 0, 0.1, offset)
    copies = [torch.zeros(n, device="cuda", dtype=BF16) for n in SIZES]
    opt = L.AdamW(params, lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1, copies=copies)
    ref = [(d(p), torch.zeros(p.numel()).double(), torch.zeros(p.numel()).double()) for p in params]
    for t in range(1, 4):
        grads = tensors(g_dtype, 100 * t, 0.3, offset)
        opt.step(grads, grad_scale=0.25)
        for i, (p, g) in enumerate(zip(params, grads)):
            r = adamw_ref(*[ref[i][0], 0.25 * d(g), ref[i][1], ref[i][2]], t, 1e-2, 0.9, 0.99, 1e-6, 0.1)
            at = slice(opt.offsets[i], opt.offsets[i] + p.numel())
            # m cancels: t steps of 2 u of its terms, which are below 0.25 max|g|;
            # v's terms are positive.  The step is below lr * 10: sqrt and the quotient
            # are within 8 u of it, and m's error moves it by lr * its share of sqrt(v)
            big = 0.25 * d(g).abs().max() if g.numel() else 0.0
            close(opt.m_flat[at], r[1], 4 * t * U * big)
            close(opt.v_flat[at], r[2], (4 * t + 4) * U * r[2])
            step = 1e-2 * 32 * t * U * (1 + big / (torch.sqrt(r[2]) + 1e-6))
            close(p, r[0], step + 4 * U * r[0].abs())
            close(copies[i], d(p), 0 * r[0] + (HALF_ULP[p_dtype] * d(p).abs() + HALF_TINY[p_dtype]
                                              if p_dtype != F32 else 0))
            # 16-bit parameters carry their rounding on; the states do not
            ref[i] = (d(p), d(opt.m_flat[at]), d(opt.v_flat[at]))
    assert opt.steps == 3
    for i, n in enumerate(SIZES):  # the padding between the tensors stays zero
        end = opt.offsets[i + 1] if i + 1 < len(SIZES) else opt.m_flat.numel()
        assert bool((opt.m_flat[opt.offsets[i] + n:end] == 0).all())


def blocks_ref(x, dither):
    """Codes' values of x (flat, 64 bits) in rows of 256, and their scales."""
    x = x.view(-1, 256)
    scale = x.abs().amax(1, keepdim=True) / 448
    a = x.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))
    e = torch.floor(torch.log2(a.clamp_min(1e-300))).clamp_min(-6)
    step = torch.exp2(e - 3)
    k = torch.round(a / step) if dither is None else torch.floor(a / step + dither)
    return torch.sign(x) * (k * step).clamp_max(448) * scale, scale, a / step, step * scale


@gpu
@pytest.mark.parametrize("dithered", [False, True])
@pytest.mark.parametrize("p_dtype,g_dtype", [(F32, F32), (BF16, BF16), (F32, F16)])
def test_adamw_8(dithered, p_dtype, g_dtype):
    params = tensors(p_dtype, 0, 0.1)
    opt = L.AdamW(params, lr=1e-2, state_bits=8)
    for t in range(1, 4):
        grads = tensors(g_dtype, 100 * t, 0.3)
        dither = torch.rand(256, generator=torch.Generator().manual_seed(t)).cuda() if dithered else None
        m0, v0 = (d(s) for s in opt.state_values())
        before = [d(p) for p in params]
        opt.step(grads, dither=dither)
        m1, v1 = (d(s) for s in opt.state_values())
        g = torch.zeros_like(m0)
        p = torch.zeros_like(m0)
        for i, n in enumerate(SIZES):
            g[opt.offsets[i]:opt.offsets[i] + n] = d(grads[i])
            p[opt.offsets[i]:opt.offsets[i] + n] = before[i]
        rp, rm, rv = adamw_ref(p, g, m0, v0, t, 1e-2, 0.9, 0.999, 1e-8, 0.01)
        for i, n in enumerate(SIZES):
            at = slice(opt.offsets[i], opt.offsets[i] + n)
            scale = 1e-2 * 32 * (1 + (m0[at].abs() + g[at].abs()) / (torch.sqrt(rv[at]) + 1e-8))
            close(params[i], rp[at], scale * U + 4 * U * rp[at].abs())
        u0 = None if dither is None else d(dither)
        # what FP32 leaves of m (its two terms may cancel) and of u = sqrt(v) (they do not)
        m_off = 4 * U * (0.9 * m0.abs() + 0.1 * g.abs())
        u_off = 8 * U * torch.sqrt(rv)
        for got, want, err, floor in ((m1, rm, m_off, 0), (torch.sqrt(v1), torch.sqrt(rv), u_off, 1)):
            ref, scale, steps, step = blocks_ref(want, u0)
            got, err = got.view(-1, 256), err.view(-1, 256)
            # the same code, or the neighbouring one where the value lies within its
            # error (and the scale's) of where the rounding turns
            turn = steps + (0.5 if u0 is None else u0)
            near = (turn - torch.round(turn)).abs() * step <= err + 2.0 ** -18 * 16 * step
            low = floor * (want.view(-1, 256) > 0) * (ref == 0) * scale * 2.0 ** -9 * (1 + 2.0 ** -8)
            assert bool(((got - ref).abs() <= 8 * U * ref.abs() + near * step * (1 + 2.0 ** -8) + low).all())
        assert bool((v1[rv > 0] > 0).all())  # never zero by rounding


@gpu
def test_adamw_8_follows_the_mean():
    """u = sqrt(v) of values without gradients falls by 0.05% a step, far below half
    a code's step.  Beside a value that holds the block's scale it stays where it is
    when rounded to nearest, and with dither falls to 0.9995^2000 = 0.368 on the
    mean: a step of about u / 12 is taken down with probability 0.0005 * 12, a
    variance of 0.0005 u^2 / 12 a step, 0.042 u0^2 over the fall; 255 positions
    with their own numbers leave a deviation of 0.2 / 16 = 0.013 u0 of the mean
    (2^-9 of u0 is the least it can fall to)."""
    start = torch.full((16, 256), 224.0)
    start[:, 0] = 448.0
    grads = torch.zeros(16, 256, device="cuda")
    grads[:, 0] = 2.0
    gen = torch.Generator(device="cuda").manual_seed(3)
    seen = []
    for dithered in (False, True):
        opt = L.AdamW([torch.zeros(4096, device="cuda")], lr=0.0, state_bits=8)
        opt.u_flat.view(16, 256).copy_(start)
        opt.u_scale.fill_(2.0 / 448)
        for _ in range(2000):
            opt.step([grads], dither=torch.rand(256, device="cuda", generator=gen) if dithered else None)
        seen.append(d(opt.state_values()[1]).sqrt().view(16, 256)[:, 1:])
    assert bool((seen[0] == 1.0).all())
    assert abs(float(seen[1].mean()) - 0.9995 ** 2000) < 5 * 0.013


@gpu
def test_adamw_many_tensors_and_none():
    n = 1100  # more than one launch takes
    params = [torch.full((1 + i % 5,), 1.0, device="cuda") for i in range(n)]
    grads = [None if i % 7 == 3 else torch.full_like(p, 1.0 + i) for i, p in enumerate(params)]
    opt = L.AdamW(params, lr=0.5, weight_decay=0.0)
    opt.step(grads)
    for i, p in enumerate(params):  # the first step is lr against the gradient's sign
        want = 1.0 if i % 7 == 3 else 0.5
        assert abs(float(p[0]) - want) < 1e-6 and bool((p == p[0]).all())
        assert (float(opt.m_flat[opt.offsets[i]]) == 0) == (i % 7 == 3)


@gpu
def test_adamw_not_finite_gradients_stay_in_their_block():
    p = torch.zeros(1024, device="cuda")
    opt = L.AdamW([p], state_bits=8)
    g = torch.ones(1024, device="cuda")
    g[300] = float("inf")
    opt.step([g])
    assert bool(p[300].isnan())
    assert bool(torch.isfinite(p[:256]).all()) and bool(torch.isfinite(p[512:]).all())
    m, v = opt.state_values()
    assert bool(torch.isfinite(m[:256]).all()) and bool(torch.isfinite(v[512:]).all())


@gpu
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dithered", [False, True])
def test_adamw_8_scales_show_what_is_not_finite(value, dithered):
    """A gradient that is not finite makes the scales of its block so, and no other's."""
    p = torch.zeros(1024, device="cuda")
    opt = L.AdamW([p], state_bits=8)
    g = torch.ones(1024, device="cuda")
    g[300] = value
    opt.step([g], dither=torch.rand(256, device="cuda") if dithered else None)
    for scale in (opt.m_scale, opt.u_scale):
        assert scale.isfinite().tolist() == [True, False, True, True]
    for state in opt.state_values():
        assert not bool(state[300].isfinite()) and bool(state[:256].isfinite().all()) and bool(state[512:].isfinite().all())


# -------------------------------------------- bounded waits, streams, refusals

@gpu
@pytest.mark.parametrize("dtype,M,N,K", [
    (BF16, 4, 256, 1024), (E4M3, 33, 200, 4096), (F16, 300, 128, 64),  # clusters that split k, single blocks
    (BF16, 4096, 4096, 1024), (E4M3, 4096, 2048, 128),                 # pairs of blocks, several tiles and one each
    (F32, 16, 256, 4096), (F32, 2000, 2000, 512), (F32, 5000, 128, 32)])
def test_a_wait_that_runs_out_is_reported(dtype, M, N, K):
    """The first block of each kernel waits for a signal that is not sent: check() names
    the barrier, once, and the next call is right."""
    x, w = randn(M, K, seed=1).to(dtype), randn(N, K, seed=2).to(dtype)
    scales = dict(x_scale=torch.ones(M, device="cuda"), w_scale=torch.ones(N, device="cuda")) if dtype == E4M3 else {}
    want = L.linear(x, w, **scales).y
    L.check()
    L.test_withhold_signal()
    L.linear(x, w, **scales)
    with pytest.raises(V.VcsrError) as e:
        L.check()
    assert e.value.status == 7 and "accumulator-full" in e.value.msg
    assert "block 0" in e.value.msg or "block 1" in e.value.msg
    L.check()
    assert torch.equal(L.linear(x, w, **scales).y, want)
    L.check()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_wait_of_the_gradient_that_runs_out_is_reported(dtype):
    dy, x, w = randn(64, 96, dtype=dtype, seed=1), randn(64, 80, dtype=dtype, seed=2), randn(96, 80, dtype=dtype, seed=3)
    want = L.linear_backward(dy, x, w)
    L.test_withhold_signal()
    L.linear_backward(dy, x, w)
    with pytest.raises(V.VcsrError) as e:
        L.check()
    assert e.value.status == 7
    assert all(torch.equal(a, b) for a, b in zip(L.linear_backward(dy, x, w), want))
    L.check()


# ------------------------------------------------------- streams and refusals

@gpu
@pytest.mark.parametrize("raw", [False, True])
def test_operators_run_on_the_given_stream(raw):
    """Work on a side stream waits for what was enqueued there: the inputs are made
    on it behind a long chain, and the results read on it."""
    side = torch.cuda.Stream()
    x, w = randn(64, 512, dtype=BF16, seed=1), randn(256, 512, dtype=BF16, seed=2)
    want = L.linear(L.rmsnorm(x, w[0].clone()).y, w).y
    torch.cuda.synchronize()
    late = torch.zeros_like(x)
    big = torch.randn(2048, 2048, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-3
        late.copy_(x)
    s = side.cuda_stream if raw else side
    y = L.rmsnorm(late, w[0].clone(), stream=s).y
    got = L.linear(y, w, stream=s).y
    side.synchronize()
    assert torch.equal(got, want)


def busy(stream):
    """Keeps `stream` at work for some milliseconds, so that what is enqueued behind is late."""
    with torch.cuda.stream(stream):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-3


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_state_values_on_the_given_stream(bits, dtype):
    """The states of a step that is still to come on a side stream, read there into
    tensors that later steps leave alone."""
    side = torch.cuda.Stream()
    p, g = randn(5000, seed=1), randn(5000, seed=2)
    busy(side)  # warm
    opt, other = (L.AdamW([p.clone()], state_bits=bits) for _ in range(2))
    other.step([g])
    torch.cuda.synchronize()
    want = [t.clone() for t in other.state_values(dtype)]
    assert bool((want[0] != 0).any())
    torch.cuda.synchronize()
    busy(side)
    opt.step([g], stream=side)
    got = opt.state_values(dtype, stream=side)
    opt.step([g], stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_adamw_dither_of_the_given_stream():
    """A strided dither that a side stream has still to write is read on that stream."""
    side = torch.cuda.Stream()
    p, g, u = randn(5000, seed=1), randn(5000, seed=2), torch.rand(256, device="cuda")
    late = torch.zeros(256, 2, device="cuda")
    opt, other = (L.AdamW([p.clone()], state_bits=8) for _ in range(2))
    # with every kernel loaded, which can wait for the whole device
    busy(side)
    late[:, 0].copy_(u)
    other.step([g], dither=late[:, 0])
    late.zero_()
    torch.cuda.synchronize()
    busy(side)
    with torch.cuda.stream(side):
        late[:, 0].copy_(u)
    opt.step([g], dither=late[:, 0], stream=side)
    side.synchronize()
    assert torch.equal(opt.m_flat.view(torch.uint8), other.m_flat.view(torch.uint8))
    with pytest.raises(V.VcsrError):
        opt.step([g], dither=torch.rand(256), stream=side)


@gpu
def test_operators_take_keywords():
    x, w, v = randn(4, 8, seed=1), randn(6, 8, seed=2), randn(8, seed=3)
    n, o = L.rmsnorm(x, v, save_rstd=True), L.linear(x, w)
    assert torch.equal(L.rmsnorm(x=x, weight=v).y, n.y) and torch.equal(L.linear(w=w, x=x).y, o.y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = L.rmsnorm_backward(dy=x, s=x, weight=v, rstd=n.rstd, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, L.rmsnorm_backward(x, x, v, n.rstd)))
    assert torch.equal(L.linear_backward(dy=o.y, x=x, w=w).dx, L.linear_backward(o.y, x, w).dx)


@gpu
def test_operators_in_a_cuda_graph():
    x, w, b = randn(16, 256, dtype=BF16, seed=1), randn(256, 256, dtype=BF16, seed=2), randn(256, dtype=BF16)
    gain = torch.ones(256, device="cuda", dtype=BF16)

    def chain():
        n = L.rmsnorm(x, gain, save_rstd=True)
        o = L.linear(n.y, w, bias=b, act="gelu", save_pre=True)
        return o.y, L.linear_backward(o.y, n.y, w, pre=o.pre, act="gelu").dw

    want = [t.clone() for t in chain()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_adamw_refuses_scales_off_their_type():
    opt = L.AdamW([randn(64)], state_bits=8)
    for name in ("m_scale", "u_scale"):
        keep = getattr(opt, name)
        setattr(opt, name, torch.zeros(8, device="cuda").view(torch.uint8)[2:])
        with pytest.raises(V.VcsrError, match=f"{name} is not aligned"):
            opt.step([randn(64)])
        setattr(opt, name, keep)
    assert opt.steps == 0


@gpu
def test_refuses_what_is_no_tensor():
    x, v = randn(4, 8), randn(8)
    opt = L.AdamW([x])
    for call in (lambda: L.linear(x, [[1.0]]), lambda: L.linear(x, x, bias=1.0), lambda: L.rmsnorm_backward(x, None, v, v),
                 lambda: L.linear_backward(x, 3, x), lambda: L.AdamW([x], copies=[3]), lambda: L.AdamW([x], copies=[None]),
                 lambda: opt.step([3]), lambda: L.dequantize(x.to(E4M3), 1.0), lambda: L.rmsnorm(x, v, out=3)):
        with pytest.raises(V.VcsrError) as e:
            call()
        assert e.value.status == 1, e.value
    assert opt.steps == 0


@gpu
def test_refusals():
    x, w, v = randn(4, 8), randn(6, 8), randn(8)

    def refused(status, fn, *args, **kw):
        with pytest.raises(V.VcsrError) as e:
            fn(*args, **kw)
        assert e.value.status == status, e.value

    refused(1, L.rmsnorm, x.cpu(), v)
    refused(1, L.rmsnorm, x, v[:7])
    refused(1, L.rmsnorm, x, v, residual=randn(4, 9))
    refused(1, L.rmsnorm, x, v, eps=-1.0)
    refused(1, L.rmsnorm, x, v, eps=float("nan"))
    refused(1, L.rmsnorm, x[0], v)
    refused(5, L.rmsnorm, x.double(), v)
    refused(5, L.rmsnorm, x.bfloat16(), v.half())
    refused(5, L.rmsnorm, x, v, out_dtype=torch.int8)
    refused(1, L.rmsnorm, x, v, out=randn(8, 4).t())
    refused(5, L.rmsnorm_backward, x, x.to(E4M3), v, randn(4))
    refused(1, L.rmsnorm_backward, x, x, v, randn(3))
    refused(1, L.linear, x, randn(6, 7))
    refused(5, L.linear, x, w.bfloat16())
    refused(5, L.linear, x, w, act="tanh")
    refused(1, L.linear, x, w, x_scale=randn(4))
    refused(1, L.linear, x.to(E4M3), w.to(E4M3))
    refused(5, L.linear, x, w, out_dtype=BF16)
    refused(5, L.linear, x.to(E4M3), w.to(E4M3), x_scale=randn(4), w_scale=randn(6), out_dtype=E4M3)
    refused(1, L.linear, x, w, bias=randn(5))
    refused(1, L.linear_backward, randn(4, 6), x, w, act="gelu")
    refused(5, L.linear_backward, x.to(E4M3), x, w)
    refused(1, L.linear_backward, randn(4, 5), x, w)
    refused(1, L.AdamW, [])
    refused(1, L.AdamW, [x.t()])
    refused(5, L.AdamW, [x], state_bits=16)
    refused(5, L.AdamW, [x, w.half()])
    refused(5, L.AdamW, [x], copies=[x])
    opt = L.AdamW([x])
    refused(1, opt.step, [])
    refused(1, opt.step, [w])
    refused(5, opt.step, [x.double()])
    refused(1, opt.step, [x], dither=torch.rand(256, device="cuda"))
    opt.betas = (1.0, 0.9)
    refused(1, opt.step, [x])
    assert opt.steps == 0
