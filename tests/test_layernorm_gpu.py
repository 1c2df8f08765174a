"""Layer norm and its gradient against their formulas in 64 bits.

Tolerances are bounds: u = 2^-24 is FP32's unit roundoff, a sum over a row goes in at
least 32 parts of dim / 32 terms and their 6 to 10 levels, so it is off by at most
(dim / 32 + 44) u of its terms' magnitude; a 16-bit result adds half a unit in its last
place."""
import pytest
import torch

import vcsr_b200 as V
from test_layers_gpu import BF16, E4M3, F16, F32, NORM_SIZES, U, busy, close, d, randn
from vcsr_b200 import layers as L

gpu = pytest.mark.gpu


def ref(x, w, b, r, eps):
    """s, mean, rstd and y in 64 bits, and bounds on what FP32 makes of the last three."""
    s = d(x) + (d(r) if r is not None else 0)
    dim = s.shape[1]
    rel = (dim / 32 + 44) * U
    mean = s.mean(1)
    c = s - mean[:, None]
    var = (c * c).mean(1) + eps
    rstd = 1 / torch.sqrt(var)
    off_mean = rel * s.abs().mean(1)
    off_c = off_mean[:, None] + U * (s.abs() + c.abs())
    off_var = 2 * (c.abs() * off_c).mean(1) + (off_c * off_c).mean(1) + rel * var
    off_rstd = rstd * (off_var / var * 0.75 + 4 * U)  # (1 - t)^-1/2 - 1 <= 0.75 t up to t = 0.4
    ww = d(w) if w is not None else torch.ones(dim).double()
    bb = d(b) if b is not None else torch.zeros(dim).double()
    y = c * rstd[:, None] * ww + bb
    off_y = ((off_c * rstd[:, None] + c.abs() * off_rstd[:, None]) * ww.abs() * (1 + 2.0 ** -10)
             + 4 * U * ((y - bb).abs() + bb.abs()))
    return s, mean, rstd, y, off_mean, off_rstd, off_y


def check(x, w, b, r, eps, y_dtype, **kw):
    out = L.layernorm(x, w, b, residual=r, eps=eps, out_dtype=y_dtype, save_stats=True, **kw)
    s, mean, rstd, y, off_mean, off_rstd, off_y = ref(x, w, b, r, eps)
    close(out.mean, mean, off_mean)
    close(out.rstd, rstd, off_rstd)
    close(out.y, y, off_y)
    if r is not None:
        close(out.sum, s, U * s.abs())
    return out


@gpu
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32), (F16, F16)])
def test_layernorm(rows, dim, x_dtype, y_dtype):
    x, r = randn(rows, dim, dtype=x_dtype, seed=1), randn(rows, dim, dtype=x_dtype, seed=2)
    w_dtype = F32 if dim % 2 else x_dtype
    w, b = randn(dim, dtype=w_dtype, seed=3), randn(dim, dtype=w_dtype, seed=4)
    for res in (None, r):
        out = check(x, w, b, res, 1e-5, y_dtype)
        assert res is not None or out.sum is x


@gpu
@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dim", [96, 333, 40000])
def test_layernorm_without_weight_or_bias(weight, bias, dim):
    x, dy = randn(9, dim, dtype=BF16, seed=1), randn(9, dim, dtype=BF16, seed=5)
    w, b = randn(dim, seed=3) if weight else None, randn(dim, seed=4) if bias else None
    out = check(x, w, b, None, 1e-5, BF16)
    g = L.layernorm_backward(dy, x, w, out.mean, out.rstd, weight_dtype=F32)
    check_grad(dy, x, w, out.mean, out.rstd, None, g)
    if not weight:
        plain = L.layernorm_backward(dy, x, None, out.mean, out.rstd)
        assert plain.dweight.dtype == plain.dbias.dtype == BF16 and torch.equal(plain.dx, g.dx)


@gpu
@pytest.mark.parametrize("shift", [100.0, -3e4])
@pytest.mark.parametrize("dim", [64, 1000, 40000])
def test_layernorm_of_rows_far_from_zero(shift, dim):
    """The spread is 1 about a mean far away: what a sum of squares less the mean's square
    would lose (all of it at 3e4: 9e8 u = 54)."""
    x, w, b = randn(7, dim, seed=1) + shift, randn(dim, seed=2), randn(dim, seed=3)
    check(x, w, b, None, 1e-5, F32)


@gpu
@pytest.mark.parametrize("rows,dim", [(20, 1), (9, 3), (31, 5), (700, 17), (33, 1001), (9, 2051), (17, 6003), (5, 9001)])
@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, BF16), (BF16, F32), (F16, F16), (BF16, E4M3)])
@pytest.mark.parametrize("pad", [0, 2])
def test_layernorm_odd_rows(rows, dim, x_dtype, y_dtype, pad):
    x, r = randn(rows, dim, dtype=x_dtype, seed=1, pad=pad), randn(rows, dim, dtype=x_dtype, seed=2, pad=pad)
    w, b = randn(dim, seed=3, offset=1), randn(dim, seed=4, offset=3)
    y = torch.zeros(rows, dim + pad, device="cuda").to(y_dtype)[:, :dim]
    sums = randn(rows, dim, dtype=x_dtype, pad=pad)
    if y_dtype == E4M3:
        out = L.layernorm(x, w, b, residual=r, eps=1e-5, out=y, sum_out=sums, save_stats=True)
        check_codes(out, *ref(x, w, b, r, 1e-5)[3::3])
    else:
        out = check(x, w, b, r, 1e-5, None, out=y, sum_out=sums)
        dy, ds = randn(rows, dim, dtype=y_dtype, seed=5, pad=pad), randn(rows, dim, dtype=x_dtype, seed=6, pad=pad)
        g = L.layernorm_backward(dy, sums, w, out.mean, out.rstd, dsum=ds)
        check_grad(dy, sums, w, out.mean, out.rstd, ds, g)
    assert out.y is y and out.sum is sums
    if pad and rows > 1:  # what lies between the rows is untouched
        gaps = sums.as_strided((rows - 1, pad), (dim + pad, 1), sums.storage_offset() + dim)
        assert bool((gaps == 77.0).all())


@gpu
@pytest.mark.parametrize("x_dtype", [F32, BF16])
@pytest.mark.parametrize("pad,offset", [(1, 0), (8, 0), (0, 1), (8, 4), (3, 5)])
def test_layernorm_strided(x_dtype, pad, offset):
    rows, dim = 37, 256
    x = randn(rows, dim, dtype=x_dtype, seed=1, pad=pad, offset=offset)
    r = randn(rows, dim, dtype=x_dtype, seed=2, pad=pad)
    w, b = randn(dim, dtype=x_dtype, seed=3), randn(dim, dtype=x_dtype, seed=4, offset=offset)
    y = randn(rows, dim, dtype=BF16, pad=pad, offset=offset)
    sums = randn(rows, dim, dtype=x_dtype, pad=pad)
    got = check(x, w, b, r, 0.0, None, out=y, sum_out=sums)
    assert got.y is y and got.sum is sums
    if pad:  # what lies between the rows is untouched
        gaps = y.as_strided((rows - 1, pad), (dim + pad, 1), y.storage_offset() + dim)
        assert bool((gaps == torch.tensor(77.0).to(BF16).item()).all())


@gpu
@pytest.mark.parametrize("dim", [64, 1000, 1001, 40000])
@pytest.mark.parametrize("which", ["x", "residual"])
def test_layernorm_sum_in_place(dim, which):
    x, r, w, b = randn(11, dim, seed=1), randn(11, dim, seed=2), randn(dim, seed=3), randn(dim, seed=4)
    s, _, _, y, _, _, off_y = ref(x, w, b, r, 1e-5)
    out = L.layernorm(x, w, b, residual=r, sum_out=x if which == "x" else r)
    close(out.y, y, off_y)
    close(x if which == "x" else r, s, U * s.abs())


def check_codes(out, y, off_y):
    """Half a step of e4m3 (2^-4 of the value, 2^-10 of the scale near zero) off y."""
    top = y.abs().amax(1)
    off_top = off_y.amax(1)
    close(out.scale, top / 448, (off_top + 4 * U * top) / 448)
    step = torch.maximum(y.abs() * 2.0 ** -4, (top / 448 * 2.0 ** -10)[:, None]) * (1 + 2.0 ** -8)
    values = d(out.y.float()) * d(out.scale)[:, None]
    assert bool(((values - y).abs() <= step + 2 * off_y + 2 * off_top[:, None] * 2.0 ** -4).all())


@gpu
@pytest.mark.parametrize("rows,dim", [(1, 16), (5, 128), (40, 1000), (3, 1001), (17, 4096), (2, 40000)])
@pytest.mark.parametrize("x_dtype", [F32, BF16, F16])
def test_layernorm_codes(rows, dim, x_dtype):
    x, r = randn(rows, dim, dtype=x_dtype, seed=1), randn(rows, dim, dtype=x_dtype, seed=2)
    w, b = randn(dim, seed=3), randn(dim, seed=4)
    check_codes(L.layernorm(x, w, b, residual=r, out_dtype=E4M3), *ref(x, w, b, r, 1e-5)[3::3])
    x[0], r[0] = 3.0, 0.0  # a row of one value is zero without a bias
    out = L.layernorm(x, w, residual=r, out_dtype=E4M3)
    assert out.scale[0] == 0 and bool((out.y[0].float() == 0).all())


@gpu
@pytest.mark.parametrize("dim", [200, 1001, 40000])
@pytest.mark.parametrize("y_dtype", [F32, BF16, E4M3])
def test_layernorm_not_finite_rows_stay_alone(dim, y_dtype):
    x, w, b = randn(6, dim, seed=1), randn(dim, seed=2), randn(dim, seed=3)
    want = L.layernorm(x, w, b, out_dtype=y_dtype)
    x[1, 3], x[4, dim - 1] = float("nan"), float("inf")
    got = L.layernorm(x, w, b, out_dtype=y_dtype)
    for i in (1, 4):  # the mean is not finite, so no distance from it is a number
        assert bool(got.y[i].float().isnan().all())
    for i in (0, 2, 3, 5):
        assert torch.equal(got.y[i].float(), want.y[i].float())
    if y_dtype == E4M3:
        assert got.scale.isnan().tolist() == [False, True, False, False, True, False]
        assert torch.equal(got.scale[[0, 2, 3, 5]], want.scale[[0, 2, 3, 5]])


@gpu
def test_layernorm_of_rows_without_values():
    x, w = randn(500, 0), randn(0)
    for _ in range(2):  # in memory that held something else
        torch.full((2000,), 5.0, device="cuda")
        out = L.layernorm(x, w, w, out_dtype=E4M3, save_stats=True)
        assert out.y.shape == (500, 0) and bool((out.scale == 0).all())
        assert bool(out.rstd.isnan().all()) and bool(out.mean.isnan().all())
    g = L.layernorm_backward(x, x, w, out.mean, out.rstd)
    assert g.dx.shape == (500, 0) and g.dweight.shape == g.dbias.shape == (0,)
    x = randn(0, 24)
    out = L.layernorm(x, randn(24), save_stats=True)
    for _ in range(2):
        torch.full((48,), 5.0, device="cuda")
        g = L.layernorm_backward(x, x, randn(24), out.mean, out.rstd)
        assert g.dx.shape == (0, 24) and bool((g.dweight == 0).all()) and bool((g.dbias == 0).all())


def check_grad(dy, s, w, mean, rstd, ds, got):
    rows, dim = s.shape
    h = (d(s) - d(mean)[:, None]) * d(rstd)[:, None]
    g = d(dy) * (d(w) if w is not None else 1.0)
    gh = (g * h).mean(1, keepdim=True)
    dx = d(rstd)[:, None] * (g - g.mean(1, keepdim=True) - h * gh) + (d(ds) if ds is not None else 0)
    k = dim / 32 + 44
    mag = (d(rstd)[:, None] * (g.abs() + k * g.abs().mean(1, keepdim=True)
                               + k * h.abs() * (g * h).abs().mean(1, keepdim=True))
           + (d(ds).abs() if ds is not None else 0))
    close(got.dx, dx, 8 * U * mag)
    close(got.dweight, (d(dy) * h).sum(0), (rows + 8) * U * (d(dy) * h).abs().sum(0))
    close(got.dbias, d(dy).sum(0), (rows + 8) * U * d(dy).abs().sum(0))


@gpu
@pytest.mark.parametrize("rows,dim", NORM_SIZES + [(5000, 128), (3001, 1000), (700, 2048), (650, 5120), (300, 5128)])
@pytest.mark.parametrize("x_dtype,dy_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32)])
def test_layernorm_backward(rows, dim, x_dtype, dy_dtype):
    s = randn(rows, dim, dtype=x_dtype, seed=1)
    dy = randn(rows, dim, dtype=dy_dtype, seed=2)
    w = randn(dim, dtype=F32 if dim % 3 else x_dtype, seed=3)
    ds = randn(rows, dim, dtype=x_dtype, seed=4)
    mean = s.float().mean(1)
    rstd = 1 / torch.sqrt((s.float() - mean[:, None]).square().mean(1) + 1e-5)
    for dsum in (None, ds):
        g = L.layernorm_backward(dy, s, w, mean, rstd, dsum=dsum)
        check_grad(dy, s, w, mean, rstd, dsum, g)
        assert g.dweight.dtype == g.dbias.dtype == w.dtype and g.dx.dtype == x_dtype
    again = L.layernorm_backward(dy, s, w, mean, rstd, dsum=ds)
    assert all(torch.equal(a, b) for a, b in zip(g, again))
    for wanted in range(4):
        part = L.layernorm_backward(dy, s, w, mean, rstd, dsum=ds, need_dweight=bool(wanted & 1),
                                    need_dbias=bool(wanted & 2))
        assert torch.equal(part.dx, g.dx)
        for bit, a, b in ((1, part.dweight, g.dweight), (2, part.dbias, g.dbias)):
            assert torch.equal(a, b) if wanted & bit else a is None


@gpu
@pytest.mark.parametrize("x_dtype", [F32, BF16])
@pytest.mark.parametrize("pads", [(1, 0, 0), (8, 8, 8), (0, 3, 5), (16, 0, 8)])
def test_layernorm_backward_strided(x_dtype, pads):
    dy, s, ds = (randn(61, 512, dtype=x_dtype, seed=i, pad=p) for i, p in enumerate(pads))
    w = randn(512, seed=3)
    out = L.layernorm(s, w, save_stats=True)
    check_grad(dy, s, w, out.mean, out.rstd, ds, L.layernorm_backward(dy, s, w, out.mean, out.rstd, dsum=ds))
    one = torch.ones((), device="cuda", dtype=x_dtype).expand(61, 512)
    check_grad(one, s, w, out.mean, out.rstd, None, L.layernorm_backward(one, s, w, out.mean, out.rstd))


@gpu
def test_layernorm_backward_by_differences():
    """The gradient of sum(c y) + sum(e s) against central differences of the forward
    formula in 64 bits: with steps of 1e-4 these are off by about 1e-8, and the gradient
    by a few u of its terms."""
    x, r, w, b = randn(5, 24, seed=1), randn(5, 24, seed=2), randn(24, seed=3), randn(24, seed=6)
    c, e = randn(5, 24, seed=4), randn(5, 24, seed=5)
    out = L.layernorm(x, w, b, residual=r, eps=1e-5, save_stats=True)
    g = L.layernorm_backward(c, out.sum, w, out.mean, out.rstd, dsum=e)
    base = {"dx": d(x), "dweight": d(w), "dbias": d(b)}

    def loss(v):
        s = v["dx"] + d(r)
        n = (s - s.mean(1, keepdim=True)) / torch.sqrt(s.var(1, unbiased=False, keepdim=True) + 1e-5)
        return float((d(c) * (n * v["dweight"] + v["dbias"])).sum() + (d(e) * s).sum())

    for name, t in base.items():
        got = d(getattr(g, name)).flatten()
        for i in range(t.numel()):
            up = {k: v.clone() for k, v in base.items()}
            down = {k: v.clone() for k, v in base.items()}
            up[name].view(-1)[i] += 1e-4
            down[name].view(-1)[i] -= 1e-4
            assert abs((loss(up) - loss(down)) / 2e-4 - float(got[i])) < 2e-5


@gpu
@pytest.mark.parametrize("raw", [False, True])
def test_layernorm_on_the_given_stream(raw):
    side = torch.cuda.Stream()
    x, w, b = randn(640, 512, dtype=BF16, seed=1), randn(512, seed=2), randn(512, seed=3)
    busy(side)
    want = L.layernorm(x, w, b, save_stats=True)
    want_g = L.layernorm_backward(x, x, w, want.mean, want.rstd)
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    busy(side)
    with torch.cuda.stream(side):
        late.copy_(x)
    s = side.cuda_stream if raw else side
    got = L.layernorm(late, w, b, save_stats=True, stream=s)
    g = L.layernorm_backward(late, late, w, got.mean, got.rstd, stream=s)
    side.synchronize()
    assert torch.equal(got.y, want.y) and all(torch.equal(p, q) for p, q in zip(g, want_g))


@gpu
def test_layernorm_in_cuda_graphs():
    """Two captured graphs of the same call, replayed in turn and at the same time."""
    x, w, b = randn(333, 1024, dtype=BF16, seed=1), randn(1024, seed=2), randn(1024, seed=3)

    def chain():
        n = L.layernorm(x, w, b, save_stats=True)
        return (n.y, *L.layernorm_backward(n.y, x, w, n.mean, n.rstd))

    want = [t.clone() for t in chain()]
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            got.append(chain())
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for made in got for p, q in zip(made, want))


@gpu
def test_layernorm_refusals():
    x, v = randn(4, 8), randn(8)
    out = L.layernorm(x, v, v, save_stats=True)

    def refused(status, fn, *args, **kw):
        with pytest.raises(V.VcsrError) as e:
            fn(*args, **kw)
        assert e.value.status == status, e.value

    refused(1, L.layernorm, x.cpu(), v)
    refused(1, L.layernorm, x, v[:7])
    refused(1, L.layernorm, x, v, v[:7])
    refused(1, L.layernorm, x, 1.0)
    refused(1, L.layernorm, x, v, v, residual=randn(4, 9))
    refused(1, L.layernorm, x, v, eps=-1.0)
    refused(1, L.layernorm, x, v, eps=float("nan"))
    refused(1, L.layernorm, x[0], v)
    refused(5, L.layernorm, x.double(), v)
    refused(5, L.layernorm, x.bfloat16(), v.half())
    refused(5, L.layernorm, x.bfloat16(), v, v.bfloat16())
    refused(5, L.layernorm, x, v, out_dtype=torch.int8)
    refused(1, L.layernorm, x, v, out=randn(8, 4).t())
    refused(5, L.layernorm_backward, x, x.to(E4M3), v, out.mean, out.rstd)
    refused(5, L.layernorm_backward, x.to(E4M3), x, v, out.mean, out.rstd)
    refused(1, L.layernorm_backward, x, x, v, randn(3), out.rstd)
    refused(1, L.layernorm_backward, x, x, v, out.mean, None)
    refused(1, L.layernorm_backward, x, None, v, out.mean, out.rstd)
    refused(5, L.layernorm_backward, x, x, None, out.mean, out.rstd, weight_dtype=BF16)
    refused(5, L.layernorm_backward, x, x, v, out.mean, out.rstd, weight_dtype=BF16)


@gpu
@pytest.mark.parametrize("rows,dim", [(700, 1000), (333, 1001), (300, 5120), (5, 40000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layernorm_gradient_over_dsum(rows, dim, dtype):
    """dx in dsum's own memory, as the C entry point allows."""
    s, dy, ds = (randn(rows, dim, dtype=dtype, seed=i) for i in range(3))
    w = randn(dim, dtype=dtype, seed=3)
    n = L.layernorm(s, w, save_stats=True)
    want = L.layernorm_backward(dy, s, w, n.mean, n.rstd, dsum=ds).dx
    a = V._LayernormGradArgs(rows, dim, dy.data_ptr(), dim, s.data_ptr(), dim, w.data_ptr(), n.mean.data_ptr(),
                             n.rstd.data_ptr(), ds.data_ptr(), dim, ds.data_ptr(), dim, None, None, None, 0,
                             L._TYPE[dtype], L._TYPE[dtype], L._TYPE[dtype])
    assert V.lib().vcsr_layernorm_grad(a, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(ds, want)


@gpu
def test_layernorm_of_some_rows():
    """A row's results are those it has among others (within one rounding: the sums of few
    rows are made by more threads), and the same bits whole and in a view."""
    x, w, b = randn(4000, 1024, dtype=BF16, seed=1), randn(1024, seed=2), randn(1024, seed=3)
    for rows in (slice(0, 1), slice(17, 20), slice(3999, 4000)):
        part = L.layernorm(x[rows], w, b, save_stats=True)
        close(part.y, d(L.layernorm(x, w, b).y[rows]), 2.0 ** -8 * d(part.y).abs())
        again = L.layernorm(x[rows].clone(), w, b, save_stats=True)
        assert torch.equal(again.y, part.y) and torch.equal(again.mean, part.mean) and torch.equal(again.rstd, part.rstd)


def stats(s):
    mean = s.float().mean(1)
    return mean, 1 / torch.sqrt((s.float() - mean[:, None]).square().mean(1) + 1e-5)


@gpu
@pytest.mark.parametrize("dim", [4104, 4608, 5120, 5632])
@pytest.mark.parametrize("x_dtype,dy_dtype", [(BF16, BF16), (F16, F32), (F32, F32)])
def test_layernorm_backward_by_width(dim, x_dtype, dy_dtype):
    """Widths whose teams take 264 to 352 threads, two or one of them a block, for several rows each."""
    s, ds = randn(700, dim, dtype=x_dtype, seed=1), randn(700, dim, dtype=x_dtype, seed=4)
    dy, w = randn(700, dim, dtype=dy_dtype, seed=2), randn(dim, seed=3)
    mean, rstd = stats(s)
    for dsum in (None, ds):
        g = L.layernorm_backward(dy, s, w, mean, rstd, dsum=dsum)
        check_grad(dy, s, w, mean, rstd, dsum, g)
        again = L.layernorm_backward(dy, s, w, mean, rstd, dsum=dsum)
        assert all(torch.equal(a, b) for a, b in zip(g, again))


# rows for several turns of every team: vectors cut at memory boundaries ((6001, 333) in teams of
# less than a warp, (700, 9001) with 32 values a thread), and short rows
MANY_TURNS = [(2001, 1501), (6001, 333), (9001, 17), (700, 9001), (1201, 5121)]


@gpu
@pytest.mark.parametrize("rows,dim", MANY_TURNS)
@pytest.mark.parametrize("x_dtype,dy_dtype", [(F32, F32), (BF16, BF16), (F32, BF16), (F16, F32)])
def test_layernorm_backward_odd_rows_in_many_turns(rows, dim, x_dtype, dy_dtype):
    s, ds = randn(rows, dim, dtype=x_dtype, seed=1), randn(rows, dim, dtype=x_dtype, seed=4)
    dy, w = randn(rows, dim, dtype=dy_dtype, seed=2), randn(dim, dtype=x_dtype, seed=3)
    mean, rstd = stats(s)
    for dsum in (None, ds):
        g = L.layernorm_backward(dy, s, w, mean, rstd, dsum=dsum)
        check_grad(dy, s, w, mean, rstd, dsum, g)
        again = L.layernorm_backward(dy, s, w, mean, rstd, dsum=dsum)
        assert all(torch.equal(a, b) for a, b in zip(g, again))


@gpu
@pytest.mark.parametrize("rows,dim", [(3001, 1001), (1200, 200), (700, 5000), (9001, 17)])
@pytest.mark.parametrize("x_dtype,dy_dtype", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_layernorm_backward_single_values_in_many_turns(rows, dim, x_dtype, dy_dtype):
    """s a value further apart than dy and dx: rows that are off 16 bytes unlike, for teams of one
    warp and more."""
    s = randn(rows, dim, dtype=x_dtype, seed=1, pad=1)
    dy, w = randn(rows, dim, dtype=dy_dtype, seed=2), randn(dim, seed=3)
    ds = randn(rows, dim, dtype=x_dtype, seed=4)
    mean, rstd = stats(s)
    for dsum in (None, ds):
        check_grad(dy, s, w, mean, rstd, dsum, L.layernorm_backward(dy, s, w, mean, rstd, dsum=dsum))


@gpu
@pytest.mark.parametrize("rows,dim", [(700, 4096), (700, 5121), (2600, 1000), (2500, 1001)])
@pytest.mark.parametrize("x_dtype,y_dtype", [(BF16, BF16), (F16, F32), (BF16, E4M3), (F32, BF16)])
@pytest.mark.parametrize("pad", [0, 1])
def test_layernorm_of_rows_that_fill_the_gpu(rows, dim, x_dtype, y_dtype, pad):
    """16 and 32 values a thread, which few rows do not get: whole, ragged, and single values (a
    residual further apart than x)."""
    x, r = randn(rows, dim, dtype=x_dtype, seed=1), randn(rows, dim, dtype=x_dtype, seed=2, pad=pad)
    w, b = randn(dim, dtype=x_dtype, seed=3), randn(dim, dtype=x_dtype, seed=4)
    if y_dtype == E4M3:
        check_codes(L.layernorm(x, w, b, residual=r, out_dtype=E4M3), *ref(x, w, b, r, 1e-5)[3::3])
    else:
        check(x, w, b, r, 1e-5, y_dtype)


@gpu
@pytest.mark.parametrize("rows,dim", [(100001, 20), (20000, 200), (1000, 4000), (700, 4096), (700, 4097)])
@pytest.mark.parametrize("x_dtype", [F32, BF16])
def test_layernorm_single_values_of_many_rows(rows, dim, x_dtype):
    """x a value further apart than residual and y, in matrices that fill the GPU: 8 values a thread
    to 4,096 a row, 16 beyond."""
    x, r = randn(rows, dim, dtype=x_dtype, seed=1, pad=1), randn(rows, dim, dtype=x_dtype, seed=2)
    w, b = randn(dim, dtype=x_dtype, seed=3), randn(dim, dtype=x_dtype, seed=4)
    check(x, w, b, r, 1e-5, x_dtype)
    check_codes(L.layernorm(x, w, b, residual=r, out_dtype=E4M3), *ref(x, w, b, r, 1e-5)[3::3])
