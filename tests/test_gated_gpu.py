"""The gated product and its gradient against their formulas in 64 bits (bounds as in
test_layers_gpu.py: a sum of K products is off by at most 2 K u sum|terms|)."""
import pytest
import torch

import vcsr_b200 as V
from test_layers_gpu import (BF16, E4M3, F16, F32, HALF_TINY, HALF_ULP, U, act_ref, busy, close, d, randn,
                             slope_ref)
from vcsr_b200 import layers as L

gpu = pytest.mark.gpu


def laid(t, dtype, pad, offset=0):
    """t as `dtype` in rows `pad` values apart, `offset` values into its storage."""
    v = torch.zeros(t.shape[0] * (t.shape[1] + pad) + offset, device="cuda").to(dtype)
    v = v[offset:].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
    v.copy_(t)
    return v


def check_gated(M, N, K, dtype, act="silu", bias=False, pre=False, pads=(0, 0, 0), offset=0, out_dtype=None):
    x, w = randn(M, K, seed=1), randn(2 * N, K, seed=2, scale=max(K, 1) ** -0.5)
    xs = ws = None
    if dtype == E4M3:
        xs = x.abs().amax(1).clamp_min(1e-3) / 448 if K else torch.ones(M, device="cuda")
        ws = w.abs().amax(1).clamp_min(1e-3) / 448 if K else torch.ones(2 * N, device="cuda")
        x, w = x / xs[:, None], w / ws[:, None]
        out_dtype = out_dtype or BF16
    else:
        out_dtype = dtype
    x, w = laid(x, dtype, pads[0], offset), laid(w, dtype, pads[1], offset)
    b = randn(2 * N, dtype=out_dtype, seed=3) if bias else None
    y = randn(M, N, dtype=out_dtype, seed=5, pad=pads[2], offset=offset)
    got = L.gated_linear(x, w, bias=b, act=act, x_scale=xs, w_scale=ws, out=y, save_pre=pre)
    assert got.y is y
    xd, wd = d(x.float()), d(w.float())
    if xs is not None:
        xd, wd = xd * d(xs)[:, None], wd * d(ws)[:, None]
    z = xd @ wd.t()
    slack = (2 * K + 8) * U * (xd.abs() @ wd.abs().t() + (d(b).abs() if bias else 0))
    if bias:
        z = z + d(b)
    g, u, off_g, off_u = z[:, :N], z[:, N:], slack[:, :N], slack[:, N:]
    a = act_ref(g, act)
    # the activations' slopes are below 1.13; FP32 erf and exp are within 4 u of 1, forms for
    # 16-bit results within 2^-13 of the value
    fast = 2.0 ** -13 if out_dtype != F32 else 0
    off_a = 1.13 * off_g + 8 * U * (g.abs() + a.abs()) + fast * a.abs()
    # FP32's u and a come rounded from one pass to the next, 16-bit ones not at all
    close(got.y, a * u, off_a * (u.abs() + off_u) + a.abs() * off_u + 4 * U * (a * u).abs())
    if pre:
        close(got.pre, z, slack)
    else:
        assert got.pre is None
    if pads[2] and M > 1:
        gaps = y.as_strided((M - 1, pads[2]), (N + pads[2], 1), y.storage_offset() + N)
        assert bool((gaps.float() == 77.0).all())
    return x, w, got


# one token to many, sizes around the tiles' edges (16, 32, 64, 128, 256), odd ones
SIZES = [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 129, 72), (3, 128, 8), (5, 257, 63), (8, 256, 512), (15, 40, 16),
         (16, 128, 128), (17, 512, 640), (31, 200, 136), (33, 384, 264), (63, 127, 64), (64, 128, 1024), (65, 130, 200),
         (100, 96, 2048), (127, 255, 65), (128, 128, 64), (129, 1, 33), (200, 777, 150), (255, 256, 192), (257, 300, 88),
         (513, 128, 128), (1001, 63, 100), (2048, 640, 320)]


@gpu
@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32, E4M3])
def test_gated_sizes(M, N, K, dtype):
    check_gated(M, N, K, dtype, bias=N % 2 == 0, pre=M % 2 == 1)
    L.check()


@gpu
@pytest.mark.parametrize("M,N,K", [(2600, 1000, 1111), (4000, 2048, 512), (9000, 260, 130)])
@pytest.mark.parametrize("dtype", [BF16, F16, E4M3])
def test_gated_many_tiles(M, N, K, dtype):
    check_gated(M, N, K, dtype, act="gelu", bias=True, pre=True)
    L.check()


@gpu
@pytest.mark.parametrize("M", [5, 300, 2100])
@pytest.mark.parametrize("dtype", [BF16, F16, F32, E4M3])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias,pre", [(False, False), (True, True)])
def test_gated_epilogues(M, dtype, act, bias, pre):
    check_gated(M, 264, 96, dtype, act, bias, pre)


@gpu
@pytest.mark.parametrize("M", [6, 130, 2100])
@pytest.mark.parametrize("dtype", [BF16, F32, E4M3])
@pytest.mark.parametrize("pads,offset", [((1, 0, 3), 0), ((16, 16, 16), 0), ((0, 3, 1), 1), ((8, 8, 8), 8), ((0, 0, 4), 0)])
def test_gated_strided(M, dtype, pads, offset):
    check_gated(M, 200, 80, dtype, pads=pads, offset=offset)


@gpu
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M", [3, 500, 2500])
def test_gated_codes_out(out_dtype, M):
    check_gated(M, 270, 200, E4M3, bias=True, pre=True, out_dtype=out_dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32, E4M3])
def test_gated_empty(dtype):
    """No values of k: act(bias) times bias; no rows, no columns: nothing."""
    for M, N in ((3, 20), (0, 20), (3, 0)):
        for K in (0, 16):
            if K and M and N:
                continue
            check_gated(M, N, K, dtype, bias=True, pre=True)
            check_gated(M, N, K, dtype)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32, E4M3])
@pytest.mark.parametrize("M", [2, 140, 2000])
@pytest.mark.parametrize("place", ["x", "g", "u"])
def test_gated_not_finite(dtype, M, place):
    """A NaN or infinity gives what the 64-bit formula gives, in every output that reads it
    and in no other."""
    N = 170
    x, w = randn(M, 80, dtype=dtype, seed=1), randn(2 * N, 80, dtype=dtype, seed=2)
    t = {"x": x, "g": w[:N], "u": w[N:]}[place]
    t[0, 3], t[1, 79] = float("inf"), float("nan")
    t[1, 5] = float("-inf")
    x[:, 7] = 2.0  # exact in every type
    w[:, 7] = 0.0
    if dtype == E4M3:
        one = dict(x_scale=torch.ones(M, device="cuda"), w_scale=torch.ones(2 * N, device="cuda"), out_dtype=F32)
    else:
        one = {}
    z = d(x.float()) @ d(w.float()).t()
    ref = act_ref(z[:, :N], "relu") * z[:, N:]
    y = d(L.gated_linear(x, w, act="relu", **one).y)
    assert torch.equal(y.isnan(), ref.isnan())
    assert torch.equal(torch.where(y.isinf(), y, torch.zeros_like(y)), torch.where(ref.isinf(), ref, torch.zeros_like(ref)))


@gpu
def test_gated_with_one_factor_is_linear():
    """u = 1 from its bias alone: act(x w_g^T + b), as linear gives it."""
    x, w = randn(70, 96, dtype=BF16, seed=1), randn(48, 96, dtype=BF16, seed=2)
    b = randn(48, dtype=BF16, seed=3)
    both = torch.cat([w, torch.zeros_like(w)])
    got = L.gated_linear(x, both, bias=torch.cat([b, torch.ones_like(b)]), act="gelu").y
    ref = act_ref(d(x) @ d(w).t() + d(b), "gelu")
    close(got, ref, 2.0 ** -12 * ref.abs() + 300 * U * (d(x).abs() @ d(w).abs().t() + 1))


def check_backward(M, N, K, dtype, act, pads=(0, 0, 0, 0)):
    dy, x = randn(M, N, dtype=dtype, seed=1, pad=pads[0]), randn(M, K, dtype=dtype, seed=2, pad=pads[1])
    w, pre = randn(2 * N, K, dtype=dtype, seed=3, pad=pads[2]), randn(M, 2 * N, dtype=dtype, seed=4, pad=pads[3])
    got = L.gated_linear_backward(dy, x, w, pre, act=act)
    g, u = d(pre)[:, :N], d(pre)[:, N:]
    dz = torch.cat([d(dy) * u * slope_ref(g, act), d(dy) * act_ref(g, act)], 1)
    # dz: a few u of its factors' magnitude (16-bit types: 2^-13 of the activation and its
    # slope), and its rounding to the type
    unit = 16 * U + (2.0 ** -12 if dtype != F32 else 0)
    off = unit * torch.cat([(d(dy) * u).abs() * (1 + g.abs()), d(dy).abs() * g.abs()], 1)
    rounded = off + (HALF_ULP[dtype] * dz.abs() + HALF_TINY[dtype] if dtype != F32 else 0)
    close(got.dx, dz @ d(w), (rounded + (4 * N + 4) * U * dz.abs()) @ d(w).abs())
    close(got.dw, dz.t() @ d(x), (rounded + (2 * M + 4) * U * dz.abs()).t() @ d(x).abs())
    close(got.db, dz.sum(0), (off + (M + 4) * U * dz.abs()).sum(0))
    again = L.gated_linear_backward(dy, x, w, pre, act=act)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for wanted in range(8):
        need = dict(need_dx=bool(wanted & 1), need_dw=bool(wanted & 2), need_db=bool(wanted & 4))
        part = L.gated_linear_backward(dy, x, w, pre, act=act, **need)
        for name, want in need.items():
            a, b = getattr(part, name[5:]), getattr(got, name[5:])
            assert a is None if not want else torch.equal(a, b), (need, name)
    L.check()


@gpu
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 64, 48), (3, 33, 65), (16, 128, 64), (65, 100, 72), (128, 256, 128),
                                   (200, 63, 190), (1000, 136, 264), (2047, 64, 40), (40, 1024, 600), (1001, 777, 1501)])
@pytest.mark.parametrize("dtype,act", [(BF16, "gelu"), (F16, "silu"), (F32, "gelu"), (F32, None), (BF16, "silu"), (F16, "relu")])
def test_gated_backward(M, N, K, dtype, act):
    check_backward(M, N, K, dtype, act)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pads", [(1, 0, 0, 3), (8, 8, 8, 8), (0, 3, 1, 0)])
def test_gated_backward_strided(dtype, pads):
    check_backward(130, 72, 96, dtype, "silu", pads)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gated_backward_of_nothing(dtype):
    for M, N, K in ((0, 8, 16), (4, 0, 16), (4, 8, 0)):
        for _ in range(2):
            torch.full((4096,), 5.0, device="cuda")  # in memory that held something else
            g = L.gated_linear_backward(randn(M, N, dtype=dtype, seed=1), randn(M, K, dtype=dtype), randn(2 * N, K, dtype=dtype),
                                        randn(M, 2 * N, dtype=dtype, seed=2))
            assert g.dx.shape == (M, K) and g.dw.shape == (2 * N, K) and g.db.shape == (2 * N,)
            assert bool((g.dx == 0).all()) and bool((g.dw == 0).all()) and (M and N or bool((g.db == 0).all()))


@gpu
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
def test_gated_backward_by_differences(act):
    """The gradient of sum(c y) against central differences of the forward formula in 64
    bits (off by about 1e-8 with steps of 1e-4)."""
    N = 5
    x, w, b, c = randn(4, 6, seed=1), randn(2 * N, 6, seed=2), randn(2 * N, seed=3), randn(4, N, seed=4)
    out = L.gated_linear(x, w, bias=b, act=act, save_pre=True)
    g = L.gated_linear_backward(c, x, w, out.pre, act=act)
    base = {"dx": d(x), "dw": d(w), "db": d(b)}

    def loss(v):
        z = v["dx"] @ v["dw"].t() + v["db"]
        return float((d(c) * act_ref(z[:, :N], act) * z[:, N:]).sum())

    for name, t in base.items():
        got = d(getattr(g, name)).flatten()
        for i in range(t.numel()):
            up = {k: v.clone() for k, v in base.items()}
            down = {k: v.clone() for k, v in base.items()}
            up[name].view(-1)[i] += 1e-4
            down[name].view(-1)[i] -= 1e-4
            assert abs((loss(up) - loss(down)) / 2e-4 - float(got[i])) < 4e-5


@gpu
@pytest.mark.parametrize("dtype,M,N,K", [
    (BF16, 4, 256, 1024), (E4M3, 33, 200, 4096), (F16, 300, 128, 64),  # clusters that split k, single blocks
    (BF16, 4096, 2048, 1024), (E4M3, 4096, 1024, 128), (F32, 16, 256, 4096)])
def test_a_wait_that_runs_out_is_reported(dtype, M, N, K):
    x, w = randn(M, K, seed=1).to(dtype), randn(2 * N, K, seed=2).to(dtype)
    scales = dict(x_scale=torch.ones(M, device="cuda"), w_scale=torch.ones(2 * N, device="cuda")) if dtype == E4M3 else {}
    want = L.gated_linear(x, w, **scales).y
    L.check()
    L.test_withhold_signal()
    L.gated_linear(x, w, **scales)
    with pytest.raises(V.VcsrError) as e:
        L.check()
    assert e.value.status == 7 and "accumulator-full" in e.value.msg
    L.check()
    assert torch.equal(L.gated_linear(x, w, **scales).y, want)
    L.check()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("raw", [False, True])
def test_gated_on_the_given_stream(dtype, raw):
    side = torch.cuda.Stream()
    x, w = randn(640, 512, dtype=dtype, seed=1), randn(256, 512, dtype=dtype, seed=2)
    busy(side)
    want = L.gated_linear(x, w, save_pre=True)
    want_g = L.gated_linear_backward(want.y, x, w, want.pre)
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    busy(side)
    with torch.cuda.stream(side):
        late.copy_(x)
    s = side.cuda_stream if raw else side
    got = L.gated_linear(late, w, save_pre=True, stream=s)
    g = L.gated_linear_backward(got.y, late, w, got.pre, stream=s)
    side.synchronize()
    assert torch.equal(got.y, want.y) and all(torch.equal(p, q) for p, q in zip(g, want_g))


@gpu
def test_gated_refusals():
    x, w = randn(4, 8), randn(12, 8)
    pre = randn(4, 12)

    def refused(status, fn, *args, **kw):
        with pytest.raises(V.VcsrError) as e:
            fn(*args, **kw)
        assert e.value.status == status, e.value

    refused(1, L.gated_linear, x.cpu(), w)
    refused(1, L.gated_linear, x, w[:11])
    refused(1, L.gated_linear, x, randn(12, 7))
    refused(1, L.gated_linear, x, [[1.0]])
    refused(5, L.gated_linear, x, w.bfloat16())
    refused(5, L.gated_linear, x, w, act="tanh")
    refused(1, L.gated_linear, x, w, x_scale=randn(4))
    refused(1, L.gated_linear, x.to(E4M3), w.to(E4M3))
    refused(1, L.gated_linear, x.to(E4M3), w.to(E4M3), x_scale=randn(4), w_scale=randn(6))
    refused(5, L.gated_linear, x, w, out_dtype=BF16)
    refused(5, L.gated_linear, x.to(E4M3), w.to(E4M3), x_scale=randn(4), w_scale=randn(12), out_dtype=E4M3)
    refused(1, L.gated_linear, x, w, bias=randn(6))
    refused(1, L.gated_linear, x, w, out=randn(4, 12))
    refused(1, L.gated_linear_backward, randn(4, 6), x, w, None)
    refused(1, L.gated_linear_backward, randn(4, 6), x, w, randn(4, 6))
    refused(5, L.gated_linear_backward, x.to(E4M3), x, w, pre)
    refused(1, L.gated_linear_backward, randn(4, 5), x, w, pre)
    refused(5, L.gated_linear_backward, randn(4, 6), x, w, pre, act="tanh")


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("M,N", [(4, 8), (300, 77)])
def test_gated_bias_gradient_over_no_k(dtype, act, M, N):
    """K = 0: dx and dw have no values, dbias sums dz as ever (bound as in check_backward)."""
    dy, pre = randn(M, N, dtype=dtype, seed=1), randn(M, 2 * N, dtype=dtype, seed=2)
    x, w = torch.empty(M, 0, device="cuda", dtype=dtype), torch.empty(2 * N, 0, device="cuda", dtype=dtype)
    for need in (True, False):
        torch.full((4096,), 5.0, device="cuda")  # in memory that held something else
        got = L.gated_linear_backward(dy, x, w, pre, act=act, need_dx=need, need_dw=need)
        g, u = d(pre)[:, :N], d(pre)[:, N:]
        dz = torch.cat([d(dy) * u * slope_ref(g, act), d(dy) * act_ref(g, act)], 1)
        unit = 16 * U + (2.0 ** -12 if dtype != F32 else 0)
        off = unit * torch.cat([(d(dy) * u).abs() * (1 + g.abs()), d(dy).abs() * g.abs()], 1)
        close(got.db, dz.sum(0), (off + (M + 4) * U * dz.abs()).sum(0))
        if need:
            assert got.dx.shape == (M, 0) and got.dw.shape == (2 * N, 0)
