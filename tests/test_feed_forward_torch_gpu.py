"""Layer norm and the gated product as torch operators with gradients."""
import pytest
import torch

from test_layers_torch_gpu import leaf
from vcsr_b200 import layers, torch_ops

gpu = pytest.mark.gpu


def doubles(*ts):
    return [None if t is None else t.detach().double().requires_grad_() for t in ts]


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
def test_layernorm_autograd(residual, weight, bias):
    """Against torch's own gradient in 64 bits: a few units of FP32's roundoff of terms
    of order 1 summed over 20 rows."""
    x, r = leaf(20, 48, seed=1), leaf(20, 48, seed=3) if residual else None
    w, b = leaf(48, seed=2) if weight else None, leaf(48, seed=4) if bias else None
    c, e = torch.randn(20, 48).cuda(), torch.randn(20, 48).cuda()
    y, s = torch_ops.layernorm(x, w, b, residual=r)
    ((y * c).sum() + (s * e).sum()).backward()
    xd, wd, bd, rd = doubles(x, w, b, r)
    sd = xd + rd if residual else xd
    yd = torch.nn.functional.layer_norm(sd, (48,), wd, bd, 1e-5)
    ((yd * c.double()).sum() + (sd * e.double()).sum()).backward()
    assert (y.double() - yd).abs().max() < 1e-5
    for a, q in ((x, xd), (w, wd), (b, bd), (r, rd)):
        if a is not None:
            assert (a.grad.double() - q.grad).abs().max() < 1e-4


@gpu
def test_layernorm_bias_of_another_type_than_x():
    x, b = leaf(20, 48, seed=1, dtype=torch.bfloat16), leaf(48, seed=4)
    y, _ = torch_ops.layernorm(x, None, b)
    y.float().sum().backward()
    assert b.grad.dtype == torch.float32 and torch.equal(b.grad, torch.full_like(b, 20.0))


@gpu
def test_layernorm_gradient_of_the_sum_alone():
    x, r, w = leaf(6, 16, seed=1), leaf(6, 16, seed=3), leaf(16, seed=2)
    c = torch.randn(6, 16, device="cuda")
    _, s = torch_ops.layernorm(x, w, residual=r)
    (s * c).sum().backward()
    assert torch.equal(x.grad, c) and torch.equal(r.grad, c) and w.grad is None


ACT = {"relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, None: lambda v: v}


@gpu
@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("bias", [False, True])
def test_gated_linear_autograd(act, bias):
    x, w, b = leaf(20, 48, seed=1), leaf(60, 48, seed=2), leaf(60, seed=3) if bias else None
    c = torch.randn(20, 30).cuda() * 0.1
    (torch_ops.gated_linear(x, w, bias=b, act=act) * c).sum().backward()
    xd, wd, bd = doubles(x, w, b)
    z = torch.nn.functional.linear(xd, wd, bd)
    (ACT[act](z[:, :30]) * z[:, 30:] * c.double()).sum().backward()
    for a, q in ((x, xd), (w, wd), (b, bd)):
        if a is not None:
            # z is below 30 and off by 1e-5; sums of up to 60 terms below 100
            assert (a.grad.double() - q.grad).abs().max() < 2e-3, act


@gpu
def test_gated_linear_with_frozen_inputs_and_without_gradients(monkeypatch):
    x, w, b = leaf(20, 48, seed=1), leaf(60, 48, seed=2), leaf(60, seed=3)
    torch_ops.gated_linear(x, w, bias=b).sum().backward()
    for wanted in range(1, 8):
        t = [v.detach().clone().requires_grad_(bool(wanted >> i & 1)) for i, v in enumerate((x, w, b))]
        torch_ops.gated_linear(*t).sum().backward()
        for v, full in zip(t, (x, w, b)):
            assert torch.equal(v.grad, full.grad) if v.requires_grad else v.grad is None
    with torch.no_grad():
        y = torch_ops.gated_linear(x, w)
    assert not y.requires_grad and torch.equal(y, layers.gated_linear(x.detach(), w.detach()).y)


@gpu
def test_results_written_in_place_are_noticed():
    w, gain = leaf(16, 16, seed=1), leaf(16, seed=2).detach()
    q = layers.block_quantize(torch.randn(16, 16, device="cuda"))
    for write in (lambda t: layers.layernorm(t, gain, residual=t.clone(), sum_out=t),
                  lambda t: layers.layernorm(t.clone(), gain, out=t),
                  lambda t: layers.gated_linear(t.clone(), torch.cat([t, t]), out=t),
                  lambda t: layers.block_linear(q.codes, q.codes, q.scale, q.scale[:1], residual=t, out=t)):
        x = leaf(16, 16, seed=3).detach()
        y = torch_ops.gated_linear(x, w)
        write(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def block(x, gain, bias, w, b, down, op):
    """A feed-forward block: x + (act(g) u) down^T, [g | u] = layernorm(x) w^T + b."""
    n, s = op.layernorm(x, gain, bias)
    return op.linear(op.gated_linear(n, w, bias=b, act="silu"), down, residual=s)


class Plain:
    @staticmethod
    def layernorm(x, gain, bias):
        return torch.nn.functional.layer_norm(x, (x.shape[1],), gain, bias, 1e-5), x

    @staticmethod
    def gated_linear(x, w, bias, act):
        z = torch.nn.functional.linear(x, w, bias)
        return ACT[act](z[:, :len(w) // 2]) * z[:, len(w) // 2:]

    @staticmethod
    def linear(x, w, residual):
        return x @ w.t() + residual


@gpu
@pytest.mark.parametrize("rows", [1, 77, 700])
def test_a_block_of_them_together(rows):
    """Two blocks forward and backward in FP32 against the same in 64 bits: values and
    gradients of order 1 to 100, each an FP32 sum of up to 700 terms."""
    dim, wide = 96, 160
    make = [(dim,), (dim,), (2 * wide, dim), (2 * wide,), (dim, wide)]
    weights = [[leaf(*s, seed=10 * k + i) for i, s in enumerate(make)] for k in range(2)]
    for ws in weights:
        for t, scale in zip(ws, (1, 1, dim ** -0.5, 1, wide ** -0.5)):
            t.data.mul_(scale)
    x = leaf(rows, dim, seed=99)
    c = torch.randn(rows, dim).cuda()

    def loss(x, weights, op, c):
        for ws in weights:
            x = block(x, *ws, op)
        return (x * c).sum()

    loss(x, weights, torch_ops, c).backward()
    layers.check()
    xd = doubles(x)[0]
    wd = [doubles(*ws) for ws in weights]
    loss(xd, wd, Plain, c.double()).backward()
    for a, q in [(x, xd)] + [p for ws, qs in zip(weights, wd) for p in zip(ws, qs)]:
        assert (a.grad.double() - q.grad).abs().max() <= 3e-5 * max(1.0, float(q.grad.abs().max()))


@gpu
def test_serving_in_8_bits_with_block_scales():
    """layernorm -> codes -> product, against the same in 64 bits: 8-bit rounding of two
    operands, each within 2^-4 of its values (below 4% in the mean square of both), leaves
    a product within 6% of its size."""
    x, gain, bias = leaf(130, 300, seed=1).detach(), leaf(300, seed=2).detach(), leaf(300, seed=3).detach()
    w = leaf(200, 300, seed=4).detach() * 300 ** -0.5
    k = layers.block_quantize(w, 128)
    q = layers.block_quantize(layers.layernorm(x, gain, bias, out_dtype=torch.bfloat16).y)
    y = layers.block_linear(q.codes, k.codes, q.scale, k.scale)
    layers.check()
    n = torch.nn.functional.layer_norm(x.double(), (300,), gain.double(), bias.double(), 1e-5)
    ref = n @ w.double().t()
    assert (y.double() - ref).norm() / ref.norm() < 0.06


@gpu
def test_a_block_in_a_cuda_graph():
    """A training step of a block captured and replayed while an eager graph of other leaves
    lives, and two captures whose replays overlap."""
    dim, wide = 96, 160
    ws = [leaf(*s, seed=i).detach() for i, s in enumerate([(dim,), (dim,), (2 * wide, dim), (2 * wide,), (dim, wide)])]
    x = leaf(200, dim, seed=9).detach()

    def step():
        n = layers.layernorm(x, ws[0], ws[1], save_stats=True)
        h = layers.gated_linear(n.y, ws[2], bias=ws[3], save_pre=True)
        y = layers.linear(h.y, ws[4], residual=x).y
        gl = layers.linear_backward(y, h.y, ws[4])
        gg = layers.gated_linear_backward(gl.dx, n.y, ws[2], h.pre)
        return (y, gl.dw, gg.dw, gg.db, *layers.layernorm_backward(gg.dx, x, ws[0], n.mean, n.rstd, dsum=y))

    want = [t.clone() for t in step()]
    alive = torch_ops.gated_linear(leaf(4, dim, seed=1), leaf(*ws[2].shape, seed=2))
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            got.append(step())
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for made in got for a, b in zip(made, want))
    alive.sum().backward()


@gpu
def test_operators_pass_opcheck():
    x, gain, b = leaf(6, 16, seed=1), leaf(16, seed=4), leaf(16, seed=5)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.vcsr.layernorm.default,
                          (x, gain, b, x.detach().clone(), 1e-6, torch.float32), test_utils=tests)
    torch.library.opcheck(torch.ops.vcsr.gated_linear.default, (x, leaf(10, 16, seed=6), leaf(10, seed=7), "silu", True),
                          test_utils=tests)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, v = torch.empty(16, 6).t(), torch.empty(32)[::2]
        y, s, mean, rstd = torch.ops.vcsr.layernorm(x, v, None, None, 1e-6, torch.bfloat16)
        assert y.shape == (6, 16) and y.dtype == torch.bfloat16 and s.shape == (0, 16)
        assert mean.shape == rstd.shape == (6,) and y.is_contiguous()
        dx, dw, db = torch.ops.vcsr.layernorm_backward(y, x, v, mean, rstd, x, torch.float32, True, False)
        assert dx.shape == (6, 16) and dx.is_contiguous() and dw.shape == (16,) and db.shape == (0,)
        w = torch.empty(16, 10).t()
        y, pre = torch.ops.vcsr.gated_linear(x, w, None, "silu", True)
        assert y.shape == (6, 5) and pre.shape == (6, 10) and y.is_contiguous()
        assert torch.ops.vcsr.gated_linear(x, w, None, "silu", False)[1].shape == (0, 10)
        dx, dw, db = torch.ops.vcsr.gated_linear_backward(y, x, w, pre, "silu", True, True, False)
        assert dx.shape == (6, 16) and dw.shape == (10, 16) and db.shape == (0,) and dw.is_contiguous()


@pytest.mark.parametrize("fake", [False, True])
def test_layernorm_refuses_codes_without_scales(fake):
    """The operator returns no scales: 8-bit rows from it could not be read."""
    from contextlib import nullcontext

    from torch._subclasses.fake_tensor import FakeTensorMode
    from vcsr_b200 import VcsrError
    with FakeTensorMode() if fake else nullcontext():
        x, v = torch.ones(4, 16), torch.ones(16)
        for call in (lambda t: torch_ops.layernorm(x, v, v, out_dtype=t),
                     lambda t: torch.ops.vcsr.layernorm(x, v, None, x.clone(), 1e-6, t)):
            with pytest.raises(VcsrError) as e:
                call(torch.float8_e4m3fn)
            assert e.value.status == 5
