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


@gpu
def test_operators_pass_opcheck():
    x, gain, b = leaf(6, 16, seed=1), leaf(16, seed=4), leaf(16, seed=5)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.vcsr.layernorm.default,
                          (x, gain, b, x.detach().clone(), 1e-6, torch.float32), test_utils=tests)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, v = torch.empty(16, 6).t(), torch.empty(32)[::2]
        y, s, mean, rstd = torch.ops.vcsr.layernorm(x, v, None, None, 1e-6, torch.bfloat16)
        assert y.shape == (6, 16) and y.dtype == torch.bfloat16 and s.shape == (0, 16)
        assert mean.shape == rstd.shape == (6,) and y.is_contiguous()
        dx, dw, db = torch.ops.vcsr.layernorm_backward(y, x, v, mean, rstd, x, torch.float32, True, False)
        assert dx.shape == (6, 16) and dx.is_contiguous() and dw.shape == (16,) and db.shape == (0,)
