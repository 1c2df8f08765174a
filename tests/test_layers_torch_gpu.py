"""The dense layer operators as torch operators with gradients, and the example that
trains with them."""
import os
import sys

import pytest
import torch

from vcsr_b200 import layers, torch_ops

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def leaf(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).cuda().to(dtype).requires_grad_()


@gpu
@pytest.mark.parametrize("residual", [False, True])
def test_rmsnorm_autograd(residual):
    """Against torch's own gradient in 64 bits: a few units of FP32's roundoff of terms
    of order 1 summed over 20 rows."""
    x, w, r = leaf(20, 48, seed=1), leaf(48, seed=2), leaf(20, 48, seed=3) if residual else None
    c, e = torch.randn(20, 48).cuda(), torch.randn(20, 48).cuda()
    y, s = torch_ops.rmsnorm(x, w, residual=r, eps=1e-5)
    ((y * c).sum() + (s * e).sum()).backward()
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    rd = r.detach().double().requires_grad_() if residual else None
    sd = xd + rd if residual else xd
    yd = sd / torch.sqrt(sd.square().mean(1, keepdim=True) + 1e-5) * wd
    ((yd * c.double()).sum() + (sd * e.double()).sum()).backward()
    assert (y.double() - yd).abs().max() < 1e-5
    for a, b in ((x, xd), (w, wd)) + (((r, rd),) if residual else ()):
        assert (a.grad.double() - b.grad).abs().max() < 1e-4


@gpu
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
def test_linear_autograd(act):
    x, w, b, r = leaf(20, 48, seed=1), leaf(30, 48, seed=2), leaf(30, seed=3), leaf(20, 30, seed=4)
    c = torch.randn(20, 30).cuda()
    (torch_ops.linear(x, w, bias=b, residual=r, act=act) * c).sum().backward()
    d = [t.detach().double().requires_grad_() for t in (x, w, b, r)]
    z = d[0] @ d[1].t() + d[2]
    f = {None: lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu,
         "silu": torch.nn.functional.silu}[act]
    ((f(z) + d[3]) * c.double()).sum().backward()
    for a, q in zip((x, w, b, r), d):
        # sums of up to 48 FP32 products of terms below 20
        assert (a.grad.double() - q.grad).abs().max() < 2e-4, act


@gpu
def test_linear_saves_nothing_without_gradients():
    x, w = leaf(8, 16).detach(), leaf(4, 16)
    with torch.no_grad():
        y = torch_ops.linear(x, w, act="gelu")
    assert not y.requires_grad
    assert torch.equal(y, layers.linear(x, w.detach(), act="gelu").y)


@gpu
def test_operators_pass_torch_opcheck():
    x, w, b = leaf(6, 16, seed=1), leaf(5, 16, seed=2), leaf(5, seed=3)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.vcsr.linear.default, (x, w, b, None, "gelu", True),
                          test_utils=tests)
    gain = leaf(16, seed=4)
    torch.library.opcheck(torch.ops.vcsr.rmsnorm.default, (x, gain, x.detach().clone(), 1e-6, torch.float32),
                          test_utils=tests)


def test_fake_shapes_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w = torch.empty(6, 16), torch.empty(5, 16)
        y, pre = torch.ops.vcsr.linear(x, w, None, None, "gelu", True)
        assert y.shape == pre.shape == (6, 5)
        y, s, rstd = torch.ops.vcsr.rmsnorm(x, torch.empty(16), None, 1e-6, torch.bfloat16)
        assert y.shape == (6, 16) and y.dtype == torch.bfloat16 and s.shape == (0, 16)
        assert rstd.shape == (6,)


def test_fake_results_are_row_major_whatever_the_inputs_are():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, w, v = torch.empty(16, 6).t(), torch.empty(16, 5).t(), torch.empty(32)[::2]
        results = [torch.ops.vcsr.rmsnorm(x, v, x, 1e-6, torch.bfloat16),
                   torch.ops.vcsr.rmsnorm_backward(x, x, v, torch.empty(6), x),
                   torch.ops.vcsr.linear(x, w, None, torch.empty(5, 6).t(), "gelu", True),
                   torch.ops.vcsr.linear_backward(torch.empty(5, 6).t(), x, w, None, "none")]
        assert all(t.is_contiguous() for ts in results for t in ts)


@gpu
def test_results_are_row_major_whatever_the_inputs_are():
    x, w, v, r = leaf(16, 6).detach().t(), leaf(16, 5).detach().t(), leaf(32).detach()[::2], leaf(5, 6).detach().t()
    y, s, rstd = torch.ops.vcsr.rmsnorm(x, v, x, 1e-6, torch.bfloat16)
    results = [(y, s), torch.ops.vcsr.rmsnorm_backward(y, s, v, rstd, s),
               torch.ops.vcsr.linear(x, w, None, r, "gelu", True), torch.ops.vcsr.linear_backward(r, x, w, None, "none")]
    assert all(t.is_contiguous() for ts in results for t in ts)


class Host:
    """The layer operators on CPU tensors, in plain operations, that note their calls."""

    def __init__(self, monkeypatch):
        self.calls = []
        for name in ("rmsnorm", "rmsnorm_backward", "linear", "linear_backward"):
            monkeypatch.setattr(layers, name, getattr(self, name))

    def rmsnorm(self, x, weight, residual=None, eps=1e-6, out_dtype=None, save_rstd=False):
        s = x if residual is None else x + residual
        rstd = (s.square().mean(1) + eps).rsqrt()
        return layers.NormOut((s * rstd[:, None] * weight).to(out_dtype), s, rstd, None)

    def rmsnorm_backward(self, dy, s, weight, rstd, dsum=None, need_dweight=True):
        self.calls.append(("rmsnorm", dict(dsum=dsum is not None, dweight=need_dweight)))
        h, g = s * rstd[:, None], dy * weight
        dx = rstd[:, None] * (g - h * (g * h).mean(1, keepdim=True))
        return dx if dsum is None else dx + dsum, (dy * h).sum(0) if need_dweight else None

    def linear(self, x, w, bias=None, residual=None, act=None, save_pre=False):
        z = x @ w.t() + (0 if bias is None else bias)
        y = (torch.nn.functional.silu(z) if act == "silu" else z.clone()) + (0 if residual is None else residual)
        return layers.LinearOut(y, z if save_pre else None)

    def linear_backward(self, dy, x, w, pre=None, act=None, need_dx=True, need_dw=True, need_db=True):
        self.calls.append(("linear", dict(dx=need_dx, dw=need_dw, db=need_db)))
        s = torch.sigmoid(pre) if act == "silu" else None
        dz = dy * s * (1 + pre * (1 - s)) if act == "silu" else dy
        return layers.LinearGrad(dz @ w if need_dx else None, dz.t() @ x if need_dw else None,
                                 dz.sum(0) if need_db else None)


class Zeros(torch.utils._python_dispatch.TorchDispatchMode):
    """Counts the tensors of zeros that are made."""
    made = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.made += "zero" in func.name()
        return func(*args, **(kwargs or {}))


def host_leaf(*shape):
    return torch.randn(*shape, dtype=torch.float64).requires_grad_()


def test_no_gradient_is_made_of_zeros(monkeypatch):
    """Results that nothing used have no gradient: no matrix of zeros stands for it."""
    host = Host(monkeypatch)
    x, gain, r, w = host_leaf(6, 16), host_leaf(16), host_leaf(6, 16), host_leaf(5, 16)
    for residual in (None, r):
        y, _ = torch_ops.rmsnorm(x, gain, residual=residual, out_dtype=torch.float64)
        z = torch_ops.linear(y, w, act="silu")
        c = torch.ones_like(z)
        with Zeros() as zeros:
            z.backward(c)
        assert zeros.made == 0
        assert host.calls[-1] == ("rmsnorm", dict(dsum=False, dweight=True))
    n = len(host.calls)
    x.grad = gain.grad = r.grad = None
    _, s = torch_ops.rmsnorm(x, gain, residual=r, out_dtype=torch.float64)
    s.backward(torch.full_like(s, 2.0))  # the sum alone: no kernel
    assert len(host.calls) == n and gain.grad is None
    assert bool((x.grad == 2.0).all()) and bool((r.grad == 2.0).all())


def test_only_wanted_gradients_are_asked_for(monkeypatch):
    """Every choice of inputs that take gradients: the backward call makes theirs and no
    other's, and they are what they are together."""
    host = Host(monkeypatch)
    make = dict(x=(6, 16), w=(5, 16), bias=(5,), residual=(6, 5))
    values = {k: torch.randn(*s, dtype=torch.float64) for k, s in make.items()}
    full = None
    for wanted in range(15, 0, -1):
        t = {k: v.clone().requires_grad_(bool(wanted >> i & 1)) for i, (k, v) in enumerate(values.items())}
        host.calls.clear()
        torch_ops.linear(**t, act="silu").sum().backward()
        flags = [t[k].requires_grad for k in ("x", "w", "bias")]
        assert host.calls == ([("linear", dict(zip(("dx", "dw", "db"), flags)))] if any(flags) else [])
        full = full or {k: v.grad for k, v in t.items()}
        for k, v in t.items():
            assert torch.equal(v.grad, full[k]) if v.requires_grad else v.grad is None
    x, gain, r = (torch.randn(*s, dtype=torch.float64) for s in ((6, 16), (16,), (6, 16)))
    for wanted in range(7, 0, -1):
        t = [v.clone().requires_grad_(bool(wanted >> i & 1)) for i, v in enumerate((x, gain, r))]
        host.calls.clear()
        y, s = torch_ops.rmsnorm(*t, out_dtype=torch.float64)
        (y.sum() + s.sum()).backward()
        assert host.calls[-1][1]["dweight"] == t[1].requires_grad
        assert [v.grad is not None for v in t] == [v.requires_grad for v in t]


@gpu
@pytest.mark.parametrize("frozen", ["x", "w", "xw"])
def test_linear_autograd_with_frozen_inputs(frozen):
    t = dict(x=leaf(20, 48, seed=1), w=leaf(30, 48, seed=2), bias=leaf(30, seed=3), residual=leaf(20, 30, seed=4))
    c = torch.randn(20, 30).cuda()
    (torch_ops.linear(**t, act="gelu") * c).sum().backward()
    some = {k: v.detach().clone().requires_grad_(k not in frozen) for k, v in t.items()}
    (torch_ops.linear(**some, act="gelu") * c).sum().backward()
    for k, v in some.items():
        assert v.grad is None if k in frozen else torch.equal(v.grad, t[k].grad)


@gpu
def test_gradient_of_the_sum_alone():
    x, gain, r = leaf(6, 16, seed=1), leaf(16, seed=2), leaf(6, 16, seed=3)
    c = torch.randn(6, 16, device="cuda")
    _, s = torch_ops.rmsnorm(x, gain, residual=r)
    (s * c).sum().backward()
    assert torch.equal(x.grad, c) and torch.equal(r.grad, c) and gain.grad is None
    assert x.grad.data_ptr() != r.grad.data_ptr()


@gpu
def test_a_step_between_forward_and_backward_is_noticed():
    """As with torch's optimizers: the weights that the backward pass saved are gone."""
    x, w, b = leaf(6, 16, seed=1), leaf(5, 16, seed=2), leaf(5, seed=3)
    half = w.detach().bfloat16().requires_grad_()
    opt = layers.AdamW([w, b], copies=[half.detach(), b.detach().bfloat16()])
    for operand, grads in ((w, [w.detach(), None]), (half, [w.detach(), b.detach()])):
        y = torch_ops.linear(x.to(operand.dtype), operand)
        opt.step(grads)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    before = b._version
    opt.step([w.detach(), None])  # what has no gradient is not written
    assert b._version == before


@gpu
def test_results_written_in_place_are_noticed():
    w, gain = leaf(16, 16, seed=1), leaf(16, seed=2).detach()
    for write in (lambda t: layers.rmsnorm(t, gain, residual=t.clone(), sum_out=t),
                  lambda t: layers.rmsnorm(t.clone(), gain, out=t),
                  lambda t: layers.linear(t.clone(), t.clone(), residual=t, out=t)):
        x = leaf(16, 16, seed=3).detach()
        y = torch_ops.linear(x, w)
        write(x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@gpu
def test_example_trains_and_serves():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import train_layer
    finally:
        sys.path.pop(0)
    losses, off = train_layer.main(rows=3000, width=64, steps=20, verbose=False)
    assert all(b == b for b in losses) and losses[-1] < 0.7 * losses[0], losses
    # two 8-bit products: each rounds its operands by up to 2^-4 of them, 3% in the mean
    # square, on a part of the answer; a wrong scale is off by 1
    assert off < 0.1, off
