"""Layer norm, the gated product and block-scaled 8-bit operands without a GPU: argument
checks come before any device work, sizes of zero are valid calls, and workspace queries
need no device."""
import ctypes

import pytest
import torch

import vcsr_b200 as V
from test_layers_cpu import P, refused
from vcsr_b200 import layers


def filled(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def norm(**kw):
    return filled(V._LayernormArgs(rows=2, dim=8, x=P, ldx=8, weight=P, bias=P, y=P, ldy=8, eps=1e-5), kw)


@pytest.mark.parametrize("status,text,kw", [
    (1, "negative", dict(rows=-1)), (1, "x is NULL", dict(x=None)), (1, "pitch of x", dict(ldx=7)),
    (1, "y is not aligned", dict(y=P + 2)), (1, "pitch of residual", dict(residual=P, ldr=3)),
    (1, "eps", dict(eps=-1.0)), (1, "eps", dict(eps=float("nan"))), (1, "scale", dict(y_dtype=3)),
    (5, "x type", dict(x_dtype=3)), (5, "weight type", dict(w_dtype=1)), (5, "y type", dict(y_dtype=4)),
    (8, "rows", dict(rows=1 << 31)), (1, "pitch of sum", dict(sum=P, lds=0)),
    (1, "bias is not aligned", dict(bias=P + 2)), (1, "weight is not aligned", dict(weight=P + 1)),
    (1, "mean is not aligned", dict(mean=P + 2)), (1, "rstd is not aligned", dict(rstd=P + 2)),
    (1, "scale is not aligned", dict(scale=P + 1, y_dtype=3))])
def test_layernorm_refuses(status, text, kw):
    refused(status, "vcsr_layernorm", norm(**kw), text)


def test_layernorm_of_nothing():
    L = V.lib()
    for kw in (dict(rows=0), dict(dim=0)):
        assert L.vcsr_layernorm(ctypes.byref(norm(**kw)), None) == 0
    assert L.vcsr_layernorm(None, None) == 1 and L.vcsr_layernorm_grad(None, None) == 1
    assert L.vcsr_layernorm_grad_workspace(0, 8) == 0 and L.vcsr_layernorm_grad_workspace(3, 8) >= 2 * 96


@pytest.mark.parametrize("status,text,kw", [
    (1, "workspace", dict(dweight=P)), (1, "workspace", dict(dbias=P)), (1, "dy is NULL", dict(dy=None)),
    (1, "s is NULL", dict(s=None)), (5, "dy type", dict(dy_dtype=3)), (5, "x type", dict(x_dtype=3)),
    (5, "weight type", dict(w_dtype=2)), (1, "rstd", dict(rstd=None)), (1, "mean", dict(mean=None)),
    (1, "pitch of dx", dict(lddx=1)), (1, "dx is NULL", dict(dx=None)), (1, "pitch of dsum", dict(dsum=P, ldds=7)),
    (1, "dbias is not aligned", dict(dbias=P + 1)), (8, "rows", dict(rows=1 << 31)),
    (1, "workspace", dict(dbias=P, workspace=P + 8, workspace_bytes=1 << 20)),
    (1, "workspace", dict(dbias=P, workspace=P, workspace_bytes=63))])
def test_layernorm_grad_refuses(status, text, kw):
    a = filled(V._LayernormGradArgs(rows=2, dim=8, dy=P, lddy=8, s=P, lds=8, weight=P, mean=P, rstd=P, dx=P, lddx=8), kw)
    refused(status, "vcsr_layernorm_grad", a, text)


def test_python_forms_refuse_cpu_tensors():
    for call in (lambda t: layers.layernorm(t, t[0]), lambda t: layers.layernorm(x=t),
                 lambda t: layers.layernorm_backward(t, t, t[0], t[0], t[0])):
        with pytest.raises(V.VcsrError) as e:
            call(torch.zeros(4, 4))
        assert e.value.status == 1
