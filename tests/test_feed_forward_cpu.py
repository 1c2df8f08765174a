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


def gated(**kw):
    return filled(V._GatedLinearArgs(M=2, N=4, K=8, x=P, ldx=8, w=P, ldw=8, y=P, ldy=4, dtype=1, out_dtype=1), kw)


@pytest.mark.parametrize("status,text,kw", [
    (1, "negative", dict(K=-1)), (8, "2^31", dict(M=1 << 31)), (8, "2 N", dict(N=1 << 30)), (5, "type 4", dict(dtype=4)),
    (5, "output type", dict(out_dtype=0)), (5, "output type", dict(dtype=3, out_dtype=3, x_scale=P, w_scale=P)),
    (5, "activation", dict(act=4)), (1, "x is NULL", dict(x=None)), (1, "w is NULL", dict(w=None)),
    (1, "y is NULL", dict(y=None)), (1, "pitch of w", dict(ldw=7)), (1, "pitch of y", dict(ldy=3)),
    (1, "scales", dict(x_scale=P)), (1, "need x_scale", dict(dtype=3)), (1, "pitch of pre", dict(pre=P, ldp=7)),
    (1, "bias is not aligned", dict(bias=P + 1)), (1, "x_scale is not aligned", dict(dtype=3, x_scale=P + 2, w_scale=P)),
    (1, "workspace", dict(x=P + 2)), (1, "workspace", dict(dtype=0, out_dtype=0)),
    (1, "workspace", dict(dtype=0, out_dtype=0, workspace=P + 16, workspace_bytes=1 << 20)),
    (8, "2^31 - 513", dict(M=(1 << 31) - 512))])
def test_gated_linear_refuses(status, text, kw):
    refused(status, "vcsr_gated_linear", gated(**kw), text)


def test_gated_linear_of_nothing():
    L = V.lib()
    for kw in (dict(M=0), dict(N=0)):
        assert L.vcsr_gated_linear(ctypes.byref(gated(**kw)), None) == 0
        assert L.vcsr_gated_linear_workspace(ctypes.byref(gated(**kw))) == 0
    assert L.vcsr_gated_linear(None, None) == 1 and L.vcsr_gated_linear_grad(None, None) == 1
    # none for aligned 16-bit operands, [g | u] for FP32 ones unless it is the caller's
    assert L.vcsr_gated_linear_workspace(ctypes.byref(gated())) == 0
    assert L.vcsr_gated_linear_workspace(ctypes.byref(gated(dtype=0, out_dtype=0))) >= 2 * 8 * 4
    assert L.vcsr_gated_linear_workspace(ctypes.byref(gated(dtype=0, out_dtype=0, pre=P, ldp=8))) == 0


@pytest.mark.parametrize("status,text,kw", [
    (1, "dy is NULL", dict(dy=None)), (1, "pre is NULL", dict(pre=None)), (5, "type 3", dict(dtype=3)),
    (5, "activation", dict(act=-1)), (1, "workspace", dict()), (1, "w is NULL", dict(w=None)),
    (1, "x is NULL", dict(x=None)), (1, "pitch of pre", dict(ldp=7)), (1, "pitch of dw", dict(lddw=7)),
    (1, "pitch of dx", dict(lddx=7)), (1, "dbias is not aligned", dict(dbias=P + 2)), (8, "2 N", dict(N=1 << 30))])
def test_gated_linear_grad_refuses(status, text, kw):
    a = filled(V._GatedLinearGradArgs(M=2, N=4, K=8, dy=P, lddy=4, pre=P, ldp=8, x=P, ldx=8, w=P, ldw=8, dx=P, lddx=8, dw=P,
                                      lddw=8), kw)
    refused(status, "vcsr_gated_linear_grad", a, text)


def block(**kw):
    return filled(V._BlockLinearArgs(M=2, N=4, K=256, x=P, ldx=256, w=P, ldw=256, x_scale=P, ldxs=2, w_scale=P, ldws=2,
                                     y=P, ldy=4), kw)


@pytest.mark.parametrize("status,text,kw", [
    (1, "negative", dict(M=-1)), (8, "2^31", dict(K=1 << 31)), (5, "output type", dict(out_dtype=3)),
    (5, "activation", dict(act=9)), (1, "x is NULL", dict(x=None)), (1, "pitch of x ", dict(ldx=255)),
    (1, "pitch of w ", dict(ldw=0)), (1, "x_scale is NULL", dict(x_scale=None)), (1, "pitch of x_scale", dict(ldxs=1)),
    (1, "pitch of w_scale", dict(ldws=1)), (1, "w_scale is not aligned", dict(w_scale=P + 1)),
    (1, "pitch of residual", dict(residual=P, ldr=3)), (1, "bias is not aligned", dict(bias=P + 2)),
    (1, "y is NULL", dict(y=None)), (1, "workspace", dict(x=P + 1)), (1, "workspace", dict(ldw=257)),
    (8, "2^31 - 513", dict(M=(1 << 31) - 512)), (8, "2^31 - 513", dict(N=(1 << 31) - 1, ldy=1 << 31))])
def test_block_linear_refuses(status, text, kw):
    refused(status, "vcsr_block_linear", block(**kw), text)


def test_block_calls_of_nothing_and_refusals():
    L = V.lib()
    for kw in (dict(M=0), dict(N=0)):
        assert L.vcsr_block_linear(ctypes.byref(block(**kw)), None) == 0
    assert L.vcsr_block_linear(None, None) == 1
    assert L.vcsr_block_linear_workspace(ctypes.byref(block())) == 0

    def quantize(rows=2, dim=200, x=P, ldx=200, dtype=0, block_rows=1, codes=P, ldc=200, scale=P, lds=2):
        return L.vcsr_block_quantize(x, ldx, rows, dim, dtype, block_rows, codes, ldc, scale, lds, None)

    def dequantize(rows=2, dim=200, codes=P, ldc=200, scale=P, lds=2, block_rows=1, out=P, ldo=200, dtype=0):
        return L.vcsr_block_dequantize(codes, ldc, scale, lds, rows, dim, block_rows, out, ldo, dtype, None)

    for call in (quantize, dequantize):
        assert call(rows=0) == 0 and call(dim=0) == 0
        assert call(rows=-1) == 1 and call(block_rows=64) == 5 and call(dtype=3) == 5 and call(rows=1 << 31) == 8
        assert call(codes=None) == 1 and call(ldc=199) == 1 and call(scale=None) == 1 and call(lds=1) == 1
        assert call(scale=P + 2) == 1
    assert quantize(x=None) == 1 and quantize(ldx=1) == 1 and quantize(x=P + 2) == 1
    assert dequantize(out=None) == 1 and dequantize(ldo=0) == 1 and dequantize(out=P + 2) == 1


def test_python_forms_of_the_products_refuse_cpu_tensors():
    t = torch.zeros(4, 4)
    for call in (lambda: layers.gated_linear(t, t), lambda: layers.gated_linear(w=t, x=t), lambda: layers.block_quantize(t),
                 lambda: layers.gated_linear_backward(t, t, t, t), lambda: layers.block_dequantize(t, t),
                 lambda: layers.block_linear(t, t, t, t)):
        with pytest.raises(V.VcsrError) as e:
            call()
        assert e.value.status == 1
