"""The dense layer operators' C entry points without a GPU: argument checks come
before any device work, sizes of zero are valid calls, and workspace queries need
no device."""
import ctypes

import numpy as np
import pytest

import vcsr_b200 as V

P = 1 << 20  # stands for an aligned device pointer; never followed


def refused(status, name, a, text):
    L = V.lib()
    assert getattr(L, name)(ctypes.byref(a), None) == status
    assert text in L.vcsr_last_error().decode()


def norm(**kw):
    a = V._RmsnormArgs(rows=2, dim=8, x=P, ldx=8, weight=P, y=P, ldy=8, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("status,text,kw", [
    (1, "negative", dict(rows=-1)), (1, "x is NULL", dict(x=None)), (1, "pitch of x", dict(ldx=7)),
    (1, "not aligned", dict(y=P + 2)), (1, "pitch of residual", dict(residual=P, ldr=3)),
    (1, "eps", dict(eps=-1.0)), (1, "scale", dict(y_dtype=3)), (5, "x type", dict(x_dtype=3)),
    (5, "weight type", dict(w_dtype=1)), (5, "y type", dict(y_dtype=4)), (8, "rows", dict(rows=1 << 31)),
    (1, "pitch of sum", dict(sum=P, lds=0))])
def test_rmsnorm_refuses(status, text, kw):
    refused(status, "vcsr_rmsnorm", norm(**kw), text)


def test_rmsnorm_of_nothing():
    L = V.lib()
    for kw in (dict(rows=0), dict(dim=0)):
        assert L.vcsr_rmsnorm(ctypes.byref(norm(**kw)), None) == 0
    assert L.vcsr_rmsnorm(None, None) == 1
    assert L.vcsr_rmsnorm_grad_workspace(0, 8) == 0 and L.vcsr_rmsnorm_grad_workspace(3, 8) >= 96


@pytest.mark.parametrize("status,text,kw", [
    (1, "workspace", dict(dweight=P)), (1, "dy is NULL", dict(dy=None)), (5, "dy type", dict(dy_dtype=3)),
    (1, "rstd", dict(rstd=None)), (1, "pitch of dx", dict(lddx=1))])
def test_rmsnorm_grad_refuses(status, text, kw):
    a = V._RmsnormGradArgs(rows=2, dim=8, dy=P, lddy=8, s=P, lds=8, weight=P, rstd=P, dx=P, lddx=8)
    for k, v in kw.items():
        setattr(a, k, v)
    refused(status, "vcsr_rmsnorm_grad", a, text)


@pytest.mark.parametrize("status,text,kw", [
    (1, "negative", dict(K=-1)), (8, "2^31", dict(M=1 << 31)), (5, "type 4", dict(dtype=4)),
    (5, "output type", dict(out_dtype=1)), (5, "activation", dict(act=4)), (1, "x is NULL", dict(x=None)),
    (1, "pitch of w", dict(ldw=7)), (1, "scales", dict(x_scale=P)), (1, "need x_scale", dict(dtype=3)),
    (1, "pitch of pre", dict(pre=P, ldp=1)), (1, "not aligned", dict(bias=P + 1))])
def test_linear_refuses(status, text, kw):
    a = V._LinearArgs(M=2, N=4, K=8, x=P, ldx=8, w=P, ldw=8, y=P, ldy=4)
    for k, v in kw.items():
        setattr(a, k, v)
    refused(status, "vcsr_linear", a, text)


def test_linear_of_nothing():
    L = V.lib()
    for kw in (dict(M=0), dict(N=0)):
        a = V._LinearArgs(M=2, N=4, K=8)
        for k, v in kw.items():
            setattr(a, k, v)
        assert L.vcsr_linear(ctypes.byref(a), None) == 0
    assert L.vcsr_linear(None, None) == 1 and L.vcsr_linear_grad(None, None) == 1


@pytest.mark.parametrize("status,text,kw", [
    (1, "dy is NULL", dict(dy=None)), (1, "pre is NULL", dict(act=2)), (5, "type 3", dict(dtype=3)),
    (1, "workspace", dict(dbias=P)), (1, "w is NULL", dict(w=None)), (1, "x is NULL", dict(x=None))])
def test_linear_grad_refuses(status, text, kw):
    a = V._LinearGradArgs(M=2, N=4, K=8, dy=P, lddy=4, x=P, ldx=8, w=P, ldw=8, dx=P, lddx=8, dw=P, lddw=8)
    for k, v in kw.items():
        setattr(a, k, v)
    refused(status, "vcsr_linear_grad", a, text)


def test_adamw_sizes_and_refusals():
    L = V.lib()
    n = np.array([1, 256, 257, 0], np.int64)
    assert L.vcsr_adamw_state_values(4, n.ctypes.data) == 256 + 256 + 512
    h = ctypes.c_void_p()
    p = np.zeros(4, np.uint64)

    def create(numel=n, params=p, p_dtype=0, copies=None, copy_dtype=0, bits=32):
        return L.vcsr_adamw_create(4, numel.ctypes.data, params.ctypes.data, p_dtype, copies, copy_dtype,
                                   bits, ctypes.byref(h), None)

    assert create() == 1 and "parameter 0" in L.vcsr_last_error().decode()
    assert create(p_dtype=3) == 5 and create(bits=16) == 5
    assert create(copies=p.ctypes.data) == 5
    assert create(numel=np.array([1, -1, 0, 0], np.int64), params=np.full(4, P, np.uint64)) == 1
    assert not h.value
    assert L.vcsr_adamw_step(None, None, None) == 1
    L.vcsr_adamw_destroy(None)


def test_python_operators_refuse_cpu_tensors():
    import torch
    from vcsr_b200 import layers
    for call in (lambda t: layers.rmsnorm(t, t[0]), lambda t: layers.linear(t, t),
                 lambda t: layers.linear_backward(t, t, t), lambda t: layers.AdamW([t]),
                 lambda t: layers.dequantize(t, t[0])):
        with pytest.raises(V.VcsrError) as e:
            call(torch.zeros(4, 4))
        assert e.value.status == 1


def test_python_operators_take_keywords():
    """The first tensor by name is refused, or taken, as it is by position."""
    import torch
    from vcsr_b200 import layers
    t = torch.zeros(4, 4)
    for fn, kw in ((layers.rmsnorm, dict(x=t, weight=t[0])), (layers.linear, dict(x=t, w=t)),
                   (layers.rmsnorm_backward, dict(dy=t, s=t, weight=t[0], rstd=t[0])),
                   (layers.linear_backward, dict(dy=t, x=t, w=t)), (layers.dequantize, dict(codes=t, scale=t[0])),
                   (layers.linear, dict(w=t))):
        with pytest.raises(V.VcsrError) as e:
            fn(**kw)
        assert e.value.status == 1 and fn.__name__ in e.value.msg


@pytest.mark.parametrize("name,kw", [("rstd", dict(rstd=P + 2)), ("scale", dict(scale=P + 1, y_dtype=3))])
def test_rmsnorm_refuses_vectors_off_their_type(name, kw):
    refused(1, "vcsr_rmsnorm", norm(**kw), f"{name} is not aligned")


@pytest.mark.parametrize("name", ["x_scale", "w_scale"])
def test_linear_refuses_scales_off_their_type(name):
    a = V._LinearArgs(M=2, N=4, K=16, x=P, ldx=16, w=P, ldw=16, y=P, ldy=4, x_scale=P, w_scale=P, dtype=3)
    setattr(a, name, P + 2)
    refused(1, "vcsr_linear", a, f"{name} is not aligned")


def test_adamw_refuses_overlapping_parameters():
    L = V.lib()
    h = ctypes.c_void_p()

    def create(numel, params):
        numel, params = np.array(numel, np.int64), np.array(params, np.uint64)
        return L.vcsr_adamw_create(len(numel), numel.ctypes.data, params.ctypes.data, 0, None, 0, 32, ctypes.byref(h), None)

    for numel, params in (([8, 4, 8], [P, P + 64, P]), ([4, 8], [P + 28, P]), ([300, 1], [P, P + 4 * 299])):
        assert create(numel, params) == 1 and "overlap" in L.vcsr_last_error().decode()
    # neighbours, and tensors without values wherever they are
    create([8, 0, 4], [P, P + 16, P + 32])
    assert "overlap" not in L.vcsr_last_error().decode()
    if h.value:
        L.vcsr_adamw_destroy(h)
