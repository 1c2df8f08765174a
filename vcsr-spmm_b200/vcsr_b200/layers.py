"""Dense layer operators beside the sparse product, on torch CUDA tensors: the
norm (rmsnorm), the product with its epilogue (linear), their gradients, and
the optimizer step over many tensors (AdamW).  The mathematics and the rules of
types and aliasing stand with the C entry points in include/vcsr_spmm.h.

    from vcsr_b200 import layers
    n = layers.rmsnorm(C, gain, residual=h, save_rstd=True)
    out = layers.linear(n.y, W, bias=b, act="gelu", save_pre=True)
    g = layers.linear_backward(dy, n.y, W, pre=out.pre, act="gelu")
    dx, dgain = layers.rmsnorm_backward(g.dx, n.sum, gain, n.rstd)
    opt = layers.AdamW([W, b, gain], lr=1e-3)
    opt.step([g.dw, g.db, dgain])

Matrices are two-dimensional; rows may be strided.  An input whose columns are
not neighbours in memory (or whose rows overlap, as an expanded gradient's do)
is copied first.  Work is enqueued on `stream`, by default the current stream
of the tensors' device, without synchronising; results and scratch are
allocated on that stream.  Wrong arguments raise VcsrError.  There is no CPU
form.
"""
from __future__ import annotations

import ctypes as C
import functools
import operator
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import (VcsrError, _AdamwStepArgs, _check, _LinearArgs, _LinearGradArgs, _RmsnormArgs,
               _RmsnormGradArgs, _stream, lib)

INVALID, UNSUPPORTED = 1, 5
F32, BF16, F16, E4M3 = range(4)
_TYPE = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16,
         torch.float8_e4m3fn: E4M3}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3}
BLOCK = 256  # values per scale of an 8-bit AdamW state

_current_stream = torch._C._cuda_getCurrentRawStream
_dtype = operator.attrgetter("dtype")
# Tells autograd, as torch's in-place operations do, that tensors hold new values: a
# backward pass that had saved the old ones raises.
_new_values = torch.autograd.graph.increment_version


def _type(dtype, name):
    try:
        return _TYPE[dtype]
    except KeyError:
        raise VcsrError(UNSUPPORTED, f"{name} has type {dtype}") from None


_current_device = torch._C._cuda_getDevice


def _operator(fn):
    """Runs fn with the first tensor's device and the given stream current."""
    name = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, stream=None, **kw):
        first = args[0] if args else kw.get(name)
        try:
            index = first.get_device()
        except AttributeError:
            index = -1
        if index < 0:
            raise VcsrError(INVALID, f"{fn.__name__} takes CUDA tensors")
        if stream is None and index == _current_device():
            return fn(*args, **kw)
        with torch.cuda.device(index):
            if stream is None:
                return fn(*args, **kw)
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream, device=first.device)
            with torch.cuda.stream(stream):
                return fn(*args, **kw)
    return call


def _matrix(t, name, like, rows, cols, dtype):
    """t as a (rows, cols) input the C entry points read: its tensor and pitch."""
    if not isinstance(t, torch.Tensor) or t.get_device() != like.get_device():
        raise VcsrError(INVALID, f"{name} must be a tensor on {like.device}")
    if t.dtype is not dtype:
        raise VcsrError(UNSUPPORTED, f"{name} has type {t.dtype}, expected {dtype}")
    if t.shape != (rows, cols):
        raise VcsrError(INVALID, f"{name} must be ({rows}, {cols}), got {tuple(t.shape)}")
    if t.is_contiguous():
        return t, cols
    s0, s1 = t.stride()
    if (s1 != 1 and cols > 1) or (s0 < cols and rows > 1):
        return t.contiguous(), cols
    return t, max(s0, cols)


def _out(t, name, like, rows, cols, dtype):
    """The output t (checked), or a new one."""
    if t is None:
        if like.dtype is dtype and like.shape == (rows, cols) and like.is_contiguous():
            return torch.empty_like(like), cols
        return like.new_empty((rows, cols), dtype=dtype), cols
    got, ld = _matrix(t, name, like, rows, cols, dtype)
    if got is not t:
        raise VcsrError(INVALID, f"the columns of {name} must be neighbours in memory")
    return t, ld


def _vector(t, name, like, n, dtype):
    if not isinstance(t, torch.Tensor) or t.get_device() != like.get_device():
        raise VcsrError(INVALID, f"{name} must be a tensor on {like.device}")
    if t.dtype is not dtype:
        raise VcsrError(UNSUPPORTED, f"{name} has type {t.dtype}, expected {dtype}")
    if t.shape != (n,):
        raise VcsrError(INVALID, f"{name} must be ({n},), got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _shape(t, name):
    if not isinstance(t, torch.Tensor):
        raise VcsrError(INVALID, f"{name} must be a tensor")
    if t.dim() != 2:
        raise VcsrError(INVALID, f"{name} must be two-dimensional, got {tuple(t.shape)}")
    return t.shape


def _workspace(n, like):
    return like.new_empty(n, dtype=torch.uint8) if n else None


def _p(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------- the norm

class NormOut(NamedTuple):
    y: torch.Tensor                 # the normalised rows (codes with an 8-bit out_dtype)
    sum: torch.Tensor               # x + residual (x itself without a residual)
    rstd: Optional[torch.Tensor]    # with save_rstd
    scale: Optional[torch.Tensor]   # one per row, 8-bit y only


@_operator
def rmsnorm(x, weight, residual=None, eps=1e-6, out_dtype=None, out=None, sum_out=None,
            save_rstd=False) -> NormOut:
    """y = s * rstd * weight, s = x + residual, rstd = 1/sqrt(mean(s^2) + eps) per
    row (vcsr_rmsnorm).  x and residual: (rows, dim) float32, bfloat16 or float16;
    weight: (dim,) of x's type or float32; out_dtype: any of the three or
    float8_e4m3fn (then y holds codes and scale their rows' scales).  sum_out may
    be x or residual itself."""
    rows, dim = _shape(x, "x")
    dt = x.dtype
    x_type = _type(dt, "x")
    x, ldx = _matrix(x, "x", x, rows, dim, dt)
    if isinstance(weight, torch.Tensor) and weight.dtype == torch.float32:
        weight = _vector(weight, "weight", x, dim, torch.float32)
    else:
        weight = _vector(weight, "weight", x, dim, dt)
    ldr = 0
    if residual is not None:
        residual, ldr = _matrix(residual, "residual", x, rows, dim, dt)
    y_dtype = out_dtype or getattr(out, "dtype", dt)
    y_type = _type(y_dtype, "out")
    y, ldy = _out(out, "out", x, rows, dim, y_dtype)
    s, lds = (None, 0)
    if residual is not None or sum_out is not None:
        s, lds = _out(sum_out, "sum_out", x, rows, dim, dt)
    rstd = x.new_empty(rows, dtype=torch.float32) if save_rstd else None
    scale = x.new_empty(rows, dtype=torch.float32) if y_type == E4M3 else None
    a = _RmsnormArgs(rows, dim, x.data_ptr(), ldx, _p(residual), ldr, weight.data_ptr(),
                     y.data_ptr(), ldy, _p(s), lds, _p(rstd), _p(scale), eps, x_type,
                     _TYPE[weight.dtype], y_type)
    _check(lib().vcsr_rmsnorm(a, _current_stream(x.get_device())))
    if out is not None or sum_out is not None:
        _new_values([t for t in (out, sum_out) if t is not None])
    return NormOut(y, x if s is None else s, rstd, scale)


@_operator
def rmsnorm_backward(dy, s, weight, rstd, dsum=None, need_dweight=True):
    """(dx, dweight) of rmsnorm from its sum and rstd (vcsr_rmsnorm_grad); dx is the
    gradient of x and of the residual, dsum (optional) the one that reached s by
    other ways.  dy: float32, bfloat16 or float16; dsum and dx are of s's type."""
    rows, dim = _shape(s, "s")
    dy_type = _type(dy.dtype, "dy")
    dt = s.dtype
    x_type = _type(dt, "s")
    s, lds = _matrix(s, "s", dy, rows, dim, dt)
    dy, lddy = _matrix(dy, "dy", dy, rows, dim, dy.dtype)
    if isinstance(weight, torch.Tensor) and weight.dtype == torch.float32:
        weight = _vector(weight, "weight", dy, dim, torch.float32)
    else:
        weight = _vector(weight, "weight", dy, dim, dt)
    rstd = _vector(rstd, "rstd", dy, rows, torch.float32)
    ldds = 0
    if dsum is not None:
        dsum, ldds = _matrix(dsum, "dsum", dy, rows, dim, dt)
    dx = torch.empty_like(s, memory_format=torch.contiguous_format)
    dw = ws = None
    n = 0
    if need_dweight:
        dw = weight.new_empty(dim)
        n = lib().vcsr_rmsnorm_grad_workspace(rows, dim)
        ws = _workspace(n, dy)
    a = _RmsnormGradArgs(rows, dim, dy.data_ptr(), lddy, s.data_ptr(), lds, weight.data_ptr(),
                         rstd.data_ptr(), _p(dsum), ldds, dx.data_ptr(), dim, _p(dw), _p(ws), n,
                         x_type, _TYPE[weight.dtype], dy_type)
    _check(lib().vcsr_rmsnorm_grad(a, _current_stream(dy.get_device())))
    return dx, dw


@_operator
def dequantize(codes, scale, out_dtype=torch.float32, squared=False):
    """codes * scale, one scale per row, as out_dtype; squared=True: its square
    (vcsr_dequantize).  codes: (rows, dim) float8_e4m3fn."""
    rows, dim = _shape(codes, "codes")
    codes, ldc = _matrix(codes, "codes", codes, rows, dim, torch.float8_e4m3fn)
    scale = _vector(scale, "scale", codes, rows, torch.float32)
    out = codes.new_empty((rows, dim), dtype=out_dtype)
    _check(lib().vcsr_dequantize(codes.data_ptr(), ldc, scale.data_ptr(), rows, dim,
                                 out.data_ptr(), dim, _type(out_dtype, "out"), int(squared),
                                 _current_stream(codes.get_device())))
    return out


# ---------------------------------------------------------------- the product

class LinearOut(NamedTuple):
    y: torch.Tensor
    pre: Optional[torch.Tensor]  # the value before the activation, with save_pre


class LinearGrad(NamedTuple):
    dx: Optional[torch.Tensor]
    dw: Optional[torch.Tensor]
    db: Optional[torch.Tensor]


def _act(act):
    try:
        return ACTIVATIONS[act]
    except KeyError:
        raise VcsrError(UNSUPPORTED, f"activation {act!r}") from None


@_operator
def linear(x, w, bias=None, residual=None, act=None, x_scale=None, w_scale=None, out_dtype=None,
           save_pre=False, out=None) -> LinearOut:
    """y = act(x w^T + bias) + residual (vcsr_linear).  x: (M, K), w: (N, K), both
    float32, bfloat16, float16, or float8_e4m3fn with x_scale (M,) and w_scale (N,);
    y, bias and residual are of x's type, or of out_dtype (bfloat16 by default) with
    8-bit operands.  act: None, "relu", "gelu" or "silu".  out may be residual itself."""
    M, K = _shape(x, "x")
    N, _ = _shape(w, "w")
    dt = x.dtype
    code = _type(dt, "x")
    x, ldx = _matrix(x, "x", x, M, K, dt)
    w, ldw = _matrix(w, "w", x, N, K, dt)
    if code == E4M3:
        if x_scale is None or w_scale is None:
            raise VcsrError(INVALID, "8-bit operands need x_scale and w_scale")
        x_scale = _vector(x_scale, "x_scale", x, M, torch.float32)
        w_scale = _vector(w_scale, "w_scale", x, N, torch.float32)
        out_dtype = out_dtype or getattr(out, "dtype", torch.bfloat16)
    else:
        if x_scale is not None or w_scale is not None:
            raise VcsrError(INVALID, "scales are for 8-bit operands")
        out_dtype = out_dtype or dt
    out_type = _type(out_dtype, "out")
    if bias is not None:
        bias = _vector(bias, "bias", x, N, out_dtype)
    ldr = 0
    if residual is not None:
        residual, ldr = _matrix(residual, "residual", x, M, N, out_dtype)
    y, ldy = _out(out, "out", x if residual is None else residual, M, N, out_dtype)
    pre = torch.empty_like(y) if save_pre and out is None else None
    if save_pre and pre is None:
        pre = x.new_empty((M, N), dtype=out_dtype)
    a = _LinearArgs(M, N, K, x.data_ptr(), ldx, w.data_ptr(), ldw, _p(x_scale), _p(w_scale),
                    _p(bias), _p(residual), ldr, y.data_ptr(), ldy, _p(pre), N, None, 0, code,
                    out_type, _act(act))
    L = lib()
    # scratch is for operands that are off 16 bytes
    size = x.element_size()
    if (x.data_ptr() | w.data_ptr() | ldx * size | ldw * size) & 15:
        n = L.vcsr_linear_workspace(a)
        if n:
            ws = _workspace(n, x)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
    _check(L.vcsr_linear(a, _current_stream(x.get_device())))
    if out is not None:
        _new_values(out)
    return LinearOut(y, pre)


@_operator
def linear_backward(dy, x, w, pre=None, act=None, need_dx=True, need_dw=True,
                    need_db=True) -> LinearGrad:
    """Gradients of linear (vcsr_linear_grad): dy (M, N), x (M, K), w (N, K) and pre
    (M, N, needed with an activation) of one type, float32, bfloat16 or float16.
    The residual's gradient is dy."""
    M, N = _shape(dy, "dy")
    K = _shape(x, "x")[1]
    dt = dy.dtype
    code = _type(dt, "dy")
    if code == E4M3:
        raise VcsrError(UNSUPPORTED, "8-bit operands have no gradient")
    act = _act(act)
    dy, lddy = _matrix(dy, "dy", dy, M, N, dt)
    x, ldx = _matrix(x, "x", dy, M, K, dt)
    w, ldw = _matrix(w, "w", dy, N, K, dt)
    ldp = 0
    if act:
        if pre is None:
            raise VcsrError(INVALID, "the gradient of an activation needs pre")
        pre, ldp = _matrix(pre, "pre", dy, M, N, dt)
    else:
        pre = None
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_dx else None
    dw = torch.empty_like(w, memory_format=torch.contiguous_format) if need_dw else None
    db = dy.new_empty(N) if need_db else None
    a = _LinearGradArgs(M, N, K, dy.data_ptr(), lddy, _p(pre), ldp, x.data_ptr(), ldx,
                        w.data_ptr(), ldw, _p(dx), K, _p(dw), K, _p(db), None, 0, code, act)
    L = lib()
    n = L.vcsr_linear_grad_workspace(a)
    if n:
        ws = _workspace(n, dy)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
    _check(L.vcsr_linear_grad(a, _current_stream(dy.get_device())))
    return LinearGrad(dx, dw, db)


def check(stream=None):
    """Synchronise and raise VcsrError (status 7) if a bounded wait of linear's or
    linear_backward's kernels on the current device ran out since the last check."""
    _check(lib().vcsr_layers_check(_stream(stream)))


def test_withhold_signal():
    """Test hook: one wait of the next product's kernel runs out on purpose
    (vcsr_layers_test_withhold_signal); check() then reports it."""
    _check(lib().vcsr_layers_test_withhold_signal())


# -------------------------------------------------------------- the optimizer

@_operator
def _values(t, dtype):
    return t.to(dtype, copy=True)


@_operator
def _dither(t, like):
    return _vector(t, "dither", like, BLOCK, torch.float32)


class AdamW:
    """AdamW over many tensors in one launch (vcsr_adamw_*).

    params: contiguous CUDA tensors of one type (float32, bfloat16 or float16), no two
    in the same memory, that keep their storage while the optimizer lives.  state_bits=32: m and v in
    m_flat, v_flat; state_bits=8: codes of m and u = sqrt(v) in m_flat, u_flat
    (float8_e4m3fn), one scale per 256 values in m_scale, u_scale.  Tensor t's
    states start at value offsets[t] of the flat buffers.  copies: 16-bit copies of
    the parameters (bfloat16 or float16, as many values each), written by every
    step.  `steps` counts the steps done; with the buffers above it is the whole
    state, to be saved and put back as such.  Step number, rates and the gradients'
    addresses go into the launch: a CUDA graph that captured a step repeats them."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 state_bits=32, copies=None):
        params = list(params)
        if not params or not all(isinstance(p, torch.Tensor) and p.is_cuda for p in params):
            raise VcsrError(INVALID, "AdamW takes a list of CUDA tensors")
        if state_bits not in (8, 32):
            raise VcsrError(UNSUPPORTED, "state_bits must be 32 or 8")
        self.device = params[0].device
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.state_bits, self.steps = state_bits, 0
        self._numel = [p.numel() for p in params]
        self._same(params, "params")
        p_type = _type(params[0].dtype, "params")
        copy_type = 0
        if copies is not None:
            copies = list(copies)
            self._same(copies, "copies")
            copy_type = _type(copies[0].dtype, "copies")
        self._keep = (params, copies or [])
        n = len(params)
        numel = np.asarray(self._numel, np.int64)
        blocks = -(-numel // BLOCK)
        self.offsets = ((np.cumsum(blocks) - blocks) * BLOCK).tolist()
        total = int(blocks.sum()) * BLOCK
        assert total == lib().vcsr_adamw_state_values(n, numel.ctypes.data)

        def zeros(count, dtype):
            return torch.zeros(count, device=self.device, dtype=dtype)

        with torch.cuda.device(self.device):
            if state_bits == 8:
                self.m_flat = zeros(total, torch.float8_e4m3fn)
                self.u_flat = zeros(total, torch.float8_e4m3fn)
                self.m_scale = zeros(total // BLOCK, torch.float32)
                self.u_scale = zeros(total // BLOCK, torch.float32)
            else:
                self.m_flat = zeros(total, torch.float32)
                self.v_flat = zeros(total, torch.float32)
            p_ptr = self._pointers(params)
            c_ptr = None if copies is None else self._pointers(copies)
            h = C.c_void_p()
            _check(lib().vcsr_adamw_create(
                n, numel.ctypes.data, p_ptr.ctypes.data, p_type,
                None if c_ptr is None else c_ptr.ctypes.data, copy_type, state_bits, C.byref(h),
                _current_stream(self.device.index)))
        self._h = h

    def _same(self, tensors, name):
        """Checks a list against the parameters; its one type."""
        if len(tensors) != len(self._numel):
            raise VcsrError(INVALID, f"{len(tensors)} {name} for {len(self._numel)} parameters")
        dev, dtype = self.device, None
        for i, (t, n) in enumerate(zip(tensors, self._numel)):
            if t is None and name == "grads":
                continue
            if not isinstance(t, torch.Tensor):
                raise VcsrError(INVALID, f"{name}[{i}] must be a tensor on {dev}")
            dtype = dtype or t.dtype
            if t.dtype != dtype:
                raise VcsrError(UNSUPPORTED, f"{name}[{i}] has type {t.dtype}, expected {dtype}")
            if t.device != dev or t.numel() != n or not t.is_contiguous():
                raise VcsrError(INVALID, f"{name}[{i}] must be contiguous on {dev} with {n} values")
        return dtype

    def _gradients(self, grads):
        """The gradients' type and addresses, checked (in whole passes over the list:
        with hundreds of small tensors the checks are most of a step), and the tensors
        that a step with them writes."""
        T = torch.Tensor
        try:
            dtypes = set(map(_dtype, grads))
            if (len(dtypes) == 1 and list(map(T.numel, grads)) == self._numel
                    and all(map(T.is_contiguous, grads))
                    and set(map(T.get_device, grads)) == {self.device.index}):
                return (dtypes.pop(), np.fromiter(map(T.data_ptr, grads), np.uint64, len(grads)),
                        self._keep[0] + self._keep[1])
        except (AttributeError, TypeError):
            pass
        dtype = self._same(grads, "grads") or torch.float32
        return dtype, self._pointers(grads), [t for ts in self._keep for g, t in zip(grads, ts)
                                              if g is not None]

    @staticmethod
    def _pointers(tensors):
        return np.fromiter((0 if t is None else t.data_ptr() for t in tensors), np.uint64,
                           len(tensors))

    def step(self, grads, lr=None, grad_scale=1.0, dither=None, stream=None):
        """One step.  grads: a contiguous tensor per parameter, all of one type (float32,
        bfloat16 or float16), or None for a parameter to leave as it is.  dither: 256 float32
        uniform numbers in [0, 1), fresh ones each step (state_bits=8; without it
        codes round to nearest)."""
        dtype, ptr, written = self._gradients(list(grads))
        if dither is not None:
            dither = _dither(dither, self.m_flat, stream=stream)
        eight = self.state_bits == 8
        second = self.u_flat if eight else self.v_flat
        a = _AdamwStepArgs(ptr.ctypes.data, _type(dtype, "grads"), self.m_flat.data_ptr(),
                           second.data_ptr(), self.m_scale.data_ptr() if eight else None,
                           self.u_scale.data_ptr() if eight else None, _p(dither),
                           self.lr if lr is None else lr, self.betas[0], self.betas[1], self.eps,
                           self.weight_decay, grad_scale, self.steps + 1)
        raw = (_current_stream(self.device.index) if stream is None
               else stream if isinstance(stream, int) else stream.cuda_stream)
        if torch.cuda.current_device() == self.device.index:
            _check(lib().vcsr_adamw_step(self._h, a, raw))
        else:
            with torch.cuda.device(self.device):
                _check(lib().vcsr_adamw_step(self._h, a, raw))
        self.steps += 1
        _new_values(written)

    def state_values(self, dtype=torch.float32, stream=None):
        """(m, v), flat: the states as values of `dtype`, in new tensors."""
        if self.state_bits == 32:
            return _values(self.m_flat, dtype, stream=stream), _values(self.v_flat, dtype, stream=stream)
        m = dequantize(self.m_flat.view(-1, BLOCK), self.m_scale, dtype, stream=stream)
        v = dequantize(self.u_flat.view(-1, BLOCK), self.u_scale, dtype, squared=True,
                       stream=stream)
        return m.view(-1), v.view(-1)

    def close(self):
        if getattr(self, "_h", None) and lib is not None:  # None while Python shuts down
            lib().vcsr_adamw_destroy(self._h)
        self._h = None

    __del__ = close
