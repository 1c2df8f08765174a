"""PyTorch operators over the C ABI: torch.ops.vcsr.spmm(plan_id, B) -> C, and the
dense layer operators with their gradients (rmsnorm, layernorm, linear and
gated_linear, below).

The reference has no Python or PyTorch binding; this one lets PyTorch code
(and graph capture by tracers, through the fake implementation below) call a
plan's C = A * B like any other operator.  spmm is forward only: no gradient is
registered (the gradient of B is the product of A's transpose, a plan of its own).
The products always run on the engine's CUDA kernels; there is no fallback when
the library or a GPU is missing.

    from vcsr_b200 import Plan, torch_ops
    plan = Plan(csr)
    pid = torch_ops.register(plan)
    C = torch.ops.vcsr.spmm(pid, B)      # B: (N, O) float32 or bfloat16, CUDA

    y, s = torch_ops.rmsnorm(C, gain, residual=h, out_dtype=torch.bfloat16)
    z = torch_ops.linear(y, W, bias=b, act="gelu")      # differentiable
"""
from __future__ import annotations

import itertools
import threading
from typing import Optional, Tuple

import torch

from . import Plan, VcsrError, layers

_plans: dict[int, Plan] = {}
_ids = itertools.count(1)
_lock = threading.Lock()


def register(plan: Plan) -> int:
    """An id under which torch.ops.vcsr.spmm finds `plan` (kept alive until
    unregister)."""
    with _lock:
        pid = next(_ids)
        _plans[pid] = plan
    return pid


def unregister(pid: int) -> None:
    with _lock:
        _plans.pop(pid, None)


def _plan(pid: int) -> Plan:
    try:
        return _plans[pid]
    except KeyError:
        raise ValueError(f"no plan registered under id {pid}") from None


@torch.library.custom_op("vcsr::spmm", mutates_args=())
def spmm(plan_id: int, B: torch.Tensor) -> torch.Tensor:
    """C = A * B for the registered plan; B is (N, O), float32 or bfloat16,
    on a CUDA device; C is (M, O) float32 on the same device."""
    plan = _plan(plan_id)
    if B.dim() != 2 or B.shape[0] != plan.N:
        raise ValueError(f"B must be ({plan.N}, O), got {tuple(B.shape)}")
    if B.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"B must be float32 or bfloat16, got {B.dtype}")
    if B.stride(1) != 1:
        B = B.contiguous()
    C = torch.empty(plan.M, B.shape[1], device=B.device, dtype=torch.float32)
    plan.spmm(B, C, stream=torch.cuda.current_stream(B.device))
    return C


@spmm.register_fake
def _spmm_fake(plan_id: int, B: torch.Tensor) -> torch.Tensor:
    plan = _plan(plan_id)
    return B.new_empty((plan.M, B.shape[1]), dtype=torch.float32)


# ------------------------------------------------------- dense layer operators

@torch.library.custom_op("vcsr::rmsnorm", mutates_args=())
def _rmsnorm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor], eps: float,
             out_dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, s, rstd) of layers.rmsnorm; s has no rows without a residual (s is x then)."""
    out = layers.rmsnorm(x, weight, residual=residual, eps=eps, out_dtype=out_dtype,
                         save_rstd=True)
    return out.y, out.sum if residual is not None else x.new_empty((0, x.shape[1])), out.rstd


@_rmsnorm.register_fake
def _(x, weight, residual, eps, out_dtype):
    rows = x.shape[0] if residual is not None else 0
    return (x.new_empty(x.shape, dtype=out_dtype), x.new_empty((rows, x.shape[1])),
            x.new_empty(x.shape[0], dtype=torch.float32))


@torch.library.custom_op("vcsr::rmsnorm_backward", mutates_args=())
def _rmsnorm_backward(dy: torch.Tensor, s: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                      dsum: Optional[torch.Tensor],
                      need_dweight: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight) of layers.rmsnorm_backward; dweight has no values unless needed."""
    dx, dw = layers.rmsnorm_backward(dy, s, weight, rstd, dsum=dsum, need_dweight=need_dweight)
    return dx, weight.new_empty(0) if dw is None else dw


@_rmsnorm_backward.register_fake
def _(dy, s, weight, rstd, dsum, need_dweight=True):
    return s.new_empty(s.shape), weight.new_empty(weight.shape if need_dweight else 0)


def _rmsnorm_setup(ctx, inputs, output):
    x, weight, residual, _, _ = inputs
    ctx.added = residual is not None
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(*output[2 if ctx.added else 1:])
    ctx.save_for_backward(output[1] if ctx.added else x, weight, output[2])


def _rmsnorm_grad(ctx, dy, ds, _):
    if dy is None:  # only s was used
        return ds, None, ds, None, None
    s, weight, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw = _rmsnorm_backward(dy, s, weight, rstd, ds if ctx.added else None, need[1])
    return dx if need[0] else None, dw if need[1] else None, dx if need[2] else None, None, None


_rmsnorm.register_autograd(_rmsnorm_grad, setup_context=_rmsnorm_setup)


def rmsnorm(x, weight, residual=None, eps=1e-6, out_dtype=None):
    """(y, s) of layers.rmsnorm, s = x + residual, with gradients of x, weight and
    residual (16- and 32-bit y)."""
    y, s, _ = _rmsnorm(x, weight, residual, eps, out_dtype or x.dtype)
    return y, (x if residual is None else s)


def _floats(out_dtype):
    """Refuses 8-bit codes, whose scales these operators do not return."""
    if out_dtype == torch.float8_e4m3fn:
        raise VcsrError(layers.UNSUPPORTED, "8-bit rows need their scales: call layers.layernorm")


@torch.library.custom_op("vcsr::layernorm", mutates_args=())
def _layernorm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
               residual: Optional[torch.Tensor], eps: float, out_dtype: torch.dtype
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, s, mean, rstd) of layers.layernorm; s has no rows without a residual (s is x then)."""
    _floats(out_dtype)
    out = layers.layernorm(x, weight, bias, residual=residual, eps=eps, out_dtype=out_dtype,
                           save_stats=True)
    return (out.y, out.sum if residual is not None else x.new_empty((0, x.shape[1])), out.mean,
            out.rstd)


@_layernorm.register_fake
def _(x, weight, bias, residual, eps, out_dtype):
    _floats(out_dtype)
    rows = x.shape[0] if residual is not None else 0
    return (x.new_empty(x.shape, dtype=out_dtype), x.new_empty((rows, x.shape[1])),
            x.new_empty(x.shape[0], dtype=torch.float32), x.new_empty(x.shape[0], dtype=torch.float32))


@torch.library.custom_op("vcsr::layernorm_backward", mutates_args=())
def _layernorm_backward(dy: torch.Tensor, s: torch.Tensor, weight: Optional[torch.Tensor],
                        mean: torch.Tensor, rstd: torch.Tensor, dsum: Optional[torch.Tensor],
                        weight_dtype: torch.dtype, need_dweight: bool = True, need_dbias: bool = True
                        ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of layers.layernorm_backward; what is not needed has no values."""
    g = layers.layernorm_backward(dy, s, weight, mean, rstd, dsum=dsum, need_dweight=need_dweight,
                                  need_dbias=need_dbias, weight_dtype=weight_dtype)
    none = [s.new_empty(0, dtype=weight_dtype) if t is None else t for t in g[1:]]
    return g.dx, *none


@_layernorm_backward.register_fake
def _(dy, s, weight, mean, rstd, dsum, weight_dtype, need_dweight=True, need_dbias=True):
    return (s.new_empty(s.shape), *(s.new_empty(s.shape[1] if need else 0, dtype=weight_dtype)
                                    for need in (need_dweight, need_dbias)))


def _layernorm_setup(ctx, inputs, output):
    x, weight, bias, residual, _, _ = inputs
    ctx.added = residual is not None
    ctx.weight_dtype = next((t.dtype for t in (weight, bias) if t is not None), x.dtype)
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(*output[2 if ctx.added else 1:])
    ctx.save_for_backward(output[1] if ctx.added else x, weight, output[2], output[3])


def _layernorm_grad(ctx, dy, ds, _, __):
    if dy is None:  # only s was used
        return ds, None, None, ds, None, None
    s, weight, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = _layernorm_backward(dy, s, weight, mean, rstd, ds if ctx.added else None,
                                     ctx.weight_dtype, need[1], need[2])
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None,
            dx if need[3] else None, None, None)


_layernorm.register_autograd(_layernorm_grad, setup_context=_layernorm_setup)


def layernorm(x, weight=None, bias=None, residual=None, eps=1e-5, out_dtype=None):
    """(y, s) of layers.layernorm, s = x + residual, with gradients of x, weight, bias and
    residual (16- and 32-bit y; an 8-bit one is refused, call layers.layernorm)."""
    y, s, _, _ = _layernorm(x, weight, bias, residual, eps, out_dtype or x.dtype)
    return y, (x if residual is None else s)


@torch.library.custom_op("vcsr::linear", mutates_args=())
def _linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor],
            residual: Optional[torch.Tensor], act: str,
            save_pre: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, pre) of layers.linear; pre has no rows unless saved."""
    out = layers.linear(x, w, bias=bias, residual=residual, act=act, save_pre=save_pre)
    return out.y, out.pre if save_pre else out.y.new_empty((0, w.shape[0]))


@_linear.register_fake
def _(x, w, bias, residual, act, save_pre):
    return (x.new_empty((x.shape[0], w.shape[0])),
            x.new_empty((x.shape[0] if save_pre else 0, w.shape[0])))


@torch.library.custom_op("vcsr::linear_backward", mutates_args=())
def _linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor,
                     pre: Optional[torch.Tensor], act: str, need_dx: bool = True, need_dw: bool = True,
                     need_db: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """layers.linear_backward; what is not needed has no values."""
    g = layers.linear_backward(dy, x, w, pre=pre, act=act, need_dx=need_dx, need_dw=need_dw,
                               need_db=need_db)
    return tuple(x.new_empty(0) if t is None else t for t in g)


@_linear_backward.register_fake
def _(dy, x, w, pre, act, need_dx=True, need_dw=True, need_db=True):
    return (x.new_empty(x.shape if need_dx else 0), w.new_empty(w.shape if need_dw else 0),
            w.new_empty(w.shape[0] if need_db else 0))


def _linear_setup(ctx, inputs, output):
    x, w, bias, residual, act, save_pre = inputs
    ctx.act = act
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, w, output[1] if save_pre else None)


def _linear_grad(ctx, dy, _):
    x, w, pre = ctx.saved_tensors
    need = ctx.needs_input_grad
    made = _linear_backward(dy, x, w, pre, ctx.act, *need[:3]) if any(need[:3]) else (None,) * 3
    return (*(g if n else None for g, n in zip(made, need)), dy if need[3] else None, None, None)


_linear.register_autograd(_linear_grad, setup_context=_linear_setup)


def linear(x, w, bias=None, residual=None, act=None):
    """y of layers.linear with gradients of x, w, bias and residual (16- and 32-bit
    operands; for 8-bit ones call layers.linear, which has no gradient)."""
    act = act or "none"
    wanted = torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                             for t in (x, w, bias))
    return _linear(x, w, bias, residual, act, wanted and act != "none")[0]


@torch.library.custom_op("vcsr::gated_linear", mutates_args=())
def _gated_linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], act: str,
                  save_pre: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, pre) of layers.gated_linear; pre has no rows unless saved."""
    out = layers.gated_linear(x, w, bias=bias, act=act, save_pre=save_pre)
    return out.y, out.pre if save_pre else out.y.new_empty((0, w.shape[0]))


@_gated_linear.register_fake
def _(x, w, bias, act, save_pre):
    return (x.new_empty((x.shape[0], w.shape[0] // 2)),
            x.new_empty((x.shape[0] if save_pre else 0, w.shape[0])))


@torch.library.custom_op("vcsr::gated_linear_backward", mutates_args=())
def _gated_linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, pre: torch.Tensor, act: str,
                           need_dx: bool = True, need_dw: bool = True, need_db: bool = True
                           ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """layers.gated_linear_backward; what is not needed has no values."""
    g = layers.gated_linear_backward(dy, x, w, pre, act=act, need_dx=need_dx, need_dw=need_dw,
                                     need_db=need_db)
    return tuple(x.new_empty(0) if t is None else t for t in g)


@_gated_linear_backward.register_fake
def _(dy, x, w, pre, act, need_dx=True, need_dw=True, need_db=True):
    return (x.new_empty(x.shape if need_dx else 0), w.new_empty(w.shape if need_dw else 0),
            w.new_empty(w.shape[0] if need_db else 0))


def _gated_linear_setup(ctx, inputs, output):
    x, w, _, act, save_pre = inputs
    ctx.act = act
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, w, output[1])


def _gated_linear_grad(ctx, dy, _):
    x, w, pre = ctx.saved_tensors
    need = ctx.needs_input_grad[:3]
    if dy is None or not any(need):
        return (None,) * 5
    made = _gated_linear_backward(dy, x, w, pre, ctx.act, *need)
    return (*(g if n else None for g, n in zip(made, need)), None, None)


_gated_linear.register_autograd(_gated_linear_grad, setup_context=_gated_linear_setup)


def gated_linear(x, w, bias=None, act="silu"):
    """y of layers.gated_linear with gradients of x, w and bias (16- and 32-bit operands; for
    8-bit ones call layers.gated_linear, which has no gradient)."""
    wanted = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias))
    return _gated_linear(x, w, bias, act or "none", wanted)[0]
