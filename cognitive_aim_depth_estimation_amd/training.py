"""Training form of the encoder's row-wise and matrix parts on the gfx950 kernels (libcogaim.so).

The model's forward (``model.py``) is inference only.  This module is what a backward pass through the encoder's norms and
MLPs needs: each operator as a pair of explicit forward and backward functions, and as a differentiable function on top.

  ===================================  ===============================================================================
  ``layer_norm_forward / _backward``   LayerNorm with its row statistics; dx, dweight, dbias
  ``linear_forward``                   ``act(x W^T + b) + residual`` or ``scale * (x W^T + b) + residual``, one kernel
  ``linear_backward_input``            ``((dy * scale) W) * act'(u)``: also through the activation below the layer
  ``linear_backward_weight``           dW, db and the scale's gradient
  ``pack8`` / ``unpack8``              activations in 8 bits for the backward pass
  ``layer_norm``, ``linear``           differentiable
  ``mlp_half``                         ``x + scale * (gelu(LN(x) W1^T + b1) W2^T + b2)``, differentiable, all it keeps in 8 bits
  ===================================  ===============================================================================

Arithmetic: matrix operands are bf16 or fp16, everything else takes bf16, fp16 or fp32 tensors; sums are fp32; an output
is rounded once, to its own type.  Norm weights, biases, LayerScale vectors, statistics and their gradients are fp32.

Tensors are ``[..., columns]`` on one ROCm device; rows may be strided (a tensor whose columns are not contiguous is copied
first).  Calls run on the current stream of the tensors' device, allocate their results and workspaces from torch's caching
allocator and never wait, so they can be captured into graphs.  The same inputs give the same bits.  Zero rows are allowed.
There is no CPU path.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["Checkpoint8", "pack8", "unpack8", "layer_norm_forward", "layer_norm_backward", "linear_forward",
           "linear_backward_input", "linear_backward_weight", "activation_backward", "layer_norm", "linear", "mlp_half"]

Tensor = torch.Tensor
_HALF = (torch.bfloat16, torch.float16)
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
HOST_PATH = os.path.join(_lib.HERE, "_host.so")


class Checkpoint8(NamedTuple):
    """Activations in 8 bits: int8 ``codes [..., D]`` and one uint8 exponent for every 32 columns, ``exponents
    [..., ceil(D / 32)]``.  A value is ``code * 2**(exponent - 127)``; the step is the smallest power of two (from 2^-126)
    for which the group's largest magnitude rounds to at most 127, so a value is off by at most half a step:
    between 1/255 and 1/127.5 of the group's largest magnitude.  A group that held an infinity or a NaN has exponent
    255 and stands for NaN."""
    codes: Tensor
    exponents: Tensor


_host = None


def _ops():
    """The compiled host side (checks, allocation, calls), bound to the loaded libcogaim.so."""
    global _host
    if _host is None:
        handle = _lib.lib()
        if not os.path.exists(HOST_PATH):
            raise _lib.CogaimError(f"{HOST_PATH} is missing: build it with `python -m cognitive_aim_depth_estimation_amd.build`")
        spec = importlib.util.spec_from_file_location("_host", HOST_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.bind({n: ctypes.cast(getattr(handle, n), ctypes.c_void_p).value for n in module.entries()}, _lib.CogaimError)
        _host = module
    return _host


def _checkpoint(t, name):
    if not isinstance(t, Checkpoint8):
        raise TypeError(f"{name} must be a Checkpoint8")
    return t


# ---- 8-bit activations -------------------------------------------------------------------------------------------
def pack8(x: Tensor) -> Checkpoint8:
    """``x [..., D]`` (bf16, fp16 or fp32) in 8 bits."""
    return Checkpoint8(*(_host or _ops()).pack8(x))


def unpack8(saved: Checkpoint8, dtype: torch.dtype = torch.float32) -> Tensor:
    """The values of an 8-bit copy: exact in fp32 and bf16, rounded once in fp16, where +-65536, which the largest finite
    numbers become in 8 bits, is held at +-65504 and anything larger is an infinity."""
    codes, exponents = _checkpoint(saved, "saved")
    return (_host or _ops()).unpack8(codes, exponents, dtype)


def activation_backward(dy: Tensor, saved: Union[Tensor, Checkpoint8], activation: str, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``dy * act'(u)`` with ``u`` itself or its 8-bit copy; activation "relu" or "gelu".  In 8 bits a u of under half its
    group's step is zero, and ReLU's gradient stops there: about 1 % of the positive ones of normally distributed rows."""
    u, codes, exponents = (None, *saved) if isinstance(saved, Checkpoint8) else (saved, None, None)
    if u is None and codes is None:
        raise TypeError("saved must be a tensor or a Checkpoint8")
    return (_host or _ops()).activation_backward(dy, u, codes, exponents, activation, out_dtype)


# ---- layer norm --------------------------------------------------------------------------------------------------
def layer_norm_forward(x: Tensor, weight: Tensor, bias: Tensor, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None,
                       checkpoint: bool = False) -> Tuple[Tensor, Tensor, Tensor, Optional[Checkpoint8]]:
    """``(y, mean, rstd, saved)``: ``y = (x - mean) * rstd * weight + bias`` of type ``out_dtype`` (default: x's), the fp32
    statistics of every row, and with ``checkpoint`` the normalised rows ``(x - mean) * rstd`` in 8 bits (else None)."""
    y, mean, rstd, codes, exponents = (_host or _ops()).layer_norm_forward(x, weight, bias, eps, out_dtype, checkpoint)
    return y, mean, rstd, Checkpoint8(codes, exponents) if checkpoint else None


def layer_norm_backward(dy: Tensor, saved: Union[Tensor, Checkpoint8], mean: Optional[Tensor], rstd: Tensor, weight: Tensor,
                        add: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``(dx, dweight, dbias)`` from ``dy`` and either the norm's input with its ``mean`` or its rows in 8 bits (``mean`` is
    not read then).  ``add`` (the gradient that flows past the norm) is added to dx.  dx is of type ``out_dtype`` (default:
    the input's, dy's with an 8-bit copy)."""
    x, codes, exponents = (None, *saved) if isinstance(saved, Checkpoint8) else (saved, None, None)
    if x is None and codes is None:
        raise TypeError("saved must be a tensor or a Checkpoint8")
    return (_host or _ops()).layer_norm_backward(dy, x, codes, exponents, mean, rstd, weight, add, out_dtype)


# ---- linear layers -----------------------------------------------------------------------------------------------
def linear_forward(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: str = "none",
                   scale: Optional[Tensor] = None, residual: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   checkpoint: bool = False, pre_activation: bool = False) -> Tuple[Tensor, Union[None, Checkpoint8, Tensor]]:
    """``(y, saved)`` for ``x [..., K]`` and ``weight [N, K]`` of one 16-bit type:  with ``u = x weight^T + bias``,
    ``y = act(u) + residual``, or ``y = scale * u + residual`` (scale: LayerScale, only without an activation).  ``y`` is of
    type ``out_dtype`` (default: x's); with ``checkpoint``, ``saved`` is u in 8 bits, with ``pre_activation`` u in x's type, both
    from the product's epilogue."""
    y, codes, exponents, pre = (_host or _ops()).linear_forward(x, weight, bias, activation, scale, residual, out_dtype, checkpoint, pre_activation)
    return y, Checkpoint8(codes, exponents) if checkpoint else pre


def linear_backward_input(dy: Tensor, weight: Tensor, activation: str = "none", saved: Optional[Checkpoint8] = None,
                          scale: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                          want_activation: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """``(dx, a)`` for ``dy [..., N]`` and ``weight [N, K]`` of one 16-bit type:  ``dx = ((dy * scale) weight) * act'(u)``,
    ``u [..., K]`` the pre-activation, kept in 8 bits (``saved``), of the activation that produced the layer's input; with
    ``want_activation``, ``a = act(u)`` in 16 bits: that input again, for ``linear_backward_weight``.  With ``scale``, the
    matrix cores take ``weight * scale`` (``dy * scale`` up to 32 rows): rounded to 16 bits for a 16-bit dx, in parts that keep
    fp32's precision for an fp32 one; in fp16 relative to the largest scale, so that a LayerScale of 1e-5 does not push
    the operand into subnormals (a small dx in fp16 still does: ask for fp32 or bf16, or scale the loss)."""
    codes, exponents = (None, None) if saved is None else _checkpoint(saved, "saved")
    return (_host or _ops()).linear_backward_input(dy, weight, activation, codes, exponents, scale, out_dtype, want_activation)


def linear_backward_weight(dy: Tensor, x: Union[Tensor, Checkpoint8], weight: Optional[Tensor] = None,
                           bias: Optional[Tensor] = None, scale: Optional[Tensor] = None, x_scale: Optional[Tensor] = None,
                           x_shift: Optional[Tensor] = None,
                           out_dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
    """``(dW, db, dscale)`` for ``dy [..., N]`` in 16 bits and the layer's input ``x [..., K]``, in dy's type or in 8 bits;
    an 8-bit copy stands for ``x_scale * copy + x_shift`` (a norm's weight and bias over its kept rows) and enters the
    product exactly whatever dy's type (with fp16, steps under 2^-33 of their column group's largest are rounded).  Without
    ``scale``, ``dW = dy^T x`` and ``db`` sums dy's rows (dscale None).  With ``scale`` (and the forward's ``weight`` and
    ``bias``), for ``y = scale * (x weight^T + bias)``: dW and db are those times scale, ``dscale`` sums ``dy * (x weight^T + bias)``.
    db and dscale are fp32, dW is of type ``out_dtype``."""
    t, codes, exponents = (None, *x) if isinstance(x, Checkpoint8) else (x, None, None)
    if t is None and codes is None:
        raise TypeError("x must be a tensor or a Checkpoint8")
    return (_host or _ops()).linear_backward_weight(dy, t, codes, exponents, weight, bias, scale, x_scale, x_shift, out_dtype)


# ---- differentiable ----------------------------------------------------------------------------------------------
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype, checkpoint):
        y, mean, rstd, saved = layer_norm_forward(x, weight, bias, eps, out_dtype, checkpoint)
        ctx.kept8 = checkpoint
        ctx.x_dtype = x.dtype
        ctx.save_for_backward(weight, rstd, *(saved if checkpoint else (x, mean)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, rstd, a, b = ctx.saved_tensors
        saved, mean = (Checkpoint8(a, b), None) if ctx.kept8 else (a, b)
        dx, dw, db = layer_norm_backward(dy, saved, mean, rstd, weight, out_dtype=ctx.x_dtype)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, None, None


def layer_norm(x: Tensor, weight: Tensor, bias: Tensor, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None,
               checkpoint: bool = False) -> Tensor:
    """Differentiable LayerNorm over the last dimension.  ``checkpoint`` keeps the normalised rows in 8 bits for the backward
    pass in place of x."""
    return _LayerNorm.apply(x, weight, bias, eps, out_dtype, checkpoint)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, scale, residual, activation, out_dtype, checkpoint):
        w = weight if weight.dtype == x.dtype else weight.to(x.dtype)
        active = activation != "none"
        y, pre = linear_forward(x, w, bias, activation, scale, residual, out_dtype, active and checkpoint, active and not checkpoint)
        kept = pack8(x) if checkpoint else None
        if not checkpoint:
            pre = (pre, None)
        ctx.activation, ctx.kept8, ctx.x_dtype, ctx.w_dtype = activation, checkpoint, x.dtype, weight.dtype
        ctx.res_dtype = None if residual is None else residual.dtype
        ctx.has = (bias is not None, scale is not None)
        ctx.save_for_backward(w, bias, scale, *(pre or (None, None)), *(kept or (x, None)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, bias, scale, pc, pe, xa, xb = ctx.saved_tensors
        need = ctx.needs_input_grad
        if ctx.activation != "none":
            du = activation_backward(dy, Checkpoint8(pc, pe) if ctx.kept8 else pc, ctx.activation, ctx.x_dtype)
        else:
            du = dy.to(ctx.x_dtype)
        dx = linear_backward_input(du, w, scale=scale)[0] if need[0] else None
        dw = db = ds = None
        if need[1] or need[2] or need[3]:
            x = Checkpoint8(xa, xb) if ctx.kept8 else xa
            more = {"weight": w, "bias": bias, "scale": scale} if scale is not None else {}
            dw, db, ds = linear_backward_weight(du, x, out_dtype=ctx.w_dtype, **more)
        dres = dy.to(ctx.res_dtype) if ctx.res_dtype is not None and need[4] else None
        return (dx, dw if need[1] else None, db if need[2] else None, ds if need[3] else None, dres, None, None, None)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: str = "none", scale: Optional[Tensor] = None,
           residual: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None, checkpoint: bool = False) -> Tensor:
    """Differentiable ``linear_forward``.  ``weight`` may be an fp32 parameter: it is rounded to x's type for the products
    and its gradient is fp32.  The backward pass reads x and, with an activation, the pre-activation, kept in x's type or,
    with ``checkpoint``, in 8 bits (where ReLU's gradient stops at values under half a step: ``activation_backward``)."""
    if weight.dtype not in _FLOATS:
        raise TypeError(f"weight must be bf16, fp16 or fp32, not {weight.dtype}")
    return _Linear.apply(x, weight, bias, scale, residual, activation, out_dtype, checkpoint)


class _MlpHalf(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, norm_bias, w1, b1, w2, b2, scale, eps, compute_dtype):
        h, _, rstd, rows = layer_norm_forward(x, norm_weight, norm_bias, eps, compute_dtype, checkpoint=True)
        v1, v2 = w1.to(compute_dtype), w2.to(compute_dtype)
        a, pre = linear_forward(h, v1, b1, "gelu", checkpoint=True)
        y, _ = linear_forward(a, v2, b2, scale=scale, residual=x, out_dtype=x.dtype)
        ctx.x_dtype, ctx.w_dtypes, ctx.compute = x.dtype, (w1.dtype, w2.dtype), compute_dtype
        ctx.save_for_backward(norm_weight, norm_bias, v1, v2, b2, scale, rstd, *rows, *pre)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        g, b, v1, v2, b2, scale, rstd, rc, re, pc, pe = ctx.saved_tensors
        rows, pre = Checkpoint8(rc, re), Checkpoint8(pc, pe)
        need = ctx.needs_input_grad
        d16 = dy.to(ctx.compute)
        second = need[5] or need[6] or need[7]
        # fp16: du and dh carry the power of two that keeps a small LayerScale out of the subnormals; `unit` undoes it on the
        # vectors that dW1, dx and the sums are multiplied by
        carried, unit = (scale, None) if scale is None or ctx.compute != torch.float16 else (_host or _ops()).scale_unit(scale)
        du, a = linear_backward_input(d16, v2, "gelu", pre, scale=carried, want_activation=second)
        dw2 = db2 = ds = dw1 = db1 = dx = dg = db = None
        if second:
            more = {"weight": v2, "bias": b2, "scale": scale} if scale is not None else {}
            dw2, db2, ds = linear_backward_weight(d16, a, out_dtype=ctx.w_dtypes[1], **more)
        if need[3] or need[4]:
            xs, xt = (g, b) if unit is None else (g * unit, b * unit)
            dw1, db1, _ = linear_backward_weight(du, rows, x_scale=xs, x_shift=xt, out_dtype=ctx.w_dtypes[0])
        if need[0] or need[1] or need[2]:
            dh = linear_backward_input(du, v1)[0]
            dx, dg, db = layer_norm_backward(dh, rows, None, rstd if unit is None else rstd * unit, g, add=dy, out_dtype=ctx.x_dtype)
        if unit is not None:
            db1, dg, db = (t if t is None else t.mul_(unit) for t in (db1, dg, db))
        got = (dx, dg, db, dw1, db1, dw2, db2, ds)
        return tuple(t if n else None for t, n in zip(got, need)) + (None, None)


def mlp_half(x: Tensor, norm_weight: Tensor, norm_bias: Tensor, w1: Tensor, b1: Tensor, w2: Tensor, b2: Tensor,
             scale: Optional[Tensor] = None, eps: float = 1e-6, compute_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The MLP half of an encoder layer (hf:372-378):  ``x + scale * (gelu(LN(x) w1^T + b1) w2^T + b2)``, differentiable in
    all its tensors.  For the backward pass it keeps the normalised rows and the hidden pre-activation in 8 bits and one
    fp32 number a row: D + H + (D + H) / 32 + 4 bytes for a row of D columns and H hidden ones, against 4 D + 2 D + 4 H for
    x, LN(x), the pre-activation and its GELU as the products read them.  ``w1``, ``w2`` may be fp32 parameters.  With fp16
    products, the gradients between the layers carry a power of two that keeps a LayerScale of 1e-5 out of fp16's
    subnormals; dy itself is rounded to fp16, so scale the loss where it is small."""
    if compute_dtype not in _HALF:
        raise TypeError(f"compute_dtype must be bf16 or fp16, not {compute_dtype}")
    for name, w in (("w1", w1), ("w2", w2)):
        if w.dtype not in _FLOATS:
            raise TypeError(f"{name} must be bf16, fp16 or fp32, not {w.dtype}")
        if w.dim() != 2:
            raise ValueError(f"{name} must be a matrix")
    if w1.shape[1] != x.shape[-1] or tuple(w2.shape) != (x.shape[-1], w1.shape[0]):
        raise ValueError(f"w1 {tuple(w1.shape)} and w2 {tuple(w2.shape)} do not go with rows of {x.shape[-1]}")
    return _MlpHalf.apply(x, norm_weight, norm_bias, w1, b1, w2, b2, scale, float(eps), compute_dtype)
