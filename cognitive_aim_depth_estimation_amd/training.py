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

import ctypes as C
import functools
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from ._lib import LinearBwdInputDesc, LinearBwdWeightDesc, LinearFwdDesc, call, ptr

__all__ = ["Checkpoint8", "pack8", "unpack8", "layer_norm_forward", "layer_norm_backward", "linear_forward",
           "linear_backward_input", "linear_backward_weight", "activation_backward", "layer_norm", "linear", "mlp_half"]

Tensor = torch.Tensor
GROUP = 32
MAX_NORM_WIDTH = 16384
MAX_LEADING_DIM = 1 << 21
_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2}


class Checkpoint8(NamedTuple):
    """Activations in 8 bits: int8 ``codes [..., D]`` and one uint8 exponent for every 32 columns, ``exponents
    [..., ceil(D / 32)]``.  A value is ``code * 2**(exponent - 127)``; the step is the smallest power of two (from 2^-126)
    for which the group's largest magnitude rounds to at most 127, so a value is off by at most half a step:
    between 1/255 and 1/127.5 of the group's largest magnitude.  A group that held an infinity or a NaN has exponent
    255 and stands for NaN."""
    codes: Tensor
    exponents: Tensor


# ---- arguments ---------------------------------------------------------------------------------------------------
def _float(t, name, types=_CODE):
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in types:
        raise TypeError(f"{name} must be one of {', '.join(str(d) for d in types)}, not {t.dtype}")
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} needs at least one column")
    return t


_HALF = (torch.bfloat16, torch.float16)


def _rows(t: Tensor) -> Tuple[Tensor, int]:
    """[rows, columns] view (or copy, when the columns are not contiguous) and its leading dimension."""
    D = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(t.numel() // D, D)
    n = t.shape[0]
    ld = t.stride(0) if n > 1 else D
    if ld < D or (D > 1 and t.stride(1) != 1):
        t = t.contiguous()
        ld = D
    return t, ld


def _vector(t, name, n, device):
    if t is None:
        return None
    if not isinstance(t, Tensor) or t.dtype != torch.float32 or t.shape != (n,):
        raise ValueError(f"{name} must be a float32 vector of {n}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the rows are on {device}")
    return t if t.stride(0) == 1 or n == 1 else t.contiguous()


def _same(t, name, shape, device):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, {tuple(shape)} is needed")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the rows are on {device}")


def _checkpoint(saved, name, shape, device):
    if not isinstance(saved, Checkpoint8):
        raise TypeError(f"{name} must be a Checkpoint8")
    codes, exponents = saved
    if codes.dtype != torch.int8 or exponents.dtype != torch.uint8:
        raise TypeError(f"{name}: codes must be int8 and exponents uint8")
    D = shape[-1]
    _same(codes, f"{name}.codes", shape, device)
    _same(exponents, f"{name}.exponents", tuple(shape[:-1]) + ((D + GROUP - 1) // GROUP,), device)
    return codes.contiguous(), exponents.contiguous()


def _out_dtype(dtype, default, types=_CODE):
    dtype = default if dtype is None else dtype
    if dtype not in types:
        raise TypeError(f"out_dtype must be one of {', '.join(str(d) for d in types)}, not {dtype}")
    return dtype


def _act(name):
    if name not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, not {name!r}")
    return _ACTIVATIONS[name]


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    """Handle of the current stream of a tensor's device."""
    if device.type != "cuda":
        raise RuntimeError("the training operators run only on a ROCm device (no CPU path)")
    # (the handle without the Python object around it, where torch offers that: 0.1 us instead of 2.8 of a call's ten)
    return _raw_stream(device.index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _on_device(fn):
    """The device of the first argument made current for a call, when it is not."""
    @functools.wraps(fn)
    def run(first, *args, **kwargs):
        t = first.codes if type(first) is Checkpoint8 else first
        if isinstance(t, Tensor) and t.is_cuda and t.get_device() != torch.cuda.current_device():
            with torch.cuda.device(t.device):
                return fn(first, *args, **kwargs)
        return fn(first, *args, **kwargs)
    return run


def _new(like, shape, dtype):
    """An empty tensor on the device of `like`."""
    return like.new_empty(shape, dtype=dtype)


def _new_checkpoint(like, lead, D):
    return Checkpoint8(_new(like, (*lead, D), torch.int8), _new(like, (*lead, (D + GROUP - 1) // GROUP), torch.uint8))


# ---- 8-bit activations -------------------------------------------------------------------------------------------
@_on_device
def pack8(x: Tensor) -> Checkpoint8:
    """``x [..., D]`` (bf16, fp16 or fp32) in 8 bits."""
    _float(x, "x")
    stream = _stream(x.device)
    out = _new_checkpoint(x, x.shape[:-1], x.shape[-1])
    v, ld = _rows(x)
    if v.shape[0]:
        call("cogaim_pack8", v.data_ptr(), _CODE[x.dtype], ld, out.codes.data_ptr(), out.exponents.data_ptr(), v.shape[0],
             v.shape[1], stream)
    return out


@_on_device
def unpack8(saved: Checkpoint8, dtype: torch.dtype = torch.float32) -> Tensor:
    """The values of an 8-bit copy: exact in fp32 and bf16, rounded once (and held at +-65504) in fp16."""
    if not isinstance(saved, Checkpoint8):
        raise TypeError("saved must be a Checkpoint8")
    dtype = _out_dtype(dtype, torch.float32)
    shape = saved.codes.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError("saved needs at least one column")
    codes, exponents = _checkpoint(saved, "saved", shape, saved.codes.device)
    stream = _stream(codes.device)
    out = _new(codes, shape, dtype)
    D = shape[-1]
    M = codes.numel() // D
    if M:
        call("cogaim_unpack8", codes.data_ptr(), exponents.data_ptr(), out.data_ptr(), _CODE[dtype], D, M, D, D, stream)
    return out


@_on_device
def activation_backward(dy: Tensor, saved: Checkpoint8, activation: str, out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``dy * act'(u)`` with ``u`` kept in 8 bits; activation "relu" or "gelu"."""
    _float(dy, "dy")
    act = _act(activation)
    if not act:
        raise ValueError("activation must be 'relu' or 'gelu'")
    out_dtype = _out_dtype(out_dtype, dy.dtype)
    codes, exponents = _checkpoint(saved, "saved", dy.shape, dy.device)
    stream = _stream(dy.device)
    out = _new(dy, dy.shape, out_dtype)
    v, ld = _rows(dy)
    M, D = v.shape
    if M:
        call("cogaim_activation_bwd", v.data_ptr(), _CODE[dy.dtype], ld, codes.data_ptr(), exponents.data_ptr(),
             out.data_ptr(), _CODE[out_dtype], D, act, M, D, stream)
    return out


# ---- layer norm --------------------------------------------------------------------------------------------------
@_on_device
def layer_norm_forward(x: Tensor, weight: Tensor, bias: Tensor, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None,
                       checkpoint: bool = False) -> Tuple[Tensor, Tensor, Tensor, Optional[Checkpoint8]]:
    """``(y, mean, rstd, saved)``: ``y = (x - mean) * rstd * weight + bias`` of type ``out_dtype`` (default: x's), the fp32
    statistics of every row, and with ``checkpoint`` the normalised rows ``(x - mean) * rstd`` in 8 bits (else None)."""
    _float(x, "x")
    D = x.shape[-1]
    if D > MAX_NORM_WIDTH:
        raise ValueError(f"layer norm of {D} columns: at most {MAX_NORM_WIDTH}")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    dev = x.device
    weight, bias = _vector(weight, "weight", D, dev), _vector(bias, "bias", D, dev)
    if weight is None or bias is None:
        raise ValueError("weight and bias are needed")
    out_dtype = _out_dtype(out_dtype, x.dtype)
    stream = _stream(dev)
    lead = x.shape[:-1]
    y = _new(x, x.shape, out_dtype)
    mean = _new(x, lead, torch.float32)
    rstd = torch.empty_like(mean)
    saved = _new_checkpoint(x, lead, D) if checkpoint else None
    v, ld = _rows(x)
    if v.shape[0]:
        call("cogaim_layernorm_train_fwd", v.data_ptr(), _CODE[x.dtype], ld, weight.data_ptr(), bias.data_ptr(), y.data_ptr(),
             _CODE[out_dtype], D, mean.data_ptr(), rstd.data_ptr(), ptr(saved.codes) if saved else None,
             ptr(saved.exponents) if saved else None, v.shape[0], D, eps, stream)
    return y, mean, rstd, saved


@_on_device
def layer_norm_backward(dy: Tensor, saved: Union[Tensor, Checkpoint8], mean: Optional[Tensor], rstd: Tensor, weight: Tensor,
                        add: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``(dx, dweight, dbias)`` from ``dy`` and either the norm's input with its ``mean`` or its rows in 8 bits (``mean`` is
    not read then).  ``add`` (the gradient that flows past the norm) is added to dx.  dx is of type ``out_dtype`` (default:
    the input's, dy's with an 8-bit copy)."""
    _float(dy, "dy")
    D, dev, lead = dy.shape[-1], dy.device, dy.shape[:-1]
    if D > MAX_NORM_WIDTH:
        raise ValueError(f"layer norm of {D} columns: at most {MAX_NORM_WIDTH}")
    weight = _vector(weight, "weight", D, dev)
    if weight is None:
        raise ValueError("weight is needed")

    def stat(t, name):
        if not isinstance(t, Tensor) or t.dtype != torch.float32:
            raise TypeError(f"{name} must be a float32 tensor")
        _same(t, name, lead, dev)
        return t.contiguous()

    rstd = stat(rstd, "rstd")
    codes = exponents = x = None
    if isinstance(saved, Checkpoint8):
        codes, exponents = _checkpoint(saved, "saved", dy.shape, dev)
        out_dtype = _out_dtype(out_dtype, dy.dtype)
    else:
        x = _float(saved, "saved")
        _same(x, "saved", dy.shape, dev)
        mean = stat(mean, "mean")
        out_dtype = _out_dtype(out_dtype, x.dtype)
    if add is not None:
        _float(add, "add")
        _same(add, "add", dy.shape, dev)
    stream = _stream(dev)
    dx = _new(dy, dy.shape, out_dtype)
    v, ld = _rows(dy)
    M = v.shape[0]
    if not M:
        return dx, torch.zeros(D, device=dev), torch.zeros(D, device=dev)
    dweight = torch.empty_like(weight)
    dbias = torch.empty_like(weight)
    nbytes = call("cogaim_layernorm_bwd_workspace_bytes", M, D)
    ws = _new(dy, nbytes, torch.uint8)
    xv, ldx = _rows(x) if x is not None else (None, 0)
    av, lda = _rows(add) if add is not None else (None, 0)
    call("cogaim_layernorm_bwd", v.data_ptr(), _CODE[dy.dtype], ld, ptr(xv), _CODE[x.dtype] if x is not None else 0, ldx,
         ptr(codes), ptr(exponents), ptr(mean) if x is not None else None, rstd.data_ptr(), weight.data_ptr(), ptr(av),
         _CODE[add.dtype] if add is not None else 0, lda, dx.data_ptr(), _CODE[out_dtype], D, dweight.data_ptr(),
         dbias.data_ptr(), M, D, ws.data_ptr(), nbytes, stream)
    return dx, dweight, dbias


# ---- linear layers -----------------------------------------------------------------------------------------------
def _matrix(w, name):
    _float(w, name, _HALF)
    if w.dim() != 2 or w.shape[0] < 1:
        raise ValueError(f"{name} must be a matrix")
    return w


def _leading(ld, name):
    if ld > MAX_LEADING_DIM:
        raise ValueError(f"rows of {name} are {ld} elements apart: at most {MAX_LEADING_DIM}")
    return ld


def _run_linear(name, desc, like, stream):
    desc = C.byref(desc)
    nbytes = call(name + "_workspace_bytes", desc)
    if nbytes < 0:
        raise ValueError(f"{name}: arguments the kernels do not take")
    ws = _new(like, nbytes, torch.uint8) if nbytes else None
    call(name, desc, ptr(ws), nbytes, stream)


@_on_device
def linear_forward(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: str = "none",
                   scale: Optional[Tensor] = None, residual: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   checkpoint: bool = False) -> Tuple[Tensor, Optional[Checkpoint8]]:
    """``(y, saved)`` for ``x [..., K]`` and ``weight [N, K]`` of one 16-bit type:  with ``u = x weight^T + bias``,
    ``y = act(u) + residual``, or ``y = scale * u + residual`` (scale: LayerScale, only without an activation).  ``y`` is of
    type ``out_dtype`` (default: x's); with ``checkpoint``, ``saved`` is u in 8 bits, packed in the product's epilogue."""
    _float(x, "x", _HALF)
    _matrix(weight, "weight")
    act = _act(activation)
    N, K = weight.shape
    dev, lead = x.device, x.shape[:-1]
    if x.shape[-1] != K or weight.dtype != x.dtype or weight.device != dev:
        raise ValueError(f"x {tuple(x.shape)} {x.dtype} on {x.device} does not go with weight {tuple(weight.shape)} {weight.dtype} on {weight.device}")
    if scale is not None and act:
        raise ValueError("scale goes with activation 'none'")
    bias, scale = _vector(bias, "bias", N, dev), _vector(scale, "scale", N, dev)
    out_dtype = _out_dtype(out_dtype, x.dtype)
    if residual is not None:
        _float(residual, "residual")
        _same(residual, "residual", tuple(lead) + (N,), dev)
    stream = _stream(dev)
    y = _new(x, (*lead, N), out_dtype)
    saved = _new_checkpoint(x, lead, N) if checkpoint else None
    xv, ldx = _rows(x)
    M = xv.shape[0]
    if M:
        wv, ldw = _rows(weight)
        rv, ldr = _rows(residual) if residual is not None else (None, 0)
        desc = LinearFwdDesc(xv.data_ptr(), wv.data_ptr(), ptr(bias), ptr(scale), ptr(rv), y.data_ptr(),
                             ptr(saved.codes) if saved else None, ptr(saved.exponents) if saved else None,
                             _leading(ldx, "x"), _leading(ldw, "weight"), _leading(ldr, "residual"), _leading(N, "y"), M, N, K,
                             _CODE[x.dtype], _CODE[residual.dtype] if residual is not None else 0, _CODE[out_dtype], act, 0)
        _run_linear("cogaim_linear_fwd", desc, x, stream)
    return y, saved


@_on_device
def linear_backward_input(dy: Tensor, weight: Tensor, activation: str = "none", saved: Optional[Checkpoint8] = None,
                          scale: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                          want_activation: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """``(dx, a)`` for ``dy [..., N]`` and ``weight [N, K]`` of one 16-bit type:  ``dx = ((dy * scale) weight) * act'(u)``,
    ``u [..., K]`` the pre-activation, kept in 8 bits (``saved``), of the activation that produced the layer's input; with
    ``want_activation``, ``a = act(u)`` in 16 bits: that input again, for ``linear_backward_weight``.  With ``scale``,
    ``weight * scale`` is rounded to 16 bits."""
    _float(dy, "dy", _HALF)
    _matrix(weight, "weight")
    act = _act(activation)
    N, K = weight.shape
    dev, lead = dy.device, dy.shape[:-1]
    if dy.shape[-1] != N or weight.dtype != dy.dtype or weight.device != dev:
        raise ValueError(f"dy {tuple(dy.shape)} {dy.dtype} on {dy.device} does not go with weight {tuple(weight.shape)} {weight.dtype} on {weight.device}")
    if bool(act) != (saved is not None):
        raise ValueError("saved is the pre-activation of an activation: give both or neither")
    if want_activation and not act:
        raise ValueError("want_activation needs an activation")
    scale = _vector(scale, "scale", N, dev)
    out_dtype = _out_dtype(out_dtype, dy.dtype)
    codes = exponents = None
    if act:
        codes, exponents = _checkpoint(saved, "saved", tuple(lead) + (K,), dev)
    stream = _stream(dev)
    dx = _new(dy, (*lead, K), out_dtype)
    a = _new(dy, (*lead, K), dy.dtype) if want_activation else None
    v, ld = _rows(dy)
    M = v.shape[0]
    if M:
        wv, ldw = _rows(weight)
        desc = LinearBwdInputDesc(v.data_ptr(), wv.data_ptr(), ptr(scale), ptr(codes), ptr(exponents), dx.data_ptr(), ptr(a),
                                  _leading(ld, "dy"), _leading(ldw, "weight"), _leading(K, "dx"), K, M, N, K, _CODE[dy.dtype],
                                  _CODE[out_dtype], act)
        _run_linear("cogaim_linear_bwd_input", desc, dy, stream)
    return dx, a


@_on_device
def linear_backward_weight(dy: Tensor, x: Union[Tensor, Checkpoint8], weight: Optional[Tensor] = None,
                           bias: Optional[Tensor] = None, scale: Optional[Tensor] = None, x_scale: Optional[Tensor] = None,
                           x_shift: Optional[Tensor] = None,
                           out_dtype: torch.dtype = torch.float32) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
    """``(dW, db, dscale)`` for ``dy [..., N]`` in 16 bits and the layer's input ``x [..., K]``, in dy's type or in 8 bits;
    an 8-bit copy stands for ``x_scale * copy + x_shift`` (a norm's weight and bias over its kept rows).  Without
    ``scale``, ``dW = dy^T x`` and ``db`` sums dy's rows (dscale None).  With ``scale`` (and the forward's ``weight`` and
    ``bias``), for ``y = scale * (x weight^T + bias)``: dW and db are those times scale, ``dscale`` sums ``dy * (x weight^T + bias)``.
    db and dscale are fp32, dW is of type ``out_dtype``."""
    _float(dy, "dy", _HALF)
    N, dev, lead = dy.shape[-1], dy.device, dy.shape[:-1]
    codes = exponents = None
    if isinstance(x, Checkpoint8):
        K = x.codes.shape[-1] if x.codes.dim() else 0
        if K < 1:
            raise ValueError("x needs at least one column")
        codes, exponents = _checkpoint(x, "x", tuple(lead) + (K,), dev)
        x = None
    else:
        _float(x, "x", _HALF)
        K = x.shape[-1]
        _same(x, "x", tuple(lead) + (K,), dev)
        if x.dtype != dy.dtype:
            raise TypeError(f"x is {x.dtype}, dy {dy.dtype}")
        if x_scale is not None or x_shift is not None:
            raise ValueError("x_scale and x_shift go with an 8-bit x")
    x_scale, x_shift = _vector(x_scale, "x_scale", K, dev), _vector(x_shift, "x_shift", K, dev)
    scale = _vector(scale, "scale", N, dev)
    if scale is not None:
        if weight is None:
            raise ValueError("scale needs the forward's weight")
        _matrix(weight, "weight")
        _same(weight, "weight", (N, K), dev)
        if weight.dtype != dy.dtype:
            raise TypeError(f"weight is {weight.dtype}, dy {dy.dtype}")
        bias = _vector(bias, "bias", N, dev)
    elif weight is not None or bias is not None:
        raise ValueError("weight and bias go with scale")
    out_dtype = _out_dtype(out_dtype, torch.float32)
    stream = _stream(dev)
    v, ld = _rows(dy)
    M = v.shape[0]
    make = dy.new_empty if M else dy.new_zeros
    dw = make((N, K), dtype=out_dtype)
    db = make(N, dtype=torch.float32)
    ds = torch.empty_like(db) if scale is not None else None
    if ds is not None and not M:
        ds.zero_()
    if M:
        xv, ldx = _rows(x) if x is not None else (None, 0)
        wv, ldw = _rows(weight) if scale is not None else (None, 0)
        desc = LinearBwdWeightDesc(v.data_ptr(), ptr(xv), ptr(codes), ptr(exponents), ptr(x_scale), ptr(x_shift), ptr(wv),
                                   ptr(bias), ptr(scale), dw.data_ptr(), db.data_ptr(), ptr(ds), _leading(ld, "dy"),
                                   _leading(ldx, "x"), _leading(ldw, "weight"), _leading(K, "dW"), M, N, K, _CODE[dy.dtype],
                                   _CODE[out_dtype], 0)
        _run_linear("cogaim_linear_bwd_weight", desc, dy, stream)
    return dw, db, ds


# ---- differentiable ----------------------------------------------------------------------------------------------
def _grad(t, like):
    return t if t is None or t.dtype == like.dtype else t.to(like.dtype)


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
        y, pre = linear_forward(x, w, bias, activation, scale, residual, out_dtype, checkpoint=activation != "none")
        kept = pack8(x) if checkpoint else None
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
            du = activation_backward(dy, Checkpoint8(pc, pe), ctx.activation, ctx.x_dtype)
        else:
            du = dy.to(ctx.x_dtype)
        dx = linear_backward_input(du, w, scale=scale)[0] if need[0] else None
        dw = db = ds = None
        if need[1] or need[2] or need[3]:
            x = Checkpoint8(xa, xb) if ctx.kept8 else xa
            more = {"weight": w, "bias": bias, "scale": scale} if scale is not None else {}
            dw, db, ds = linear_backward_weight(du, x, out_dtype=ctx.w_dtype if ctx.w_dtype in _CODE else torch.float32, **more)
        dres = dy.to(ctx.res_dtype) if ctx.res_dtype is not None and need[4] else None
        return (dx, dw if need[1] else None, db if need[2] else None, ds if need[3] else None, dres, None, None, None)


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: str = "none", scale: Optional[Tensor] = None,
           residual: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None, checkpoint: bool = False) -> Tensor:
    """Differentiable ``linear_forward``.  ``weight`` may be an fp32 parameter: it is rounded to x's type for the products
    and its gradient is fp32.  A pre-activation is always kept in 8 bits; ``checkpoint`` keeps x in 8 bits as well."""
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
        du, a = linear_backward_input(d16, v2, "gelu", pre, scale=scale, want_activation=second)
        dw2 = db2 = ds = dw1 = db1 = dx = dg = db = None
        if second:
            more = {"weight": v2, "bias": b2, "scale": scale} if scale is not None else {}
            dw2, db2, ds = linear_backward_weight(d16, a, out_dtype=ctx.w_dtypes[1], **more)
        if need[3] or need[4]:
            dw1, db1, _ = linear_backward_weight(du, rows, x_scale=g, x_shift=b, out_dtype=ctx.w_dtypes[0])
        if need[0] or need[1] or need[2]:
            dh = linear_backward_input(du, v1)[0]
            dx, dg, db = layer_norm_backward(dh, rows, None, rstd, g, add=dy, out_dtype=ctx.x_dtype)
        got = (dx, dg, db, dw1, db1, dw2, db2, ds)
        return tuple(t if n else None for t, n in zip(got, need)) + (None, None)


def mlp_half(x: Tensor, norm_weight: Tensor, norm_bias: Tensor, w1: Tensor, b1: Tensor, w2: Tensor, b2: Tensor,
             scale: Optional[Tensor] = None, eps: float = 1e-6, compute_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The MLP half of an encoder layer (hf:372-378):  ``x + scale * (gelu(LN(x) w1^T + b1) w2^T + b2)``, differentiable in
    all its tensors.  For the backward pass it keeps the normalised rows and the hidden pre-activation in 8 bits and one
    fp32 number a row: D + H + (D + H) / 32 + 4 bytes for a row of D columns and H hidden ones, against 4 D + 2 D + 4 H for
    x, LN(x), the pre-activation and its GELU as the products read them.  ``w1``, ``w2`` may be fp32 parameters."""
    if compute_dtype not in _HALF:
        raise TypeError(f"compute_dtype must be bf16 or fp16, not {compute_dtype}")
    for name, w in (("w1", w1), ("w2", w2)):
        _float(w, name)
        if w.dim() != 2:
            raise ValueError(f"{name} must be a matrix")
    _float(x, "x")
    if w1.shape[1] != x.shape[-1] or tuple(w2.shape) != (x.shape[-1], w1.shape[0]):
        raise ValueError(f"w1 {tuple(w1.shape)} and w2 {tuple(w2.shape)} do not go with rows of {x.shape[-1]}")
    return _MlpHalf.apply(x, norm_weight, norm_bias, w1, b1, w2, b2, scale, float(eps), compute_dtype)
