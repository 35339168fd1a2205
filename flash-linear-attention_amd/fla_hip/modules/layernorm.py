"""Layer / RMS normalisation with the residual stream, with the interface of the reference's fla/modules/layernorm.py: ``layer_norm_fwd`` /
``layer_norm_bwd``, the differentiable ``layer_norm`` / ``rms_norm`` and the ``LayerNorm`` / ``RMSNorm`` layers (one group; weights as torch's).  All compute
is done by ``gdn_layer_norm_fwd``, ``gdn_layer_norm_bwd`` and ``gdn_sum_rows`` of the HIP library.

What is normalised is the residual stream as it is handed on, in the stream's own type, with ``prenorm`` and without (the reference normalises the sum before it is
rounded): the backward sees the numbers the forward saw and keeps one tensor of them, and every call equals an addition followed by a normalisation.  With a stream of 16 bits that is
one rounding more than the sum in 32 bits would have; an fp32 stream has none."""
from __future__ import annotations

import torch
import torch.nn as nn

from fla_hip import _lib
from fla_hip.ops.gated_delta_rule._common import differentiable_once, dtype_code, launch, no_forward_mode, ptr, require_gpu, restored, sum_rows


def _stream_dtype(x: torch.Tensor, residual: torch.Tensor | None, residual_dtype: torch.dtype | None) -> torch.dtype:
    dt = residual.dtype if residual is not None else (residual_dtype or x.dtype)
    if dt not in (x.dtype, torch.float32):
        raise NotImplementedError(f'the residual stream of {x.dtype} rows is kept in that type or in fp32, not in {dt}')
    return dt


def _params(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None):
    """weight and bias in one type that the kernels take: the rows' or fp32."""
    D = x.shape[-1]
    for name, p in (('weight', weight), ('bias', bias)):
        if p is not None and tuple(p.shape) != (D,):
            raise ValueError(f'{name} must be [{D}], got {tuple(p.shape)}')
    dts = {p.dtype for p in (weight, bias) if p is not None}
    dt = dts.pop() if len(dts) == 1 else torch.float32
    if dt != x.dtype:
        dt = torch.float32
    weight, bias = (p if p is None else p.to(dt).contiguous() for p in (weight, bias))
    return weight, bias, dtype_code(dt)


def _check_rows(x: torch.Tensor, dtype: torch.dtype) -> None:
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f'x must be [rows, D], got {tuple(x.shape)}')
    if x.shape[1] * dtype.itemsize >= 65536:
        raise RuntimeError("This layer norm doesn't support feature dim >= 64KB.")


def layer_norm_fwd(
    x: torch.Tensor,
    weight: torch.Tensor | None,
    bias: torch.Tensor | None,
    eps: float = 1e-5,
    residual: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    residual_dtype: torch.dtype | None = None,
    is_rms_norm: bool = False,
):
    """``x`` is ``[rows, D]``.  Returns ``(y, mean, rstd, residual_out)``: ``mean`` is ``None`` for RMS norm, ``residual_out`` (what was normalised) is ``x``
    itself when no residual stream was asked for."""
    _check_rows(x, x.dtype)
    dev = require_gpu(x, *(t for t in (weight, bias, residual) if t is not None))
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f'residual must be shaped as x {tuple(x.shape)}, got {tuple(residual.shape)}')
    rows, D = x.shape
    stream_dtype = _stream_dtype(x, residual, residual_dtype)
    weight, bias, w_code = _params(x, weight, bias)
    x = x.contiguous()
    y = torch.empty_like(x)
    if residual is not None or stream_dtype != x.dtype:
        residual = residual if residual is None else residual.contiguous()
        stream = torch.empty(rows, D, dtype=stream_dtype, device=dev)
    else:
        stream = None
    rstd = torch.empty(rows, dtype=torch.float32, device=dev)
    mean = None if is_rms_norm else torch.empty_like(rstd)
    launch(_lib.load().gdn_layer_norm_fwd, dev, ptr(x), ptr(residual), ptr(weight), ptr(bias), ptr(y), ptr(stream), ptr(mean), ptr(rstd), rows, D, eps,
           dtype_code(x.dtype), dtype_code(stream_dtype), w_code, int(bool(is_rms_norm)))
    if out_dtype is not None and out_dtype != y.dtype:
        y = y.to(out_dtype)
    return y, mean, rstd, x if stream is None else stream


def layer_norm_bwd(
    dy: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor | None,
    bias: torch.Tensor | None,
    eps: float = 1e-5,
    mean: torch.Tensor | None = None,
    rstd: torch.Tensor | None = None,
    dresidual: torch.Tensor | None = None,
    has_residual: bool = False,
    is_rms_norm: bool = False,
    x_dtype: torch.dtype | None = None,
    needs: tuple = (True, True, True, True),
):
    """Gradients ``(dx, dw, db, dresidual_in)`` of ``layer_norm_fwd``.  ``x`` is what was normalised (the forward's fourth result), ``mean`` / ``rstd`` the
    forward's row statistics, ``dresidual`` the gradient of the residual stream handed on (prenorm).  ``dx`` comes in ``x_dtype`` (default: dy's type),
    ``dresidual_in`` in x's, ``None`` unless ``has_residual``.  ``needs``: which of dx, dw, db and dresidual_in are wanted at all."""
    dt = x_dtype or dy.dtype
    _check_rows(x, dt)
    dev = require_gpu(dy, x, *(t for t in (weight, bias, mean, rstd, dresidual) if t is not None))
    rows, D = x.shape
    if dy.shape != x.shape or (dresidual is not None and dresidual.shape != x.shape):
        raise ValueError(f'dy and dresidual must be shaped as x {tuple(x.shape)}, got {tuple(dy.shape)}' + ('' if dresidual is None else f' and {tuple(dresidual.shape)}'))
    if rstd is None or (mean is None and not is_rms_norm):
        raise ValueError('layer_norm_bwd needs the row statistics of the forward (rstd, and mean for layer norm)')
    for name, s in (('rstd', rstd), ('mean', mean)):
        if s is not None and (s.shape != (rows,) or s.dtype != torch.float32):
            raise ValueError(f'{name} must be [{rows}] fp32, got {tuple(s.shape)} {s.dtype}')
    if x.dtype not in (dt, torch.float32):
        raise NotImplementedError(f'the residual stream of {dt} rows is kept in that type or in fp32, not in {x.dtype}')
    w_k, _, w_code = _params(dy.to(dt) if dy.dtype != dt else dy, weight, None)
    dy, x = dy.to(dt).contiguous(), x.contiguous()
    dresidual = dresidual if dresidual is None else dresidual.to(x.dtype).contiguous()
    mean, rstd = mean if mean is None else mean.contiguous(), rstd.contiguous()
    need_x, need_w, need_b, need_res = needs[0], needs[1] and weight is not None, needs[2] and bias is not None, needs[3] and has_residual
    shared = x.dtype == dt
    dx = torch.empty(rows, D, dtype=dt, device=dev) if need_x or (need_res and shared) else None
    dres = torch.empty(rows, D, dtype=x.dtype, device=dev) if need_res and not shared else None
    lib = _lib.load()
    kinds = int(need_w) + int(need_b)
    parts = lib.gdn_layer_norm_bwd_parts(rows, D, dtype_code(dt))
    part = torch.empty(parts, kinds, D, dtype=torch.float32, device=dev) if kinds else None
    launch(lib.gdn_layer_norm_bwd, dev, ptr(dy), ptr(x), ptr(w_k), ptr(mean), ptr(rstd), ptr(dresidual), ptr(dx), ptr(dres), ptr(part), rows, D, parts,
           int(need_w), int(need_b), dtype_code(dt), dtype_code(x.dtype), w_code, int(bool(is_rms_norm)))
    dw = db = None
    if kinds == 2 and weight.dtype == bias.dtype:
        dw, db = sum_rows(part, weight.dtype)
    elif kinds:
        sums = sum_rows(part, torch.float32 if kinds == 2 else (weight if need_w else bias).dtype)
        dw, db = sums[0].to(weight.dtype) if need_w else None, sums[-1].to(bias.dtype) if need_b else None
    return dx if need_x else None, dw, db, (dx if shared else dres) if need_res else None


class LayerNormFunction(torch.autograd.Function):
    """Forward and backward kernels as one differentiable function."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, prenorm, residual_in_fp32, is_rms_norm):
        shape = x.shape
        y, mean, rstd, stream = _run(x, weight, bias, residual, eps, residual_in_fp32, is_rms_norm)
        ctx.save_for_backward(stream, weight, bias, mean, rstd)
        ctx.shape, ctx.eps, ctx.is_rms_norm, ctx.has_residual, ctx.x_dtype = shape, eps, is_rms_norm, residual is not None, x.dtype
        ctx.rows, ctx.device = stream.shape, x.device
        ctx.dtypes = (stream.dtype, *(None if t is None else t.dtype for t in (weight, bias)))
        ctx.set_materialize_grads(False)
        if not prenorm:
            return y.view(shape)
        # (without a residual stream of its own the stream is x: a view, so that autograd sees an output and not the input again)
        return y.view(shape), stream.view(shape)

    @staticmethod
    @differentiable_once
    def backward(ctx, dy, dstream=None):
        if dy is None and dstream is None:
            return (None,) * 8
        need_x, need_w, need_b, need_res = ctx.needs_input_grad[:4]
        rows, dtypes = ctx.rows, (*ctx.dtypes, torch.float32, torch.float32)
        shapes = (rows, rows[1:], rows[1:], rows[:1], rows[:1])
        stream, weight, bias, mean, rstd = (restored(t, dt, shape, ctx.device) for t, dt, shape in zip(ctx.saved_tensors, dtypes, shapes))
        dy = torch.zeros(rows, dtype=ctx.x_dtype, device=stream.device) if dy is None else dy.reshape(rows)
        dstream = None if dstream is None else dstream.reshape(rows)
        dx, dw, db, dres = layer_norm_bwd(dy, stream, weight, bias, ctx.eps, mean, rstd, dstream, ctx.has_residual, ctx.is_rms_norm, ctx.x_dtype,
                                          (need_x, need_w, need_b, need_res))
        return (None if dx is None else dx.view(ctx.shape), dw, db, None if dres is None else dres.view(ctx.shape)) + (None,) * 4


def _run(x, weight, bias, residual, eps, residual_in_fp32, is_rms_norm):
    if x.dim() == 0:
        raise ValueError('x must be [..., D]')
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f'residual must be shaped as x {tuple(x.shape)}, got {tuple(residual.shape)}')
    D = x.shape[-1]
    return layer_norm_fwd(x.reshape(-1, D) if D else x.reshape(0, 0), weight, bias, eps, None if residual is None else residual.reshape(-1, D),
                          residual_dtype=torch.float32 if residual_in_fp32 else None, is_rms_norm=is_rms_norm)


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None,
    bias: torch.Tensor | None,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
    prenorm: bool = False,
    residual_in_fp32: bool = False,
    is_rms_norm: bool = False,
):
    """Layer norm of ``x (+ residual)`` over the last dimension.  ``prenorm``: returns ``(y, stream)`` with ``stream = x + residual`` in the residual's type
    (without one: x's, or fp32 with ``residual_in_fp32``).  ``x`` bf16, fp16 or fp32; the stream in x's type or fp32."""
    out = _lib.host().layer_norm(x, weight, bias, residual, eps, prenorm, residual_in_fp32, is_rms_norm)
    if out is not None:
        return out
    no_forward_mode('layer_norm', x, weight, bias, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return LayerNormFunction.apply(x, weight, bias, residual, eps, prenorm, residual_in_fp32, is_rms_norm)
    y, _, _, stream = _run(x, weight, bias, residual, eps, residual_in_fp32, is_rms_norm)
    return (y.view(x.shape), stream.view(x.shape)) if prenorm else y.view(x.shape)


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None,
    bias: torch.Tensor | None,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
    prenorm: bool = False,
    residual_in_fp32: bool = False,
):
    """The same with the mean left where it is: ``y = r / sqrt(mean(r^2) + eps) * weight + bias``."""
    return layer_norm(x, weight, bias, residual, eps, prenorm, residual_in_fp32, True)


class LayerNorm(nn.Module):
    _is_rms = False

    def __init__(self, hidden_size: int, elementwise_affine: bool = True, bias: bool = False, eps: float = 1e-5, device=None, dtype=None):
        super().__init__()
        self.hidden_size, self.elementwise_affine, self.eps = hidden_size, elementwise_affine, eps
        self.register_parameter('weight', None)
        self.register_parameter('bias', None)
        if elementwise_affine:
            self.weight = nn.Parameter(torch.empty(hidden_size, device=device, dtype=dtype))
            if bias:
                self.bias = nn.Parameter(torch.empty(hidden_size, device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self):
        if self.elementwise_affine:
            nn.init.ones_(self.weight)
            if self.bias is not None:
                nn.init.zeros_(self.bias)

    def __repr__(self) -> str:
        s = f'{self.__class__.__name__}({self.hidden_size}'
        if not self.elementwise_affine:
            s += f', elementwise_affine={self.elementwise_affine}'
        return s + f', eps={self.eps})'

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, prenorm: bool = False, residual_in_fp32: bool = False):
        return layer_norm(x, self.weight, self.bias, residual, self.eps, prenorm, residual_in_fp32, self._is_rms)


class RMSNorm(LayerNorm):
    _is_rms = True
