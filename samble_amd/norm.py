"""Layer normalisation on the MI355X kernels (csrc/layernorm.hip): `layer_norm` beside `attention.batch_norm`, and the module
`LayerNorm`.  Normalises any one axis of a tensor in fp32, fp16 or bf16 -- the channels of this package's (B, C, N) tensors
(`dim=1`) or the last axis -- with an optional residual added in the same pass, forward and backward.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from . import _lib
from .ops import ELEMENT_TYPES as TYPES
from .ops import _differentiated, _need_gpu, _on, _p


def _slices(t: torch.Tensor, dim: int):
    """(outer, C, inner) view of t around axis `dim` -> (tensor, outer stride, channel stride); copied where the leading axes do
    not collapse into one stride, or the axes behind (rows: the axis itself) are not contiguous."""
    if t.is_contiguous():
        inner = 1
        for n in t.shape[dim + 1:]:
            inner *= n
        return t, t.shape[dim] * inner, inner
    C = t.shape[dim]
    inner = 1
    for n in t.shape[dim + 1:]:
        inner *= n
    expect, plain = 1, True
    for a in range(t.dim() - 1, dim, -1):
        if t.shape[a] != 1:
            plain = plain and t.stride(a) == expect
            expect *= t.shape[a]
    if inner == 1:
        plain = plain and (C == 1 or t.stride(dim) == 1)
    lead = [a for a in range(dim) if t.shape[a] != 1]
    for a, b in zip(lead, lead[1:]):
        plain = plain and t.stride(a) == t.shape[b] * t.stride(b)
    if not plain:
        t = t.contiguous()
    os = t.stride(lead[-1]) if lead else 0
    return t, os, (t.stride(dim) if inner > 1 else 1)


def _extent(t: torch.Tensor, dim: int):
    outer = inner = 1
    for n in t.shape[:dim]:
        outer *= n
    for n in t.shape[dim + 1:]:
        inner *= n
    return outer, t.shape[dim], inner


def _weight_type(x, weight, bias) -> int:
    for t in (weight, bias):
        if t is not None:
            return TYPES[t.dtype]
    return TYPES[x.dtype]


def stage_layer_norm_fwd(x: torch.Tensor, weight, bias, eps: float, dim: int, residual=None, stats: bool = True):
    """-> (y, s, mean, rstd): s = x + residual in x's type (x itself without a residual), mean / rstd (outer * inner) fp32
    (None unless `stats`)."""
    _need_gpu(x, weight, bias, residual)
    outer, C, inner = _extent(x, dim)
    with _on(x.device) as stream:
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        s = torch.empty_like(y) if residual is not None else x
        n = outer * inner
        mean, rstd = torch.empty((2, n), dtype=torch.float32, device=x.device).unbind(0) if stats else (None, None)
        if n:
            xv, x_os, x_cs = _slices(x, dim)
            rv, r_os, r_cs = _slices(residual, dim) if residual is not None else (None, 0, 0)
            _lib.call("samble_layer_norm_fwd", TYPES[x.dtype], _weight_type(x, weight, bias), xv.data_ptr(), x_os, x_cs, _p(rv),
                      r_os, r_cs, _p(weight), _p(bias), outer, C, inner, float(eps), y.data_ptr(),
                      _p(s) if residual is not None else None, _p(mean), _p(rstd), stream)
    return y, s, mean, rstd


def stage_layer_norm_bwd(s: torch.Tensor, dy: torch.Tensor, weight, mean: torch.Tensor, rstd: torch.Tensor, dim: int, extra=None,
                         want_weight_grads: bool = True, w_dtype=None):
    """-> (ds, dweight | None, dbias | None); `extra`: a gradient that reaches s from elsewhere, added to ds."""
    _need_gpu(s, dy, weight, mean, rstd, extra)
    outer, C, inner = _extent(s, dim)
    w_dtype = weight.dtype if weight is not None else (w_dtype or s.dtype)
    with _on(s.device) as stream:
        ds = torch.empty_like(s, memory_format=torch.contiguous_format)
        if outer * inner == 0:
            zero = lambda: torch.zeros(C, dtype=w_dtype, device=s.device) if want_weight_grads else None  # noqa: E731
            return ds, zero(), zero()
        dw, db = torch.empty((2, C), dtype=w_dtype, device=s.device).unbind(0) if want_weight_grads else (None, None)
        sv, s_os, s_cs = _slices(s, dim)
        gv, g_os, g_cs = _slices(dy, dim)
        ev, e_os, e_cs = _slices(extra, dim) if extra is not None else (None, 0, 0)
        nbytes = _lib.query("samble_layer_norm_workspace_bytes", TYPES[s.dtype], C, outer, inner) if want_weight_grads else 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=s.device) if want_weight_grads else None
        _lib.call("samble_layer_norm_bwd", TYPES[s.dtype], TYPES[w_dtype], sv.data_ptr(), s_os, s_cs, gv.data_ptr(), g_os, g_cs,
                  _p(ev), e_os, e_cs, _p(weight), mean.data_ptr(), rstd.data_ptr(), outer, C, inner, ds.data_ptr(), _p(dw),
                  _p(db), _p(ws), nbytes, stream)
    return ds, dw, db


class _LayerNorm(torch.autograd.Function):
    # (no autocast decorators: no torch arithmetic runs in either direction, the kernels take the types they are given)
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, dim):
        y, s, mean, rstd = stage_layer_norm_fwd(x, weight, bias, eps, dim, residual)
        ctx.save_for_backward(s, weight, mean, rstd)
        ctx.dim = dim
        ctx.b_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, s)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, extra=None):
        s, weight, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        if dy is None:      # only the sum was used
            zero = lambda need, like: torch.zeros(s.shape[ctx.dim], dtype=like, device=s.device) if need else None  # noqa: E731
            return (extra if need_x else None, zero(need_w, weight.dtype if weight is not None else None),
                    zero(need_b, ctx.b_dtype), extra if need_r else None, None, None)
        ds, dw, db = stage_layer_norm_bwd(s, dy.to(s.dtype), weight, mean, rstd, ctx.dim,
                                          None if extra is None else extra.to(s.dtype), need_w or need_b, ctx.b_dtype)
        return ds if need_x else None, dw if need_w else None, db if need_b else None, ds if need_r else None, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               dim: int = -1, residual: Optional[torch.Tensor] = None):
    """(x - mean) / sqrt(var + eps) * weight + bias over axis `dim` (biased variance), differentiable in every tensor (reverse
    mode; dual tensors of forward mode are refused).

    x: fp32, fp16 or bf16, any shape; weight / bias (C,) of x's type or fp32, of one type, either may be None.  residual: x's
    shape and type; then s = x + residual (rounded to x's type) is what is normalised, and (y, s) is returned -- gradients
    that reach s join in the backward pass.  Statistics and sums are fp32.  Rows of any width and any number of channels
    (to 2^30; gradients of weight and bias below 2^26);
    leading axes may be strided.  A NaN or infinity stays in its own row."""
    if not isinstance(x, torch.Tensor) or x.dim() == 0:
        raise ValueError("layer_norm: x must be a tensor with at least one axis")
    if x.dtype not in TYPES:
        raise ValueError(f"layer_norm: x must be float32, float16 or bfloat16, got {x.dtype}")
    if not -x.dim() <= dim < x.dim():
        raise ValueError(f"layer_norm: axis {dim} of a tensor with {x.dim()} axes")
    dim %= x.dim()
    C = x.shape[dim]
    if C == 0:
        raise ValueError("layer_norm: the normalised axis is empty")
    if C > 1 << 30:
        raise ValueError(f"layer_norm: at most 2^30 values in a slice, got {C}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != (C,) or t.dtype not in (x.dtype, torch.float32) or t.device != x.device:
            raise ValueError(f"layer_norm: {name} must be ({C},) of type {x.dtype} or float32 on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("layer_norm: weight and bias must share one type")
    if C >= 1 << 26 and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (weight, bias)):
        raise ValueError(f"layer_norm: gradients of weight and bias below 2^26 channels, got {C}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("layer_norm: residual must have x's shape, type and device")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    _need_gpu(x, weight, bias, residual)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    if _differentiated(x, weight, bias, residual):
        return _LayerNorm.apply(x, weight, bias, residual, float(eps), dim)
    y, s, _, _ = stage_layer_norm_fwd(x, weight, bias, eps, dim, residual, stats=False)
    return y if residual is None else (y, s)


class LayerNorm(nn.Module):
    """`layer_norm` with learned weight and bias (C,) (state_dict keys and initial values of nn.LayerNorm(C)); `dim`: the
    normalised axis, 1 for (B, C, N) tensors.  forward(x, residual=None) -> y, or (y, x + residual)."""

    def __init__(self, channels: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, dim: int = -1,
                 device=None, dtype=None):
        super().__init__()
        if channels < 1:
            raise ValueError("LayerNorm: channels must be positive")
        self.channels, self.eps, self.dim = channels, eps, dim
        kw = dict(device=device, dtype=dtype)
        self.weight = nn.Parameter(torch.ones(channels, **kw)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(channels, **kw)) if elementwise_affine and bias else None

    def forward(self, x, residual=None):
        return layer_norm(x, self.weight, self.bias, self.eps, self.dim, residual)

    def extra_repr(self):
        return f"{self.channels}, eps={self.eps}, dim={self.dim}, affine={self.weight is not None}"
