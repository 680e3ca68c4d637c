"""Layer norm and its gradient on the MI355X, with the residual addition in front of it.

``layer_norm(x, weight, bias)`` normalises the last dimension as
``torch.nn.functional.layer_norm`` does; with ``residual`` it first forms ``x + residual``, the
stream that a pre-LN block hands on (model/transformer.py:54-57 of mini-megatron), and
returns both, in one pass over memory.  ``out_dtype`` lets an fp32 stream reach the bf16 linears
without a cast of its own.  ``LayerNorm`` is the module, a ``torch.nn.LayerNorm`` with the same
parameters and state_dict.  Weight gradients are summed over tokens in an order that depends on
the sizes alone, so training runs repeat bit for bit.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _as_rows(t: torch.Tensor, hidden: int) -> torch.Tensor:
    """t as [rows, hidden] with dense rows; a view where its strides allow."""
    t = t.reshape(t.numel() // max(hidden, 1), hidden)
    return t if hidden == 1 or t.stride(1) == 1 else t.contiguous()


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _call(fn, args, device: torch.device, what: str) -> None:
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            _lib.check(fn(ctypes.addressof(args), torch._C._cuda_getCurrentRawStream(index)),
                       what)
        return
    _lib.check(fn(ctypes.addressof(args), torch._C._cuda_getCurrentRawStream(index)), what)


def _forward(x, residual, weight, bias, eps, out_dtype, stats: bool):
    """(y, sum or None, x as rows, mean, rstd)"""
    hidden = x.shape[-1]
    x2 = _as_rows(x, hidden)
    rows = x2.shape[0]
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    mean = rstd = r2 = total = None
    if residual is not None:
        r2 = _as_rows(residual, hidden)
        total = torch.empty(x.shape, dtype=torch.promote_types(x.dtype, residual.dtype),
                            device=x.device)
    if stats:
        mean, rstd = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    if x.numel():
        args = _lib.LayerNormArgs(
            x2.data_ptr(), _ptr(r2), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(total),
            _ptr(mean), _ptr(rstd), rows, hidden, x2.stride(0),
            0 if r2 is None else r2.stride(0), eps, _DTYPES[x.dtype],
            0 if r2 is None else _DTYPES[r2.dtype], _DTYPES[out_dtype])
        _call(_lib.load().mi_adamw_layer_norm, args, x.device, "mi_adamw_layer_norm")
    return y, total, x2, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, out_dtype):
        y, total, rows, mean, rstd = _forward(x, residual, weight, bias, eps, out_dtype, True)
        ctx.set_materialize_grads(False)
        # the sum as the output that it is: a view of it would keep it, and with it this node
        ctx.save_for_backward(rows if total is None else total, weight, mean, rstd)
        ctx.shape, ctx.x_dtype = x.shape, x.dtype
        ctx.residual_dtype = None if residual is None else residual.dtype
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        normalised, weight, mean, rstd = ctx.saved_tensors
        need_x, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        if dy is None and dsum is None:
            return (None,) * 6
        hidden = normalised.shape[-1]
        # a saved-tensor hook may give them back at other strides
        rows = _as_rows(normalised, hidden)
        weight, mean, rstd = (t if t is None else t.contiguous() for t in (weight, mean, rstd))
        n = rows.shape[0]
        device = rows.device
        if dy is None:
            dy = torch.zeros(ctx.shape, dtype=torch.float32, device=device)
        dy2 = _as_rows(dy, hidden)
        ds2 = None if dsum is None else _as_rows(dsum, hidden)
        dx = dr = dw = db = partials = None
        types = [t for t, need in ((ctx.x_dtype, need_x), (ctx.residual_dtype, need_r)) if need]
        if types:
            dx = torch.empty(ctx.shape, dtype=types[0], device=device)
            if types[-1] != types[0]:
                dr = torch.empty(ctx.shape, dtype=types[-1], device=device)
        if need_w:
            dw = torch.empty(hidden, dtype=torch.float32, device=device)
        if need_b:
            db = torch.empty(hidden, dtype=torch.float32, device=device)
        if not rows.numel():
            dw, db = (None if t is None else t.zero_() for t in (dw, db))
        elif dx is not None or dw is not None or db is not None:
            lib = _lib.load()
            if dw is not None or db is not None:
                partials = torch.empty(lib.mi_adamw_layer_norm_grad_workspace(n, hidden),
                                       dtype=torch.uint8, device=device)
            args = _lib.LayerNormGradArgs(
                rows.data_ptr(), dy2.data_ptr(), _ptr(ds2), _ptr(weight), mean.data_ptr(),
                rstd.data_ptr(), _ptr(dx), _ptr(dr), _ptr(dw), _ptr(db), _ptr(partials), n,
                hidden, rows.stride(0), dy2.stride(0), 0 if ds2 is None else ds2.stride(0),
                _DTYPES[rows.dtype], _DTYPES[dy2.dtype], 0 if dx is None else _DTYPES[dx.dtype],
                0 if dr is None else _DTYPES[dr.dtype])
            _call(lib.mi_adamw_layer_norm_grad, args, device, "mi_adamw_layer_norm_grad")
        # one tensor serves both addends where their types agree, as an addition's backward gives
        return (dx if need_x else None, (dr if dr is not None else dx) if need_r else None, dw, db,
                None, None)


def refuse_records(what: str, *tensors) -> None:
    """What is lost without a word otherwise: a forward-mode tangent, which the kernels do not
    compute, and the launches in a trace, which would record the outputs' allocation alone."""
    if torch.jit.is_tracing():
        raise NotImplementedError(f"{what} cannot be recorded by torch.jit.trace")
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def _check(x, weight, bias, eps, residual, out_dtype) -> None:
    if x.dim() == 0:
        raise RuntimeError("layer_norm needs at least one dimension to normalise")
    if x.device.type != "cuda":
        raise RuntimeError(f"mi_adamw.layer_norm runs on a ROCm GPU only; got a {x.device.type} "
                           "tensor")
    for name, t in (("x", x), ("residual", residual)):
        if t is not None and t.dtype not in _DTYPES:
            raise NotImplementedError(f"layer_norm: {name} of {t.dtype} is not supported (fp32 and "
                                      "bf16 are)")
    if out_dtype not in _DTYPES:
        raise NotImplementedError(f"layer_norm: out_dtype {out_dtype} is not supported (fp32 and "
                                  "bf16 are)")
    if residual is not None and (residual.shape != x.shape or residual.device != x.device):
        raise ValueError("layer_norm: residual needs x's shape and device")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != x.shape[-1:] or t.device != x.device:
            raise ValueError(f"layer_norm: {name} needs the shape of x's last dimension "
                             f"({x.shape[-1]}) and x's device, got {tuple(t.shape)}")
        if t.dtype != torch.float32:
            raise NotImplementedError(f"layer_norm: {name} of {t.dtype} is not supported (fp32 "
                                      "master parameters only)")
    if not (0 <= eps <= _lib.FP32_MAX):
        raise ValueError(f"layer_norm: eps should be >= 0 and finite in fp32 but is: {eps}")
    if x.shape[-1] > 1 << 24 or (x.numel() and x.numel() // x.shape[-1] >= 1 << 23):
        raise NotImplementedError("layer_norm: at most 2^23 - 1 rows of 2^24 values")
    refuse_records("mi_adamw.layer_norm", x, weight, bias, residual)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, *, residual: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None):
    """Layer norm over x's last dimension: ``y``, or ``(y, x + residual)`` with a residual.

    x, residual: fp32 or bf16 on a ROCm GPU, any leading shape; rows dense at any stride
                 (other layouts are copied first).  The sum has their promoted type, and what
                 is normalised is the sum as it is returned.
    weight, bias: fp32 [hidden], or None.
    out_dtype:   y's type; by default x's, or fp32 inside an autocast region, as torch's.
    """
    if _lib._host is not None:
        out = _lib._host.layer_norm(x, weight, bias, eps, residual, out_dtype)
        if out is not None:
            return out
    if out_dtype is None:
        out_dtype = torch.float32 if torch.is_autocast_enabled("cuda") else x.dtype
    _check(x, weight, bias, eps, residual, out_dtype)
    _lib.load()
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, residual, weight, bias)):
        return _LayerNorm.apply(x, residual, weight, bias, eps, out_dtype)
    y, total, _, _, _ = _forward(x, residual, weight, bias, eps, out_dtype, False)
    return y if residual is None else (y, total)


class LayerNorm(torch.nn.LayerNorm):
    """torch.nn.LayerNorm (its constructor, parameters and state_dict) on ``layer_norm``.
    ``forward(x, residual=None)``; out_dtype as there."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None, *,
                 out_dtype: torch.dtype | None = None) -> None:
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        self.out_dtype = out_dtype

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        dims = len(self.normalized_shape)
        if tuple(x.shape[-dims:]) != tuple(self.normalized_shape):
            raise RuntimeError(f"Given normalized_shape={list(self.normalized_shape)}, expected "
                               f"input with shape [*, {', '.join(map(str, self.normalized_shape))}]"
                               f", but got input of size{list(x.shape)}")
        if dims == 1:
            return layer_norm(x, self.weight, self.bias, self.eps, residual=residual,
                              out_dtype=self.out_dtype)
        lead = x.shape[:-dims]

        def flat(t, shape):
            return None if t is None else t.reshape(shape)

        hidden = math.prod(self.normalized_shape)
        out = layer_norm(x.reshape(*lead, hidden), flat(self.weight, (hidden,)),
                         flat(self.bias, (hidden,)), self.eps,
                         residual=flat(residual, (*lead, hidden)), out_dtype=self.out_dtype)
        return out.view(x.shape) if residual is None else tuple(t.view(x.shape) for t in out)
