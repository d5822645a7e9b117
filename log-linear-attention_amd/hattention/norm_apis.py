"""Layer norm with the residual stream's addition (MI355X).

The norm of a hybrid stack's residual stream, next to the gated RMSNorm that closes
the Mamba-2 layer (``mamba_layer.GatedRMSNorm``).  One launch forward, two backward
(libhattn_hip.so: ``hattn_layer_norm_fwd`` / ``hattn_layer_norm_bwd``).  No counterpart
in the reference.
"""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from hattention import _lib

MAX_N = 16384


def _forward(x, residual, weight, bias, eps, keep):
    """(y, s or x, mean, rstd); the statistics where ``keep``."""
    dev = _lib.require_device(x, residual, weight, bias)
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    n = x.shape[-1]
    rows = x.numel() // n
    y = torch.empty_like(x)
    s = torch.empty_like(residual) if residual is not None else None
    stat = torch.empty(2, rows, dtype=torch.float32, device=dev) if keep else None
    if rows:
        param = weight if weight is not None else bias
        _lib.launch(dev, _lib.load().hattn_layer_norm_fwd, x.data_ptr(), _lib.ptr(residual),
                    _lib.ptr(weight), _lib.ptr(bias), y.data_ptr(), _lib.ptr(s), _lib.ptr(stat),
                    stat[1].data_ptr() if keep else 0, rows, n, eps, _lib.dtype_code(x),
                    _lib.dtype_code(residual) if residual is not None else 2,
                    _lib.dtype_code(param) if param is not None else 2)
    return y, s if s is not None else x, stat


class LayerNormFunction(torch.autograd.Function):
    """(y, s) of :func:`layer_norm`; s is None without a residual."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        ctx.set_materialize_grads(False)
        y, s, stat = _forward(x, residual, weight, bias, eps, True)
        ctx.save_for_backward(s, weight, stat)
        ctx.has_residual = residual is not None
        ctx.x_dtype = x.dtype
        ctx.bias_dtype = bias.dtype if bias is not None else None
        return y, s if residual is not None else None

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        s, weight, stat = ctx.saved_tensors
        need_x, need_r, need_w, need_b, _ = ctx.needs_input_grad
        if dy is None:  # only the sum was used
            if ds is None:
                return None, None, None, None, None
            return (ds.to(ctx.x_dtype) if need_x else None, ds if need_r else None,
                    None, None, None)
        dy = dy.contiguous()
        ds = ds.contiguous() if ds is not None else None
        n = s.shape[-1]
        rows = s.numel() // n
        dev = s.device
        # x and the residual have the same gradient: one tensor where they have one dtype
        same = ctx.x_dtype == s.dtype
        dx = torch.empty(s.shape, dtype=ctx.x_dtype, device=dev) \
            if need_x or (need_r and same) else None
        dres = torch.empty_like(s) if need_r and not same else None
        dw = torch.empty(n, dtype=weight.dtype, device=dev) if need_w else None
        db = torch.empty(n, dtype=ctx.bias_dtype, device=dev) if need_b else None
        if rows:
            lib = _lib.load()
            ws, ws_ptr, ws_bytes = _lib.workspace(
                lib.hattn_layer_norm_bwd_workspace(rows, n) if need_w or need_b else 0, dev)
            param = weight if weight is not None else db
            _lib.launch(dev, lib.hattn_layer_norm_bwd, s.data_ptr(), _lib.ptr(weight),
                        stat.data_ptr(), stat[1].data_ptr(), dy.data_ptr(), _lib.ptr(ds),
                        _lib.ptr(dx), _lib.ptr(dres), _lib.ptr(dw), _lib.ptr(db), rows, n,
                        _lib.DTYPE_CODES[ctx.x_dtype], _lib.dtype_code(s),
                        _lib.dtype_code(param) if param is not None else 2, ws_ptr, ws_bytes)
        else:
            dw = dw.zero_() if dw is not None else None
            db = db.zero_() if db is not None else None
        return (dx if need_x else None, (dx if same else dres) if need_r else None, dw, db, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
               eps: float = 1e-5):
    """Layer norm over the last dimension, ``y = (s - mean) rstd weight + bias``.

    x [..., n] (bf16, fp16 or fp32; n <= 16384); weight, bias [n], of one dtype; ``s`` is x,
    or with ``residual`` (x's shape; x's dtype or fp32) the sum ``x + residual`` rounded to
    the residual's dtype.  Returns y in x's dtype, or with a residual ``(y, s)``: s goes on
    as the residual stream.  The sums over a row and over the rows are held in fp32;
    dweight and dbias are summed in a fixed order.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension")
    n = x.shape[-1]
    if n > MAX_N:
        raise NotImplementedError(f"n={n} above {MAX_N}")
    _lib.dtype_code(x)
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            if p.shape != (n,):
                raise ValueError(f"{name} must be [{n}]")
            _lib.dtype_code(p)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one dtype")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError("residual must have x's shape")
        if residual.dtype not in (x.dtype, torch.float32):
            raise NotImplementedError(f"residual in {residual.dtype} with x in {x.dtype}")
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    if torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, residual, weight, bias)):
        y, s = LayerNormFunction.apply(x, residual, weight, bias, eps)
    else:
        y, s, _ = _forward(x, residual, weight, bias, eps, False)
    return (y, s) if residual is not None else y
