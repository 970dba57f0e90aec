"""Operators of the block around the scan: group norm, dropout and dense layers.

They cover what a BidirectionalMamba block computes outside its scans
(src/selectssm/selectssm.py:306-362) with norm_type "group", the output
projection and the MLP with its dropout:

* :func:`group_norm_act`  activation(group norm of channels-last x)
* :func:`dropout_act`     residual + activation(dropout(x))
* :func:`dense_act`       residual + activation(dropout(x @ kernel + bias))

Each is differentiable once.  PyTorch holds the memory, the stream and the
autograd graph; the arithmetic runs in the kernels of ``libselectssm_b200.so``.

Dropout takes its random bits from ``rng = (seed, offset)``, two integers or an
int64 CUDA tensor of the two (which a captured CUDA graph reads afresh at every
replay).  The mask is a function of them and of an element's row and column
only, so it is never stored, and the same ``rng`` gives the same mask in every
operator over the same (rows, columns).  A step that needs another mask takes
another offset.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _dense, _dtype_code, _ptr, _require_cuda, ctypes_byref

__all__ = ["group_norm_act", "dropout_act", "dense_act"]

_U64 = (1 << 64) - 1


def _act_code(activation):
    try:
        return _lib.ACT_CODES[activation]
    except KeyError:
        raise ValueError(f"unknown activation {activation!r}; one of silu, gelu, relu or None") from None


def _drop_of(rate):
    """Dropped values of 65536, the resolution of the kernels' 16-bit draws."""
    if not 0.0 <= rate <= 1.0:
        raise ValueError(f"dropout rate must be in [0, 1], got {rate}")
    return round(rate * 65536)


def _rng_of(rng, drop, device):
    """(seed, offset, device tensor or None)."""
    if drop == 0:
        return 0, 0, None
    if rng is None:
        raise ValueError("dropout needs rng = (seed, offset)")
    if torch.is_tensor(rng):
        if rng.dtype != torch.int64 or rng.shape != (2,) or rng.device != device:
            raise ValueError(f"rng must be an int64 tensor of two values on {device}, got {rng.dtype} "
                             f"{tuple(rng.shape)} on {rng.device}")
        return 0, 0, rng.contiguous()
    seed, offset = rng
    return int(seed) & _U64, int(offset) & _U64, None


def _same_device(x, **others):
    _require_cuda(x, *others.values())
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")


def _matrix(t):
    """(2-D view with unit stride along the last axis, row stride); copies only
    when the leading axes do not collapse to one stride."""
    cols = t.shape[-1]
    rows = t.numel() // cols if cols else 0
    if t.numel() == 0 or t.is_contiguous():
        return t.reshape(rows, cols), cols
    if t.stride(-1) == 1 or cols == 1:
        # axes of one element have no stride of their own
        lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1]
        if all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:])):
            step = lead[-1][1] if lead else cols
            if step >= cols:
                return t.as_strided((rows, cols), (step, 1)), step
    return t.reshape(rows, cols).contiguous(), cols


def _stream_of(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _workspace(nbytes, device):
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


def _residual_of(residual, shape, dtype):
    if residual is None:
        return None
    if residual.shape != shape:
        try:
            residual = residual.expand(shape)  # autograd sums a broadcast residual's gradient
        except RuntimeError:
            raise ValueError(f"residual {tuple(residual.shape)} does not broadcast to {tuple(shape)}") from None
    return residual.to(dtype)


# ----------------------------------------------------------------------------- dropout
class _DropoutActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, drop, rng, act):
        seed, offset, rng_t = rng
        x2, xs = _matrix(x)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        p = _drop_params(x2, drop, seed, offset, rng_t, act)
        p.x, p.x_stride, p.y = x2.data_ptr(), xs, y.data_ptr()
        if residual is not None:
            r2, p.res_stride = _matrix(residual)
            p.residual = r2.data_ptr()
        if x.numel():
            _lib.check(_lib.load().ssm_dropout_act_fwd(ctypes_byref(p), _stream_of(x)), "ssm_dropout_act_fwd")
        ctx.save_for_backward(x2 if act else None, rng_t)
        ctx.cfg = (x.shape, x.dtype, drop, seed, offset, act, xs)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, rng_t = ctx.saved_tensors
        shape, dtype, drop, seed, offset, act, xs = ctx.cfg
        dx = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty(shape, dtype=dtype, device=dy.device)
            if dx.numel():
                d2, ds = _matrix(dy.to(dtype))
                p = _drop_params(d2, drop, seed, offset, rng_t, act)
                p.x, p.x_stride = _ptr(x2), xs
                p.dy, p.dy_stride, p.dx = d2.data_ptr(), ds, dx.data_ptr()
                _lib.check(_lib.load().ssm_dropout_act_bwd(ctypes_byref(p), _stream_of(dy)), "ssm_dropout_act_bwd")
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def _drop_params(x2, drop, seed, offset, rng_t, act):
    p = _lib.SSMDropoutParams()
    p.rows, p.dim = x2.shape
    p.dtype, p.act, p.drop = _dtype_code(x2), act, drop
    p.seed, p.offset, p.rng = seed, offset, _ptr(rng_t)
    return p


def dropout_act(x, rate, rng, activation=None, residual=None):
    """residual + activation(dropout(x)) over the last axis of x.

    x: (..., dim), float32 or bfloat16, rows at any stride.  ``rate`` in [0, 1]
    is taken to the nearest 65536th, kept values are divided by the keep
    probability that leaves.  ``residual`` broadcasts to x."""
    _same_device(x, residual=residual)
    _dtype_code(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last axis of at least one element, got {tuple(x.shape)}")
    act, drop = _act_code(activation), _drop_of(rate)
    rng = _rng_of(rng, drop, x.device)
    return _DropoutActFn.apply(x, _residual_of(residual, x.shape, x.dtype), drop, rng, act)


# ----------------------------------------------------------------------------- group norm
class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, groups, eps, act):
        x3 = _dense(x).view(x.shape[0], -1, x.shape[-1]) if x.numel() else x.reshape(x.shape[0], 0, x.shape[-1])
        scale32 = None if scale is None else _dense(scale.float())
        bias32 = None if bias is None else _dense(bias.float())
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((x.shape[0], groups, 2), dtype=torch.float32, device=x.device)
        p = _gn_params(x3, scale32, bias32, stats, groups, eps, act)
        p.y = y.data_ptr()
        lib = _lib.load()
        if x.numel():
            ws = _workspace(lib.ssm_group_norm_fwd_workspace_bytes(ctypes_byref(p)), x.device)
            p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
            _lib.check(lib.ssm_group_norm_act_fwd(ctypes_byref(p), _stream_of(x)), "ssm_group_norm_act_fwd")
        ctx.save_for_backward(x3, scale32, bias32, stats)
        ctx.cfg = (x.shape, groups, eps, act)
        ctx.dtypes = (None if scale is None else scale.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x3, scale32, bias32, stats = ctx.saved_tensors
        shape, groups, eps, act = ctx.cfg
        dim = x3.shape[2]
        dy = _dense(dy.to(x3.dtype))
        dx = torch.empty(shape, dtype=x3.dtype, device=x3.device)
        dscale, dbias = (torch.empty(dim, dtype=torch.float32, device=x3.device) for _ in range(2))
        p = _gn_params(x3, scale32, bias32, stats, groups, eps, act)
        p.dy, p.dx, p.dscale, p.dbias = dy.data_ptr(), dx.data_ptr(), dscale.data_ptr(), dbias.data_ptr()
        lib = _lib.load()
        ws = _workspace(lib.ssm_group_norm_bwd_workspace_bytes(ctypes_byref(p)), x3.device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(lib.ssm_group_norm_act_bwd(ctypes_byref(p), _stream_of(x3)), "ssm_group_norm_act_bwd")
        del ws
        sdt, bdt = ctx.dtypes
        return (dx, None if sdt is None else dscale.to(sdt), None if bdt is None else dbias.to(bdt), None, None, None)


def _gn_params(x3, scale32, bias32, stats, groups, eps, act):
    p = _lib.SSMGroupNormParams()
    p.batch, p.seqlen, p.dim = x3.shape
    p.groups, p.dtype, p.act, p.eps = groups, _dtype_code(x3), act, eps
    p.x, p.scale, p.bias, p.stats = x3.data_ptr(), _ptr(scale32), _ptr(bias32), stats.data_ptr()
    return p


def group_norm_act(x, scale=None, bias=None, groups=32, eps=1e-6, activation=None):
    """activation(flax.linen.GroupNorm(x)), channels last (selectssm.py:306-313).

    x: (batch, ..., dim), float32 or bfloat16.  Each batch row's mean and
    variance are taken over all middle axes and the dim / groups channels of a
    group.  ``scale`` and ``bias``: (dim,) or None for ones and zeros."""
    _same_device(x, scale=scale, bias=bias)
    _dtype_code(x)
    if x.dim() < 2 or x.shape[-1] < 1:
        raise ValueError(f"x must be (batch, ..., dim), got {tuple(x.shape)}")
    dim = x.shape[-1]
    if groups < 1 or dim % groups:
        raise ValueError(f"groups={groups} must divide dim={dim}")
    for name, t in (("scale", scale), ("bias", bias)):
        if t is not None and t.shape != (dim,):
            raise ValueError(f"{name} must be ({dim},), got {tuple(t.shape)}")
    return _GroupNormActFn.apply(x, scale, bias, int(groups), float(eps), _act_code(activation))


# ----------------------------------------------------------------------------- dense layer
class _DenseActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias, residual, act, drop, rng, grad):
        seed, offset, rng_t = rng
        x2, xs = _matrix(x)
        w = _dense(kernel.to(x.dtype))
        b = None if bias is None else _dense(bias)
        out_shape = (*x.shape[:-1], kernel.shape[1])
        y = torch.empty(out_shape, dtype=x.dtype, device=x.device)
        pre = torch.empty((x2.shape[0], kernel.shape[1]), dtype=x.dtype, device=x.device) if grad and act else None
        p = _dense_params(x2, xs, w, b, drop, seed, offset, rng_t, act)
        p.y, p.pre = y.data_ptr(), _ptr(pre)
        if residual is not None:
            r2, p.res_stride = _matrix(residual)
            p.residual = r2.data_ptr()
        lib = _lib.load()
        if y.numel():
            ws = _workspace(lib.ssm_dense_fwd_workspace_bytes(ctypes_byref(p)), x.device)
            p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
            _lib.check(lib.ssm_dense_act_fwd(ctypes_byref(p), _stream_of(x)), "ssm_dense_act_fwd")
        if grad:
            ctx.save_for_backward(x2, w, b, pre, rng_t)
        ctx.cfg = (x.shape, xs, drop, seed, offset, act, kernel.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dres = dy if ctx.needs_input_grad[3] else None
        if not any(ctx.needs_input_grad[:3]):
            return None, None, None, dres, None, None, None, None
        x2, w, b, pre, rng_t = ctx.saved_tensors
        shape, xs, drop, seed, offset, act, kdtype = ctx.cfg
        d2, ds = _matrix(dy.to(x2.dtype))
        p = _dense_params(x2, xs, w, b, drop, seed, offset, rng_t, act)
        p.pre, p.dy, p.dy_stride = _ptr(pre), d2.data_ptr(), ds
        p.dkernel_dtype = _lib.SSM_BF16 if kdtype == torch.bfloat16 else _lib.SSM_F32
        dx = torch.empty(shape, dtype=x2.dtype, device=x2.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(w.shape, dtype=kdtype, device=x2.device) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(b) if ctx.needs_input_grad[2] else None
        p.dx, p.dkernel, p.dbias = _ptr(dx), _ptr(dw), _ptr(db)
        lib = _lib.load()
        ws = _workspace(lib.ssm_dense_bwd_workspace_bytes(ctypes_byref(p)), x2.device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(lib.ssm_dense_act_bwd(ctypes_byref(p), _stream_of(x2)), "ssm_dense_act_bwd")
        del ws
        return dx, dw, db, dres, None, None, None, None


def _dense_params(x2, xs, w, b, drop, seed, offset, rng_t, act):
    p = _lib.SSMDenseParams()
    p.rows, p.fin = x2.shape
    p.fout = w.shape[1]
    p.dtype, p.act, p.drop = _dtype_code(x2), act, drop
    p.bias_dtype = p.dkernel_dtype = p.dtype if b is None else _dtype_code(b)
    p.seed, p.offset, p.rng = seed, offset, _ptr(rng_t)
    p.x, p.x_stride, p.kernel, p.bias = x2.data_ptr(), xs, w.data_ptr(), _ptr(b)
    return p


def dense_act(x, kernel, bias=None, activation=None, residual=None, rate=0.0, rng=None):
    """residual + activation(dropout(x @ kernel + bias)) (selectssm.py:345-362).

    x: (..., fin), float32 or bfloat16, rows at any stride; kernel: Flax's
    (fin, fout), converted to x's type; bias: (fout,); ``residual`` broadcasts
    to the (..., fout) output.  Products are summed in fp32; float32 operands
    keep fp32 accuracy.  ``rate`` and ``rng`` as in :func:`dropout_act`, over
    rows of fout columns.  For the backward an activation's input is kept in
    x's type."""
    _same_device(x, kernel=kernel, bias=bias, residual=residual)
    _dtype_code(x), _dtype_code(kernel)
    if kernel.dim() != 2 or x.dim() < 1 or x.shape[-1] != kernel.shape[0] or min(kernel.shape) < 1:
        raise ValueError(f"x {tuple(x.shape)} and kernel {tuple(kernel.shape)} do not match (..., fin) @ (fin, fout)")
    fout = kernel.shape[1]
    if bias is not None:
        _dtype_code(bias)
        if bias.shape != (fout,):
            raise ValueError(f"bias must be ({fout},), got {tuple(bias.shape)}")
    act, drop = _act_code(activation), _drop_of(rate)
    rng = _rng_of(rng, drop, x.device)
    residual = _residual_of(residual, (*x.shape[:-1], fout), x.dtype)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, kernel, bias))
    return _DenseActFn.apply(x, kernel, bias, residual, act, drop, rng, grad)
