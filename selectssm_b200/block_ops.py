"""Operators of the block around the scan: group norm, dropout and dense layers.

They cover what a BidirectionalMamba block computes outside its scans
(src/selectssm/selectssm.py:306-362) with norm_type "group", the output
projection and the MLP with its dropout:

* :func:`group_norm_act`  activation(group norm of channels-last x)
* :func:`dropout_act`     residual + activation(dropout(x))
* :func:`dense_act`       residual + activation(dropout(x @ kernel + bias))

Each is differentiable once, in reverse mode; forward-mode tangents are refused
with autograd's NotImplementedError.  PyTorch holds the memory, the stream and the
autograd graph; the arithmetic runs in the kernels of ``libselectssm_b200.so``.

Dropout takes its random bits from ``rng = (seed, offset)``, two integers or an
int64 CUDA tensor of the two (which a captured CUDA graph reads afresh at every
replay).  The mask is a function of them and of an element's row and column
only, so it is never stored, and the same ``rng`` gives the same mask in every
operator over the same (rows, columns).  A step that needs another mask takes
another offset.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DT, _dense, _dtype_code, _ptr, _require_cuda, ctypes_byref

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


def _check_devices(x, *others):
    _require_cuda(x, *others)
    device = x.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"operands on {t.device} and {device}")


def _rows_of(t):
    """(t, row stride) as rows of the last axis with unit stride in it; copies
    only when the leading axes do not collapse to one stride."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, cols
    if t.stride(-1) == 1 or cols == 1:
        # axes of one element have no stride of their own
        lead = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1]
        if all(a[1] == b[0] * b[1] for a, b in zip(lead, lead[1:])):
            step = lead[-1][1] if lead else cols
            if step >= cols:
                return t, step
    return t.contiguous(), cols


def _stream_of(t):
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _workspace(nbytes, t):
    return t.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _residual_of(residual, shape, dtype):
    if residual.shape != shape:
        try:
            residual = residual.expand(shape)  # autograd sums a broadcast residual's gradient
        except RuntimeError:
            raise ValueError(f"residual {tuple(residual.shape)} does not broadcast to {tuple(shape)}") from None
    return residual.to(dtype)


def _records(*tensors):
    """Whether the call is autograd's business: it will ask for a gradient, or an
    operand carries a forward-mode tangent, which autograd refuses (a direct call
    would lose it)."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    # outside every dual level (the usual case) no operand is looked at
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


# Each operator has a plain function that makes the call and an autograd
# function around it; without a gradient to record or a tangent to refuse the
# former is called directly, which halves the host's time for a single token.

# ----------------------------------------------------------------------------- dropout
def _dropout_forward(x, residual, drop, rng, act):
    y = x.new_empty(x.shape)
    if not x.numel():
        return y
    x, xs = _rows_of(x)
    res, rs = (None, 0) if residual is None else _rows_of(residual)
    dim = x.shape[-1]
    p = _lib.SSMDropoutParams(x.numel() // dim, dim, _DT[x.dtype], act, drop, rng[0], rng[1], _ptr(rng[2]), xs, rs, 0,
                              x.data_ptr(), _ptr(res), y.data_ptr())
    _lib.check(_lib.load().ssm_dropout_act_fwd(ctypes_byref(p), _stream_of(x)), "ssm_dropout_act_fwd")
    return y


class _DropoutActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, drop, rng, act):
        ctx.save_for_backward(x if act else None, rng[2])
        ctx.cfg = (drop, rng[:2], act)
        return _dropout_forward(x, residual, drop, rng, act)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, rng_t = ctx.saved_tensors
        drop, rng, act = ctx.cfg
        dx = None
        if ctx.needs_input_grad[0]:
            dx = dy.new_empty(dy.shape)
            if dx.numel():
                d, ds = _rows_of(dy)
                x, xs = _rows_of(x) if act else (None, 0)
                dim = dy.shape[-1]
                p = _lib.SSMDropoutParams(dy.numel() // dim, dim, _DT[dy.dtype], act, drop, *rng, _ptr(rng_t), xs, 0, ds,
                                          _ptr(x), None, None, d.data_ptr(), dx.data_ptr())
                _lib.check(_lib.load().ssm_dropout_act_bwd(ctypes_byref(p), _stream_of(dy)), "ssm_dropout_act_bwd")
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout_act(x, rate, rng, activation=None, residual=None):
    """residual + activation(dropout(x)) over the last axis of x.

    x: (..., dim), float32 or bfloat16, rows at any stride.  ``rate`` in [0, 1]
    is taken to the nearest 65536th, kept values are divided by the keep
    probability that leaves.  ``residual`` broadcasts to x and is converted to x's
    type, in which the sum is returned."""
    _check_devices(x, residual)
    _dtype_code(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last axis of at least one element, got {tuple(x.shape)}")
    act, drop = _act_code(activation), _drop_of(rate)
    rng = _rng_of(rng, drop, x.device)
    if residual is not None:
        residual = _residual_of(residual, x.shape, x.dtype)
    if _records(x, residual):
        return _DropoutActFn.apply(x, residual, drop, rng, act)
    return _dropout_forward(x, residual, drop, rng, act)


# ----------------------------------------------------------------------------- group norm
def _gn_params(x, scale, bias, y, stats, groups, eps, act):
    batch, dim = x.shape[0], x.shape[-1]
    seqlen = x.numel() // (batch * dim) if batch else 0
    return _lib.SSMGroupNormParams(batch, seqlen, dim, groups, _DT[x.dtype], act, eps, x.data_ptr(), _ptr(scale),
                                   _ptr(bias), _ptr(y), _ptr(stats))


def _group_norm_forward(x, scale, bias, groups, eps, act, keep_stats):
    """y and, with keep_stats, the statistics; x, scale and bias are dense, the latter float32."""
    y = x.new_empty(x.shape)
    stats = x.new_empty((x.shape[0], groups, 2), dtype=torch.float32) if keep_stats else None
    if x.numel():
        p = _gn_params(x, scale, bias, y, stats, groups, eps, act)
        lib, ref = _lib.load(), ctypes_byref(p)
        ws = _workspace(lib.ssm_group_norm_fwd_workspace_bytes(ref), x)
        if ws is not None:
            p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(lib.ssm_group_norm_act_fwd(ref, _stream_of(x)), "ssm_group_norm_act_fwd")
    return y, stats


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale, bias, groups, eps, act):
        x = _dense(x)
        y, stats = _group_norm_forward(x, scale, bias, groups, eps, act, True)
        ctx.save_for_backward(x, scale, bias, stats)
        ctx.cfg = (groups, eps, act)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, scale, bias, stats = ctx.saved_tensors
        groups, eps, act = ctx.cfg
        dim = x.shape[-1]
        dy = _dense(dy)
        dx = x.new_empty(x.shape)
        sums = x.new_empty((2, dim), dtype=torch.float32)
        p = _gn_params(x, scale, bias, None, stats, groups, eps, act)
        p.dy, p.dx, p.dscale, p.dbias = dy.data_ptr(), dx.data_ptr(), sums.data_ptr(), sums.data_ptr() + 4 * dim
        lib, ref = _lib.load(), ctypes_byref(p)
        ws = _workspace(lib.ssm_group_norm_bwd_workspace_bytes(ref), x)
        if ws is not None:
            p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(lib.ssm_group_norm_act_bwd(ref, _stream_of(x)), "ssm_group_norm_act_bwd")
        return dx, None if scale is None else sums[0], None if bias is None else sums[1], None, None, None


def group_norm_act(x, scale=None, bias=None, groups=32, eps=1e-6, activation=None):
    """activation(flax.linen.GroupNorm(x)), channels last (selectssm.py:306-313).

    x: (batch, ..., dim), float32 or bfloat16.  Each batch row's mean and
    variance are taken over all middle axes and the dim / groups channels of a
    group.  ``scale`` and ``bias``: (dim,) or None for ones and zeros."""
    _check_devices(x, scale, bias)
    _dtype_code(x)
    if x.dim() < 2 or x.shape[-1] < 1:
        raise ValueError(f"x must be (batch, ..., dim), got {tuple(x.shape)}")
    dim = x.shape[-1]
    if groups < 1 or dim % groups:
        raise ValueError(f"groups={groups} must divide dim={dim}")
    for name, t in (("scale", scale), ("bias", bias)):
        if t is not None and t.shape != (dim,):
            raise ValueError(f"{name} must be ({dim},), got {tuple(t.shape)}")
    # converted outside, so that autograd returns the gradients in their types
    scale = scale if scale is None else scale.float().contiguous()
    bias = bias if bias is None else bias.float().contiguous()
    if _records(x, scale, bias):
        return _GroupNormActFn.apply(x, scale, bias, groups, eps, _act_code(activation))
    return _group_norm_forward(_dense(x), scale, bias, groups, eps, _act_code(activation), False)[0]


# ----------------------------------------------------------------------------- dense layer
_status = {}  # device index -> (pinned word, the same as a C integer)


def _status_word(index):
    """Address of the word in which the device's dense kernels say that a bounded
    wait gave up (the outputs that it held up are NaN).  It lies in host memory, so
    that asking for it waits for nothing: what an earlier call has left there by
    now is raised here."""
    word = _status.get(index)
    if word is None:
        t = torch.zeros(1, dtype=torch.int32, pin_memory=True)
        word = _status.setdefault(index, (t, ctypes.c_int32.from_address(t.data_ptr())))
    code = word[1].value
    if code:
        word[1].value = 0
        _lib.check(code, f"an earlier dense_act call on cuda:{index}")
    return word[0].data_ptr()


def _dense_params(x, xs, w, b, drop, rng, act):
    code = _DT[x.dtype]
    fin, fout = w.shape
    p = _lib.SSMDenseParams(x.numel() // fin, fin, fout, code, code if b is None else _DT[b.dtype], code, act, drop,
                            rng[0], rng[1], _ptr(rng[2]), xs, 0, 0, x.data_ptr(), w.data_ptr(), _ptr(b))
    p.status = _status_word(x.get_device())
    return p


def _dense_forward(x, w, bias, residual, act, drop, rng, keep_pre):
    """y and, with keep_pre, the activation's input; w and bias are dense, w of x's type."""
    shape = (*x.shape[:-1], w.shape[1])
    y = x.new_empty(shape)
    pre = x.new_empty(shape) if keep_pre else None
    if y.numel():
        x, xs = _rows_of(x)
        p = _dense_params(x, xs, w, bias, drop, rng, act)
        p.y = y.data_ptr()
        if keep_pre:
            p.pre = pre.data_ptr()
        if residual is not None:
            residual, p.res_stride = _rows_of(residual)
            p.residual = residual.data_ptr()
        lib, ref = _lib.load(), ctypes_byref(p)
        ws = _workspace(lib.ssm_dense_fwd_workspace_bytes(ref), x)
        if ws is not None:
            p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(lib.ssm_dense_act_fwd(ref, _stream_of(x)), "ssm_dense_act_fwd")
    return y, pre


class _DenseActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kernel, bias, residual, act, drop, rng):
        w = kernel.to(x.dtype).contiguous()
        need = any(ctx.needs_input_grad[:3])
        y, pre = _dense_forward(x, w, bias, residual, act, drop, rng, need and act != 0)
        if need:
            ctx.save_for_backward(x, w, bias, pre, rng[2])
        ctx.cfg = (drop, rng[:2], act, kernel.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dres = dy if ctx.needs_input_grad[3] else None
        if not any(ctx.needs_input_grad[:3]):
            return None, None, None, dres, None, None, None
        x, w, bias, pre, rng_t = ctx.saved_tensors
        drop, rng, act, kdtype = ctx.cfg
        d, ds = _rows_of(dy)
        xc, xs = _rows_of(x)
        p = _dense_params(xc, xs, w, bias, drop, (*rng, rng_t), act)
        p.pre, p.dy, p.dy_stride = _ptr(pre), d.data_ptr(), ds
        p.dkernel_dtype = _DT[kdtype]
        dx = x.new_empty(x.shape) if ctx.needs_input_grad[0] else None
        dw = w.new_empty(w.shape, dtype=kdtype) if ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        p.dx, p.dkernel, p.dbias = _ptr(dx), _ptr(dw), _ptr(db)
        lib, ref = _lib.load(), ctypes_byref(p)
        ws = _workspace(lib.ssm_dense_bwd_workspace_bytes(ref), x)
        if ws is not None:
            p.workspace, p.workspace_bytes = ws.data_ptr(), ws.numel()
        _lib.check(lib.ssm_dense_act_bwd(ref, _stream_of(x)), "ssm_dense_act_bwd")
        return dx, dw, db, dres, None, None, None


def dense_act(x, kernel, bias=None, activation=None, residual=None, rate=0.0, rng=None):
    """residual + activation(dropout(x @ kernel + bias)) (selectssm.py:345-362).

    x: (..., fin), float32 or bfloat16, rows at any stride; kernel: Flax's
    (fin, fout), converted to x's type; bias: (fout,); ``residual`` broadcasts
    to the (..., fout) output and is converted to x's type, in which the sum is
    returned.  Products are summed in fp32; float32 operands keep fp32 accuracy.
    ``rate`` and ``rng`` as in :func:`dropout_act`, over rows of fout columns.
    For the backward an activation's input is kept in x's type, and the gradient
    before the two products is rounded to it.

    The kernels' waits are bounded.  Should one give up, the outputs that it held
    up are NaN and the next dense call on the device raises SSMLibraryError."""
    _check_devices(x, kernel, bias, residual)
    _dtype_code(x), _dtype_code(kernel)
    if kernel.dim() != 2 or x.dim() < 1 or x.shape[-1] != kernel.shape[0] or min(kernel.shape) < 1:
        raise ValueError(f"x {tuple(x.shape)} and kernel {tuple(kernel.shape)} do not match (..., fin) @ (fin, fout)")
    fout = kernel.shape[1]
    if bias is not None:
        _dtype_code(bias)
        if bias.shape != (fout,):
            raise ValueError(f"bias must be ({fout},), got {tuple(bias.shape)}")
        bias = bias if bias.is_contiguous() else bias.contiguous()
    act, drop = _act_code(activation), _drop_of(rate)
    rng = _rng_of(rng, drop, x.device)
    if residual is not None:
        residual = _residual_of(residual, (*x.shape[:-1], fout), x.dtype)
    if _records(x, kernel, bias, residual):
        return _DenseActFn.apply(x, kernel, bias, residual, act, drop, rng)
    kernel = kernel if kernel.dtype == x.dtype else kernel.to(x.dtype)
    return _dense_forward(x, kernel.contiguous(), bias, residual, act, drop, rng, False)[0]
