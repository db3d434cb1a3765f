"""Residual add + RMSNorm over the sm_100a kernels ``ss_rmsnorm_fwd`` / ``ss_rmsnorm_bwd``.

The reference's ``RMSNorm.forward`` (modules/rms_norm.py:21-30) computes, in fp32 and cast back,
``x * rsqrt(mean(x^2) + eps) * (1 + weight)``, and its ``Block`` adds the residual stream after
the mixer (models/causal_lm.py:30-37).  ``rms_norm_fn(x, weight, residual=...,
prenorm=True)`` does both in one pass — the sum (the next residual stream, rounded to the
I/O dtype as the reference's in-place add) and its normalisation — and is differentiable in
x, residual and weight.  ``rms_norm(module, x, ...)`` takes a reference ``RMSNorm`` module
(its ``weight`` and ``eps``).

``block_norm_fn`` (``ss_block_norm_fwd`` / ``ss_block_norm_bwd``) is for models whose blocks have a
norm behind them as well, a gate, or a scale on the residual branch (the reference's have none): the
norm after the block, the gate, the scaled residual add and the norm before the next block in one
pass each way.
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .selective_scan_interface import _cuda_device


def _rows(t, dim):
    t2 = t.reshape(-1, dim)
    return t2 if t2.stride(-1) == 1 else t2.contiguous()


class RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, unit_offset, prenorm):
        _cuda_device(x, weight, residual)
        dim = x.shape[-1]
        io = x.dtype
        xr = _rows(x, dim)
        rr = None
        if residual is not None:
            if residual.shape != x.shape:
                raise ValueError("residual must have the shape of x")
            rr = _rows(residual if residual.dtype == io else residual.to(io), dim)
        w = weight.to(torch.float32).contiguous()
        rows = xr.shape[0]
        y = torch.empty((rows, dim), dtype=io, device=x.device)
        h = torch.empty((rows, dim), dtype=io, device=x.device) if rr is not None else None
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        args = L.RmsNormArgs(rows, dim, L.dtype_code(io), int(bool(unit_offset)), float(eps),
                             xr.data_ptr(), xr.stride(0), L.ptr(rr), rr.stride(0) if rr is not None else 0,
                             w.data_ptr(), y.data_ptr(), y.stride(0),
                             L.ptr(h), h.stride(0) if h is not None else 0, rstd.data_ptr())
        with torch.cuda.device(x.device):
            L.check(L.lib().ss_rmsnorm_fwd(args, L.stream_of(x.device)), "ss_rmsnorm_fwd")
        hh = h if h is not None else xr
        ctx.save_for_backward(hh, w, rstd)
        ctx.meta = (x.shape, weight.dtype, residual is not None, bool(unit_offset), bool(prenorm))
        y = y.reshape(x.shape)
        if prenorm:
            return y, (h if h is not None else xr).reshape(x.shape)
        return y

    @staticmethod
    def backward(ctx, dy, *dh_out):
        hh, w, rstd = ctx.saved_tensors
        shape, wdtype, has_res, unit, prenorm = ctx.meta
        dim = shape[-1]
        io = hh.dtype
        rows = hh.shape[0]
        dyr = _rows(dy.to(io), dim)
        dhin = None
        if prenorm and dh_out and dh_out[0] is not None:
            dhin = _rows(dh_out[0].to(io), dim)
        dh = torch.empty((rows, dim), dtype=io, device=hh.device)
        dw = torch.empty(dim, dtype=torch.float32, device=hh.device)
        args = L.RmsNormBwdArgs(rows, dim, L.dtype_code(io), int(unit), hh.data_ptr(), hh.stride(0),
                                w.data_ptr(), rstd.data_ptr(), dyr.data_ptr(), dyr.stride(0),
                                L.ptr(dhin), dhin.stride(0) if dhin is not None else 0,
                                dh.data_ptr(), dh.stride(0), dw.data_ptr())
        with torch.cuda.device(hh.device):
            L.check(L.lib().ss_rmsnorm_bwd(args, L.stream_of(hh.device)), "ss_rmsnorm_bwd")
        dh = dh.reshape(shape)
        return dh, dw.to(wdtype), (dh if has_res else None), None, None, None


def rms_norm_fn(x, weight, residual=None, eps=1e-6, unit_offset=True, prenorm=False):
    """RMSNorm of ``x + residual`` (of ``x`` when residual is None) over the last dimension,
    scaled by ``1 + weight`` (unit_offset, the reference's convention) or ``weight``.
    Returns y, or (y, x + residual) with prenorm — the sum being the next residual stream."""
    return RMSNormFn.apply(x, weight, residual, eps, unit_offset, prenorm)


def rms_norm(norm, x, residual=None, prenorm=False):
    """A reference ``RMSNorm`` module's forward (modules/rms_norm.py:21-30) through the fused
    kernel, optionally adding ``residual`` first (see rms_norm_fn)."""
    return rms_norm_fn(x, norm.weight, residual, norm.eps, True, prenorm)


_ACTIVATIONS = {None: 0, "silu": 1, "sigmoid": 2}


_pack_block_fwd, _pack_block_bwd = (L.packer(st) for st in (L.BlockNormArgs, L.BlockNormBwdArgs))


def _row_at(t):
    """Address and row stride of a (rows, dim) tensor."""
    return (0, 0) if t is None else (t.data_ptr(), t.stride(0))


def _like(t):
    return None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=1024)
def _block_work(n, dim, io):
    return int(L.lib().ss_block_norm_work_elems(n, dim, io))


def _block_rows(t, dtype, dim):
    if t is None or (t.dtype == dtype and t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= dim):
        return t
    t = _rows(t if t.dtype == dtype else t.to(dtype), dim)
    return t if t.stride(0) >= dim else t.contiguous()  # rows that share memory


def _f32(t):
    return t if t is None or (t.dtype == torch.float32 and t.is_contiguous()) else t.to(torch.float32).contiguous()


def _block_args(rows, cols, call, h, x, rstd):
    """The fields of ss_block_norm_args; h, x (packed) and rstd are addresses."""
    (y, residual, gate), (post, pre, scale) = rows, cols
    io, activation, eps, pre_eps, unit, const = call
    n, dim = y.shape
    return (n, dim, io, unit, activation, eps, pre_eps, const, y.data_ptr(), y.stride(0), residual.data_ptr(),
            residual.stride(0), *_row_at(gate), _address(post), _address(pre), _address(scale), h, dim, x, dim, rstd)


def _address(t):
    return 0 if t is None else t.data_ptr()


def _block_forward(y, residual, post, pre, gate, scale, call, train):
    """Returns (x | None, h, rows, columns, rstd | None)."""
    dev = _cuda_device(y, residual, post, pre, gate, scale)
    dim, io = y.shape[-1], y.dtype
    rows = _block_rows(y, io, dim), _block_rows(residual, io, dim), _block_rows(gate, io, dim)
    cols = _f32(post), _f32(pre), _f32(scale)
    h = _like(y)
    x = None if pre is None else _like(y)
    rstd = torch.empty((rows[0].shape[0], 2), dtype=torch.float32, device=dev) if train else None
    L.launch("ss_block_norm_fwd", _pack_block_fwd(*_block_args(rows, cols, call, h.data_ptr(), _address(x), _address(rstd))),
             dev)
    return x, h, rows, cols, rstd


def _block_backward(ctx, *grads):
    y, residual, gate, post, pre, scale, rstd = ctx.saved_tensors
    (n, dim), io, dev = y.shape, y.dtype, y.device
    dx, dh = grads if pre is not None else (None, grads[0])
    if dx is None and dh is None:
        return (None,) * 7
    if pre is not None and dx is None:
        dx = torch.zeros_like(y)
    dx, dh = _block_rows(dx, io, dim), _block_rows(dh, io, dim)
    dy, dres, dgate = _like(y), _like(residual), _like(gate)
    work = torch.empty(_block_work(n, dim, ctx.call[0]), dtype=torch.float32, device=dev)
    dpost, dpre, dscale = _like(post), _like(pre), _like(scale)
    L.launch("ss_block_norm_bwd", _pack_block_bwd(
        *_block_args((y, residual, gate), (post, pre, scale), ctx.call, 0, 0, rstd.data_ptr()), *_row_at(dx), *_row_at(dh),
        dy.data_ptr(), dim, dres.data_ptr(), dim, _address(dgate), dim, _address(dpost), _address(dpre), _address(dscale),
        work.data_ptr()), dev)
    grads = dy, dres, dpost, dpre, dgate, dscale
    if ctx.casts is not None:
        grads = (t if t is None else _as_leaf(t, *c) for t, c in zip(grads, ctx.casts))
    return (*grads, None)


def _as_leaf(t, shape, dtype):
    t = t if t.shape == shape else t.reshape(shape)
    return t if t.dtype == dtype else t.to(dtype)


_block_backward_once = once_differentiable(_block_backward)


class BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, post_weight, pre_weight, gate, scale, call):
        x, h, rows, cols, rstd = _block_forward(y, residual, post_weight, pre_weight, gate, scale, call, True)
        ctx.save_for_backward(*rows, *cols, rstd)
        ctx.set_materialize_grads(False)
        ctx.call = call
        # what came in another shape or type than it is saved in
        had, kept = (y, residual, post_weight, pre_weight, gate, scale), (*rows[:2], *cols[:2], rows[2], cols[2])
        ctx.casts = None if all(a is b for a, b in zip(had, kept)) else [None if t is None else (t.shape, t.dtype) for t in had]
        return h if x is None else (x, h)

    @staticmethod
    def backward(ctx, *grads):
        # create_graph: the gradients may be used, not differentiated again
        return (_block_backward_once if torch.is_grad_enabled() else _block_backward)(ctx, *grads)


def block_norm_fn(y, residual, post_weight=None, pre_weight=None, gate=None, residual_scale=None, activation="silu",
                  eps=1e-6, pre_eps=None, unit_offset=True):
    """What stands between two blocks, in one pass over the block's output ``y`` (..., dim):

        h = residual + residual_scale * act(gate) * RMSNorm(y; post_weight)
        x = RMSNorm(h; pre_weight)

    post_weight (dim,): the norm after the block (none when None); gate (y's shape), through
    ``activation`` ("silu", "sigmoid" or None: as it is); residual_scale: a (dim,) tensor or a number;
    pre_weight (dim,): the norm before the next block.  Norms scale by 1 + weight (unit_offset) or
    weight.  residual and gate are taken in y's dtype (cast to it where they come in another: an fp32
    residual beside a 16-bit y is rounded first), and x and h are returned in it; between, everything is
    computed in fp32 and rounded once, x from the unrounded h.  dim is at most 8192.  Returns (x, h), or h
    alone without pre_weight; differentiable in every tensor, once (a second or a forward-mode derivative
    raises)."""
    shape = y.shape
    if residual.shape != shape or (gate is not None and gate.shape != shape):
        raise ValueError("residual and gate must have the shape of y")
    dim = shape[-1] if len(shape) else 0
    if dim < 1:
        raise ValueError("y must have a last dimension of at least 1")
    if dim > L.MAX_BLOCK_NORM_DIM:
        raise NotImplementedError(f"rows of {dim} values (at most {L.MAX_BLOCK_NORM_DIM})")
    scale, const = (residual_scale, 1.0) if isinstance(residual_scale, torch.Tensor) else (
        None, 1.0 if residual_scale is None else float(residual_scale))
    for t, name in ((post_weight, "post_weight"), (pre_weight, "pre_weight"), (scale, "residual_scale")):
        if t is not None and tuple(t.shape) != (dim,):
            raise ValueError(f"{name} must be ({dim},), got {tuple(t.shape)}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation {activation!r} (one of {list(_ACTIVATIONS)})")
    call = (L.dtype_code(y.dtype), _ACTIVATIONS[activation], float(eps), float(eps if pre_eps is None else pre_eps),
            int(bool(unit_offset)), const)
    tensors = y, residual, post_weight, pre_weight, gate, scale
    if L.differentiated(tensors):
        return BlockNormFn.apply(*tensors, call)
    x, h, *_ = _block_forward(*tensors, call, False)
    return h if x is None else (x, h)
