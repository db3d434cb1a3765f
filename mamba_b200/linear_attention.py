"""Linear attention with a decay per head, over the sm_100a kernels ``ss_linear_fwd`` /
``ss_linear_bwd`` / ``ss_linear_step``.

The selective scan's sibling with a matrix state (the reference has no counterpart): per batch row
and head,

    S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T        (key_dim x value_dim, fp32)
    o_t = scale * q_t S_t

* ``linear_attention_fn``   over a sequence, in chunks; differentiable in q, k, v, log_decay and
  initial_state, and through the final state;
* ``linear_attention_step`` for one token, updating the state in place;
* ``linear_attention_forward`` / ``linear_attention_prefill`` / ``linear_attention_block_step`` run a
  module that holds the projections (see ``linear_attention_forward``), as the LM path and the
  ``Decoder`` do for layers with a ``linear_attn``.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .selective_scan_interface import _cuda_device


def _unit(t):
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _strides(t):
    return t.data_ptr(), *t.stride()[:-1]


def _decay(log_decay, io):
    return log_decay if log_decay.dtype in (torch.float32, io) else log_decay.to(torch.float32)


def _scale(scale, key_dim):
    s = key_dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(s) or s == 0.0:
        raise ValueError(f"scale must be finite and not zero, got {s}")
    return s


def _check_heads(q, k, v, lead):
    """q, k: (*lead, key_heads, key_dim), v: (*lead, heads, value_dim)."""
    n = len(lead) + 2
    names = "(batch, seqlen, heads, dim)" if n == 4 else "(batch, heads, dim)"
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != n:
            raise ValueError(f"{name} must be {names}, got shape {tuple(t.shape)}")
        if tuple(t.shape[:-2]) != tuple(lead):
            raise ValueError(f"q, k and v must share their leading shape: {name} has {tuple(t.shape)}")
    if q.shape != k.shape:
        raise ValueError(f"q and k must have the same shape, got {tuple(q.shape)} and {tuple(k.shape)}")
    heads, key_heads = v.shape[-2], k.shape[-2]
    if key_heads < 1 or heads < 1 or heads % key_heads:
        raise ValueError(f"the heads of v ({heads}) must be a multiple of those of q and k ({key_heads})")
    if min(k.shape[-1], v.shape[-1]) < 1:
        raise ValueError("head sizes must be at least 1")
    if max(k.shape[-1], v.shape[-1]) > L.MAX_LINEAR_DIM:
        raise NotImplementedError(f"head sizes above {L.MAX_LINEAR_DIM}: {k.shape[-1]}, {v.shape[-1]}")


def _check_state(t, shape, name):
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")


class _Call:
    """Validated, normalised operands of one sequence call."""

    def __init__(self, q, k, v, log_decay, scale, initial_state, seq_lens):
        self.device = _cuda_device(q, k, v, log_decay, initial_state, seq_lens)
        io = v.dtype
        L.dtype_code(io)
        _check_heads(q, k, v, tuple(v.shape[:2]) if v.dim() == 4 else (0, 0))
        self.b, self.l, self.h, self.dv = v.shape
        self.hk, self.dk = k.shape[2:]
        self.io, self.scale = io, _scale(scale, self.dk)
        if tuple(log_decay.shape) not in ((self.h,), (self.b, self.l, self.h)):
            raise ValueError(f"log_decay must be ({self.h},) or {(self.b, self.l, self.h)}, got {tuple(log_decay.shape)}")
        self.q, self.k, self.v = (_unit(t if t.dtype == io else t.to(io)) for t in (q, k, v))
        self.g = _decay(log_decay, io)
        if self.g.dim() == 3 and self.g.stride(0) == 0 and self.g.stride(1) == 0:
            self.g = self.g.contiguous()  # an expanded tensor still has a gradient for every token
        self.state = None
        if initial_state is not None:
            _check_state(initial_state, (self.b, self.h, self.dk, self.dv), "initial_state")
            self.state = initial_state.to(torch.float32).contiguous()
        self.lens = None
        if seq_lens is not None:
            if tuple(seq_lens.shape) != (self.b,) or seq_lens.is_floating_point() or seq_lens.dtype == torch.bool:
                raise ValueError(f"seq_lens must be ({self.b},) integers, got {seq_lens.dtype} {tuple(seq_lens.shape)}")
            self.lens = seq_lens.clamp(0, self.l).to(torch.int32).contiguous() if seq_lens.dtype != torch.int32 \
                else seq_lens.contiguous()

    def args(self, o=None, state_out=None):
        g = (0, 0, self.g.stride(0)) if self.g.dim() == 1 else self.g.stride()
        return L.LinearArgs(
            self.b, self.l, self.h, self.hk, self.dk, self.dv, L.dtype_code(self.io), L.dtype_code(self.g.dtype),
            self.scale, *_strides(self.q), *_strides(self.k), *_strides(self.v), self.g.data_ptr(), *g,
            L.ptr(self.lens), L.ptr(self.state), L.ptr(state_out), *((None, 0, 0, 0) if o is None else _strides(o)),
            None)

    def work(self, args, backward):
        n = int(L.lib().ss_linear_work_bytes(args, int(backward)))
        return torch.empty(n, dtype=torch.uint8, device=self.device) if n else None

    def forward(self, want_final):
        o = torch.empty((self.b, self.l, self.h, self.dv), dtype=self.io, device=self.device)
        final = None
        if want_final:
            final = torch.empty((self.b, self.h, self.dk, self.dv), dtype=torch.float32, device=self.device)
        args = self.args(o, final)
        work = self.work(args, False)
        args.work = L.ptr(work)
        with torch.cuda.device(self.device):
            L.check(L.lib().ss_linear_fwd(args, L.stream_of(self.device)), "ss_linear_fwd")
            L.maybe_check_status(self.device, "ss_linear_fwd")
        return o, final

    def backward(self, dout, dfinal, final, want_decay, want_state):
        new = lambda t, dtype=None: torch.empty(t.shape, dtype=dtype or t.dtype, device=self.device)  # noqa: E731
        dout = _unit(dout if dout.dtype == self.io else dout.to(self.io))
        dfinal = None if dfinal is None else dfinal.to(torch.float32).contiguous()
        dq, dk, dv = new(self.q), new(self.k), new(self.v)
        dg = new(self.g) if want_decay else None
        ds = torch.empty((self.b, self.h, self.dk, self.dv), dtype=torch.float32, device=self.device) \
            if want_state else None
        args = L.LinearBwdArgs(self.args(None, final), *_strides(dout), L.ptr(dfinal), *_strides(dq), *_strides(dk),
                               *_strides(dv), L.ptr(dg), L.ptr(ds), None)
        work = self.work(args.f, True)
        args.work = L.ptr(work)
        with torch.cuda.device(self.device):
            L.check(L.lib().ss_linear_bwd(args, L.stream_of(self.device)), "ss_linear_bwd")
            L.maybe_check_status(self.device, "ss_linear_bwd")
        return dq, dk, dv, dg, ds


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, seq_lens, want_final):
        c = _Call(q, k, v, log_decay, scale, initial_state, seq_lens)
        o, final = c.forward(want_final)
        ctx.set_materialize_grads(False)
        # the final state is needed again for the decays' gradient through it
        ctx.save_for_backward(c.q, c.k, c.v, c.g, c.state, c.lens, final)
        ctx.scale = c.scale
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (q, k, v, log_decay, initial_state))
        return (o, final) if want_final else o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal=None):
        q, k, v, g, state, lens, final = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 8
        c = _Call(q, k, v, g, ctx.scale, state, lens)
        if dout is None:
            dout = torch.zeros_like(v)
        grads = c.backward(dout, dfinal, final, ctx.needs_input_grad[3], ctx.needs_input_grad[5])
        dq, dk, dv, dg, ds = (t if t is None or t.dtype == d else t.to(d)
                              for t, d in zip(grads, ctx.dtypes))
        return dq, dk, dv, dg, None, ds, None, None


def linear_attention_fn(q, k, v, log_decay, scale=None, initial_state=None, seq_lens=None, return_final_state=False):
    """Linear attention with a decay per head over a sequence.

    q, k: (batch, seqlen, key_heads, key_dim); v: (batch, seqlen, heads, value_dim), heads a multiple
    of key_heads (head j reads key head j // (heads // key_heads)); head sizes up to 128.
    log_decay: (batch, seqlen, heads), or (heads,) for one decay per head at every token; its values
    are the logarithms of the decays (<= 0; -inf resets the state).  scale: of the outputs
    (key_dim ** -0.5 when None).  initial_state: (batch, heads, key_dim, value_dim), zeros when None.
    seq_lens: (batch,) integers; the tokens behind a row's length are ignored (whatever they hold),
    their outputs and gradients are zero.  Returns o (batch, seqlen, heads, value_dim) in v's dtype,
    and with return_final_state the state after each row's last token, fp32.
    float32, bfloat16 and float16; the state is fp32 throughout."""
    return LinearAttentionFn.apply(q, k, v, log_decay, scale, initial_state, seq_lens, bool(return_final_state))


@torch.no_grad()
def linear_attention_step(state, q, k, v, log_decay, scale=None):
    """One token of ``linear_attention_fn``; updates ``state`` (batch, heads, key_dim, value_dim) fp32 in
    place.  q, k: (batch, key_heads, key_dim); v: (batch, heads, value_dim); log_decay: (batch, heads)
    or (heads,).  Returns o (batch, heads, value_dim) in v's dtype."""
    dev = _cuda_device(state, q, k, v, log_decay)
    io = v.dtype
    L.dtype_code(io)
    _check_heads(q, k, v, tuple(v.shape[:1]) if v.dim() == 3 else (0,))
    b, h, dv = v.shape
    hk, dk = k.shape[1:]
    _check_state(state, (b, h, dk, dv), "state")
    if state.dtype != torch.float32 or not state[:1].is_contiguous() or (b > 1 and state.stride(0) < h * dk * dv):
        raise ValueError("state must be float32 with contiguous (heads, key_dim, value_dim) rows")
    if tuple(log_decay.shape) not in ((h,), (b, h)):
        raise ValueError(f"log_decay must be ({h},) or {(b, h)}, got {tuple(log_decay.shape)}")
    q, k, v = (_unit(t if t.dtype == io else t.to(io)) for t in (q, k, v))
    g = _decay(log_decay, io)
    gs = (0, g.stride(0)) if g.dim() == 1 else g.stride()
    o = torch.empty((b, h, dv), dtype=io, device=dev)
    args = L.LinearStepArgs(b, h, hk, dk, dv, L.dtype_code(io), L.dtype_code(g.dtype), _scale(scale, dk),
                            state.data_ptr(), state.stride(0) if b > 1 else h * dk * dv, *_strides(q), *_strides(k),
                            *_strides(v), g.data_ptr(), *gs, *_strides(o))
    with torch.cuda.device(dev):
        L.check(L.lib().ss_linear_step(args, L.stream_of(dev)), "ss_linear_step")
    return o


# ------------------------------------------------------------------------------------- modules
def _projected(block, x):
    """q, k, v, log_decay of a mixer module's input (..., d_model)."""
    lead = x.shape[:-1]
    q = block.q_proj(x).reshape(*lead, block.num_key_heads, -1)
    k = block.k_proj(x).reshape(*lead, block.num_key_heads, -1)
    v = block.v_proj(x).reshape(*lead, block.num_heads, -1)
    decay = getattr(block, "decay_proj", None)
    if decay is None:
        return q, k, v, block.log_decay
    return q, k, v, torch.nn.functional.logsigmoid(decay(x))


def linear_attention_forward(block, hidden_states, seq_lens=None):
    """Forward of a linear-attention mixer module over hidden_states (batch, seqlen, d_model).
    ``block`` has num_heads, num_key_heads, the projections q_proj, k_proj, v_proj, output_proj and
    either decay_proj (d_model -> num_heads; the log decay is logsigmoid of it) or a fixed
    log_decay (num_heads,)."""
    o = linear_attention_fn(*_projected(block, hidden_states), seq_lens=seq_lens)
    return block.output_proj(o.flatten(-2))


@torch.no_grad()
def linear_attention_prefill(block, hidden_states):
    """The module's forward over a prompt from a zero state: (output, state fp32)."""
    o, state = linear_attention_fn(*_projected(block, hidden_states), return_final_state=True)
    return block.output_proj(o.flatten(-2)), state


@torch.no_grad()
def linear_attention_block_step(block, hidden, state):
    """One token (batch, d_model) through the module; updates the state in place."""
    o = linear_attention_step(state, *_projected(block, hidden))
    return block.output_proj(o.flatten(-2))
