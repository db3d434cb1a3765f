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

import functools
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .selective_scan_interface import _cuda_device


_pack_fwd, _pack_bwd, _pack_step = (L.packer(st) for st in (L.LinearArgs, L.LinearBwdArgs, L.LinearStepArgs))
_NONE4 = (0, 0, 0, 0)


def _as(t, dtype):
    return t if t.dtype == dtype else t.to(dtype)


def _at(t):
    """Address and the strides but the innermost."""
    return t.data_ptr(), *t.stride()[:-1]


def _p(t):
    return 0 if t is None else t.data_ptr()


def _decay(log_decay, io):
    return log_decay if log_decay.dtype in (torch.float32, io) else log_decay.to(torch.float32)


def _scale(scale, key_dim):
    s = key_dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(s) or s == 0.0:
        raise ValueError(f"scale must be finite and not zero, got {s}")
    return s


def _check_heads(q, k, v, n):
    """q, k: (..., key_heads, key_dim), v: (..., heads, value_dim), n axes each.  Returns their sizes."""
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != n or len(ks) != n or len(vs) != n:
        names = "(batch, seqlen, heads, dim)" if n == 4 else "(batch, heads, dim)"
        raise ValueError(f"q, k and v must be {names}, got {tuple(qs)}, {tuple(ks)} and {tuple(vs)}")
    if qs != ks:
        raise ValueError(f"q and k must have the same shape, got {tuple(qs)} and {tuple(ks)}")
    if ks[:-2] != vs[:-2]:
        raise ValueError(f"q, k and v must share their leading shape, got {tuple(ks)} and {tuple(vs)}")
    (hk, dk), (h, dv) = ks[-2:], vs[-2:]
    if hk < 1 or h < 1 or h % hk:
        raise ValueError(f"the heads of v ({h}) must be a multiple of those of q and k ({hk})")
    if dk < 1 or dv < 1:
        raise ValueError("head sizes must be at least 1")
    if dk > L.MAX_LINEAR_DIM or dv > L.MAX_LINEAR_DIM:
        raise NotImplementedError(f"head sizes above {L.MAX_LINEAR_DIM}: {dk}, {dv}")
    return h, hk, dk, dv


def _check_state(t, shape, name):
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")


@functools.lru_cache(maxsize=1024)
def _work_bytes(sizes, io, decay, backward):
    args = L.LinearArgs(*sizes, io, decay)
    return int(L.lib().ss_linear_work_bytes(args, backward))


def _work(c, backward, device):
    n = _work_bytes(c[:6], c[6], c[7], backward)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _whole(t):
    """t with rows of whole 16-byte units, as the tensor-core kernel's copies need them: itself where it has them."""
    if t.shape[-1] % 8:
        return torch.nn.functional.pad(t, (0, -t.shape[-1] % 8))
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _prepare(q, k, v, log_decay, scale, initial_state, seq_lens):
    """Validated, normalised operands: (tensors, (sizes, type codes, scale)), tensors q, k, v, log_decay,
    initial_state, seq_lens."""
    _cuda_device(q, k, v, log_decay, initial_state, seq_lens)
    io = v.dtype
    io_code = L.dtype_code(io)
    h, hk, dk, dv = _check_heads(q, k, v, 4)
    b, l = v.shape[:2]
    scale = _scale(scale, dk)
    if tuple(log_decay.shape) not in ((h,), (b, l, h)):
        raise ValueError(f"log_decay must be ({h},) or {(b, l, h)}, got {tuple(log_decay.shape)}")
    q, k, v = _as(q, io), _as(k, io), _as(v, io)
    if q.stride(-1) != 1 or k.stride(-1) != 1 or v.stride(-1) != 1:
        q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, v))
    g = _decay(log_decay, io)
    if g.dim() == 3 and g.stride(0) == 0 and g.stride(1) == 0:
        g = g.contiguous()  # an expanded tensor still has a gradient for every token
    if initial_state is not None:
        _check_state(initial_state, (b, h, dk, dv), "initial_state")
        initial_state = _as(initial_state, torch.float32).contiguous()
    if seq_lens is not None:
        if tuple(seq_lens.shape) != (b,) or seq_lens.is_floating_point() or seq_lens.dtype == torch.bool:
            raise ValueError(f"seq_lens must be ({b},) integers, got {seq_lens.dtype} {tuple(seq_lens.shape)}")
        if seq_lens.dtype != torch.int32:
            seq_lens = seq_lens.clamp(0, l).to(torch.int32)
        seq_lens = seq_lens.contiguous()
    return (q, k, v, g, initial_state, seq_lens), (b, l, h, hk, dk, dv, io_code, L.dtype_code(g.dtype), scale)


def _inputs(t, c, state_out):
    """The leading fields of ss_linear_args."""
    q, k, v, g, state, lens = t
    gs = (0, 0, g.stride(0)) if g.dim() == 1 else g.stride()
    return (*c, *_at(q), *_at(k), *_at(v), g.data_ptr(), *gs, _p(lens), _p(state), _p(state_out))


def _forward(t, c, want_final):
    b, l, h, _, dk, dv = c[:6]
    v = t[2]
    dev = v.device
    o = torch.empty_like(v, memory_format=torch.contiguous_format)
    final = torch.empty((b, h, dk, dv), dtype=torch.float32, device=dev) if want_final else None
    work = _work(c, 0, dev)
    L.launch("ss_linear_fwd", _pack_fwd(*_inputs(t, c, final), *_at(o), _p(work)), dev)
    L.maybe_check_status(dev, "ss_linear_fwd")
    return o, final


def _backward(t, c, dout, dfinal, final, want_decay, want_state):
    q, k, v, g = t[:4]
    dev = v.device
    new = functools.partial(torch.empty_like, memory_format=torch.contiguous_format)
    dout = _as(dout, v.dtype)
    if v.dtype != torch.float32:
        dout = _whole(dout)
    elif dout.stride(-1) != 1:
        dout = dout.contiguous()
    if dfinal is not None:
        dfinal = _as(dfinal, torch.float32).contiguous()
    dq, dk, dv = new(q), new(k), new(v)
    dg = new(g) if want_decay else None
    ds = new(t[4]) if want_state else None
    work = _work(c, 1, dev)
    L.launch("ss_linear_bwd", _pack_bwd(*_inputs(t, c, final), *_NONE4, 0, *_at(dout), _p(dfinal), *_at(dq), *_at(dk),
                                        *_at(dv), _p(dg), _p(ds), _p(work)), dev)
    L.maybe_check_status(dev, "ss_linear_bwd")
    return dq, dk, dv, dg, ds


def _backward_of(ctx, dout, dfinal=None):
    *t, final = ctx.saved_tensors
    if dout is None and dfinal is None:
        return (None,) * 8
    if dout is None:
        dout = torch.zeros_like(t[2])
    grads = _backward(t, ctx.call, dout, dfinal, final, ctx.needs_input_grad[3], ctx.needs_input_grad[5])
    dq, dk, dv, dg, ds = (x if x is None else _as(x, d) for x, d in zip(grads, ctx.dtypes))
    return dq, dk, dv, dg, None, ds, None, None


_backward_once = once_differentiable(_backward_of)


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial_state, seq_lens, want_final):
        t, c = _prepare(q, k, v, log_decay, scale, initial_state, seq_lens)
        o, final = _forward(t, c, want_final)
        ctx.set_materialize_grads(False)
        # the final state is needed again for the decays' gradient through it; where that is not asked for, a caller
        # may go on to step the state in place
        ctx.save_for_backward(*t, final if ctx.needs_input_grad[3] else None)
        ctx.call = c
        ctx.dtypes = tuple(None if x is None else x.dtype for x in (q, k, v, log_decay, initial_state))
        return (o, final) if want_final else o

    @staticmethod
    def backward(ctx, *grads):
        # create_graph: the gradients may be used, not differentiated again
        return (_backward_once if torch.is_grad_enabled() else _backward_of)(ctx, *grads)


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

    float32, bfloat16 and float16; the state is fp32 throughout.  Tokens are summed in chunks, so one that holds
    an infinity or NaN reaches the outputs of up to 127 tokens before it.  16-bit inputs run on the tensor cores; for
    that, inputs whose rows are not whole 16-byte units (head sizes off a multiple of 8, odd strides) are
    copied first.  q and k are taken in v's dtype.  Differentiable once (a second or a forward-mode
    derivative raises)."""
    want = bool(return_final_state)
    cut = None
    if v.dtype in (torch.bfloat16, torch.float16) and v.dim() == k.dim() == q.dim() == 4 and v.numel():
        if (q.shape[3] | k.shape[3] | v.shape[3]) % 8:  # padded below: the sizes that were passed are checked first
            _cuda_device(q, k, v, log_decay, initial_state, seq_lens)
            h, _, dk, dv = _check_heads(q, k, v, 4)
            scale = _scale(scale, dk)
            cut = dk, dv
            if initial_state is not None:
                _check_state(initial_state, (v.shape[0], h, dk, dv), "initial_state")
                initial_state = torch.nn.functional.pad(initial_state, (0, -dv % 8, 0, -dk % 8))
        q, k, v = _whole(_as(q, v.dtype)), _whole(_as(k, v.dtype)), _whole(v)
    if L.differentiated((q, k, v, log_decay, initial_state)):
        out = LinearAttentionFn.apply(q, k, v, log_decay, scale, initial_state, seq_lens, want)
        o, final = out if want else (out, None)
    else:
        o, final = _forward(*_prepare(q, k, v, log_decay, scale, initial_state, seq_lens), want)
    if cut:
        o = o[..., :cut[1]].contiguous()
        final = final[..., :cut[0], :cut[1]].contiguous() if want else None
    return (o, final) if want else o


def linear_attention_step(state, q, k, v, log_decay, scale=None):
    """One token of ``linear_attention_fn``; updates ``state`` (batch, heads, key_dim, value_dim) fp32 in
    place.  q, k: (batch, key_heads, key_dim); v: (batch, heads, value_dim); log_decay: (batch, heads)
    or (heads,).  Returns o (batch, heads, value_dim) in v's dtype.  Not differentiable."""
    dev = _cuda_device(state, q, k, v, log_decay)
    io = v.dtype
    io_code = L.dtype_code(io)
    h, hk, dk, dv = _check_heads(q, k, v, 3)
    b, n = v.shape[0], h * dk * dv
    _check_state(state, (b, h, dk, dv), "state")
    ss = state.stride()
    if state.dtype != torch.float32 or (b > 1 and ss[0] < n) or (
            ss[1:] != (dk * dv, dv, 1) and not state[:1].is_contiguous()):
        raise ValueError("state must be float32 with contiguous (heads, key_dim, value_dim) rows")
    if tuple(log_decay.shape) not in ((h,), (b, h)):
        raise ValueError(f"log_decay must be ({h},) or {(b, h)}, got {tuple(log_decay.shape)}")
    q, k, v = _as(q, io), _as(k, io), _as(v, io)
    if q.stride(-1) != 1 or k.stride(-1) != 1 or v.stride(-1) != 1:
        q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, v))
    g = _decay(log_decay, io)
    gs = (0, g.stride(0)) if g.dim() == 1 else g.stride()
    o = torch.empty_like(v, memory_format=torch.contiguous_format)
    L.launch("ss_linear_step", _pack_step(b, h, hk, dk, dv, io_code, L.dtype_code(g.dtype), _scale(scale, dk),
                                          state.data_ptr(), ss[0] if b > 1 else n, *_at(q), *_at(k), *_at(v),
                                          g.data_ptr(), *gs, o.data_ptr(), h * dv, dv), dev)
    L.written((state,))
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
