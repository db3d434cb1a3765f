"""Plain float64 restatements of the sequence operators (linear attention, norms around a block,
beam selection), differentiable where the operators are, for the tests."""
import math

import torch


def linear_ref(q, k, v, log_decay, scale, s0=None, lens=None):
    """The recurrence token by token.  Returns (o, final state)."""
    b, l, h, dv = v.shape
    dk, rep = q.shape[-1], h // q.shape[2]
    q, k = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
    g = log_decay if log_decay.dim() == 3 else log_decay.expand(b, l, h)
    S = v.new_zeros(b, h, dk, dv) if s0 is None else s0
    outs = []
    for t in range(l):
        new = torch.exp(g[:, t])[..., None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        o = scale * (q[:, t, :, None, :] @ new).squeeze(-2)
        if lens is None:
            S = new
        else:
            live = (t < lens).view(b, 1, 1, 1)
            S = torch.where(live, new, S)
            o = torch.where(live[..., 0], o, torch.zeros_like(o))
        outs.append(o)
    return (torch.stack(outs, 1) if outs else v.new_zeros(b, 0, h, dv)), S


def block_norm_ref(y, residual, post=None, pre=None, gate=None, scale=None, act="silu", eps=1e-6, pre_eps=None,
                   unit=True):
    def rms(t, w, e):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + e) * (w + 1 if unit else w)

    u = y if post is None else rms(y, post, eps)
    if gate is not None:
        u = u * {"silu": gate * torch.sigmoid(gate), "sigmoid": torch.sigmoid(gate), None: gate}[act]
    if scale is not None:
        u = u * scale
    h = residual + u
    return (None if pre is None else rms(h, pre, eps if pre_eps is None else pre_eps)), h


def beam_ref(logits, scores, k, finished=None, eos=None):
    """Lists of (score, beam, token) per batch row, by sorting every candidate (Python floats)."""
    rows = []
    for b in range(logits.shape[0]):
        cand = []
        for w in range(logits.shape[1]):
            x = logits[b, w].double().tolist()
            s = float(scores[b, w])
            done = finished is not None and bool(finished[b, w])
            top = max(x) if not any(math.isnan(v) for v in x) else math.nan
            lse = math.nan if math.isnan(top) or math.isinf(top) else top + math.log(math.fsum(math.exp(v - top) for v in x))
            for t, v in enumerate(x):
                c = (s if t == eos else -math.inf) if done else s + (v - lse)
                if math.isnan(c) or math.isnan(s) or s == math.inf:
                    c = -math.inf
                cand.append((-c, w, t))
        cand.sort()
        rows.append([(-c, w, t) for c, w, t in cand[:k]])
    return rows
