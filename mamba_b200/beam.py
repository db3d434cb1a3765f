"""Beam search's step over the sm_100a kernels ``ss_beam_select`` and ``ss_reorder``: the best
continuations over the beams and the vocabulary, and the beams' states put in their new order in
place.  ``mamba_b200.beam_search`` runs a model with them; the reference has no counterpart (its
``generate`` is a stub, models/causal_lm.py:61-62)."""
from __future__ import annotations

import operator

import torch

from . import _lib as L
from .selective_scan_interface import _cuda_device


_nbytes, _rows_of = operator.attrgetter("nbytes"), operator.methodcaller("size", 0)
_pack_beam, _pack_reorder = L.packer(L.BeamArgs), L.packer(L.ReorderArgs)


def beam_select(logits, scores, num_select=None, finished=None, eos_token_id=None):
    """The num_select best continuations of every batch row.

    logits: (batch, beams, vocab) in float32, bfloat16 or float16; scores: (batch, beams) fp32 sums of
    log probabilities.  A candidate's score is scores + log_softmax(logits).  finished (batch, beams)
    bool: such a beam offers itself alone, at eos_token_id with its score unchanged, and its logits
    are not read.  Candidates that are not a number count as -inf, as does every candidate of a beam
    whose score is NaN or +inf.  Returns (scores, parents, tokens), each (batch, num_select), in falling
    order of score, equal candidates in order of (beam, token); scores fp32, indices int64.  Candidates
    are compared in fp64; a beam's log-softmax is good to 1e-7 (its exponentials are fp32), so candidates
    of different beams that are nearer than that may change places against exact arithmetic.
    num_select (beams when None) and beams are at most 32."""
    dev = _cuda_device(logits, scores, finished)
    if logits.dim() != 3:
        raise ValueError(f"logits must be (batch, beams, vocab), got {tuple(logits.shape)}")
    b, w, vocab = logits.shape
    k = w if num_select is None else int(num_select)
    if w < 1 or vocab < 1 or not 1 <= k <= w * vocab:
        raise ValueError(f"num_select {k} of {w} beams x {vocab} tokens")
    if w > L.MAX_BEAMS or k > L.MAX_BEAMS:
        raise NotImplementedError(f"beams {w} and num_select {k} are at most {L.MAX_BEAMS}")
    if tuple(scores.shape) != (b, w):
        raise ValueError(f"scores must be {(b, w)}, got {tuple(scores.shape)}")
    if (finished is not None) != (eos_token_id is not None):
        raise ValueError("finished and eos_token_id go together")
    eos = 0
    if finished is not None:
        if tuple(finished.shape) != (b, w) or finished.dtype != torch.bool:
            raise ValueError(f"finished must be {(b, w)} bool, got {finished.dtype} {tuple(finished.shape)}")
        eos = int(eos_token_id)
        if not 0 <= eos < vocab:
            raise ValueError(f"eos_token_id {eos} of {vocab} tokens")
        finished = finished.contiguous()
    io = L.dtype_code(logits.dtype)
    x = logits if (logits.stride(-1) == 1 or vocab == 1) and min(logits.stride()) >= 0 else logits.contiguous()
    s = scores if scores.dtype == torch.float32 and scores.is_contiguous() else scores.to(torch.float32).contiguous()
    out = torch.empty((b, k), dtype=torch.float32, device=dev)
    parents = torch.empty((b, k), dtype=torch.int64, device=dev)
    tokens = torch.empty((b, k), dtype=torch.int64, device=dev)
    work = torch.empty(int(L.lib().ss_beam_work_bytes(b, w, vocab, k)), dtype=torch.uint8, device=dev)
    L.launch("ss_beam_select", _pack_beam(b, w, vocab, k, io, eos, x.data_ptr(), x.stride(0), x.stride(1), s.data_ptr(),
                                          0 if finished is None else finished.data_ptr(), out.data_ptr(),
                                          parents.data_ptr(), tokens.data_ptr(), work.data_ptr()), dev)
    return out, parents, tokens


def reorder_states(states, parents):
    """Put per-beam rows in their new order, in place: for every tensor of ``states`` ((batch * beams, ...)
    contiguous, rows of a multiple of 4 bytes) and every batch row, row w becomes what row
    parents[:, w] was.  parents: (batch, beams) int64 (its beams may be a slice of a wider result of
    ``beam_select``).  A parent outside the beams leaves its row as it was, and the next
    ``check_device_status`` raises.  Tensors that share memory are refused."""
    _cuda_device(parents)
    if parents.dim() != 2 or parents.dtype != torch.int64:
        raise ValueError(f"parents must be (batch, beams) int64, got {parents.dtype} {tuple(parents.shape)}")
    b, w = parents.shape
    if w < 1:
        raise ValueError("parents must name at least one beam")
    if w > L.MAX_BEAMS:
        raise NotImplementedError(f"{w} beams are more than {L.MAX_BEAMS}")
    total = b * w
    if not isinstance(states, (list, tuple)):
        states = list(states)
    # whole columns of checks at a time: a model's dozens of states pass in a few microseconds
    if min(map(torch.Tensor.dim, states), default=1) < 1 or not set(map(_rows_of, states)) <= {total} or not all(
            map(torch.Tensor.is_contiguous, states)):
        raise ValueError(f"a state must have {total} contiguous rows, got {[tuple(t.shape) for t in states]}")
    if states and set(map(torch.Tensor.get_device, states)) != {parents.get_device()}:
        raise RuntimeError("states and parents on different devices")
    sizes = list(map(_nbytes, states))
    rows = sorted(zip(map(torch.Tensor.data_ptr, states), sizes))
    if 0 in sizes:
        rows = [r for r in rows if r[1]]
    end, step = 0, 4 * total
    for at, n in rows:
        if n % step or at % 4:
            raise NotImplementedError(f"rows of {n / total} bytes at address {at} (multiples of 4 are supported)")
        if at < end:
            raise ValueError("states must not share memory")
        end = at + n
    # rows of parents that share memory (one order for the whole batch) are laid out first
    p = parents if (parents.stride(1) == 1 or w == 1) and (parents.stride(0) >= w or b <= 1) else parents.contiguous()
    L.written(states)
    for i in range(0, len(rows), L.MAX_REORDER):
        part = rows[i:i + L.MAX_REORDER]
        none = (0,) * (L.MAX_REORDER - len(part))
        L.launch("ss_reorder", _pack_reorder(b, w, len(part), p.data_ptr(), p.stride(0) if b > 1 else w,
                                             *[at for at, _ in part], *none, *[n // total for _, n in part], *none),
                 parents.device)
