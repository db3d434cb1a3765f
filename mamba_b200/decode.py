"""Decoding for MambaSimple models: a prompt prefill that leaves per-layer states, single-token
steps that continue from them, and ``generate`` and ``beam_search`` for CausalLM-shaped models.

The reference has no decode path: ``CausalLM.generate`` is a stub (models/causal_lm.py:61-62)
and ``MambaSimple`` has no step, so continuing a sequence there means re-running the whole
forward over it for every new token.  Here a block keeps two states per sequence:

* conv state (batch, d_inner, K-1) fp32 — the last K-1 inputs of its causal convolution;
* SSM state  (batch, d_inner, d_state) fp32 — h of the selective scan
  (a layer with a ``linear_attn`` mixer: its state (batch, heads, key_dim, value_dim) fp32),

and a new token costs the block's input and output projections plus one fused mixer kernel
(``ss_mamba_step``: the conv step, the x and delta projections, the SSM step and the SiLU(z)
gate).  The prefill runs the fused block path
(``mamba_inner_prefill``: conv kernel, batched GEMMs, scan with ``return_last_state``); each
block's residual add is fused with the next RMSNorm (``rms_norm(..., prenorm=True)``); and the
per-token model step of ``Decoder`` is captured once in a CUDA graph and replayed, so a decode
step is one graph launch rather than a dozen kernel launches per layer from Python.

Models are duck-typed on the reference's structure (models/causal_lm.py:20-58): ``embedding``,
``layers`` (each with ``norm``, ``mamba``), ``norm``, ``lm_head``; each ``mamba`` has
MambaSimple's parameter names (modules/mamba_simple.py:33-85); layers may hold a ``linear_attn``
mixer, a ``post_norm``, a ``gate_proj`` and a ``residual_scale`` instead (see lm.py).  Dropout is not
applied (inference).

``beam_search`` keeps the beams as rows of the decoder's batch: after each selection
(``beam_select``) the layers' states are put in the beams' new order in place (``reorder_states``), so
the captured step goes on at the same addresses.
"""
from __future__ import annotations

import torch

from . import _lib as L
from .beam import beam_select, reorder_states
from .inner import mamba_inner_prefill
from .linear_attention import linear_attention_block_step, linear_attention_prefill
from .lm import branch_parts, join_residual
from .norm import rms_norm_fn
from .selective_scan_interface import _cuda_device


class _BlockParams:
    """A MambaSimple block's parameters in the form the step kernels take, computed once."""

    def __init__(self, blk):
        self.blk = blk
        self.d = blk.D.shape[0]
        self.n = blk.log_A.shape[1]
        self.R = blk.delta_proj.weight.shape[1]
        self.A = (-torch.exp(blk.log_A.detach().float())).contiguous()
        self.D = blk.D.detach().float().contiguous()
        self.dt_bias = blk.delta_proj.bias.detach().float().contiguous()
        w = blk.short_conv.weight.detach()
        self.conv_w = w.reshape(w.shape[0], -1).float().contiguous()
        self.conv_b = None if blk.short_conv.bias is None else blk.short_conv.bias.detach().float().contiguous()
        self.K = self.conv_w.shape[1]


@torch.no_grad()
def mamba_simple_prefill(block, hidden_states, params: _BlockParams | None = None):
    """Block forward over a prompt (batch, L, d_model) from zero states.  Returns
    (output (batch, L, d_model), conv_state, ssm_state)."""
    p = params or _BlockParams(block)
    xz = block.input_proj(hidden_states)
    return mamba_inner_prefill(xz, p.conv_w, p.conv_b, block.ssm_param_proj.weight, block.delta_proj.weight,
                               block.delta_proj.bias, block.output_proj.weight, block.output_proj.bias, p.A, p.D,
                               True)


def mamba_mixer_step(xz, conv_state, ssm_state, p: _BlockParams, x_proj_weight, delta_proj_weight):
    """The mixer of one decode step (conv step, x projection, delta projection, SSM step, gate)
    in one kernel (``ss_mamba_step``): xz (batch, 2 d) -> y (batch, d); both states update in
    place."""
    _cuda_device(xz, conv_state, ssm_state, x_proj_weight, delta_proj_weight)
    b = xz.shape[0]
    io = xz.dtype
    if xz.stride(-1) != 1:
        xz = xz.contiguous()
    Wx = x_proj_weight if x_proj_weight.dtype == io else x_proj_weight.to(io)
    Wdt = delta_proj_weight if delta_proj_weight.dtype == io else delta_proj_weight.to(io)
    Wx, Wdt = Wx.contiguous(), Wdt.contiguous()
    for t, shape in ((conv_state, (b, p.d, p.K - 1)), (ssm_state, (b, p.d, p.n))):
        if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"state must be a contiguous fp32 {shape} tensor")
    y = torch.empty((b, p.d), dtype=io, device=xz.device)
    args = L.MambaStepArgs(b, p.d, p.n, p.K, p.R, L.dtype_code(io), 1, xz.data_ptr(), xz.stride(0),
                           L.ptr(conv_state) if p.K > 1 else None, p.conv_w.data_ptr(), L.ptr(p.conv_b),
                           Wx.data_ptr(), Wdt.data_ptr(), p.dt_bias.data_ptr(), p.A.data_ptr(), p.D.data_ptr(),
                           ssm_state.data_ptr(), y.data_ptr(), y.stride(0))
    with torch.cuda.device(xz.device):
        L.check(L.lib().ss_mamba_step(args, L.stream_of(xz.device)), "ss_mamba_step")
    return y


@torch.no_grad()
def mamba_simple_step(block, hidden, conv_state, ssm_state, params: _BlockParams | None = None):
    """One token (batch, d_model) through a block; updates both states in place.  Three kernels:
    the input projection (GEMM), the fused mixer step, the output projection (GEMM)."""
    p = params or _BlockParams(block)
    xz = block.input_proj(hidden)                                    # (b, 2 d)
    y = mamba_mixer_step(xz, conv_state, ssm_state, p, block.ssm_param_proj.weight, block.delta_proj.weight)
    return block.output_proj(y)


class _MambaLayer:
    """A decoder's MambaSimple layer: its mixer, and where its parameters and states stand in the decoder's lists."""

    def __init__(self, mixer, dec, dev):
        self.mixer, self.at = mixer, len(dec.params)
        p = _BlockParams(mixer)
        dec.params.append(p)
        dec.conv_states.append(torch.zeros(dec.batch, p.d, p.K - 1, device=dev))
        dec.ssm_states.append(torch.zeros(dec.batch, p.d, p.n, device=dev))

    def states(self, dec):
        return dec.conv_states[self.at], dec.ssm_states[self.at]

    def prefill(self, dec, x):
        y, *states = mamba_simple_prefill(self.mixer, x, dec.params[self.at])
        return y, states

    def step(self, dec, x):
        return mamba_simple_step(self.mixer, x, *self.states(dec), dec.params[self.at])


class _LinearLayer:
    """A decoder's linear-attention layer: its mixer, and where its state stands in the decoder's list."""

    def __init__(self, mixer, dec, dev):
        self.mixer, self.at = mixer, len(dec.linear_states)
        heads, key_heads = mixer.num_heads, mixer.num_key_heads
        dec.linear_states.append(torch.zeros(dec.batch, heads, mixer.k_proj.weight.shape[0] // key_heads,
                                             mixer.v_proj.weight.shape[0] // heads, device=dev))

    def states(self, dec):
        return (dec.linear_states[self.at],)

    def prefill(self, dec, x):
        y, state = linear_attention_prefill(self.mixer, x)
        return y, [state]

    def step(self, dec, x):
        return linear_attention_block_step(self.mixer, x, *self.states(dec))


class Decoder:
    """Incremental decoding of a CausalLM-shaped model for a fixed batch size.

    ``prefill(input_ids)`` runs the prompt and returns the last position's logits;
    ``step(token_ids)`` feeds one token per sequence and returns the next logits (fp32);
    ``reorder(parents)`` puts the states of beams in a new order.
    With ``cuda_graph`` the step is captured on first use and replayed afterwards."""

    def __init__(self, model, batch: int, cuda_graph: bool = True):
        self.model = model
        self.batch = batch
        dev = model.lm_head.weight.device
        # per layer of its kind: MambaSimple parameters and states, linear-attention states.  The lists may be
        # assigned to, or an item replaced, until the step is captured
        self.params, self.conv_states, self.ssm_states, self.linear_states = [], [], [], []
        self.mixers = [_LinearLayer(layer.linear_attn, self, dev) if getattr(layer, "linear_attn", None) is not None
                       else _MambaLayer(layer.mamba, self, dev) for layer in model.layers]
        # fp32 norm weights, cast once (a per-call cast would be one more kernel per layer and step)
        norms = [layer.norm for layer in model.layers] + [model.norm]
        *self.norms, self.final_norm = [(n.weight.detach().float().contiguous(), n.eps) for n in norms]
        self.parts = [self._cast(branch_parts(layer, n)) for layer, n in zip(model.layers, norms[1:])]
        self.cuda_graph = cuda_graph
        self.graph = None
        self.tok = torch.zeros(batch, dtype=torch.long, device=dev)
        self.logits = None

    @staticmethod
    def _cast(parts):
        return parts and tuple(t.detach().float().contiguous() if isinstance(t, torch.Tensor) else t for t in parts)

    @property
    def states(self):
        """The states of all layers, in the layers' order."""
        return [s for m in self.mixers for s in m.states(self)]

    @torch.no_grad()
    def prefill(self, input_ids, repeat: int = 1):
        """Runs a prompt (batch / repeat, L); each row's states go to ``repeat`` rows of the batch (its beams).
        Returns the last position's logits (batch / repeat, vocab)."""
        if input_ids.shape[0] * repeat != self.batch:
            raise ValueError(f"batch {input_ids.shape[0]} x {repeat} != decoder batch {self.batch}")

        def mixer(m, x):
            y, states = m.prefill(self, x)
            for own, new in zip(m.states(self), states):
                own.unflatten(0, (-1, repeat)).copy_(new[:, None])
            return y

        return self._run(self.model.embedding(input_ids), mixer)

    def _run(self, h, mixer):
        """Logits from embeddings (batch, [L,] d_model): the last position's where there are several."""
        norms = [*self.norms, self.final_norm]
        w, eps = norms[0]
        x, res = rms_norm_fn(h, w, None, eps, True, True)
        last = len(self.mixers) - 1
        for i, m in enumerate(self.mixers):
            y = mixer(m, x)
            if i == last and y.dim() == 3:
                x, y, res = x[:, -1], y[:, -1], res[:, -1]
            w, eps = norms[i + 1]
            if i == last and self.parts[i] is None:
                x = rms_norm_fn(y, w, res, eps)
            else:  # the residual add of this block fused with the next norm
                x, res = join_residual(self.parts[i], x, y, res, w, eps)
        return self.model.lm_head(x).float()

    def _step_eager(self, tok):
        return self._run(self.model.embedding(tok), lambda m, x: m.step(self, x))

    def reorder(self, parents):
        """parents (batch / beams, beams) int64: row w of a prompt's beams becomes what row parents[:, w] was."""
        reorder_states(self.states, parents)

    @torch.no_grad()
    def step(self, token_ids):
        if not self.cuda_graph:
            return self._step_eager(token_ids)
        self.tok.copy_(token_ids)
        if self.graph is None:
            self._capture()
        self.graph.replay()
        return self.logits

    def _capture(self):
        # warm-up on a side stream (library handles, cuBLAS workspaces), states saved around it
        saved = [t.clone() for t in self.states]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                self._step_eager(self.tok)
        torch.cuda.current_stream().wait_stream(s)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = self._step_eager(self.tok)
        for t, v in zip(self.states, saved):
            t.copy_(v)


def _sample(logits, temperature, top_k, generator):
    if temperature == 0:
        return logits.argmax(-1)
    logits = logits / temperature
    if top_k is not None:
        kth = torch.topk(logits, top_k, dim=-1).values[:, -1:]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    return torch.multinomial(torch.softmax(logits, -1), 1, generator=generator).squeeze(-1)


@torch.no_grad()
def generate(model, input_ids, max_new_tokens: int = 50, temperature: float = 1.0, top_k: int | None = None,
             cuda_graph: bool = True, generator: torch.Generator | None = None):
    """Continue every sequence of ``input_ids`` (batch, L) by ``max_new_tokens`` tokens —
    the signature of the reference's stub CausalLM.generate (models/causal_lm.py:61), with
    ``temperature = 0`` meaning greedy.  Returns (batch, L + max_new_tokens) token ids."""
    dec = Decoder(model, input_ids.shape[0], cuda_graph=cuda_graph)
    out = [input_ids]
    logits = dec.prefill(input_ids)
    for i in range(max_new_tokens):
        tok = _sample(logits, temperature, top_k, generator)
        out.append(tok[:, None])
        if i + 1 < max_new_tokens:
            logits = dec.step(tok)
    return torch.cat(out, 1)


@torch.no_grad()
def beam_search(model, input_ids, num_beams: int, max_new_tokens: int = 50, eos_token_id: int | None = None,
                length_penalty: float = 1.0, cuda_graph: bool = True):
    """The most probable continuation found with ``num_beams`` beams for every sequence of ``input_ids``
    (batch, L).  A beam that emits eos_token_id is finished and keeps its place and its score, its row
    filled with eos_token_id.  The beams of a prompt are ranked by score / length ** length_penalty, length
    counting new tokens up to the first eos.  Returns (ids (batch, L + T) of the best beam, its ranking
    score (batch,)), T <= max_new_tokens (less when every beam has finished)."""
    if num_beams < 1:
        raise ValueError(f"num_beams {num_beams}")
    b, l = input_ids.shape
    if max_new_tokens < 1:
        return input_ids, torch.zeros(b, device=input_ids.device)
    w, dev = num_beams, input_ids.device
    dec = Decoder(model, b * w, cuda_graph=cuda_graph)
    logits = dec.prefill(input_ids, repeat=w)
    # the first step chooses among one beam's tokens: the others are copies of it
    scores = torch.full((b, w), float("-inf"), device=dev)
    scores[:, 0] = 0.0
    logits = logits[:, None].expand(b, w, logits.shape[-1])
    done = torch.zeros(b, w, dtype=torch.bool, device=dev)
    length = torch.zeros(b, w, dtype=torch.long, device=dev)
    ids = input_ids[:, None].expand(b, w, l)
    for i in range(max_new_tokens):
        marks = (None, None) if eos_token_id is None else (done, eos_token_id)
        scores, parents, tokens = beam_select(logits, scores, None, *marks)
        ids = torch.cat([ids.gather(1, parents[..., None].expand_as(ids)), tokens[..., None]], -1)
        done, length = done.gather(1, parents), length.gather(1, parents)
        length = length + (~done)
        if eos_token_id is not None:
            done = done | (tokens == eos_token_id)
            if bool(done.all()):
                break
        if i + 1 < max_new_tokens:
            if i > 0:  # after the prompt every beam has the same states
                dec.reorder(parents)
            logits = dec.step(tokens.flatten()).unflatten(0, (b, w))
    rank = scores / length.clamp(min=1).float() ** length_penalty
    best = rank.argmax(-1)
    rows = torch.arange(b, device=dev)
    return ids[rows, best], rank[rows, best]
