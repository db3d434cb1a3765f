"""A CausalLM-shaped model's forward through the fused paths.

The reference's ``CausalLM.forward`` (models/causal_lm.py:50-58) runs, per block,
``h = h + dropout(mamba(norm(h)))`` (Block.forward, :30-37) with a PyTorch RMSNorm, the
MambaSimple block (permute copies, separate conv / SiLU / gate kernels) and an in-place
residual add, then a final RMSNorm and the tied lm_head.  ``causal_lm_forward(model, ids)``
computes the same logits from the same parameters with:

* ``rms_norm(..., residual=..., prenorm=True)`` — the residual add of one block fused with the
  RMSNorm that starts the next (and with the final norm);
* ``mamba_simple_forward`` — the fused block (conv + SiLU kernel, batched GEMMs, gated scan).

It is differentiable end to end (training) and applies the blocks' dropout modules as the
reference does.  The model is duck-typed on the reference's module tree.

Layers may also hold what the reference's do not:

* ``linear_attn`` in place of ``mamba``: a linear-attention mixer (``linear_attention_forward``);
* ``post_norm`` (an RMSNorm behind the block), ``gate_proj`` (a projection of the block's input whose
  SiLU gates the block's output) and ``residual_scale`` (a (d_model,) parameter or a number on the
  block's branch): they run with the residual add and the next norm in one pass (``block_norm_fn``).
"""
from __future__ import annotations

from .inner import mamba_simple_forward
from .linear_attention import linear_attention_forward
from .norm import block_norm_fn, rms_norm, rms_norm_fn


def branch_parts(layer, norm):
    """(post weight, gate projection, residual scale, epsilons) of a layer whose branch has any of them, else
    None; ``norm`` is the RMSNorm that follows the layer."""
    post, gate = getattr(layer, "post_norm", None), getattr(layer, "gate_proj", None)
    scale = getattr(layer, "residual_scale", None)
    if post is None and gate is None and scale is None:
        return None
    return (None if post is None else post.weight), gate, scale, (norm if post is None else post).eps, norm.eps


def join_residual(parts, x, y, residual, weight, eps):
    """The next block's input and residual stream from block output y, block input x and the residual stream:
    the plain residual add and norm, or the layer's post norm, gate and scale with them."""
    if parts is None:
        return rms_norm_fn(y, weight, residual, eps, True, True)
    post, gate, scale, post_eps, pre_eps = parts
    return block_norm_fn(y, residual, post, weight, None if gate is None else gate(x), scale, "silu", post_eps, pre_eps)


def mixer_forward(layer, x):
    mixer = getattr(layer, "linear_attn", None)
    return mamba_simple_forward(layer.mamba, x) if mixer is None else linear_attention_forward(mixer, x)


def causal_lm_hidden(model, input_ids):
    """Final normalised hidden states (batch, L, d_model)."""
    h = model.embedding(input_ids)
    layers = list(model.layers)
    if not layers:
        return rms_norm(model.norm, h)
    x, res = rms_norm(layers[0].norm, h, prenorm=True)
    for i, layer in enumerate(layers):
        y = mixer_forward(layer, x)
        drop = getattr(layer, "dropout", None)
        if drop is not None:
            y = drop(y)
        last = i + 1 == len(layers)
        norm = model.norm if last else layers[i + 1].norm
        parts = branch_parts(layer, norm)
        if last and parts is None:
            return rms_norm(norm, y, residual=res)
        x, res = join_residual(parts, x, y, res, norm.weight, norm.eps)
    return x


def causal_lm_forward(model, input_ids):
    """Logits (batch, L, vocab) of a reference CausalLM (models/causal_lm.py:50-58)."""
    return model.lm_head(causal_lm_hidden(model, input_ids))
