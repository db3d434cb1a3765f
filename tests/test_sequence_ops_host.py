"""Host-side checks of the sequence operators that need no GPU: the arguments they refuse, in Python
(with the device check taken out, on CPU tensors: every refusal comes before the library is called)
and at the C boundary (dummy pointers: rejected before any device access), and the sizes of their workspaces."""
import ctypes

import pytest
import torch

import mamba_b200
import mamba_b200._lib as L
from mamba_b200 import beam as beam_mod
from mamba_b200 import linear_attention as la_mod
from mamba_b200 import norm as norm_mod


@pytest.fixture
def on_cpu(monkeypatch):
    for m in (beam_mod, la_mod, norm_mod):
        monkeypatch.setattr(m, "_cuda_device", lambda *t: torch.device("cpu"))


def test_cpu_tensors_fail_loudly():
    t = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        mamba_b200.linear_attention_fn(t, t, t, torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        mamba_b200.linear_attention_step(torch.zeros(1, 2, 8, 8), t[:, 0], t[:, 0], t[:, 0], torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        mamba_b200.block_norm_fn(t, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        mamba_b200.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        mamba_b200.reorder_states([torch.zeros(2, 3)], torch.zeros(1, 2, dtype=torch.int64))


def _qkv(**kw):
    a = dict(q=(2, 5, 2, 8), k=(2, 5, 2, 8), v=(2, 5, 4, 6), g=(2, 5, 4))
    a.update(kw)
    return [torch.zeros(*a[n]) for n in ("q", "k", "v", "g")]


@pytest.mark.parametrize("kw,error", [
    (dict(q=(2, 5, 8)), ValueError), (dict(v=(2, 5, 6)), ValueError), (dict(q=(2, 4, 2, 8)), ValueError),
    (dict(k=(2, 5, 2, 7)), ValueError), (dict(q=(2, 5, 3, 8), k=(2, 5, 3, 8)), ValueError),
    (dict(q=(2, 5, 0, 8), k=(2, 5, 0, 8)), ValueError), (dict(q=(2, 5, 2, 0), k=(2, 5, 2, 0)), ValueError),
    (dict(q=(2, 5, 2, 129), k=(2, 5, 2, 129)), NotImplementedError), (dict(v=(2, 5, 4, 130)), NotImplementedError),
    (dict(g=(2, 5, 2)), ValueError), (dict(g=(2,)), ValueError), (dict(g=(5, 4)), ValueError)])
def test_linear_attention_refuses_shapes(on_cpu, kw, error):
    with pytest.raises(error):
        mamba_b200.linear_attention_fn(*_qkv(**kw))


@pytest.mark.parametrize("kw,error", [
    (dict(scale=0.0), ValueError), (dict(scale=float("nan")), ValueError), (dict(scale=float("inf")), ValueError),
    (dict(initial_state=torch.zeros(2, 4, 6, 8)), ValueError), (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(seq_lens=torch.zeros(2)), ValueError), (dict(seq_lens=torch.zeros(2, dtype=torch.bool)), ValueError)])
def test_linear_attention_refuses_options(on_cpu, kw, error):
    with pytest.raises(error):
        mamba_b200.linear_attention_fn(*_qkv(), **kw)


def test_linear_attention_refuses_types(on_cpu):
    q, k, v, g = _qkv()
    with pytest.raises(NotImplementedError):
        mamba_b200.linear_attention_fn(q, k, v.double(), g)


@pytest.mark.parametrize("state,g", [(torch.zeros(2, 4, 6, 8), (2, 4)), (torch.zeros(2, 4, 8, 6).double(), (2, 4)),
                                     (torch.zeros(2, 4, 6, 8).transpose(2, 3), (2, 4)), (torch.zeros(2, 4, 8, 6), (2, 2)),
                                     (torch.zeros(1, 4, 8, 6).expand(2, 4, 8, 6), (2, 4))])
def test_linear_step_refuses(on_cpu, state, g):
    with pytest.raises(ValueError):
        mamba_b200.linear_attention_step(state, torch.zeros(2, 2, 8), torch.zeros(2, 2, 8), torch.zeros(2, 4, 6), torch.zeros(*g))


@pytest.mark.parametrize("kw,error", [
    (dict(residual=torch.zeros(3, 7)), ValueError), (dict(gate=torch.zeros(1, 8)), ValueError),
    (dict(post_weight=torch.zeros(7)), ValueError), (dict(pre_weight=torch.zeros(1, 8)), ValueError),
    (dict(residual_scale=torch.zeros(())), ValueError), (dict(activation="relu"), ValueError),
    (dict(y=torch.zeros(2, 8193), residual=torch.zeros(2, 8193)), NotImplementedError),
    (dict(y=torch.zeros(3, 8).double()), NotImplementedError), (dict(y=torch.zeros(3, 0), residual=torch.zeros(3, 0)), ValueError)])
def test_block_norm_refuses(on_cpu, kw, error):
    args = dict(y=torch.zeros(3, 8), residual=torch.zeros(3, 8))
    args.update(kw)
    with pytest.raises(error):
        mamba_b200.block_norm_fn(**args)


@pytest.mark.parametrize("kw,error", [
    (dict(logits=torch.zeros(2, 9)), ValueError), (dict(scores=torch.zeros(2, 2)), ValueError), (dict(num_select=0), ValueError),
    (dict(num_select=28), ValueError), (dict(logits=torch.zeros(2, 3, 0)), ValueError),
    (dict(logits=torch.zeros(2, 33, 9), scores=torch.zeros(2, 33)), NotImplementedError),
    (dict(logits=torch.zeros(2, 3, 90), num_select=33), NotImplementedError),
    (dict(finished=torch.zeros(2, 3, dtype=torch.bool)), ValueError), (dict(eos_token_id=1), ValueError),
    (dict(finished=torch.zeros(2, 3, dtype=torch.bool), eos_token_id=9), ValueError),
    (dict(finished=torch.zeros(2, 3, dtype=torch.bool), eos_token_id=-1), ValueError),
    (dict(finished=torch.zeros(2, 3), eos_token_id=1), ValueError), (dict(logits=torch.zeros(2, 3, 9).double()), NotImplementedError)])
def test_beam_select_refuses(on_cpu, kw, error):
    args = dict(logits=torch.zeros(2, 3, 9), scores=torch.zeros(2, 3))
    args.update(kw)
    with pytest.raises(error):
        mamba_b200.beam_select(**args)


_S = torch.zeros(6, 4)


@pytest.mark.parametrize("states,parents,error", [
    ([torch.zeros(5, 4)], torch.zeros(2, 3, dtype=torch.int64), ValueError),
    ([torch.zeros(4, 6).t()], torch.zeros(2, 3, dtype=torch.int64), ValueError),
    ([torch.zeros(6, 3, dtype=torch.uint8)], torch.zeros(2, 3, dtype=torch.int64), NotImplementedError),
    ([torch.zeros(6, 3, dtype=torch.float16)], torch.zeros(2, 3, dtype=torch.int64), NotImplementedError),
    ([_S], torch.zeros(2, 3, dtype=torch.int32), ValueError), ([_S], torch.zeros(6, dtype=torch.int64), ValueError),
    ([_S], torch.zeros(2, 0, dtype=torch.int64), ValueError), ([_S, _S], torch.zeros(2, 3, dtype=torch.int64), ValueError),
    ([torch.zeros(33, 4)], torch.zeros(1, 33, dtype=torch.int64), NotImplementedError),
    ([torch.zeros(13, dtype=torch.float16)[1:].view(6, 2)], torch.zeros(2, 3, dtype=torch.int64), NotImplementedError)])
def test_reorder_refuses(on_cpu, states, parents, error):
    with pytest.raises(error):
        mamba_b200.reorder_states(states, parents)


def _linear_args(**kw):
    a = L.LinearArgs()
    a.batch, a.seqlen, a.heads, a.key_heads, a.key_dim, a.value_dim, a.scale = 1, 300, 4, 2, 64, 64, 0.5
    a.io_dtype = a.decay_dtype = L.SS_BF16
    for f in ("q", "k", "v", "log_decay", "o", "work"):
        setattr(a, f, 0x1000)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), 1), (dict(heads=3), 1), (dict(key_heads=0), 1), (dict(key_dim=0), 1), (dict(scale=0.0), 1),
    (dict(scale=float("inf")), 1), (dict(q=None), 1), (dict(log_decay=None), 1), (dict(o=None), 1), (dict(key_dim=129), 2),
    (dict(value_dim=129), 2), (dict(io_dtype=7), 2), (dict(decay_dtype=L.SS_F16), 2), (dict(batch=0), 0),
    (dict(scale=1e-40), 1), (dict(seqlen=2 ** 30 + 1), 2), (dict(work=0x1008), 1), (dict(work=None), 1)])
def test_c_boundary_of_linear_attention(kw, status):
    assert L.lib().ss_linear_fwd(ctypes.byref(_linear_args(**kw)), None) == status


def test_c_boundary_null_arguments():
    for f in ("ss_linear_fwd", "ss_linear_bwd", "ss_linear_step", "ss_block_norm_fwd", "ss_block_norm_bwd", "ss_beam_select",
              "ss_reorder"):
        assert getattr(L.lib(), f)(None, None) == L.SS_ERR_INVALID, f


def test_c_boundary_missing_gradients():
    g = L.LinearBwdArgs()
    g.f = _linear_args()
    assert L.lib().ss_linear_bwd(ctypes.byref(g), None) == L.SS_ERR_INVALID
    b = L.BlockNormBwdArgs()
    b.f.rows, b.f.dim, b.f.y, b.f.residual, b.f.y_row_stride, b.f.residual_row_stride = 2, 8, 0x1000, 0x1000, 8, 8
    assert L.lib().ss_block_norm_bwd(ctypes.byref(b), None) == L.SS_ERR_INVALID


def test_c_boundary_alignment_and_limits():
    b = L.BlockNormArgs()
    b.rows, b.dim, b.y_row_stride, b.residual_row_stride, b.h_row_stride = 2, 8, 8, 8, 8
    b.y = b.residual = b.h = 0x1000
    b.rstd = 0x1004
    assert L.lib().ss_block_norm_fwd(ctypes.byref(b), None) == L.SS_ERR_INVALID
    s = L.BeamArgs(1, 1, 2 ** 30 + 1, 1, L.SS_F16, 0, 0x1000, 2 ** 30 + 1, 2 ** 30 + 1, 0x1000, None, 0x1000, 0x1000, 0x1000,
                   0x1000)
    assert L.lib().ss_beam_select(ctypes.byref(s), None) == L.SS_ERR_UNSUPPORTED
    s.vocab, s.work = 100, 0x1008
    assert L.lib().ss_beam_select(ctypes.byref(s), None) == L.SS_ERR_INVALID


def test_workspace_sizes():
    lib = L.lib()
    assert lib.ss_beam_work_bytes(0, 4, 100, 4) == 0 and lib.ss_beam_work_bytes(1, 4, 100, 0) == 0
    assert lib.ss_beam_work_bytes(1, 4, 100, 4) == 4 * (16 + 4 * 8)      # one slice a beam
    assert lib.ss_block_norm_work_elems(0, 768, L.SS_BF16) == 0
    assert lib.ss_block_norm_work_elems(5, 768, L.SS_BF16) == 2 * 2 * 768  # two CTAs of four rows
    assert lib.ss_linear_work_bytes(ctypes.byref(_linear_args(batch=-1)), 0) == 0
    # many heads: one segment, nothing but the backward's row sums and the groups' parts
    a = _linear_args(batch=64, heads=8, key_heads=4)
    assert lib.ss_linear_work_bytes(ctypes.byref(a), 0) == 0
    assert lib.ss_linear_work_bytes(ctypes.byref(a), 1) >= 2 * 64 * 8 * 300 * 4 * (1 + 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q,k,v,state", [((1, 5, 2, 60), (1, 5, 2, 64), (1, 5, 2, 64), None),
                                         ((1, 5, 2, 33), (1, 5, 2, 40), (1, 5, 2, 57), None),
                                         ((1, 5, 2, 33), (1, 5, 2, 33), (1, 5, 2, 57), (1, 2, 40, 64)),
                                         ((1, 5, 2, 64), (1, 5, 2, 64), (1, 5, 2, 57), (1, 2, 64, 64)),
                                         ((1, 5, 2, 33), (1, 5, 2, 33), (1, 5, 2, 57), (1, 2, 33, 64)),
                                         ((1, 4, 2, 33), (1, 4, 2, 33), (1, 5, 2, 57), None),
                                         ((1, 5, 3, 33), (1, 5, 3, 33), (1, 5, 2, 57), None),
                                         ((1, 5, 2, 33), (1, 5, 2, 33), (1, 5, 57), None)])
def test_shapes_that_padding_would_hide(on_cpu, dtype, q, k, v, state):
    """Head sizes that come to the same multiple of 8: refused by the sizes that were passed, in every type."""
    q, k, v = (torch.zeros(*s, dtype=dtype) for s in (q, k, v))
    with pytest.raises(ValueError):
        mamba_b200.linear_attention_fn(q, k, v, torch.zeros(2), initial_state=None if state is None else torch.zeros(*state))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_limits_of_head_sizes_name_what_was_passed(on_cpu, dtype):
    q, v = torch.zeros(1, 5, 2, 130, dtype=dtype), torch.zeros(1, 5, 2, 16, dtype=dtype)
    with pytest.raises(NotImplementedError, match="130"):
        mamba_b200.linear_attention_fn(q, q, v, torch.zeros(2))


def test_what_goes_through_the_autograd_functions():
    import torch.autograd.forward_ad as forward_ad

    plain, leaf = torch.zeros(2), torch.zeros(2).requires_grad_()
    assert not L.differentiated((plain, None)) and L.differentiated((None, leaf))
    with torch.no_grad():
        assert not L.differentiated((leaf,))
        with forward_ad.dual_level():
            assert L.differentiated((plain,))
    assert not L.differentiated((plain,))


def test_workspaces_of_sizes_beyond_the_limits_are_empty():
    """Sizes that the calls refuse, up to the largest int: no size (and no overflow on the way to one)."""
    lib = L.lib()
    for kw in (dict(seqlen=2 ** 31 - 1), dict(seqlen=2 ** 30 + 1), dict(batch=2 ** 23, heads=4), dict(batch=2 ** 31 - 1, heads=2 ** 31 - 1, key_heads=1)):
        a = _linear_args(**kw)
        assert lib.ss_linear_work_bytes(ctypes.byref(a), 0) == 0 and lib.ss_linear_work_bytes(ctypes.byref(a), 1) == 0, kw
        assert lib.ss_linear_fwd(ctypes.byref(a), None) != L.SS_OK
    assert lib.ss_linear_work_bytes(ctypes.byref(_linear_args(batch=1, heads=1, key_heads=1, seqlen=2 ** 30)), 1) > 2 ** 33
    for sizes in ((1, 1, 2 ** 31 - 1, 1), (1, 32, 2 ** 26, 4), (1, 33, 100, 4), (1, 4, 100, 33), (2 ** 31 - 1, 32, 2 ** 31 - 1, 32)):
        assert lib.ss_beam_work_bytes(*sizes) == 0, sizes
    assert lib.ss_beam_work_bytes(1, 32, 2 ** 25, 32) > 0
