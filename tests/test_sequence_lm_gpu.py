"""The sequence operators together, as a model uses them: a CausalLM-shaped model with linear-attention and
MambaSimple layers, norms behind the blocks, gates and residual scales — its forward and gradients
against a float64 composition, prompt + single tokens against the full forward, and beam search over
the decoder against the same search on full forwards.

Tolerances: fp32 runs sum in other orders than the reference: 1e-4 of the largest magnitude (the model's
values are about 1, its sums a few hundred terms long); bf16 a few roundings of 2^-8 a layer, of values
that the norms bring back to 1: 5e-2 of the largest magnitude, as the other model tests."""
import pytest
import torch

from common import assert_close
from sequence_ref import block_norm_ref, linear_ref
from torch_ref import MambaSimpleRef, RMSNormRef

pytestmark = pytest.mark.gpu


class LinearMixer(torch.nn.Module):
    def __init__(self, dm, heads, key_heads, dk, dv, fixed=False):
        super().__init__()
        self.num_heads, self.num_key_heads = heads, key_heads
        self.q_proj = torch.nn.Linear(dm, key_heads * dk, bias=False)
        self.k_proj = torch.nn.Linear(dm, key_heads * dk, bias=False)
        self.v_proj = torch.nn.Linear(dm, heads * dv, bias=False)
        if fixed:
            self.log_decay = torch.nn.Parameter(-torch.rand(heads))
        else:
            self.decay_proj = torch.nn.Linear(dm, heads)
        self.output_proj = torch.nn.Linear(heads * dv, dm, bias=False)

    def forward(self, x):  # float64
        lead = x.shape[:2]
        q, k = (p(x).reshape(*lead, self.num_key_heads, -1) for p in (self.q_proj, self.k_proj))
        v = self.v_proj(x).reshape(*lead, self.num_heads, -1)
        g = torch.nn.functional.logsigmoid(self.decay_proj(x)) if hasattr(self, "decay_proj") else self.log_decay
        return self.output_proj(linear_ref(q, k, v, g, q.shape[-1] ** -0.5)[0].flatten(-2))


class Layer(torch.nn.Module):
    def __init__(self, dm, kind):
        super().__init__()
        self.norm = RMSNormRef(dm, eps=1e-5)
        if kind == "mamba":
            self.mamba = MambaSimpleRef(dm, state_dim=16, conv_bias=True)
        else:
            self.linear_attn = LinearMixer(dm, 4, 2, 16, 24, fixed=kind == "fixed")
            self.post_norm = RMSNormRef(dm, eps=1e-4)
            self.gate_proj = torch.nn.Linear(dm, dm)
            self.residual_scale = torch.nn.Parameter(0.5 + 0.1 * torch.randn(dm))


class Model(torch.nn.Module):
    def __init__(self, kinds, vocab=53, dm=32):
        super().__init__()
        self.embedding = torch.nn.Embedding(vocab, dm)
        self.layers = torch.nn.ModuleList([Layer(dm, k) for k in kinds])
        self.norm = RMSNormRef(dm, eps=1e-5)
        self.lm_head = torch.nn.Linear(dm, vocab, bias=False)
        for n in self.modules():
            if isinstance(n, RMSNormRef):
                torch.nn.init.normal_(n.weight, 0, 0.1)

    def reference(self, ids):
        """The same model from plain operations, in the parameters' type (float64 here)."""
        h = self.embedding(ids)
        x = block_norm_ref(torch.zeros_like(h), h, pre=self.layers[0].norm.weight, pre_eps=1e-5)[0]
        for i, layer in enumerate(self.layers):
            nxt = self.norm if i + 1 == len(self.layers) else self.layers[i + 1].norm
            if hasattr(layer, "mamba"):
                x, h = block_norm_ref(layer.mamba(x), h, pre=nxt.weight, pre_eps=1e-5)
            else:
                x, h = block_norm_ref(layer.linear_attn(x), h, layer.post_norm.weight, nxt.weight, layer.gate_proj(x),
                                      layer.residual_scale, eps=1e-4, pre_eps=1e-5)
        return self.lm_head(x)


KINDS = ["linear", "mamba", "fixed"]


def make(dtype, seed=0):
    torch.manual_seed(seed)
    m = Model(KINDS)
    ref = Model(KINDS)
    ref.load_state_dict(m.state_dict())
    return m.to(dtype).cuda(), ref.double().cuda()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 5e-2), (torch.float16, 5e-2)])
def test_forward_and_gradients(dtype, tol):
    from mamba_b200 import causal_lm_forward

    m, ref = make(dtype)
    with torch.no_grad():
        for p, q in zip(m.parameters(), ref.parameters()):
            q.copy_(p.double())
    ids = torch.randint(0, 53, (2, 150), generator=torch.Generator().manual_seed(1)).cuda()
    g = torch.randn(2, 150, 53, generator=torch.Generator().manual_seed(2)).cuda()
    logits = causal_lm_forward(m, ids)
    want = ref.reference(ids)
    assert logits.dtype == dtype
    assert_close("logits", logits, want, 0, tol * float(want.detach().abs().max()))
    (logits.float() * g).sum().backward()
    (want * g.double()).sum().backward()
    for (name, p), q in zip(m.named_parameters(), ref.parameters()):
        assert_close(name, p.grad, q.grad, 0, 2 * tol * float(q.grad.abs().max()))


@pytest.mark.parametrize("cuda_graph", [True, False])
def test_decoder_continues_the_prompt(cuda_graph):
    from mamba_b200 import Decoder, causal_lm_forward

    m, _ = make(torch.float32)
    ids = torch.randint(0, 53, (3, 40), generator=torch.Generator().manual_seed(3)).cuda()
    with torch.no_grad():
        full = causal_lm_forward(m, ids)
    dec = Decoder(m, 3, cuda_graph=cuda_graph)
    tol = 1e-4 * float(full.abs().max())
    assert_close("prompt", dec.prefill(ids[:, :25]), full[:, 24], 0, tol)
    for t in range(25, 40):
        assert_close(f"step {t}", dec.step(ids[:, t]), full[:, t], 0, tol)


def test_prompt_states_go_to_every_beam():
    from mamba_b200 import Decoder

    m, _ = make(torch.float32)
    ids = torch.randint(0, 53, (2, 20), generator=torch.Generator().manual_seed(4)).cuda()
    one, many = Decoder(m, 2, cuda_graph=False), Decoder(m, 6, cuda_graph=False)
    assert torch.equal(one.prefill(ids), many.prefill(ids, repeat=3))
    for a, b in zip(one.states, many.states):
        assert torch.equal(a.repeat_interleave(3, 0), b)
    with pytest.raises(ValueError):
        many.prefill(ids, repeat=2)


def _search(m, ids, w, steps, eos, penalty):
    """Beam search with a full forward for every beam and step (fp64 scores)."""
    from mamba_b200 import causal_lm_forward

    out = []
    for row in ids:
        beams = [(0.0, row.tolist(), False, 0)]
        for _ in range(steps):
            with torch.no_grad():
                logits = causal_lm_forward(m, torch.tensor([b[1] for b in beams], device="cuda"))[:, -1].double()
            logp = torch.log_softmax(logits, -1).tolist()
            cand = []
            for i, (s, seq, done, n) in enumerate(beams):
                if done:
                    cand.append((-s, i, eos, seq + [eos], True, n))
                else:
                    cand += [(-(s + lp), i, t, seq + [t], t == eos, n + 1) for t, lp in enumerate(logp[i])]
            beams = [(-c[0], c[3], c[4], c[5]) for c in sorted(cand, key=lambda c: c[:3])[:w]]
            if all(b[2] for b in beams):
                break
        out.append(max(beams, key=lambda b: b[0] / max(b[3], 1) ** penalty))
    return out


@pytest.mark.parametrize("cuda_graph", [True, False])
@pytest.mark.parametrize("w,eos,penalty", [(1, None, 1.0), (4, None, 1.0), (5, 7, 0.6), (3, 11, 1.0)])
def test_beam_search(cuda_graph, w, eos, penalty):
    """The same beams as a search on full forwards; the scores are sums of log probabilities of fp32 logits that
    differ by 1e-4 at most, over 8 tokens."""
    from mamba_b200 import beam_search

    m, _ = make(torch.float32, seed=w)
    ids = torch.randint(0, 53, (2, 9), generator=torch.Generator().manual_seed(5 + w)).cuda()
    got, score = beam_search(m, ids, w, 8, eos, penalty, cuda_graph=cuda_graph)
    for i, (s, seq, _, n) in enumerate(_search(m, ids, w, 8, eos, penalty)):
        row = got[i].tolist()
        assert row[:len(seq)] == seq and all(t == eos for t in row[len(seq):])
        assert abs(float(score[i]) - s / max(n, 1) ** penalty) <= 1e-3


def test_beam_search_refuses_and_stops():
    from mamba_b200 import beam_search

    m, _ = make(torch.float32)
    ids = torch.zeros(1, 3, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError):
        beam_search(m, ids, 0)
    with pytest.raises(NotImplementedError):
        beam_search(m, ids, 33)
    assert torch.equal(beam_search(m, ids, 2, 0)[0], ids)
