"""Beam selection against a sort of every candidate (Python floats), and the in-place reordering.

Tokens and parents are compared exactly; scores are fp32 roundings of fp64 sums that are good to
1e-7, so one step of fp32 (2^-23 relative) apart at most, plus that."""
import math

import pytest
import torch

from sequence_ref import beam_ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(logits, scores, k=None, finished=None, eos=None):
    from mamba_b200 import beam_select

    k = k or logits.shape[1]
    s, p, t = beam_select(logits.cuda() if not logits.is_cuda else logits, scores.cuda(), k,
                          None if finished is None else finished.cuda(), eos)
    want = beam_ref(logits.cpu(), scores, k, finished, eos)
    for b, row in enumerate(want):
        assert list(zip(p[b].tolist(), t[b].tolist())) == [(w, v) for _, w, v in row], b
        for got, (c, _, _) in zip(s[b].tolist(), row):
            assert got == c or abs(got - c) <= 2.0 ** -23 * abs(c) + 2e-7, (b, got, c)


def make(b, w, vocab, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (2.5 * torch.randn(b, w, vocab, generator=g)).to(dtype), -10 - 3 * torch.rand(b, w, generator=g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,w,vocab,k", [(1, 1, 1, 1), (2, 3, 5, 3), (1, 4, 2, 8), (3, 2, 31, 4), (2, 4, 1000, 8), (1, 32, 77, 32),
                                         (2, 5, 1025, 10), (1, 4, 20011, 4), (2, 2, 4096, 32), (1, 1, 50280, 7)])
def test_sizes(dtype, b, w, vocab, k):
    check(*make(b, w, vocab, dtype, vocab), k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_finished_beams(dtype):
    logits, scores = make(4, 3, 200, dtype, 1)
    done = torch.tensor([[0, 1, 0], [1, 1, 1], [0, 0, 0], [1, 0, 1]]).bool()
    logits[done] = float("nan")  # a finished beam's logits are not read
    check(logits, scores, 6, done, 7)
    check(logits, scores, 3, done, 0)
    check(logits, scores, 3, done, 199)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_candidates_go_by_index(dtype):
    logits = torch.zeros(1, 4, 300, dtype=dtype)
    scores = torch.tensor([[-1.0, -1.0, -2.0, -1.0]])
    check(logits, scores, 4)
    check(logits, scores, 32)
    logits[:, :, 100::3] = -0.0
    check(logits, scores, 32)
    logits[0, :, 250] = 1
    logits[0, :, 17] = 1
    check(logits, scores, 8)


def test_first_step_of_a_search():
    """All beams alike, one of them alive."""
    logits, _ = make(2, 1, 500, torch.bfloat16, 2)
    check(logits.expand(2, 4, 500), torch.tensor([[0.0, -math.inf, -math.inf, -math.inf]] * 2), 4)
    check(logits.expand(2, 4, 500), torch.zeros(2, 4), 8)


def test_masked_and_broken_logits():
    logits, scores = make(6, 2, 100, torch.float32, 3)
    logits[0, :, 5:] = -math.inf          # fewer tokens than candidates
    logits[1, 0] = -math.inf              # nothing allowed in a beam
    logits[2] = -math.inf                 # nor in a row
    logits[3, 0, 9] = math.nan
    logits[4, 1, 9] = math.inf
    scores[5, 0] = math.nan
    check(logits, scores, 12)
    scores[5] = torch.tensor([math.inf, -math.inf])
    check(logits, scores, 12)


def test_ascending_logits():
    """Every element enters the lists: the worst order for them."""
    check(torch.linspace(-5, 5, 3000).expand(1, 2, 3000).contiguous(), torch.tensor([[-1.0, -1.5]]), 8)


def test_strided_logits():
    logits, scores = make(2, 3, 200, torch.bfloat16, 4)
    wide = torch.randn(2, 3, 333).bfloat16()
    wide[..., 33:233] = logits
    check(wide.cuda()[..., 33:233], scores, 5)
    check(logits.cuda().transpose(0, 1).contiguous().transpose(0, 1), scores, 5)


@pytest.mark.parametrize("w", [1, 2, 4, 5, 8, 16, 32])
@pytest.mark.parametrize("shape,dtype", [((7, 16), torch.float32), ((5, 3), torch.float32), ((64, 64), torch.bfloat16),
                                         ((6,), torch.float16), ((2,), torch.int64)])
def test_reorder(w, shape, dtype):
    from mamba_b200 import reorder_states

    b = 3
    g = torch.Generator().manual_seed(w)
    parents = torch.randint(0, w, (b, w + 2), generator=g).cuda()[:, :w]
    states = [(100 * torch.randn(b * w, *shape, generator=g)).to(dtype).cuda() for _ in range(3)]
    rows = (parents + w * torch.arange(b, device="cuda")[:, None]).flatten()
    want = [t[rows] for t in states]
    reorder_states(states, parents)
    for a, c in zip(states, want):
        assert torch.equal(a, c)


def test_reorder_many_tensors_and_bad_parents():
    from mamba_b200 import check_device_status, reorder_states

    states = [torch.randn(4, 5, device="cuda") for _ in range(70)]
    before = [t.clone() for t in states]
    reorder_states(states, torch.tensor([[1, 0], [0, 0]], device="cuda"))
    for a, c in zip(states, before):
        assert torch.equal(a, c[[1, 0, 2, 2]])
    check_device_status()
    kept = [t.clone() for t in states]
    reorder_states(states, torch.tensor([[5, 0], [1, -1]], device="cuda"))
    with pytest.raises(RuntimeError, match="parent"):
        check_device_status()
    for a, c in zip(states, kept):
        assert torch.equal(a, c[[0, 0, 3, 3]])
    reorder_states([torch.zeros(0, 3, device="cuda")], torch.zeros(0, 2, dtype=torch.int64, device="cuda"))
    reorder_states([], torch.zeros(1, 2, dtype=torch.int64, device="cuda"))


def test_selection_and_reordering_in_a_graph():
    from mamba_b200 import beam_select, reorder_states

    logits, scores = (t.cuda() for t in make(2, 4, 3000, torch.bfloat16, 6))
    state = torch.randn(8, 40, device="cuda")
    start = state.clone()

    def step():
        out = beam_select(logits, scores)
        reorder_states([state], out[1])
        return out

    want = step()
    after = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    state.copy_(start)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(state, after)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,w,vocab,k", [(1, 2, 50, 4), (2, 3, 6000, 32), (3, 2, 7, 9)])
def test_candidates_that_are_equal_though_their_logits_are_not(dtype, b, w, vocab, k):
    """Logits whose difference is lost beside the sum of exponentials, or beside the beam's score: such candidates
    are equal in fp64, and go by index like any others."""
    tiny = torch.rand(b, w, vocab, generator=torch.Generator().manual_seed(vocab)) * 1e-20
    if dtype != torch.float16:  # whose smallest number is 6e-8
        check(tiny.to(dtype), -torch.arange(1.0, w + 1).expand(b, w), k)
        tiny[..., 3] = 1.0
        check(tiny.to(dtype), -torch.arange(1.0, w + 1).expand(b, w), k)
    logits, _ = make(b, w, vocab, dtype, 9)
    for low in (-3e38, -1e30, 1e25):
        check(logits, torch.full((b, w), low), k)
        scores = torch.full((b, w), low)
        scores[:, 0] = -4.0
        check(logits, scores, k)


@pytest.mark.parametrize("b,w", [(3, 2), (4, 1), (1, 5)])
def test_reorder_by_one_order_for_the_batch(b, w):
    """Parents expanded over the batch (a batch stride of 0), and overlapping rows of a wider tensor."""
    from mamba_b200 import reorder_states

    order = torch.arange(w - 1, -1, -1, device="cuda")
    wide = torch.cat([order, order])
    for p in (order.expand(b, w), torch.as_strided(wide, (b, w), (0, 1)), torch.as_strided(torch.zeros(b + w, dtype=torch.int64, device="cuda"), (b, w), (1, 1))):
        s = torch.randn(b * w, 3, 5, device="cuda")
        want = s.view(b, w, 3, 5)[torch.arange(b, device="cuda")[:, None], p].flatten(0, 1)
        reorder_states([s], p)
        assert torch.equal(s, want)
