"""Linear attention with a decay per head against the recurrence in float64, token by token.

Tolerances.  Every result is a sum of products; ``magnitude`` is the same sum with every factor's
absolute value, computed by running the reference on absolute values (its gradients are sums of
positive products too).  With u the half step of the I/O dtype, the result is rounded once (u |want|),
and of each product's factors at most the weighted score and the carried state, or one of them twice,
are rounded to 16 bits on the way: 2 u magnitude, for gradients of grouped heads as well (they are
summed in fp32).  fp32 sums of n terms add n 2^-24 magnitude at most; n here is below 1024 and an
exponential adds 2^-22, so 1024 * 2^-24 = 2^-14 covers the fp32 path in the worst case; random signs
leave about sqrt(n), and 2^-17 magnitude is asked for.  States are fp32 results: with 16-bit I/O one
factor of each product is split into two 16-bit parts (u^2), so 2^-14 magnitude holds with bf16 (u^2 =
2^-16) and is asked of all types there."""
import pytest
import torch

from sequence_ref import linear_ref

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(b, l, h, hk, dk, dv, dtype, *, per_head=False, state=False, lens=None, seed=0, bias=2.0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = dict(q=rn(b, l, hk, dk).to(dtype), k=rn(b, l, hk, dk).to(dtype), v=rn(b, l, h, dv).to(dtype))
    if per_head:
        t["g"] = -torch.nn.functional.softplus(rn(h) - bias)
    else:
        t["g"] = (-torch.nn.functional.softplus(rn(b, l, h) - bias)).to(dtype)
    t["s0"] = rn(b, h, dk, dv) if state else None
    t["lens"] = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    t["do"], t["dF"] = rn(b, l, h, dv).to(dtype), rn(b, h, dk, dv)
    return {k: None if v is None else v.cuda() for k, v in t.items()}


def reference(t, scale, want_final, absolute=False):
    """o, final and the gradients in float64 (of the inputs' absolute values: the magnitudes)."""
    f = (lambda x: x.double().abs()) if absolute else (lambda x: x.double())
    leaves = [f(t[n]).requires_grad_() for n in ("q", "k", "v")]
    g = t["g"].double().requires_grad_()
    s0 = None if t["s0"] is None else f(t["s0"]).requires_grad_()
    if t["lens"] is not None:  # what stands behind a row's end is not part of the mathematics
        live = torch.arange(t["v"].shape[1], device="cuda")[None] < t["lens"][:, None]
        clean = [torch.where(live[..., None, None], x, 0.0) for x in leaves]
        gg = torch.where(live[..., None], g, 0.0) if g.dim() == 3 else g
    else:
        clean, gg = leaves, g
    o, final = linear_ref(*clean, gg, scale, s0, t["lens"])
    loss = (torch.where(live[..., None, None], f(t["do"]), 0.0) * o).sum() if t["lens"] is not None else (f(t["do"]) * o).sum()
    if want_final:
        loss = loss + (f(t["dF"]) * final).sum()
    every = leaves + [g] + ([s0] if s0 is not None else [])
    grads = torch.autograd.grad(loss, every, allow_unused=True)
    return o.detach(), final.detach(), [torch.zeros_like(x) if d is None else d for d, x in zip(grads, every)]


def close(name, got, want, mag, dtype, factor):
    """|got - want| <= (half a step of got's dtype) |want| + factor * magnitude, everywhere."""
    err = (got.double() - want).abs()
    tol = HALF[got.dtype] * want.abs() * 1.001 + factor * mag + 1e-30
    bad = err / tol
    bad = torch.where(err == 0, 0.0, bad)
    assert bool(torch.isfinite(got.double()).all()), f"{name}: not finite"
    worst = float(bad.max()) if bad.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} of the tolerance"


def decay_magnitude(t, scale, mags, mag_final, want_final):
    """Magnitude of the decays' gradient: the telescoped sum of |q| dq + |k| dk, and <dF, S>."""
    q, k = t["q"].double().abs(), t["k"].double().abs()
    h = t["v"].shape[2]
    rep = h // q.shape[2]
    # per key head the magnitudes of the group's parts are summed; each part is at most that
    x = sum((torch.where(torch.isfinite(a), a, 0.0) * m).sum(-1) for a, m in ((q, mags[0]), (k, mags[1])))
    x = x.repeat_interleave(rep, 2).flip(1).cumsum(1).flip(1)
    if want_final:
        x = x + (t["dF"].double().abs() * mag_final).sum((-1, -2))[:, None]
    return x if t["g"].dim() == 3 else x.sum((0, 1))


def check(t, scale=0.3, want_final=True, tensors=None):
    from mamba_b200 import linear_attention_fn

    dtype = t["v"].dtype
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    s0 = None if t["s0"] is None else t["s0"].detach().requires_grad_()
    out = linear_attention_fn(*(tensors(leaves) if tensors else leaves), scale=scale, initial_state=s0,
                              seq_lens=t["lens"], return_final_state=want_final)
    o, final = out if want_final else (out, None)
    seeds = [t["do"]] + ([t["dF"]] if want_final else [])
    every = leaves + ([s0] if s0 is not None else [])
    grads = torch.autograd.grad([o] + ([final] if want_final else []), every, seeds, allow_unused=True)
    want_o, want_f, want_g = reference(t, scale, want_final)
    mag_o, mag_f, mag_g = reference(t, scale, want_final, absolute=True)
    f32 = dtype == torch.float32
    soft = 2.0 ** -17 if f32 else 2 * HALF[dtype] + 2.0 ** -17
    hard = 2.0 ** -17 if f32 else 2.0 ** -14
    close("o", o, want_o, mag_o, dtype, soft)
    if want_final:
        assert final.dtype == torch.float32
        close("final", final, want_f, mag_f, dtype, hard)
    for name, got, want, mag in zip(("dq", "dk", "dv"), grads, want_g, mag_g):
        assert got.dtype == dtype
        close(name, got, want, mag, dtype, soft)
    close("dlog_decay", grads[3], want_g[3], decay_magnitude(t, scale, mag_g, mag_f, want_final), dtype, soft)
    if s0 is not None:
        close("dinitial_state", grads[4], want_g[4], mag_g[4], dtype, hard)


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,h,hk,dk,dv", [(2, 1, 2, 2, 64, 64), (1, 2, 3, 1, 8, 16), (2, 63, 2, 2, 64, 64),
                                           (1, 64, 2, 1, 128, 128), (2, 65, 4, 2, 64, 128), (1, 129, 2, 2, 128, 64),
                                           (2, 200, 2, 1, 40, 57), (1, 300, 1, 1, 33, 128), (1, 257, 2, 2, 1, 1),
                                           (1, 130, 6, 2, 72, 24)])
def test_sizes(dtype, b, l, h, hk, dk, dv):
    check(make(b, l, h, hk, dk, dv, dtype, state=True, seed=l))
    check(make(b, l, h, hk, dk, dv, dtype, seed=l + 1), want_final=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [-3.0, 0.0, 7.0])
def test_decays_from_forgetful_to_lasting(dtype, bias):
    check(make(1, 200, 2, 2, 64, 64, dtype, state=True, bias=bias, seed=5))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_decay_per_head(dtype):
    check(make(2, 150, 4, 2, 64, 64, dtype, per_head=True, state=True, seed=6))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[100, 0, 1, 170], [64, 128, 129, 65]])
def test_padded_rows(dtype, lens):
    """Rows end anywhere, one of them before its first token; what stands behind is NaN or infinite."""
    t = make(4, 170, 2, 1, 64, 64, dtype, state=True, lens=lens, seed=7)
    for i, n in enumerate(lens):
        for name in ("q", "k", "v", "g"):
            t[name][i, n:] = float("nan") if i % 2 else float("inf")
    check(t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_resets(dtype):
    """A log decay of -inf forgets what came before; its own gradient is zero."""
    t = make(1, 190, 2, 2, 64, 64, dtype, state=True, seed=8)
    t["g"][0, [0, 5, 6, 100, 128, 189]] = float("-inf")
    from mamba_b200 import linear_attention_fn

    g = t["g"].clone().requires_grad_()
    o, final = linear_attention_fn(t["q"], t["k"], t["v"], g, 0.3, t["s0"], None, True)
    want_o, want_f, _ = reference(t, 0.3, True)
    mag_o, mag_f, _ = reference(t, 0.3, True, absolute=True)
    soft = 2.0 ** -17 if dtype == torch.float32 else 2 * HALF[dtype] + 2.0 ** -17
    close("o", o, want_o, mag_o, dtype, soft)
    close("final", final, want_f, mag_f, dtype, 2.0 ** -17 if dtype == torch.float32 else 2.0 ** -14)
    (dg,) = torch.autograd.grad([o, final], [g], [t["do"], t["dF"]])
    assert bool(torch.isfinite(dg).all()) and float(dg[0, [0, 5, 6, 100, 128, 189]].abs().max()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_inputs(dtype):
    """(batch, heads, seqlen, dim) storage, a slice of a wider projection, an expanded decay."""
    t = make(2, 140, 4, 4, 64, 64, dtype, state=True, seed=9)

    def views(leaves):
        q, k, v, g = leaves
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.cat([k, v], -1)
        return q, wide[..., :64], wide[..., 64:], g.transpose(0, 2).contiguous().transpose(0, 2)

    check(t, tensors=views)


@pytest.mark.parametrize("dtype", DTYPES)
def test_misaligned_inputs(dtype):
    """Rows that start off the 16-byte boundary."""
    t = make(1, 70, 2, 2, 64, 64, dtype, seed=10)

    def views(leaves):
        q, k, v, g = leaves
        pad = lambda x: torch.cat([x.new_zeros(*x.shape[:-1], 1), x], -1)[..., 1:]  # noqa: E731
        return pad(q), pad(k), pad(v), g

    check(t, tensors=views)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sequence_is_its_halves(dtype):
    """A long row with few heads (cut into segments that run side by side) against the same row in two
    calls with the state carried over: the same sums in another grouping, so 2 roundings apart."""
    from mamba_b200 import linear_attention_fn

    t = make(1, 5000, 2, 1, 64, 64, dtype, state=True, bias=5.0, seed=11)
    o, f = linear_attention_fn(t["q"], t["k"], t["v"], t["g"], None, t["s0"], None, True)
    cut = 2113
    a, s = linear_attention_fn(t["q"][:, :cut], t["k"][:, :cut], t["v"][:, :cut], t["g"][:, :cut], None, t["s0"], None, True)
    c, s = linear_attention_fn(t["q"][:, cut:], t["k"][:, cut:], t["v"][:, cut:], t["g"][:, cut:], None, s, None, True)
    two = torch.cat([a, c], 1)
    rel = lambda x, y: float((x.double() - y.double()).norm() / y.double().norm())  # noqa: E731
    # relative 2-norms: independent roundings of u each (4 of them for 16 bits), fp32 sums below 1e-5
    assert rel(o, two) <= (1e-5 if dtype == torch.float32 else 4 * HALF[dtype])
    assert rel(f, s) <= 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,h,hk,dk,dv,lens", [(1, 4100, 1, 1, 128, 128, None), (1, 3333, 2, 1, 64, 128, None),
                                                 (2, 2600, 2, 2, 128, 64, [2600, 1301]), (3, 2050, 1, 1, 48, 40, [0, 2050, 300])])
def test_many_chunks_in_segments(dtype, b, l, h, hk, dk, dv, lens):
    """Few heads and many chunks a segment, decays that reach across segments, against the recurrence."""
    check(make(b, l, h, hk, dk, dv, dtype, state=True, bias=5.0, lens=lens, seed=l))


@pytest.mark.parametrize("sizes", [(1.0, 1.0, 1.0), (100.0, 60.0, 1e-3), (1e-3, 1e-4, 100.0), (1e-2, 100.0, 1e-3),
                                   (200.0, 1e-2, 1e-2)])
def test_range_of_fp16(sizes):
    """Scores far above and below what fp16 holds (6.1e-5 is its smallest normal number, 65504 its largest),
    of inputs that it holds; the outputs' scale is chosen so that they are normal numbers again.  The tolerance
    has fp16's smallest step (2^-24, half of it a rounding) beside the relative one: inputs of 1e-4 already
    carry that step, results below 2^-14 are rounded by it, and gradients reach down there."""
    from mamba_b200 import linear_attention_fn

    t = make(2, 300, 2, 1, 64, 64, torch.float16, seed=31)
    for n, x in zip(("q", "k", "v"), sizes):
        t[n] = (t[n].float() * x).half()
    scale = 0.1 / (sizes[0] * sizes[1] * sizes[2])
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    o, f = linear_attention_fn(*leaves, scale=scale, return_final_state=True)
    want_o, want_f, _ = reference(t, scale, False)
    mag_o, mag_f, _ = reference(t, scale, False, absolute=True)
    soft = 2 * HALF[torch.float16] + 2.0 ** -17
    close("o", o, want_o, mag_o + 2.0 ** -15, torch.float16, soft)
    close("final", f, want_f, mag_f, torch.float16, 2.0 ** -14)
    # seeds that keep the gradients in range: dq is about 1 / q of o.do, and so on
    do = (t["do"].float() * min(1.0, *sizes)).half()
    grads = torch.autograd.grad(o, leaves, do)
    ref = [x.detach().double().requires_grad_() for x in leaves]
    want = torch.autograd.grad(linear_ref(*ref, scale)[0], ref, do.double())
    pos = [x.detach().double().abs().requires_grad_() for x in leaves[:3]]
    mags = torch.autograd.grad(linear_ref(*pos, leaves[3].detach().double(), scale)[0], pos, do.double().abs())
    for name, got, w, m in zip(("dq", "dk", "dv"), grads, want, mags):
        close(name, got, w, m + 2.0 ** -15, torch.float16, soft)


@pytest.mark.parametrize("dtype", DTYPES)
def test_results_do_not_vary(dtype):
    from mamba_b200 import linear_attention_fn

    t = make(1, 1500, 4, 2, 64, 64, dtype, state=True, seed=12)

    def once():
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "s0")]
        o, f = linear_attention_fn(*leaves[:4], None, leaves[4], None, True)
        return [o, f, *torch.autograd.grad([o, f], leaves, [t["do"], t["dF"]])]

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_gradient_against_differences():
    """fp32 gradients against central differences of the operator itself along random directions."""
    from mamba_b200 import linear_attention_fn

    t = make(2, 90, 2, 1, 24, 20, torch.float32, state=True, lens=[90, 41], seed=13)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "s0")]

    def loss(ls):
        o, f = linear_attention_fn(*ls[:4], 0.3, ls[4], t["lens"], True)
        return (o.double() * t["do"].double()).sum() + (f.double() * t["dF"].double()).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in range(5):
        d = torch.randn(leaves[i].shape, generator=gen, device="cuda")
        d = d / d.norm()
        with torch.no_grad():
            hi, lo = ([x + s * d if j == i else x for j, x in enumerate(leaves)] for s in (1e-2, -1e-2))
            num = float(loss(hi) - loss(lo)) / 2e-2
        # third-order term of the difference (step^2 = 1e-4 of the gradient's scale) and fp32 noise / step
        assert abs(num - float((grads[i] * d).sum())) <= 2e-3 * float(grads[i].norm()) + 2e-3


def test_only_the_final_state_is_used():
    from mamba_b200 import linear_attention_fn

    t = make(2, 70, 2, 2, 16, 16, torch.float32, seed=14)
    leaves = [t[n].detach().requires_grad_() for n in ("k", "v")]
    _, f = linear_attention_fn(t["q"], *leaves, t["g"], return_final_state=True)
    got = torch.autograd.grad(f, leaves, t["dF"])
    ref = [x.detach().double().requires_grad_() for x in leaves]
    _, rf = linear_ref(t["q"].double(), *ref, t["g"].double(), 1.0)
    for a, b in zip(got, torch.autograd.grad(rf, ref, t["dF"].double())):
        assert float((a.double() - b).abs().max()) <= 2.0 ** -17 * float(b.abs().max()) * 16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hk", [4, 2, 1])
def test_gradients_without_the_decays(dtype, hk):
    """A fixed decay (no gradient asked for), own and shared key heads, one leaf at a time."""
    from mamba_b200 import linear_attention_fn

    t = make(2, 150, 4, hk, 64, 64, dtype, state=True, seed=32 + hk)
    all_of = [t[n].detach().requires_grad_() for n in ("q", "k", "v")]
    together = torch.autograd.grad(linear_attention_fn(*all_of, t["g"], 0.3, t["s0"]), all_of, t["do"])
    _, _, want = reference(t, 0.3, False)
    _, _, mags = reference(t, 0.3, False, absolute=True)
    soft = 2.0 ** -17 if dtype == torch.float32 else 2 * HALF[dtype] + 2.0 ** -17
    for i, name in enumerate(("dq", "dk", "dv")):
        close(name, together[i], want[i], mags[i], dtype, soft)
        args = [x.requires_grad_(j == i) for j, x in enumerate(t[n].detach().clone() for n in ("q", "k", "v"))]
        (alone,) = torch.autograd.grad(linear_attention_fn(*args, t["g"], 0.3, t["s0"]), [args[i]], t["do"])
        assert torch.equal(alone, together[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_broadcast_output_gradients(dtype):
    """The gradient of a sum (all strides zero) and of a sum over heads."""
    from mamba_b200 import linear_attention_fn

    t = make(2, 70, 4, 2, 32, 32, dtype, seed=36)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    o = linear_attention_fn(*leaves)
    for do in (torch.ones((), device="cuda", dtype=dtype).expand_as(o), t["do"][:, :, :1].expand_as(o)):
        a = torch.autograd.grad(o, leaves, do, retain_graph=True)
        b = torch.autograd.grad(o, leaves, do.contiguous(), retain_graph=True)
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dk,dv,per_head", [(33, 57, False), (128, 100, True)])
def test_rows_off_16_bytes_on_the_fp32_units(dtype, dk, dv, per_head):
    """LinearAttentionFn takes its operands as they are: 16-bit rows that TMA cannot copy."""
    from mamba_b200 import LinearAttentionFn

    t = make(2, 150, 4, 2, dk, dv, dtype, per_head=per_head, state=True, lens=[150, 77], seed=37)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "s0")]
    o, f = LinearAttentionFn.apply(*leaves[:4], 0.3, leaves[4], t["lens"], True)
    grads = torch.autograd.grad([o, f], leaves, [t["do"], t["dF"]])
    want_o, want_f, want = reference(t, 0.3, True)
    mag_o, mag_f, mags = reference(t, 0.3, True, absolute=True)
    close("o", o, want_o, mag_o, dtype, 2.0 ** -17)
    close("final", f, want_f, mag_f, dtype, 2.0 ** -17)
    for i, name in ((0, "dq"), (1, "dk"), (2, "dv"), (4, "dinitial_state")):
        close(name, grads[i], want[i], mags[i], dtype, 2.0 ** -17)
    close("dlog_decay", grads[3], want[3], decay_magnitude(t, 0.3, mags, mag_f, True), dtype, 2.0 ** -17)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 state entries (8.7 GB): the last row steps and moves as it does alone."""
    from mamba_b200 import linear_attention_step, reorder_states

    b, h, d = 3302, 40, 128
    state = torch.empty(b, h, d, d, device="cuda")
    assert state.numel() > 2 ** 31
    state[-2:] = torch.randn(2, h, d, d, device="cuda")
    state[:-2] = 0.0
    alone = state[-2:].clone()
    q, k, v = (torch.randn(b, h, d, device="cuda") for _ in range(3))
    g = -torch.rand(h, device="cuda")
    o = linear_attention_step(state, q, k, v, g)
    assert torch.equal(o[-2:], linear_attention_step(alone, q[-2:], k[-2:], v[-2:], g)) and torch.equal(state[-2:], alone)
    reorder_states([state], torch.tensor([[1, 0]], device="cuda").expand(b // 2, 2).contiguous())
    assert torch.equal(state[-2:], alone.flip(0))
    del state
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_calls(dtype):
    from mamba_b200 import linear_attention_fn

    t = make(2, 0, 2, 2, 16, 16, dtype, state=True)
    o, f = linear_attention_fn(t["q"], t["k"], t["v"], t["g"], 0.5, t["s0"], None, True)
    assert o.shape == (2, 0, 2, 16) and torch.equal(f, t["s0"])
    t = make(0, 5, 2, 2, 16, 16, dtype)
    o, f = linear_attention_fn(t["q"], t["k"], t["v"], t["g"], return_final_state=True)
    assert o.shape == (0, 5, 2, 16) and f.shape == (0, 2, 16, 16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,h,hk,dk,dv,per_head", [(1, 2, 2, 64, 64, False), (3, 6, 2, 128, 128, True), (2, 3, 1, 33, 57, False),
                                                  (5, 4, 4, 128, 64, True), (1, 1, 1, 1, 1, False), (70, 2, 1, 16, 100, False)])
def test_step(dtype, b, h, hk, dk, dv, per_head):
    """Tokens one by one against the float64 recurrence; the state is fp32 arithmetic throughout
    (a step: three roundings of 2^-24 each), the output rounded once."""
    from mamba_b200 import linear_attention_step

    t = make(b, 5, h, hk, dk, dv, dtype, per_head=per_head, state=True, seed=b + dk)
    s = t["s0"].clone()
    at = lambda x, i: x[:, i] if x.dim() > 1 else x  # noqa: E731
    outs = [linear_attention_step(s, t["q"][:, i], t["k"][:, i], t["v"][:, i], at(t["g"], i), 0.3) for i in range(5)]
    want_o, want_f = linear_ref(*(t[n].double() for n in ("q", "k", "v", "g")), 0.3, t["s0"].double())
    mag_o, mag_f = linear_ref(*(t[n].double().abs() for n in ("q", "k", "v")), t["g"].double(), 0.3, t["s0"].double().abs())
    close("o", torch.stack(outs, 1), want_o, mag_o, dtype, 2.0 ** -18)
    close("state", s, want_f, mag_f, dtype, 2.0 ** -20)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_continue_a_prompt(dtype):
    from mamba_b200 import linear_attention_fn, linear_attention_step

    t = make(2, 90, 4, 2, 64, 64, dtype, seed=21)
    whole, f = linear_attention_fn(t["q"], t["k"], t["v"], t["g"], return_final_state=True)
    _, s = linear_attention_fn(*(t[n][:, :80] for n in ("q", "k", "v", "g")), return_final_state=True)
    for i in range(80, 90):
        o = linear_attention_step(s, t["q"][:, i], t["k"][:, i], t["v"][:, i], t["g"][:, i])
        err = float((o.double() - whole[:, i].double()).norm() / whole[:, i].double().norm())
        assert err <= (1e-5 if dtype == torch.float32 else 4 * HALF[dtype])
    assert float((s - f).norm() / f.norm()) <= 1e-4


def test_step_on_strided_state_rows():
    """A slice of a larger cache (batch stride wider than the state); the rows between stay as they are."""
    from mamba_b200 import linear_attention_step

    t = make(3, 1, 2, 2, 16, 16, torch.float32, state=True, seed=22)
    cache = torch.full((3, 5, 16, 16), 7.0, device="cuda")
    cache[:, 1:3] = t["s0"]
    packed = t["s0"].clone()
    args = t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"][:, 0]
    o = linear_attention_step(cache[:, 1:3], *args)
    assert torch.equal(o, linear_attention_step(packed, *args))
    assert torch.equal(cache[:, 1:3], packed) and bool((cache[:, [0, 3, 4]] == 7).all())


def test_gradients_of_an_empty_sequence():
    from mamba_b200 import linear_attention_fn

    for dtype in DTYPES:
        t = make(2, 0, 2, 1, 16, 16, dtype, state=True)
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "s0")]
        o, f = linear_attention_fn(*leaves[:4], 0.5, leaves[4], None, True)
        grads = torch.autograd.grad([o, f], leaves, [t["do"], t["dF"]])
        assert all(g.shape == x.shape for g, x in zip(grads, leaves))
        # the state passes through; its gradient carries the scale and its reciprocal, exact at a power of two
        assert torch.equal(grads[4], t["dF"])


def test_a_state_that_a_backward_needs_cannot_be_stepped():
    from mamba_b200 import linear_attention_fn, linear_attention_step

    t = make(1, 20, 2, 2, 16, 16, torch.float32, seed=25)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    o, f = linear_attention_fn(*leaves, return_final_state=True)
    with torch.no_grad():
        linear_attention_step(f, t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"][:, 0])
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(o.sum() + f.sum(), leaves)
    with torch.inference_mode():
        s = torch.zeros(1, 2, 16, 16, device="cuda")
        linear_attention_step(s, t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"][:, 0])
        assert float(s.abs().max()) > 0


def test_a_second_derivative_is_refused():
    from mamba_b200 import block_norm_fn, linear_attention_fn

    t = make(1, 20, 2, 2, 16, 16, torch.float32, seed=29)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    y, w = torch.randn(3, 16, device="cuda").requires_grad_(), torch.zeros(16, device="cuda")
    for out, xs in ((linear_attention_fn(*leaves), leaves), (block_norm_fn(y, y.detach(), w), [y])):
        plain = torch.autograd.grad(out.square().sum(), xs, retain_graph=True)
        grads = torch.autograd.grad(out.square().sum(), xs, create_graph=True)
        for a, b in zip(plain, grads):
            assert torch.equal(a, b)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grads[0].sum(), xs)


def test_two_streams_at_once():
    from mamba_b200 import linear_attention_fn

    ts = [make(1, 2000, 2, 1, 64, 64, torch.bfloat16, state=True, seed=26 + i) for i in range(2)]

    def once(t):
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "s0")]
        o, f = linear_attention_fn(*leaves[:4], None, leaves[4], None, True)
        return [o, f, *torch.autograd.grad([o, f], leaves, [t["do"], t["dF"]])]

    want = [once(t) for t in ts]
    streams = [torch.cuda.Stream() for _ in ts]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for t, s in zip(ts, streams):
            with torch.cuda.stream(s):
                got.append(once(t))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for a, b in zip(g, want[i % 2]):
            assert torch.equal(a, b)


def test_runs_on_another_stream_and_in_a_graph():
    from mamba_b200 import linear_attention_fn

    t = make(2, 300, 2, 2, 64, 64, torch.bfloat16, state=True, seed=23)
    call = lambda: linear_attention_fn(t["q"], t["k"], t["v"], t["g"], None, t["s0"], None, True)  # noqa: E731
    o, f = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, f2 = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o2) and torch.equal(f, f2)
    graphs = []
    for _ in range(2):  # two graphs alive at once, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    t["v"].mul_(0.5)
    want = call()
    for graph, out in graphs + graphs:
        graph.replay()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_training_step_in_a_graph():
    from mamba_b200 import linear_attention_fn

    t = make(2, 200, 4, 2, 64, 64, torch.bfloat16, seed=24)
    leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]
    step = lambda: torch.autograd.grad(linear_attention_fn(*leaves), leaves, t["do"])  # noqa: E731
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l", [(0, 5), (2, 0)])
def test_decays_of_heads_have_a_zero_gradient_without_tokens(dtype, b, l):
    """No rows, or no tokens: the gradient of one decay per head is not empty, and is zero (exactly; the
    allocator is left with NaN where the call finds its memory)."""
    from mamba_b200 import linear_attention_fn

    for decay_dtype in {torch.float32, dtype}:
        t = make(b, l, 4, 2, 16, 16, dtype, per_head=True, state=True)
        leaves = [t["g"].to(decay_dtype).requires_grad_(), t["s0"].requires_grad_()]
        o, f = linear_attention_fn(t["q"], t["k"], t["v"], leaves[0], 0.5, leaves[1], None, True)
        held = [torch.full((n,), float("nan"), device="cuda") for n in (1, 4, 64, 128, 256) for _ in range(8)]
        del held
        dg, ds = torch.autograd.grad([o, f], leaves, [t["do"], t["dF"]])
        assert dg.dtype == decay_dtype and torch.equal(dg, torch.zeros_like(leaves[0])) and torch.equal(ds, t["dF"])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_new_thread_runs_the_same_kernels(dtype):
    """The first call that a thread makes (as autograd's do), every buffer at hand already: forward and backward
    give the bits of any other call."""
    import threading

    from mamba_b200 import linear_attention_fn

    t = make(1, 150, 2, 1, 64, 64, dtype, state=True, seed=41)
    got = []

    def once():
        with torch.no_grad():
            o, f = linear_attention_fn(t["q"], t["k"], t["v"], t["g"], None, t["s0"], None, True)
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "s0")]
        out = linear_attention_fn(*leaves[:4], None, leaves[4], None, True)
        got.append([o, f, *torch.autograd.grad(list(out), leaves, [t["do"], t["dF"]])])

    once()
    once()
    torch.cuda.synchronize()
    del got[0]  # its memory serves the next call
    thread = threading.Thread(target=once)
    thread.start()
    thread.join()
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dq,dk,dv,state", [(60, 64, 64, None), (33, 40, 57, None), (33, 33, 57, (40, 64)), (64, 64, 57, (64, 64))])
def test_shapes_that_padding_would_hide(dtype, dq, dk, dv, state):
    """Operands and states of another size than their counterparts', equal to it in multiples of 8, are refused."""
    from mamba_b200 import linear_attention_fn

    z = lambda d: torch.zeros(1, 20, 2, d, dtype=dtype, device="cuda")  # noqa: E731
    s = None if state is None else torch.zeros(1, 2, *state, device="cuda")
    with pytest.raises(ValueError):
        linear_attention_fn(z(dq), z(dk), z(dv), torch.zeros(2, device="cuda"), initial_state=s, return_final_state=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_state_that_no_backward_needs_can_be_stepped(dtype):
    """With fixed decays no gradient reads the final state: it may be stepped in place before the backward, which
    gives the same bits."""
    from mamba_b200 import linear_attention_fn, linear_attention_step

    t = make(1, 150, 2, 1, 16, 24, dtype, state=True, seed=42)

    def once(step):
        leaves = [t[n].detach().requires_grad_() for n in ("q", "k", "v", "s0")]
        o, f = linear_attention_fn(*leaves[:3], t["g"], 0.3, leaves[3], None, True)
        if step:
            with torch.no_grad():
                linear_attention_step(f, t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"][:, 0])
        return torch.autograd.grad([o, f], leaves, [t["do"], t["dF"]])

    for a, b in zip(once(True), once(False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,h,hk", [(1, 150, 2, 1), (1, 1, 2, 2), (2, 150, 1, 1), (1, 1, 1, 1)])
def test_strides_of_axes_of_one_do_not_matter(dtype, b, l, h, hk):
    """The stride of an axis of one element is never stepped along: whatever it is, forward and backward run the same
    kernels, and give the bits of the contiguous call."""
    from mamba_b200 import linear_attention_fn

    t = make(b, l, h, hk, 64, 64, dtype, seed=43)

    def odd(x):
        return torch.as_strided(x, x.shape, [7 if n == 1 else s for n, s in zip(x.shape[:-1], x.stride())] + [1])

    def once(view):
        leaves = [view(t[n]).detach().requires_grad_() for n in ("q", "k", "v")] + [t["g"].detach().requires_grad_()]
        o = linear_attention_fn(*leaves)
        return [o, *torch.autograd.grad(o, leaves, t["do"])]

    for x, y in zip(once(odd), once(lambda x: x)):
        assert torch.equal(x, y)


def decay_gradient(t, scale):
    """dlog_decay of the outputs alone in float64, from every pair of tokens: the weight of (i, j) holds the decays of
    j < t <= i.  Also the same sum of absolute values, and the largest sum over a token's own pairs.  A reset is -1e5."""
    q, k = (t[n].double().repeat_interleave(t["v"].shape[2] // t[n].shape[2], 2) for n in ("q", "k"))
    b, l, h, _ = t["v"].shape
    g = t["g"].double().clamp(min=-1e5).expand(b, l, h)
    G = g.cumsum(1).transpose(1, 2)
    D = torch.exp(torch.where(torch.ones(l, l, device="cuda").tril() > 0, G[..., :, None] - G[..., None, :], -torch.inf))
    pair = lambda x, y: torch.einsum("bihd,bjhd->bhij", x, y)  # noqa: E731
    N = scale * D * pair(q, k) * pair(t["do"].double(), t["v"].double())

    def spanning(x):  # sum over j < t <= i
        left = torch.nn.functional.pad(x, (1, 0)).cumsum(-1)[..., :-1]              # [i, t]: j < t
        return left.flip(-2).cumsum(-2).flip(-2).diagonal(dim1=-2, dim2=-1).transpose(1, 2)

    return spanning(N), spanning(N.abs()), float((N.abs().sum(-1) + N.abs().sum(-2)).max())


def own_decay_gradient(t, scale):
    from mamba_b200 import linear_attention_fn

    g = t["g"].detach().requires_grad_()
    return torch.autograd.grad(linear_attention_fn(t["q"], t["k"], t["v"], g, scale), g, t["do"])[0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias,b,l,h,hk,dk,dv", [(-3.0, 1, 200, 2, 2, 64, 64), (0.0, 2, 333, 4, 2, 128, 64), (2.0, 1, 129, 2, 1, 40, 57),
                                                 (7.0, 1, 200, 2, 2, 64, 64), (0.0, 1, 2600, 2, 2, 128, 64), (5.0, 1, 2600, 2, 1, 64, 128),
                                                 (-3.0, 1, 2600, 2, 2, 64, 64)])
def test_decays_gradient_of_every_row_and_head(dtype, bias, b, l, h, hk, dk, dv):
    """The relative 2-norm of dlog_decay's error, per row and head.  The gradient is what is left of the suffix sums of
    two runs' dot products, so it holds only if the runs weight and round alike.  16 bits: each pair's weighted score
    is rounded once, the same in both runs (half a step u at most, u / sqrt 3 in the mean square), the result once
    more: sqrt(2/3) u where they are independent, and 2 u is asked for.  fp32: a dot product of some 128 fp32 terms is
    off by 2^-24 sqrt(128), a suffix of n of them by sqrt(n) as much; of pairs that span a token with decays of
    e^-3 a twentieth of that product is left, 2^-20.5 sqrt(200) 20 = 2^-12.4."""
    t = make(b, l, h, hk, dk, dv, dtype, bias=bias, seed=l + int(bias))
    want, _, _ = decay_gradient(t, 0.3)
    got = own_decay_gradient(t, 0.3).double()
    bound = 2.0 ** -12 if dtype == torch.float32 else 2 * HALF[dtype]
    off = lambda x: ((x - want).norm(dim=1) / want.norm(dim=1)).max()  # noqa: E731
    assert float(off(got)) <= bound, f"{float(off(got)):.3g} of the norm, {bound:.3g} asked for"
    assert float(off(0 * got)) > bound and float(off(-got)) > bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("l,hk", [(150, 16), (1500, 4)])
def test_one_decay_per_heads_gradient(dtype, l, hk):
    """The same for one decay per head: a value per head, so the norm is over the 16 heads.  The sum over tokens is
    one over more independent roundings, of a value that is rounded once itself (fp32 here)."""
    t = make(2, l, 16, hk, 64, 64, dtype, per_head=True, seed=l)
    want = decay_gradient(t, 0.3)[0].sum((0, 1))
    got = own_decay_gradient(t, 0.3).double()
    bound = 2.0 ** -12 if dtype == torch.float32 else 2 * HALF[dtype]
    off = lambda x: float((x - want).norm() / want.norm())  # noqa: E731
    assert off(got) <= bound and off(0 * got) > bound and off(-got) > bound, off(got)


def with_resets(n, dtype, bias=2.0, state=False):
    """n resets among the tokens of the second chunk of 128."""
    t = make(1, 300, 2, 1, 64, 64, dtype, bias=bias, state=state, seed=50 + n)
    at = 128 + torch.randperm(128, generator=torch.Generator().manual_seed(n))[:n].cuda()
    t["g"][0, at] = float("-inf")
    return t, at


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 12, 40, 90, 128])
def test_decays_gradient_between_resets(dtype, n):
    """Every value against its own pairs: what stands behind a reset has to cancel out of the suffix sums.  With u the
    half step of 16 bits, a pair's product is off by u (its score), the result by u; 2^-17 for fp32's sums.  The
    products that cancel are sums of some 128 fp32 terms (2^-24 sqrt 128 of M, the largest sum over a token's pairs),
    some 300 of them in a suffix: 2^-16 M."""
    t, at = with_resets(n, dtype)
    want, local, M = decay_gradient(t, 0.3)
    got = own_decay_gradient(t, 0.3).double()
    u = HALF[dtype]
    tol = (u * 1.01 * (local + want.abs()) if dtype != torch.float32 else 2.0 ** -17 * local) + 2.0 ** -16 * M
    worst = lambda x: float(((x - want).abs() / tol).max())  # noqa: E731
    assert float(got[0, at].abs().max()) == 0
    assert worst(got) <= 1, worst(got)
    assert worst(0 * got) > 1 and worst(-got) > 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2, 40, 128])
@pytest.mark.parametrize("bias", [-2.0, 5.0])
def test_gradients_with_resets(dtype, n, bias):
    """Outputs, states and the other gradients where resets stand, few or all of a chunk's tokens, in the middle of
    tokens that forget or last."""
    from mamba_b200 import linear_attention_fn

    t, _ = with_resets(n, dtype, bias, state=True)
    leaves = [t[x].detach().requires_grad_() for x in ("q", "k", "v", "s0")]
    out = linear_attention_fn(*leaves[:3], t["g"], 0.3, leaves[3], None, True)
    grads = torch.autograd.grad(list(out), leaves, [t["do"], t["dF"]])
    t["g"] = t["g"].double().clamp(min=-1e5)
    want_o, want_f, want = reference(t, 0.3, True)
    mag_o, mag_f, mags = reference(t, 0.3, True, absolute=True)
    f32 = dtype == torch.float32
    soft, hard = (2.0 ** -17, 2.0 ** -17) if f32 else (2 * HALF[dtype] + 2.0 ** -17, 2.0 ** -14)
    close("o", out[0], want_o, mag_o, dtype, soft)
    close("final", out[1], want_f, mag_f, dtype, hard)
    for name, got, w, m, f in zip(("dq", "dk", "dv", "dinitial_state"), grads, want[:3] + want[4:], mags[:3] + mags[4:],
                                  (soft, soft, soft, hard)):
        close(name, got, w, m, dtype, f)
