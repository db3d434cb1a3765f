"""The norms around a block against float64.

Tolerances: outputs and elementwise gradients are computed in fp32 and rounded once: half a step of
the result, plus fp32 noise of 2^-18 of the row's largest term (a mean of up to 8192 squares in
fp32, summed in short pieces, is good to 2^-20; a rsqrt, a sigmoid and a few products follow).  In
the gradients the terms that cancel are bounded by the same sums of absolute values, taken as the
largest magnitude in the row.  Column gradients: fp32 sums over the rows, 2^-16 of the sum of absolute terms."""
import pytest
import torch

from sequence_ref import block_norm_ref

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def run(shape, dtype, *, post=True, pre=True, gate=True, scale="vector", act="silu", unit=True, seed=0, view=None,
        eps=1e-6, pre_eps=None):
    from mamba_b200 import block_norm_fn

    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = shape[-1]
    t = dict(y=rn(*shape).to(dtype), residual=rn(*shape).to(dtype), gate=rn(*shape).to(dtype) if gate else None,
             post=0.3 * rn(d) if post else None, pre=0.3 * rn(d) if pre else None,
             scale=(0.5 + 0.2 * rn(d)) if scale == "vector" else None)
    names = [n for n, v in t.items() if v is not None]
    t = {n: None if v is None else v.cuda().requires_grad_() for n, v in t.items()}
    const = scale if isinstance(scale, float) else None
    use = {n: view(v) if view is not None and v is not None and v.dim() > 1 else v for n, v in t.items()}
    out = block_norm_fn(use["y"], use["residual"], use["post"], use["pre"], use["gate"],
                        use["scale"] if const is None else const, act, eps, pre_eps, unit)
    x, h = out if pre else (None, out)
    dx, dh = rn(*shape).to(dtype).cuda(), rn(*shape).to(dtype).cuda()
    outs, seeds = ([x, h], [dx, dh]) if pre else ([h], [dh])
    grads = dict(zip(names, torch.autograd.grad(outs, [t[n] for n in names], seeds)))
    r = {n: None if v is None else v.detach().double().requires_grad_() for n, v in t.items()}
    rx, rh = block_norm_ref(r["y"], r["residual"], r["post"], r["pre"], r["gate"], r["scale"] if const is None else const,
                            act, eps, pre_eps, unit)
    routs, rseeds = ([rx, rh], [dx.double(), dh.double()]) if pre else ([rh], [dh.double()])
    want = dict(zip(names, torch.autograd.grad(routs, [r[n] for n in names], rseeds)))
    if not dx.numel():
        return

    def close(name, got, ref, mag):
        err = (got.double() - ref).abs()
        tol = HALF[got.dtype] * 1.001 * ref.abs() + mag
        assert bool((err <= tol).all()), f"{name}: {float((err / tol).max()):.3g} of the tolerance"

    row = lambda v: v.abs().amax(-1, keepdim=True) * 2.0 ** -18  # noqa: E731
    close("h", h, rh.detach(), row(rh.detach()) + row(r["residual"].detach()))
    if pre:
        close("x", x, rx.detach(), row(rx.detach()) + row(r["residual"].detach()))
    for n in ("y", "residual", "gate"):
        if n in grads:
            assert grads[n].dtype == dtype
            close("d" + n, grads[n], want[n], 8 * row(want[n]) + 8 * row(want["residual"]))
    for n in ("post", "pre", "scale"):
        if n in grads:  # the sum of absolute terms is at most sqrt(rows) times their 2-norm, and that about |sum| for random signs
            rows = dx.numel() // d
            close("d" + n, grads[n], want[n], 2.0 ** -16 * rows ** 0.5 * (8 + want[n].abs()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (2, 5, 64), (7, 100), (4, 33, 768), (9, 1000), (5, 1024), (3, 2049),
                                   (6, 2560), (2, 4096), (3, 5120), (2, 6144), (3, 8192), (2, 8191), (0, 64)])
def test_lengths(dtype, shape):
    run(shape, dtype, seed=shape[-1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(gate=False), dict(scale=None), dict(scale=0.7), dict(post=False), dict(pre=False),
                                dict(post=False, pre=False), dict(act="sigmoid"), dict(act=None), dict(unit=False),
                                dict(gate=False, scale=None), dict(eps=1e-2, pre_eps=1e-5)])
@pytest.mark.parametrize("dim", [200, 2600])
def test_options(dtype, kw, dim):
    run((19, dim), dtype, seed=dim, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(dtype):
    """More rows than the persistent grids hold, and not a multiple of them."""
    run((7141, 768), dtype, seed=3)
    run((5003, 72), dtype, seed=4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("rows,dim", [(5003, 128), (5001, 260), (2500, 512), (1300, 1100), (1301, 1536), (700, 2048), (700, 2564),
                                      (700, 4096), (650, 5000), (601, 8192)])
def test_several_rows_a_warp(dtype, gate, rows, dim):
    """Every kernel's row loop: the next row is fetched while one is computed, and the last has no next."""
    run((rows, dim), dtype, gate=gate, seed=dim)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_misaligned_rows(dtype):
    run((6, 96), dtype, seed=5, view=lambda v: torch.cat([v, v], -1)[:, :96])
    run((6, 96), dtype, seed=6, view=lambda v: torch.cat([v[:, :1], v], -1)[:, 1:])


def test_a_row_of_any_stride_and_rows_that_share_memory():
    from mamba_b200 import block_norm_fn

    g = torch.Generator().manual_seed(6)
    y, res, w = (torch.randn(*s, generator=g).cuda() for s in ((40, 1), (40,), (40,)))
    a = block_norm_fn(y.t(), res[None], w, w)              # one row, strides (1, 1)
    b = block_norm_fn(y.t().contiguous(), res[None], w, w)
    c = block_norm_fn(y.flatten(), res, w, w)              # no row axis at all
    for i in range(2):
        assert torch.equal(a[i], b[i]) and torch.equal(c[i], b[i][0])
    leaf = res.clone().requires_grad_()
    rows = torch.randn(5, 40, generator=g).cuda()
    h = block_norm_fn(rows, leaf.expand(5, 40), w)         # one residual row for all
    assert torch.equal(h, block_norm_fn(rows, res.repeat(5, 1), w))
    dh = torch.randn(5, 40, generator=g).cuda()
    (d,) = torch.autograd.grad(h, [leaf], dh)
    assert torch.allclose(d, dh.sum(0), rtol=0, atol=1e-5)  # five fp32 terms of about 1


def test_expanded_gate_and_its_gradient():
    from mamba_b200 import block_norm_fn

    g = torch.Generator(device="cuda").manual_seed(7)
    y, r = (torch.randn(2, 9, 64, generator=g, device="cuda") for _ in range(2))
    z = torch.randn(2, 1, 64, generator=g, device="cuda").requires_grad_()
    h = block_norm_fn(y, r, torch.zeros(64, device="cuda"), gate=z.expand(2, 9, 64))
    (got,) = torch.autograd.grad(h.sum(), z)
    zd = z.detach().double().requires_grad_()
    _, rh = block_norm_ref(y.double(), r.double(), torch.zeros(64, dtype=torch.float64, device="cuda"), gate=zd.expand(2, 9, 64))
    (want,) = torch.autograd.grad(rh.sum(), zd)
    assert got.shape == want.shape and float((got.double() - want).abs().max()) <= 2.0 ** -18 * 9 * 8


def test_only_one_output_is_used():
    from mamba_b200 import block_norm_fn

    g = torch.Generator(device="cuda").manual_seed(8)
    y, r = (torch.randn(5, 64, generator=g, device="cuda").requires_grad_() for _ in range(2))
    w = torch.zeros(64, device="cuda")
    x, h = block_norm_fn(y, r, w, w)
    for out, pick in ((x, 0), (h, 1)):
        got = torch.autograd.grad(out.sum(), [y, r], retain_graph=True)
        yd, rd = (t.detach().double().requires_grad_() for t in (y, r))
        want = torch.autograd.grad(block_norm_ref(yd, rd, w.double(), w.double())[pick].sum(), [yd, rd])
        for a, b in zip(got, want):
            assert float((a.double() - b).abs().max()) <= 2.0 ** -16 * float(b.abs().max())


def test_column_gradients_do_not_vary():
    from mamba_b200 import block_norm_fn

    g = torch.Generator(device="cuda").manual_seed(9)
    y, r = (torch.randn(4000, 768, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = [torch.zeros(768, device="cuda").requires_grad_() for _ in range(3)]
    once = lambda: torch.autograd.grad(block_norm_fn(y, r, w[0], w[1], residual_scale=w[2])[0].float().square().sum(), w)  # noqa: E731
    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


def test_captured_training_step():
    from mamba_b200 import block_norm_fn

    g = torch.Generator(device="cuda").manual_seed(10)
    y, r, z = (torch.randn(300, 256, generator=g, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    w = torch.zeros(256, device="cuda").requires_grad_()

    def step():
        x, h = block_norm_fn(y, r, w, w, gate=z)
        return torch.autograd.grad([x, h], [y, r, z, w], [torch.ones_like(x), torch.ones_like(h)])

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
