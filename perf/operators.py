"""The sequence-model operators beside the selective scan, as cases to measure: linear attention
with a decay per head (prompt, training step, single token), the norms around a block with its gate
and residual scale, and a beam-search step (selection over beams and vocabulary, reordering of the
layers' states).

``run`` computes a case in plain torch (32-bit arithmetic, 64-bit where sums are long or an order
between near-equal values decides) while ``own`` is false, and through ``mamba_b200`` while it is
true.  ``exact`` computes the same outputs in 64 bits from the definitions."""
import torch

own = False
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a short prompt of one request: launch latency, one partial tile
        dict(name="linear_prompt_short", op="linear", grad=False, dtype="bf16", b=1, l=100, h=12, hk=12, dk=64, dv=64,
             decay="token", state=True, lens=False),
        # one long document, few heads: the grid must come from the time axis
        dict(name="linear_prompt_long", op="linear", grad=False, dtype="bf16", b=1, l=16384, h=16, hk=16, dk=128,
             dv=128, decay="head", state=True, lens=False),
        # a training step at the width and batch of the 24-layer model (1536 = 24 heads of 64)
        dict(name="linear_train", op="linear", grad=True, dtype="bf16", b=8, l=2048, h=24, hk=24, dk=64, dv=64,
             decay="token", state=False, lens=False),
        # training with keys and queries shared by groups of heads, wide keys, a length off the tile
        dict(name="linear_train_groups", op="linear", grad=True, dtype="fp16", b=4, l=1999, h=16, hk=4, dk=128, dv=64,
             decay="token", state=False, lens=False),
        # fp32, odd head sizes, padded rows (one of them empty), carried state
        dict(name="linear_train_odd", op="linear", grad=True, dtype="fp32", b=3, l=777, h=6, hk=3, dk=40, dv=57,
             decay="token", state=True, lens=True),
        # one token of one request
        dict(name="linear_step_one", op="linear_step", dtype="bf16", b=1, h=24, hk=24, dk=64, dv=64, decay="token"),
        # one token of a full serving batch: the states fill the memory traffic
        dict(name="linear_step_batch", op="linear_step", dtype="bf16", b=64, h=40, hk=8, dk=128, dv=128, decay="head"),
        # the norms of a decode step
        dict(name="norm_decode", op="norm", grad=False, dtype="bf16", rows=64, dim=768, gate=True, scale=True),
        # the norms of a training step at the 24-layer model's width
        dict(name="norm_train", op="norm", grad=True, dtype="bf16", rows=16384, dim=768, gate=True, scale=True),
        # a wider model in fp32, rows off the tile, no gate
        dict(name="norm_train_wide", op="norm", grad=True, dtype="fp32", rows=4099, dim=2560, gate=False, scale=True),
        # a beam step of one request on the 24-layer model's states
        dict(name="beam_one", op="beam", dtype="bf16", b=1, w=4, k=4, vocab=50280, layers=24, dim=1536, done=False),
        # a beam step of a batch of requests, some beams finished
        dict(name="beam_batch", op="beam", dtype="fp32", b=24, w=8, k=8, vocab=50280, layers=8, dim=1536, done=True),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_step", "norm", "beam"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("linear", "linear_step"):
        hk = _log_int(rng, 1, 16)
        h = hk * rng.choice([1, 1, 2, 4])
        dk = rng.choice([64, 128, rng.randint(8, 128)])
        dv = rng.choice([64, 128, rng.randint(8, 128)])
        if op == "linear_step":
            return dict(op=op, dtype=dtype, b=_log_int(rng, 1, 64), h=min(h, 40 // hk * hk), hk=hk, dk=dk, dv=dv,
                        decay=rng.choice(["token", "head"]))
        b = _log_int(rng, 1, 8)
        grad = rng.random() < 0.5
        # tokens x heads x (dk + dv) up to half of the largest training case
        most = (25_000_000 if dtype == "fp32" else 50_000_000) // (b * h * (dk + dv))
        return dict(op=op, grad=grad, dtype=dtype, b=b, l=_log_int(rng, 1, max(2, min(16384, most // (2 if grad else 1)))),
                    h=h, hk=hk, dk=dk, dv=dv, decay="token" if grad else rng.choice(["token", "head"]),
                    state=rng.random() < 0.5, lens=b > 1 and rng.random() < 0.5)
    if op == "norm":
        dim = rng.choice([768, 2560, _log_int(rng, 32, 5120)])
        return dict(op=op, grad=rng.random() < 0.6, dtype=dtype, rows=_log_int(rng, 1, 12_000_000 // dim), dim=dim,
                    gate=rng.random() < 0.6, scale=rng.random() < 0.6)
    w = rng.randint(2, 8)
    return dict(op=op, dtype=dtype, b=_log_int(rng, 1, 24), w=w, k=w * rng.choice([1, 1, 2]), vocab=_log_int(rng, 100, 50280),
                layers=rng.randint(1, 8), dim=_log_int(rng, 64, 1536), done=rng.random() < 0.5)


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rn(*s, dtype=dt):
        return torch.randn(*s, generator=g, device="cuda").to(dtype)

    s = dict(case=case)
    if case["op"] in ("linear", "linear_step"):
        b, h, hk, dk, dv = (case[x] for x in ("b", "h", "hk", "dk", "dv"))
        seq = (b, case["l"]) if case["op"] == "linear" else (b,)
        s["q"], s["k"], s["v"] = rn(*seq, hk, dk), rn(*seq, hk, dk), rn(*seq, h, dv)
        # heads of different memory: log decays around -0.7 ... -0.002
        bias = torch.linspace(0.0, 6.0, h, device="cuda")
        if case["decay"] == "token":
            s["log_decay"] = (-torch.nn.functional.softplus(rn(*seq, h, dtype=torch.float32) - bias)).to(dt)
        else:
            s["log_decay"] = -torch.nn.functional.softplus(-bias + 0.3 * rn(h, dtype=torch.float32))
        s["scale"] = dk ** -0.5
        if case["op"] == "linear_step":
            s["state"] = rn(b, h, dk, dv, dtype=torch.float32)
            return s
        s["state"] = rn(b, h, dk, dv, dtype=torch.float32) if case["state"] else None
        s["lens"] = None
        if case["lens"]:
            lens = torch.randint(0, case["l"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
            lens[0], lens[-1] = case["l"], 0
            s["lens"] = lens
        if case["grad"]:
            s["dout"] = rn(b, case["l"], h, dv)
            s["dfinal"] = rn(b, h, dk, dv, dtype=torch.float32) if case["state"] else None
            s["leaves"] = [t for t in (s["q"], s["k"], s["v"], s["log_decay"], s["state"]) if t is not None]
            for t in s["leaves"]:
                t.requires_grad_()
        return s
    if case["op"] == "norm":
        r, d = case["rows"], case["dim"]
        s["y"], s["residual"] = rn(r, d), rn(r, d)
        s["gate"] = rn(r, d) if case["gate"] else None
        s["post_weight"], s["pre_weight"] = 0.1 * rn(d, dtype=torch.float32), 0.1 * rn(d, dtype=torch.float32)
        s["scale"] = 0.5 + 0.1 * rn(d, dtype=torch.float32) if case["scale"] else None
        if case["grad"]:
            s["dx"], s["dh"] = rn(r, d), rn(r, d)
            s["leaves"] = [t for t in (s["y"], s["residual"], s["gate"], s["post_weight"], s["pre_weight"], s["scale"])
                           if t is not None]
            for t in s["leaves"]:
                t.requires_grad_()
        return s
    b, w, d = case["b"], case["w"], case["dim"]
    s["logits"] = rn(b, w, case["vocab"], dtype=torch.float32).mul_(2.5).to(dt)
    s["scores"] = -20.0 - 3.0 * torch.rand(b, w, generator=g, device="cuda")
    s["done"] = torch.rand(b, w, generator=g, device="cuda") < 0.25 if case["done"] else None
    s["eos"] = 2 if case["done"] else None
    # a layer's convolution state (3 inputs) and scan state (16 per channel), a row per beam;
    # the first w of k selected candidates continue as beams
    s["states"] = [rn(b * w, d, n, dtype=torch.float32) for _ in range(case["layers"]) for n in (3, 16)]
    return s


# --------------------------------------------------------------------------------------- run
def run(s):
    case = s["case"]
    op = case["op"]
    if op == "linear":
        if own:
            import mamba_b200
            out = mamba_b200.linear_attention_fn(s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"],
                                                 initial_state=s["state"], seq_lens=s["lens"],
                                                 return_final_state=case["state"])
            o, final = out if case["state"] else (out, None)
        else:
            o, final = _linear(s["q"], s["k"], s["v"], s["log_decay"], s["scale"], s["state"], s["lens"])
        res = dict(o=o)
        if case["state"]:
            res["final"] = final
        return _with_grads(s, res, [o] + [final] * case["state"], lambda: [s["dout"]] + [s["dfinal"]] * case["state"])
    if op == "linear_step":
        if own:
            import mamba_b200
            o = mamba_b200.linear_attention_step(s["state"], s["q"], s["k"], s["v"], s["log_decay"], scale=s["scale"])
        else:
            o = _linear_step(s["state"], s["q"], s["k"], s["v"], s["log_decay"], s["scale"])
        return dict(o=o, state=s["state"])
    if op == "norm":
        if own:
            import mamba_b200
            x, h = mamba_b200.block_norm_fn(s["y"], s["residual"], s["post_weight"], s["pre_weight"], gate=s["gate"],
                                            residual_scale=s["scale"], eps=EPS)
        else:
            x, h = _norm(s["y"], s["residual"], s["post_weight"], s["pre_weight"], s["gate"], s["scale"])
        return _with_grads(s, dict(x=x, h=h), [x, h], lambda: [s["dx"], s["dh"]])
    if own:
        import mamba_b200
        scores, parents, tokens = mamba_b200.beam_select(s["logits"], s["scores"], num_select=case["k"],
                                                         finished=s["done"], eos_token_id=s["eos"])
        mamba_b200.reorder_states(s["states"], parents[:, :case["w"]])
    else:
        scores, parents, tokens = _beam_select(s["logits"], s["scores"], case["k"], s["done"], s["eos"])
        _reorder(s["states"], parents[:, :case["w"]])
    return dict(scores=scores, parents=parents, tokens=tokens, states=s["states"])


def _with_grads(s, res, outs, seeds):
    if s["case"]["grad"]:
        res["grads"] = list(torch.autograd.grad(outs, s["leaves"], seeds()))
    return {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in res.items()}


def _linear(q, k, v, log_decay, scale, s0, lens, chunk=64):
    """S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale q_t S_t, over chunks: the pairs inside a
    chunk, the chunk's own states, and every chunk's state from the earlier ones' at once."""
    b, l, h, dv = v.shape
    dk, dtype = q.shape[-1], v.dtype
    n = -(-l // chunk)
    valid = torch.ones(b, l, dtype=torch.bool, device=v.device)
    if lens is not None:
        valid = torch.arange(l, device=v.device)[None] < lens[:, None]
    keep = valid[..., None, None]
    g = log_decay.double().clamp(min=-1e4).expand(b, l, h) * valid[..., None]

    def cut(t):  # (b, l, heads, d) -> (b, h, chunks, chunk, d)
        t = torch.where(keep, t.float(), 0.0).repeat_interleave(h // t.shape[2], 2)
        t = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, n * chunk - l))
        return t.reshape(b, n, chunk, h, -1).permute(0, 3, 1, 2, 4)

    q, k, v = cut(q) * scale, cut(k), cut(v)
    g = torch.nn.functional.pad(g, (0, 0, 0, n * chunk - l)).reshape(b, n, chunk, h).permute(0, 3, 1, 2)
    G = g.cumsum(-1)                                                       # (b, h, n, chunk)
    T = G[..., -1]
    low = torch.ones(chunk, chunk, dtype=torch.bool, device=v.device).tril()
    D = torch.where(low, G[..., :, None] - G[..., None, :], -torch.inf).exp().float()
    o = ((q @ k.transpose(-1, -2)) * D) @ v
    S = (k * (T[..., None] - G).exp().float()[..., None]).transpose(-1, -2) @ v   # (b, h, n, dk, dv)
    end = T.cumsum(-1)
    past = torch.ones(n, n, dtype=torch.bool, device=v.device).tril(-1)
    W = torch.where(past, (end - T)[..., :, None] - end[..., None, :], -torch.inf).exp().float()
    H = (W @ S.flatten(-2)).unflatten(-1, (dk, dv))
    last = ((end[..., -1:] - end).exp().float()[..., None, :] @ S.flatten(-2)).reshape(b, h, dk, dv)
    if s0 is not None:
        H = H + (end - T).exp().float()[..., None, None] * s0[:, :, None]
        last = last + end[..., -1].exp().float()[..., None, None] * s0
    o = o + (q * G.exp().float()[..., None]) @ H
    o = o.permute(0, 2, 3, 1, 4).reshape(b, n * chunk, h, dv)[:, :l]
    return torch.where(keep, o, 0.0).to(dtype), last


def _linear_step(state, q, k, v, log_decay, scale):
    h = v.shape[1]
    q, k = (t.float().repeat_interleave(h // t.shape[1], 1) for t in (q, k))
    a = log_decay.float().exp().expand(v.shape[:2])
    state.mul_(a[..., None, None]).add_(k[..., :, None] * v.float()[..., None, :])
    return (scale * (q[..., None, :] @ state)[..., 0, :]).to(v.dtype)


def _rms(t, weight):
    return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * (1 + weight)


def _norm(y, residual, post_weight, pre_weight, gate, scale):
    u = _rms(y.float(), post_weight)
    if gate is not None:
        u = u * (gate.float() * torch.sigmoid(gate.float()))
    if scale is not None:
        u = u * scale
    h = residual.float() + u
    return _rms(h, pre_weight).to(y.dtype), h.to(y.dtype)


def _beam_select(logits, scores, k, done, eos):
    b, w, vocab = logits.shape
    x = logits.double()
    cand = scores.double()[..., None] + (x - x.logsumexp(-1, keepdim=True))
    if done is not None:  # a finished beam goes on as itself, at its end token
        only = torch.full_like(cand, -torch.inf)
        only[..., eos] = scores.double()
        cand = torch.where(done[..., None], only, cand)
    best, at = cand.flatten(1).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    return best.float(), at // vocab, at % vocab


def _reorder(states, parents):
    b, w = parents.shape
    rows = (parents + w * torch.arange(b, device=parents.device)[:, None]).flatten()
    for t in states:
        t.copy_(t[rows])


# ------------------------------------------------------------------------------------- exact
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _exact_linear(case, s)
    if op == "linear_step":
        rep = case["h"] // case["hk"]
        q, k = (torch.repeat_interleave(s[x].double(), rep, dim=1) for x in "qk")
        a = torch.exp(s["log_decay"].double()).expand(case["b"], case["h"])
        state = torch.einsum("bh,bhij->bhij", a, s["state"].double()) + torch.einsum("bhi,bhj->bhij", k, s["v"].double())
        return dict(o=s["scale"] * torch.einsum("bhi,bhij->bhj", q, state), state=state)
    if op == "norm":
        return _exact_norm(case, s)
    return _exact_beam(case, s)


def _exact_linear(case, s):
    """Every pair (i, j) of a row's tokens at once, one batch row and one key head at a time."""
    b, l, h, hk, dk, dv = (case[x] for x in ("b", "l", "h", "hk", "dk", "dv"))
    rep, scale, grad = h // hk, s["scale"], case["grad"]
    q, k, v = (s[x].double() for x in "qkv")
    gd = s["log_decay"].double().expand(b, l, h)
    zeros = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    o, final = zeros(b, l, h, dv), zeros(b, h, dk, dv)
    dq, dkk, dv_, dg, ds = zeros(b, l, hk, dk), zeros(b, l, hk, dk), zeros(b, l, h, dv), zeros(b, l, h), zeros(b, h, dk, dv)
    lens = [l] * b if s["lens"] is None else s["lens"].tolist()
    for i in range(b):
        n = lens[i]
        for j in range(h):
            Q, K, V = q[i, :n, j // rep], k[i, :n, j // rep], v[i, :n, j]
            G = gd[i, :n, j].cumsum(0)
            total = G[-1] if n else zeros(())
            D = torch.exp((G[:, None] - G[None, :]).tril_()).tril_()
            P = scale * (Q @ K.T)
            M = P * D
            o[i, :n, j] = M @ V
            to_end = torch.exp(total - G)
            final[i, j] = (K * to_end[:, None]).T @ V
            S0 = None if s["state"] is None else s["state"][i, j].double()
            if S0 is not None:
                o[i, :n, j] += scale * torch.exp(G)[:, None] * (Q @ S0)
                final[i, j] += torch.exp(total) * S0
            if not grad:
                del D, P, M
                continue
            dO = s["dout"][i, :n, j].double()
            dA = dO @ V.T
            N = M * dA
            dG = N.sum(1) - N.sum(0)
            dv_[i, :n, j] = M.T @ dO
            E = scale * D * dA
            dq[i, :n, j // rep] += E @ K
            dkk[i, :n, j // rep] += E.T @ Q
            if S0 is not None:
                F = s["dfinal"][i, j].double()
                c = scale * torch.exp(G)[:, None] * (dO @ S0.T)
                dq[i, :n, j // rep] += c
                dG += (Q * c).sum(1)
                ds[i, j] = (scale * Q * torch.exp(G)[:, None]).T @ dO + torch.exp(total) * F
                c = to_end[:, None] * (V @ F.T)
                dkk[i, :n, j // rep] += c
                dv_[i, :n, j] += to_end[:, None] * (K @ F)
                z = (K * c).sum(1)
                dG -= z
                if n:
                    dG[-1] += z.sum() + torch.exp(total) * (F * S0).sum()
            dg[i, :n, j] = dG.flip(0).cumsum(0).flip(0)
    res = dict(o=o)
    if case["state"]:
        res["final"] = final
    if grad:
        res["grads"] = [dq, dkk, dv_, dg] + [ds] * case["state"]
    return res


def _exact_norm(case, s):
    y, r = s["y"].double(), s["residual"].double()
    d = y.shape[-1]
    wp, wn = 1 + s["post_weight"].double(), 1 + s["pre_weight"].double()
    sc = s["scale"].double() if case["scale"] else torch.ones(d, dtype=torch.float64, device="cuda")
    ry = 1 / torch.sqrt((y * y).sum(-1, keepdim=True) / d + EPS)
    n = y * ry
    act = slope = torch.ones((), dtype=torch.float64, device="cuda")
    if case["gate"]:
        z = s["gate"].double()
        sig = 1 / (1 + torch.exp(-z))
        act, slope = z * sig, sig * (1 + z * (1 - sig))
    h = r + sc * act * wp * n
    rh = 1 / torch.sqrt((h * h).sum(-1, keepdim=True) / d + EPS)
    res = dict(x=h * rh * wn, h=h)
    if case["grad"]:
        dx = s["dx"].double()
        t = dx * wn
        dh = s["dh"].double() + rh * (t - h * rh * rh * (t * h).sum(-1, keepdim=True) / d)
        t = dh * sc * act * wp
        dy = ry * (t - n * (t * n).sum(-1, keepdim=True) / d)
        grads = [dy, dh] + ([dh * sc * wp * n * slope] if case["gate"] else [])
        grads += [(dh * sc * act * n).sum(0), (dx * h * rh).sum(0)]
        res["grads"] = grads + ([(dh * act * wp * n).sum(0)] if case["scale"] else [])
    return res


def _exact_beam(case, s):
    b, w, vocab, k = (case[x] for x in ("b", "w", "vocab", "k"))
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    cand = (x - lse) + s["scores"].double()[:, :, None]
    if case["done"]:
        at_end = torch.arange(vocab, device="cuda")[None, None] == s["eos"]
        kept = torch.where(at_end, s["scores"].double()[:, :, None], -torch.inf)
        cand = torch.where(s["done"][:, :, None], kept, cand)
    cand = cand.reshape(b, -1)
    taken, index, best, at = torch.zeros_like(cand, dtype=torch.bool), torch.arange(w * vocab, device="cuda"), [], []
    for _ in range(k):  # the largest that is left, the first of its equals
        m = torch.where(taken, -torch.inf, cand).amax(-1, keepdim=True)
        i = torch.where((cand == m) & ~taken, index, w * vocab).amin(-1, keepdim=True)
        taken.scatter_(1, i, True)
        best.append(m)
        at.append(i)
    best, at = torch.cat(best, 1), torch.cat(at, 1)
    parents = at // vocab
    rows = (torch.arange(b, device="cuda")[:, None] * w + parents[:, :w]).reshape(-1)
    return dict(scores=best, parents=parents, tokens=at - parents * vocab,
                states=[t.index_select(0, rows) for t in s["states"]])


# -------------------------------------------------------------------------------------- work
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op in ("linear", "linear_step"):
        b, h, hk, dk, dv = (case[x] for x in ("b", "h", "hk", "dk", "dv"))
        tokens = b * case.get("l", 1)
        qk, vv, states = 2 * tokens * hk * dk, tokens * h * dv, b * h * dk * dv * 4
        decay = tokens * h * es if case["decay"] == "token" else 4 * h
        # a token of a head: its state decayed, its outer product added, its query's product
        flops = 5 * tokens * h * dk * dv
        if op == "linear_step":
            return dict(bytes=(qk + 2 * vv) * es + decay + 2 * states, flops=flops)
        nbytes = (qk + 2 * vv) * es + decay + (2 * states if case["state"] else 0)
        if case["grad"]:  # dout read, the four inputs' gradients written, both states' gradients
            nbytes += (qk + 2 * vv) * es + decay + (2 * states if case["state"] else 0)
            flops *= 3.4  # the forward's, and four more products of the state's size with its two decays
        return dict(bytes=nbytes, flops=flops)
    if op == "norm":
        r, d = case["rows"], case["dim"]
        n, cols = (3 if case["gate"] else 2), 2 + case["scale"]
        nbytes = r * d * es * (n + 2) + 4 * d * cols
        if case["grad"]:  # the gradients of x and h read, those of the inputs written
            nbytes += r * d * es * (n + 2) + 4 * d * cols
        return dict(bytes=nbytes, flops=r * d * (10 + 30 * case["grad"]))
    n = case["b"] * case["w"]
    return dict(bytes=n * case["vocab"] * es + 2 * n * case["layers"] * case["dim"] * 19 * 4, flops=4 * n * case["vocab"])
