"""Causal convolution with a carried state (`ops.mamba_ops.causal_conv`, `causal_conv_step`): the torch statement and
the kernels against the definition in 64 bits.

Tolerances, from the arithmetic: a result of type t is rounded once, by at most eps_t / 2 of its value. Before that,
with u = 2^-24 and m = |b| + sum |w||s| (a sum of k + 1 products is off by at most (k + 2) u m <= 10 u m), SiLU (slope
at most 1.1, the quick exponential and division within 8 u plus |x| u of relative error, |x| <= m) adds at most
12 u + m u of |pre| <= m: together at most 2^-19 m (1 + m). A gradient row is a sum of k such terms times |w|; a sum
over n rows in any order is off by at most n u of the sum of magnitudes."""
import pytest
import torch

from burn_dragon_b200.ops import mamba_ops as MO

U = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def definition(x, w, bias, state, lengths, silu):
    """Row by row, in the inputs' type: y, the state behind every sequence, and sum |w||s| + |b| at every output."""
    B, T, C = x.shape
    k = w.shape[1]
    y, mag, ends = [], [], []
    for b in range(B):
        n = T if lengths is None else max(0, min(T, int(lengths[b])))
        seq = torch.cat([state[b] if state is not None else x.new_zeros(k - 1, C), x[b, :n]])
        pre = [sum((w[:, j] * seq[t + j] for j in range(k)), bias if bias is not None else x.new_zeros(C)) for t in range(n)]
        m = [sum(((w[:, j] * seq[t + j]).abs() for j in range(k)), bias.abs() if bias is not None else x.new_zeros(C)) for t in range(n)]
        rows = torch.stack(pre) if n else x.new_zeros(0, C)
        rows = rows / (1 + torch.exp(-rows)) if silu else rows
        y.append(torch.cat([rows, x.new_zeros(T - n, C)]))
        mag.append(torch.cat([torch.stack(m) if n else x.new_zeros(0, C), x.new_zeros(T - n, C)]).detach())
        ends.append(seq[n:n + k - 1])
    return torch.stack(y), torch.stack(ends), torch.stack(mag)


def make(device, dtype, B, T, C, k, bias, carry, lengths, view):
    g = torch.Generator().manual_seed(B * 1000 + T * 10 + C + k)
    r = lambda *s: torch.randn(*s, generator=g)
    wide = r(B, T, C + 24).to(dtype).to(device)
    x = wide[..., 8:8 + C] if view else wide[..., :C].contiguous()
    w, b = (r(C, k) / k ** 0.5).to(device), (r(C) * 0.1).to(device) if bias else None
    state = r(B, k - 1, C).to(dtype).to(device) if carry else None
    n = None
    if lengths:
        n = torch.randint(0, T + 1, (B,), generator=g)
        n[0] = T if B > 1 else 0
        if B > 2:
            n[2] = 1
        n = n.to(device)
    return x, w, b, state, n


def within(got, want, bound, name):
    eps = torch.finfo(got.dtype).eps
    err = (got.double() - want).abs()
    lim = eps / 2 * want.abs() + bound + 1e-30
    if got.dtype == torch.float16:
        lim = lim + 2.0 ** -25                              # half a step of the subnormal numbers
    assert bool((err <= lim).all()), (name, (err / lim).max().item())


SHAPES = [
    (1, 1, 1, 4, True, True, False, False),
    (2, 5, 8, 4, False, False, False, False),
    (3, 2, 16, 4, True, True, True, False),               # fewer rows than the state holds
    (3, 70, 40, 4, True, True, True, True),               # two tiles, a view into wider rows
    (2, 131, 33, 3, True, False, True, False),            # an odd width: element by element
    (2, 65, 24, 2, False, True, False, True),
    (2, 67, 48, 8, True, True, True, False),
    (1, 40, 8, 1, True, False, False, False),
    (4, 1, 264, 5, True, True, True, False),
    (3, 300, 64, 4, True, True, True, True),              # tiles with nothing to test inside, and ragged ends
    (2, 260, 130, 3, True, False, False, False),
    (1, 250, 36, 2, True, True, False, False),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("silu", [True, False])
def test_outputs_and_gradients(device, dtype, shape, silu):
    B, T, C, k, bias, carry, lengths, view = shape
    x, w, b, state, n = make(device, dtype, *shape)
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, state)]
    y, end = MO.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], lengths=n, activation="silu" if silu else None)
    assert y.dtype == dtype and end.shape == (B, k - 1, C) and end.dtype == dtype
    exact = [t.detach().double().requires_grad_() if t is not None else None for t in (x, w, b, state)]
    y0, end0, mag = definition(*exact, n, silu)
    within(y.detach(), y0.detach(), 2.0 ** -19 * mag * (1 + mag), "y")
    assert torch.equal(end.double(), end0.detach().to(end.dtype).double())
    dy, dend = torch.randn_like(x), torch.randn_like(end)
    ask = [t for t in leaves if t is not None]
    got = torch.autograd.grad([y, end], ask, [dy, dend], allow_unused=True)
    want = torch.autograd.grad([y0, end0], [t for t in exact if t is not None], [dy.double(), dend.double()], allow_unused=True)
    live = 1.0 if n is None else (torch.arange(T, device=device) < n[:, None])[..., None].double()
    gmag = dy.double().abs() * (1 + mag) * live                               # |d pre| and its error's scale
    sums = gmag.sum((0, 1)) if T else torch.zeros(C, device=device, dtype=torch.float64)
    reach = torch.nn.functional.pad(gmag, (0, 0, k - 1, k - 1)).unfold(1, k, 1) @ w.double().abs().max(0).values.flip(0) if T else 0
    big = max(1.0, float(x.double().abs().max()) if x.numel() else 1.0, float(state.double().abs().max()) if carry and k > 1 else 1.0)
    rel = (B * T + 40) * U + 2.0 ** -18
    names = [m for m, t in zip(("x", "w", "bias", "state"), leaves) if t is not None]
    for name, g, e in zip(names, got, want):
        if e is None or e.numel() == 0:
            continue
        if name in ("x", "state"):
            span = reach[:, k - 1:] if name == "x" else reach[:, :k - 1]
            bound = 2.0 ** -18 * span * max(1.0, float(w.abs().max()))
            # the new state's gradient joins in 32 bits; the torch statement rounds each of the two parts to the rows' type
            if device == "cpu" and dend.numel():
                bound = bound + torch.finfo(dtype).eps * (e.abs() + float(dend.abs().max()))
            within(g, e, bound, "d " + name)
        elif name == "w":
            within(g, e, rel * big * sums[:, None], "d w")
        else:
            within(g, e, rel * sums, "d bias")


@pytest.mark.parametrize("device", DEVICES)
def test_what_pads_a_batch_is_not_read(device):
    x, w, b, state, _ = make(device, torch.float32, 3, 37, 24, 4, True, True, False, False)
    n = torch.tensor([37, 0, 9], device=device)
    x[1] = float("nan")
    x[2, 9:] = float("inf")
    dy = torch.randn_like(x)
    dy[2, 9:] = float("nan")
    leaves = [t.detach().requires_grad_() for t in (x, w, b, state)]
    y, end = MO.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], lengths=n)
    assert torch.isfinite(y).all() and torch.isfinite(end).all()
    assert (y[1] == 0).all() and (y[2, 9:] == 0).all() and torch.equal(end[1], state[1])
    if device == "cuda":
        for g in torch.autograd.grad(y, leaves, dy):
            assert torch.isfinite(g).all()
    # lengths outside [0, T] count as the nearer bound
    y2, end2 = MO.causal_conv(x, w, b, state=state, lengths=torch.tensor([99, -5, 9], device=device))
    assert torch.equal(y2, y) and torch.equal(end2, end)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,C", [(torch.float32, 20), (torch.bfloat16, 40), (torch.float16, 7)])
def test_single_tokens_and_segments_continue_a_prompt(device, dtype, C):
    x, w, b, _, _ = make(device, dtype, 5, 23, C, 4, True, False, False, False)
    with torch.no_grad():
        whole, end = MO.causal_conv(x, w, b)
        first, st = MO.causal_conv(x[:, :10], w, b)
        second, st = MO.causal_conv(x[:, 10:20], w, b, state=st)
        rows = [first, second]
        for t in range(20, 23):
            before = st.clone()
            y, new = MO.causal_conv_step(x[:, t], st, w, b)
            assert torch.equal(st, before)
            y2, same = MO.causal_conv_step(x[:, t], st, w, b, out=st)
            assert same is st and torch.equal(st, new) and torch.equal(y, y2)
            rows.append(y[:, None])
    got, eps = torch.cat(rows, 1), torch.finfo(dtype).eps
    assert torch.equal(st, end)
    assert ((got.double() - whole.double()).abs() <= eps * whole.double().abs() + 2.0 ** -18 * 12).all()
    active = torch.tensor([True, False, True, False, True], device=device)
    bad = x[:, 0].clone()
    bad[1] = float("nan")
    with torch.no_grad():
        y, new = MO.causal_conv_step(bad, st, w, b, active=active)
        ref, moved = MO.causal_conv_step(x[:, 0], st, w, b)
        kept = st.clone()
        MO.causal_conv_step(bad, kept, w, b, active=active, out=kept)
    assert torch.equal(y[active], ref[active]) and (y[~active] == 0).all()
    assert torch.equal(new[active], moved[active]) and torch.equal(new[~active], st[~active]) and torch.equal(kept, new)


@pytest.mark.parametrize("device", DEVICES)
def test_empty_batches_and_prompts(device):
    w, b = torch.randn(8, 4, device=device), torch.randn(8, device=device)
    y, end = MO.causal_conv(torch.zeros(0, 5, 8, device=device), w, b)
    assert y.shape == (0, 5, 8) and end.shape == (0, 3, 8)
    st = torch.randn(2, 3, 8, device=device, requires_grad=True)
    x = torch.zeros(2, 0, 8, device=device, requires_grad=True)
    w.requires_grad_()
    y, end = MO.causal_conv(x, w, b, state=st)
    assert y.shape == (2, 0, 8) and torch.equal(end, st)
    gw, gs = torch.autograd.grad(end, (w, st), torch.ones_like(end), allow_unused=True)
    assert (gw is None or (gw == 0).all()) and (gs == 1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w = torch.zeros(2, 6, 8, device=device), torch.zeros(8, 4, device=device)
    bad = [
        (dict(x=x[0]), "x:"), (dict(x=x.long()), "x:"), (dict(w=torch.zeros(7, 4, device=device)), "w:"),
        (dict(w=torch.zeros(8, 9, device=device)), "w:"), (dict(bias=torch.zeros(7, device=device)), "bias"),
        (dict(state=torch.zeros(2, 4, 8, device=device)), "state"), (dict(state=torch.zeros(2, 3, 8, device=device).half()), "state"),
        (dict(lengths=torch.zeros(3, device=device, dtype=torch.int64)), "lengths"), (dict(lengths=torch.zeros(2, device=device)), "lengths"),
        (dict(activation="relu"), "activation"), (dict(bias=torch.zeros(8, device="meta")), "bias"),
    ]
    for change, message in bad:
        args = {**dict(x=x, w=w), **change}
        with pytest.raises(ValueError, match=message):
            MO.causal_conv(args.pop("x"), args.pop("w"), args.pop("bias", None), **args)
    st = torch.zeros(2, 3, 8, device=device)
    for change, message in [(dict(state=st[:1]), "state"), (dict(active=torch.ones(2, device=device)), "active"),
                            (dict(out=st.half()), "out"), (dict(out=st[:, :1].expand(2, 3, 8)), "out"),
                            (dict(out=torch.zeros(64, device=device).as_strided((2, 3, 8), (12, 4, 1))), "overlap")]:
        args = {**dict(state=st), **change}
        with pytest.raises(ValueError, match=message):
            MO.causal_conv_step(x[:, 0], args.pop("state"), w, **args)
    pool = torch.zeros(3, 3, 8, device=device)
    with pytest.raises(ValueError, match="overlaps"):
        MO.causal_conv_step(x[:, 0], pool[:2], w, out=pool[1:])
    with pytest.raises(ValueError, match="gradient"):
        MO.causal_conv_step(x[:, 0].requires_grad_(), st, w)


@pytest.mark.gpu
def test_two_runs_give_the_same_bits_and_replay_from_a_graph():
    x, w, b, state, n = make("cuda", torch.bfloat16, 4, 300, 264, 4, True, True, True, True)
    dy = torch.randn_like(x)

    def grads():
        leaves = [t.detach().requires_grad_() for t in (x, w, b, state)]
        y, end = MO.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], lengths=n)
        return [y.detach(), end.detach(), *torch.autograd.grad(y, leaves, dy)]

    first, second = grads(), grads()
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y, end = MO.causal_conv(x, w, b, state=state, lengths=n)
        y1, st1 = MO.causal_conv_step(x[:, 0], end, w, b)
    x.mul_(0.5)
    n.clamp_(max=100)
    graph.replay()
    with torch.no_grad():
        want, want_end = MO.causal_conv(x, w, b, state=state, lengths=n)
        want1, want_st1 = MO.causal_conv_step(x[:, 0], want_end, w, b)
    assert torch.equal(y, want) and torch.equal(end, want_end) and torch.equal(y1, want1) and torch.equal(st1, want_st1)


@pytest.mark.gpu
def test_offsets_past_31_bits():
    """Rows of a view whose last row starts more than 2^31 elements in; only the rows that are read exist in full."""
    B, T, C = 3, 9, 16
    wide = torch.zeros(B, 2 ** 30 + 64, device="cuda", dtype=torch.bfloat16)
    x = wide[:, 2 ** 30 - T * 8:].as_strided((B, T, C), (2 ** 30 + 64, 8, 1), 2 ** 30 - T * 8)
    wide[:, 2 ** 30 - T * 8:] = torch.randn(B, T * 8 + 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(C, 4, device="cuda")
    with torch.no_grad():
        y, end = MO.causal_conv(x, w)
        want, want_end = MO.causal_conv(x.contiguous(), w)
    assert torch.equal(y, want) and torch.equal(end, want_end)
