"""Selective scan (`ops.selective_scan`): the torch statement and the kernels against the recurrence in 64 bits.

Tolerances are carried along with the recurrence (u = 2^-24). x = dt' A is off by at most (24 + T) u |x| (the step: a
sum, an exponential and a logarithm; two products; T for the sum of the steps of a segment that is skipped over), its
exponential by 4 u more, an input dt' u B by 24 u. So a state with magnitude H_t = a H_{t-1} + |dt' u B_t| is off by E_t
with E_t = a E_{t-1} + delta H_t, delta = (24 + (24 + T) |x|) u, and so are the states of the reverse recurrence. What is
made of them is off by the sum of their errors, and a sum of n terms by n u of the sum of its magnitudes. A result of type
t is rounded once, by eps_t / 2 of its value."""
import pytest
import torch

from burn_dragon_b200.ops import mamba_ops as MO
from burn_dragon_b200.ops import norm_rotate as NR
from burn_dragon_b200.ops import selective_scan as S

U = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def definition(p, n, softplus, dy, dhT):
    """Values and bounds {name: (value, bound)} of y, h and every gradient, from float64 inputs."""
    u, raw, A, Bm, Cm = p["u"], p["dt"], p["A"], p["B"], p["C"]
    B, T, D = u.shape
    N = A.shape[1]
    dev = u.device
    live = torch.ones(B, T, 1, dtype=torch.bool, device=dev) if n is None else (torch.arange(T, device=dev) < n[:, None])[..., None]
    zero = lambda t: torch.where(live, t, 0.0)                                                           # noqa: E731
    u, Bm, Cm, dy = zero(u), zero(Bm), zero(Cm), zero(dy)
    raw = zero(raw) + (p["dt_bias"] if p["dt_bias"] is not None else 0.0)
    slope = torch.where(raw > 20, 1.0, torch.sigmoid(raw)) if softplus else torch.ones_like(raw)
    dt = zero(torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20)))) if softplus else raw)
    skip = p["D"] if p["D"] is not None else torch.zeros(D, dtype=u.dtype, device=dev)
    x = dt[..., None] * A
    a, delta = torch.exp(x), (24 + (24 + T) * x.abs()) * U
    b = (dt * u)[..., None] * Bm[:, :, None]
    h = p["h0"] if p["h0"] is not None else u.new_zeros(B, D, N)
    hs, Hs, Es = [h], [h.abs()], [torch.zeros_like(h)]
    for t in range(T):
        H = a[:, t] * Hs[-1] + b[:, t].abs()
        Es.append(a[:, t] * Es[-1] + delta[:, t] * H)
        Hs.append(H)
        hs.append(a[:, t] * hs[-1] + b[:, t])
    got = {"h": (hs[-1], Es[-1])}
    hs, Hs, Es = (torch.stack(v, 1) for v in (hs, Hs, Es))
    c4, b4 = Cm.abs()[:, :, None], Bm.abs()[:, :, None]
    ymag = (c4 * Hs[:, 1:]).sum(-1)
    got["y"] = zero((hs[:, 1:] * Cm[:, :, None]).sum(-1) + skip * u), zero((c4 * Es[:, 1:]).sum(-1) + (N + 8) * U * ymag + 4 * U * (skip * u).abs())
    r = dhT if dhT is not None else torch.zeros_like(h)
    R, E = r.abs(), torch.zeros_like(h)
    g, G, EG, rs, Rs, ER = ([None] * T for _ in range(6))
    for t in range(T - 1, -1, -1):
        c = Cm[:, t, None] * dy[:, t, :, None]
        g[t], G[t] = c + r, c.abs() + R
        EG[t] = E + 4 * U * G[t]
        r, R = a[:, t] * g[t], a[:, t] * G[t]
        E = a[:, t] * EG[t] + delta[:, t] * R
        rs[t], Rs[t], ER[t] = r, R, E
    got["d_h0"] = r, E
    g, G, EG, rs, Rs, ER = (torch.stack(v, 1) for v in (g, G, EG, rs, Rs, ER))
    q, Q = rs * hs[:, :-1], Rs * Hs[:, :-1]
    EQ = Rs * Es[:, :-1] + ER * Hs[:, :-1] + 2 * U * Q
    gb, GB = (g * Bm[:, :, None]).sum(-1), (G * b4).sum(-1)
    EGB = (EG * b4).sum(-1) + (N + 8) * U * GB
    aq, AQ = (q * A).sum(-1), (Q * A.abs()).sum(-1)
    EAQ = (EQ * A.abs()).sum(-1) + (N + 8) * U * AQ
    dd, DD = (aq + u * gb) * slope, AQ + u.abs() * GB
    EDD = EAQ + u.abs() * EGB + 64 * U * DD
    rows = B * T + 64
    got["d_dt"] = zero(dd), zero(EDD)
    got["d_u"] = zero(dt * gb + skip * dy), zero(dt.abs() * (EGB + 64 * U * GB) + 4 * U * (skip * dy).abs())
    got["d_A"] = (q * dt[..., None]).sum((0, 1)), ((EQ + (rows + 32) * U * Q) * dt.abs()[..., None]).sum((0, 1))
    w = (dt * u).abs()[..., None]
    got["d_B"] = (g * (dt * u)[..., None]).sum(2), ((EG + (D + 32) * U * G) * w).sum(2)
    got["d_C"] = (hs[:, 1:] * dy[..., None]).sum(2), ((Es[:, 1:] + (D + 8) * U * Hs[:, 1:]) * dy.abs()[..., None]).sum(2)
    got["d_D"] = (dy * u).sum((0, 1)), rows * U * (dy * u).abs().sum((0, 1))
    got["d_dt_bias"] = zero(dd).sum((0, 1)), zero(EDD + rows * U * DD).sum((0, 1))
    return got


def make(device, dtype, B, T, D, N, ragged, carry, softplus, extras, view):
    g = torch.Generator().manual_seed(7 * B + T + D + N)
    r = lambda *s: torch.randn(*s, generator=g)                                                          # noqa: E731
    wide = r(B, T, 2 * D + 2 * N + 8).to(dtype)
    if not softplus:
        wide[..., D:2 * D] = torch.rand(B, T, D, generator=g).to(dtype) * 0.2
    wide = wide.to(device)
    u, dt, Bm, Cm, _ = wide.split([D, D, N, N, 8], -1)
    if not view:
        u, dt, Bm, Cm = (t.contiguous() for t in (u, dt, Bm, Cm))
    p = dict(u=u, dt=dt, A=-(torch.rand(D, N, generator=g) * N + 0.1).to(device), B=Bm, C=Cm,
             D=r(D).to(device) if extras else None, dt_bias=(r(D) - 3 if softplus else 0.1 * r(D).abs()).to(device) if extras else None,
             h0=r(B, D, N).to(device) if carry else None)
    n = None
    if ragged:
        n = torch.randint(0, T + 1, (B,), generator=g)
        n[0] = T if B == 1 else 0
        n[-1] = T
        n = n.to(device)
    dy = torch.randn(B, T, D, generator=g).to(dtype).to(device)
    dhT = r(B, D, N).to(device) if carry else None
    return p, n, dy, dhT


def call(p, n, softplus, fn=S.selective_scan):
    return fn(p["u"], p["dt"], p["A"], p["B"], p["C"], p["D"], dt_bias=p["dt_bias"], dt_softplus=softplus, h0=p["h0"], lengths=n)


def within(got, want, bound, name):
    err = (got.double() - want).abs()
    lim = torch.finfo(got.dtype).eps / 2 * want.abs() + bound + (2.0 ** -25 if got.dtype == torch.float16 else 1e-30)
    assert got.shape == want.shape and bool((err <= lim).all()), (name, (err / lim).max().item())


# B, T, D, N, lengths, carried state (and its gradient), softplus, D and dt_bias, views into wider rows
CASES = [
    (1, 1, 1, 1, False, False, True, False, False),
    (2, 5, 24, 16, False, True, True, True, False),
    (3, 37, 72, 16, True, True, True, True, True),
    (2, 16, 65, 8, True, False, False, True, True),         # an odd width, no softplus
    (2, 33, 40, 5, False, True, True, True, False),
    (1, 300, 96, 16, False, True, True, True, False),       # few channels: the sequence is cut into segments
    (2, 150, 33, 24, True, True, True, False, True),
    (1, 47, 48, 64, True, True, True, True, False),
    (4, 18, 136, 33, True, True, False, True, False),
    (6, 20, 4000, 16, False, False, True, True, False),     # enough channels for two a lane
    (9, 50, 1200, 16, True, False, True, True, True),       # many warps, the sequence whole
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_outputs_and_gradients(device, dtype, case):
    B, T, D, N, ragged, carry, softplus, extras, view = case
    if device == "cpu" and D >= 1000 and dtype != torch.float32:
        pytest.skip("once is enough for the torch statement at this size")
    p, n, dy, dhT = make(device, dtype, *case)
    leaves = {k: t.detach().requires_grad_() if t is not None else None for k, t in p.items()}
    y, h = call(leaves, n, softplus)
    assert y.dtype == dtype and y.is_contiguous() and h.dtype == torch.float32
    want = definition({k: t.double() if t is not None else None for k, t in p.items()}, n, softplus, dy.double(),
                      dhT.double() if dhT is not None else None)
    within(y.detach(), *want["y"], "y")
    within(h.detach(), *want["h"], "h")
    with torch.no_grad():
        y2, h2 = call(p, n, softplus)                        # the form that keeps nothing for a backward pass
    assert torch.equal(y2, y) and torch.equal(h2, h)
    ask = {k: t for k, t in leaves.items() if t is not None}
    outs, grads = ([y, h], [dy, dhT]) if carry else ([y], [dy])
    for name, got in zip(ask, torch.autograd.grad(outs, list(ask.values()), grads)):
        within(got, *want["d_" + name], "d " + name)


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_agree_with_differences(device):
    """Central differences of sum(y w) + sum(h v) along a random direction, in float64 (the torch statement), against the
    gradients of the fp32 call. The difference quotient is off by a step^2 term (1e-8 here), the gradients by what
    the bounds above allow (a sum of about 10^4 terms of size 1: below 1e-3 of their norm)."""
    p, n, dy, dhT = make(device, torch.float32, 2, 40, 24, 16, True, True, True, True, False)
    leaves = {k: t.detach().requires_grad_() for k, t in p.items()}
    y, h = call(leaves, n, True)
    grads = torch.autograd.grad([y, h], list(leaves.values()), [dy, dhT])
    g = torch.Generator().manual_seed(1)
    for k, grad in zip(p, grads):
        way = torch.randn(p[k].shape, generator=g).to(device).double()
        value = []
        for s in (1e-4, -1e-4):
            moved = {m: t.double() + (s * way if m == k else 0) for m, t in p.items()}
            y2, h2 = call(moved, n, True, S.selective_scan_reference)
            value.append((y2 * dy.double()).sum() + (h2 * dhT.double()).sum())
        quotient = float(value[0] - value[1]) / 2e-4
        scale = float(grad.double().norm() * way.norm())
        assert abs(float((grad.double() * way).sum()) - quotient) <= 1e-4 * scale, k


@pytest.mark.parametrize("device", DEVICES)
def test_what_pads_a_batch_is_not_read(device):
    p, _, dy, _ = make(device, torch.float32, 4, 45, 40, 16, False, True, True, True, False)
    n = torch.tensor([45, 0, 17, 32], device=device)
    for k in ("u", "dt", "B", "C"):
        p[k][1] = float("nan")
        p[k][2, 17:] = float("inf")
        p[k][3, 32:] = float("nan")
    dy[1], dy[2, 17:] = float("nan"), float("inf")
    leaves = {k: t.detach().requires_grad_() for k, t in p.items()}
    y, h = call(leaves, n, True)
    assert torch.isfinite(y).all() and torch.isfinite(h).all() and torch.equal(h[1], p["h0"][1])
    assert (y[1] == 0).all() and (y[2, 17:] == 0).all() and (y[3, 32:] == 0).all()
    if device == "cuda":
        grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
        assert all(torch.isfinite(t).all() for t in grads.values())
        assert all((grads[k][2, 17:] == 0).all() and (grads[k][1] == 0).all() for k in ("u", "dt", "B", "C"))
    y2, h2 = call(p, torch.tensor([99, -3, 17, 32], device=device), True)
    assert torch.equal(y2, y) and torch.equal(h2, h)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N", [16, 7])
def test_segments_and_single_tokens_continue_a_prompt(device, N):
    p, _, _, _ = make(device, torch.float32, 3, 60, 40, N, False, False, True, True, False)
    part = lambda lo, hi, h: call({k: t[:, lo:hi] if k in ("u", "dt", "B", "C") else (h if k == "h0" else t) for k, t in p.items()}, None, True)  # noqa: E731
    with torch.no_grad():
        y, h = call(p, None, True)
        y1, h1 = part(0, 23, None)
        y2, h2 = part(23, 57, h1)
        rows, st = [], h2
        for t in range(57, 60):
            row = [p[k][:, t] for k in ("u", "dt")] + [p["A"]] + [p[k][:, t] for k in ("B", "C")]
            before = st.clone()
            yt, new = S.selective_scan_step(*row, st, p["D"], dt_bias=p["dt_bias"], dt_softplus=True)
            assert torch.equal(st, before)
            yt2, same = S.selective_scan_step(*row, st, p["D"], dt_bias=p["dt_bias"], dt_softplus=True, out=st)
            assert same is st and torch.equal(st, new) and torch.equal(yt, yt2)
            rows.append(yt[:, None])
        whole = torch.cat([y1, y2, *rows], 1)
        want = definition({k: t.double() if t is not None else None for k, t in p.items()}, None, True, torch.zeros_like(y).double(), None)
        within(whole, *want["y"], "y")
        within(st, *want["h"], "h")
        active = torch.tensor([True, False, True], device=device)
        bad = row[0].clone()
        bad[1] = float("nan")
        pool = torch.zeros(4, 2, 40, N, device=device)                     # states of two layers side by side
        pool[:3, 1] = st
        yt, new = S.selective_scan_step(bad, *row[1:], st, p["D"], dt_bias=p["dt_bias"], dt_softplus=True, active=active)
        ref, moved = S.selective_scan_step(*row, st, p["D"], dt_bias=p["dt_bias"], dt_softplus=True)
        S.selective_scan_step(bad, *row[1:], pool[:3, 1], p["D"], dt_bias=p["dt_bias"], dt_softplus=True, active=active, out=pool[:3, 1])
    assert torch.equal(yt[active], ref[active]) and (yt[~active] == 0).all()
    assert torch.equal(new[active], moved[active]) and torch.equal(new[~active], st[~active])
    assert torch.equal(pool[:3, 1], new) and (pool[:, 0] == 0).all() and (pool[3] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,D,N", [(torch.bfloat16, 79, 1030, 16), (torch.float32, 82, 2048, 5), (torch.float16, 21, 1000, 61)])
def test_single_tokens_of_many_streams(dtype, B, D, N):
    """Enough streams that a lane group takes four of them; one row of the recurrence, with and without its extras."""
    for extras in (True, False):
        p, _, _, _ = make("cuda", dtype, B, 1, D, N, False, True, True, extras, True)
        want = definition({k: t.double() if t is not None else None for k, t in p.items()}, None, True, torch.zeros(B, 1, D, device="cuda").double(),
                          None)
        active = torch.rand(B, device="cuda") < 0.7
        with torch.no_grad():
            row = [p["u"][:, 0], p["dt"][:, 0], p["A"], p["B"][:, 0], p["C"][:, 0]]
            y, h = S.selective_scan_step(*row, p["h0"], p["D"], dt_bias=p["dt_bias"], dt_softplus=True)
            some, kept = S.selective_scan_step(*row, p["h0"], p["D"], dt_bias=p["dt_bias"], dt_softplus=True, active=active)
            inplace = p["h0"].clone()
            S.selective_scan_step(*row, inplace, p["D"], dt_bias=p["dt_bias"], dt_softplus=True, active=active, out=inplace)
        within(y[:, None], *want["y"], "y")
        within(h, *want["h"], "h")
        assert torch.equal(some[active], y[active]) and (some[~active] == 0).all()
        assert torch.equal(kept[active], h[active]) and torch.equal(kept[~active], p["h0"][~active]) and torch.equal(inplace, kept)


@pytest.mark.parametrize("device", DEVICES)
def test_steps_past_the_softplus_threshold_and_vanishing_decays(device):
    p, _, _, _ = make(device, torch.float32, 1, 20, 16, 16, False, True, True, False, False)
    p["dt"] = torch.where(torch.rand(p["dt"].shape).to(device) < 0.5, 30.0, -40.0)
    p["A"] = p["A"] * 10                                                    # exp(dt A) is 0 in 32 bits, or 1 - 10^-15
    leaves = {k: t.detach().requires_grad_() if t is not None else None for k, t in p.items()}
    y, h = call(leaves, None, True)
    want = definition({k: t.double() if t is not None else None for k, t in p.items()}, None, True, torch.ones_like(y).double(), None)
    within(y.detach(), *want["y"], "y")
    ask = {k: t for k, t in leaves.items() if t is not None}
    for name, got in zip(ask, torch.autograd.grad(y, list(ask.values()), torch.ones_like(y))):
        value, bound = want["d_" + name]
        within(got, value, bound + 2.0 ** -120, "d " + name)


@pytest.mark.parametrize("device", DEVICES)
def test_empty_batches_and_prompts(device):
    A = -torch.ones(8, 4, device=device)
    z = lambda *s: torch.zeros(*s, device=device)                                                        # noqa: E731
    y, h = S.selective_scan(z(0, 3, 8), z(0, 3, 8), A, z(0, 3, 4), z(0, 3, 4))
    assert y.shape == (0, 3, 8) and h.shape == (0, 8, 4)
    h0 = torch.randn(2, 8, 4, device=device, requires_grad=True)
    y, h = S.selective_scan(z(2, 0, 8), z(2, 0, 8), A, z(2, 0, 4), z(2, 0, 4), z(8), h0=h0)
    assert y.shape == (2, 0, 8) and torch.equal(h, h0)
    assert (torch.autograd.grad(h.sum(), h0)[0] == 1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    z = lambda *s: torch.zeros(*s, device=device)                                                        # noqa: E731
    ok = dict(u=z(2, 5, 8), dt=z(2, 5, 8), A=z(8, 4), Bm=z(2, 5, 4), Cm=z(2, 5, 4))
    bad = [
        (dict(u=z(5, 8)), "u:"), (dict(u=z(2, 5, 8).long()), "u:"), (dict(dt=z(2, 5, 7)), "dt"), (dict(dt=z(2, 5, 8).half()), "dt"),
        (dict(A=z(7, 4)), "A:"), (dict(A=z(8, 65)), "A:"), (dict(A=z(8, 0)), "A:"), (dict(Bm=z(2, 5, 3)), "B:"), (dict(Cm=z(2, 4, 4)), "C:"),
        (dict(D=z(4)), "D:"), (dict(dt_bias=z(7)), "dt_bias"), (dict(h0=z(2, 8, 3)), "h0"), (dict(h0=z(2, 8, 4).half()), "h0"),
        (dict(lengths=z(2)), "lengths"), (dict(lengths=z(3).long()), "lengths"), (dict(D=torch.zeros(8, device="meta")), "D is on"),
    ]
    for change, message in bad:
        with pytest.raises(ValueError, match=message):
            S.selective_scan(**{**ok, **change})
    row = dict(u=z(2, 8), dt=z(2, 8), A=z(8, 4), Bm=z(2, 4), Cm=z(2, 4), h=z(2, 8, 4))
    for change, message in [(dict(h=z(1, 8, 4)), "h:"), (dict(h=z(2, 8, 4).half()), "h:"), (dict(active=z(2)), "active"),
                            (dict(out=z(1, 8, 4).expand(2, 8, 4)), "out"), (dict(u=z(2, 8).requires_grad_()), "gradient")]:
        with pytest.raises(ValueError, match=message):
            S.selective_scan_step(**{**row, **change})
    pool = z(3, 8, 4)
    with pytest.raises(ValueError, match="overlaps"):
        S.selective_scan_step(**{**row, "h": pool[:2], "out": pool[1:]})


def layer(x, w, lengths, state):
    """A state-space layer between its projections: convolution, then norm and rotation of B and C by learned angles, then
    the scan; `state` = (convolution's rows, last angle, scan's state)."""
    D, N = w["A"].shape
    xbc, dt, turn = x.split([D + 2 * N, D, N // 2], -1)
    conv, ang, h = state
    if x.dim() == 2:
        xbc, conv = MO.causal_conv_step(xbc, conv, w["conv"], w["conv_b"])
        u, Bm, Cm = xbc.split([D, N, N], -1)
        ang = ang + turn.float()
        Cm, Bm = NR.norm_rotate(Cm[:, None, None], Bm[:, None, None], w["c"], w["b"], angles=ang[:, None])
        y, h = S.selective_scan_step(u, dt, w["A"], Bm[:, 0, 0], Cm[:, 0, 0], h, w["D"], dt_bias=w["bias"], dt_softplus=True)
        return y, (conv, ang, h)
    xbc, conv = MO.causal_conv(xbc, w["conv"], w["conv_b"], state=conv, lengths=lengths)
    u, Bm, Cm = xbc.split([D, N, N], -1)
    if lengths is not None:
        turn = torch.where((torch.arange(x.shape[1], device=x.device) < lengths[:, None])[..., None], turn, 0.0)
    ang = (ang[:, None] if ang is not None else 0.0) + turn.float().cumsum(1)
    Cm, Bm = NR.norm_rotate(Cm.unsqueeze(2), Bm.unsqueeze(2), w["c"], w["b"], angles=ang, lengths=lengths)
    y, h = S.selective_scan(u, dt, w["A"], Bm.squeeze(2), Cm.squeeze(2), w["D"], dt_bias=w["bias"], dt_softplus=True, h0=h, lengths=lengths)
    return y, (conv, ang[:, -1], h)


def layer_weights(device, D, N):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(device)                                               # noqa: E731
    return dict(conv=r(D + 2 * N, 4) / 2, conv_b=0.1 * r(D + 2 * N), c=1 + 0.1 * r(N), b=1 + 0.1 * r(N), A=-(r(D, N).abs() * 4 + 0.2), D=r(D),
                bias=r(D) - 3)


@pytest.mark.parametrize("device", DEVICES)
def test_the_operators_together_as_a_layer(device):
    """A ragged batch of prompts through conv, norm + rotation and scan, then single tokens: the same rows as the float64
    layer run on each whole sequence. Errors of one operator pass through the next (gain at most about 30 at these
    magnitudes), each below 1e-5: 1e-3 of the outputs' scale holds them."""
    D, N, T = 40, 16, 33
    w = layer_weights(device, D, N)
    x = torch.randn(3, T, 2 * D + 2 * N + N // 2, generator=torch.Generator().manual_seed(5)).to(device)
    n = torch.tensor([30, 7, 19], device=device)
    with torch.no_grad():
        y, st = layer(x[:, :30], w, n, (None, None, None))
        rows = torch.arange(3, device=device)
        tail = [layer(x[rows, n], w, None, st)]
        tail.append(layer(x[rows, n + 1], w, None, tail[0][1]))
        exact = {k: t.double() for k, t in w.items()}
        for b in range(3):
            m = int(n[b])
            want, _ = layer(x[b:b + 1, :m + 2].double(), exact, None, (None, None, None))
            got = torch.cat([y[b, :m], tail[0][0][b:b + 1], tail[1][0][b:b + 1]])
            assert (got.double() - want[0]).abs().max() <= 1e-3 * want.abs().max()
            assert (y[b, m:] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_the_layer_has_gradients_of_all_its_weights(device):
    D, N = 24, 16
    w = {k: t.requires_grad_() for k, t in layer_weights(device, D, N).items()}
    x = torch.randn(2, 40, 2 * D + 2 * N + N // 2, generator=torch.Generator().manual_seed(6)).to(device).requires_grad_()
    n = torch.tensor([40, 22], device=device)
    dy = torch.randn(2, 40, D, generator=torch.Generator().manual_seed(8)).to(device)
    y, _ = layer(x, w, n, (None, None, None))
    got = torch.autograd.grad(y, [x, *w.values()], dy)
    we = {k: t.detach().double().requires_grad_() for k, t in w.items()}
    xe = x.detach().double().requires_grad_()
    ye, _ = layer(xe, we, n, (None, None, None))
    want = torch.autograd.grad(ye, [xe, *we.values()], dy.double())
    for name, a, e in zip(["x", *w], got, want):
        assert (a.double() - e).norm() <= 1e-4 * e.norm(), name


@pytest.mark.gpu
def test_two_runs_give_the_same_bits_and_replay_from_a_graph():
    p, n, dy, dhT = make("cuda", torch.bfloat16, 2, 200, 72, 16, True, True, True, True, True)

    def grads():
        leaves = {k: t.detach().requires_grad_() for k, t in p.items()}
        y, h = call(leaves, n, True)
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], list(leaves.values()), [dy, dhT])]

    assert all(torch.equal(a, b) for a, b in zip(grads(), grads()))
    graphs = []
    with torch.no_grad():
        row = [p[k][:, 3] for k in ("u", "dt")] + [p["A"]] + [p[k][:, 3] for k in ("B", "C")]
        for _ in range(2):                                                  # two graphs, each with scratch of its own
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y, h = call(p, n, True)
                y1, h1 = S.selective_scan_step(*row, h, p["D"], dt_bias=p["dt_bias"], dt_softplus=True)
            graphs.append((graph, y, h, y1, h1))
    p["u"].mul_(0.5)
    n.clamp_(max=120)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs[0][0].replay()
    with torch.cuda.stream(side):
        graphs[1][0].replay()
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        y, h = call(p, n, True)
        y1, h1 = S.selective_scan_step(*row, h, p["D"], dt_bias=p["dt_bias"], dt_softplus=True)
    for g in graphs:
        assert all(torch.equal(a, b) for a, b in zip(g[1:], (y, h, y1, h1)))


@pytest.mark.gpu
def test_long_sequences_and_other_streams():
    """Segments of many tiles, on a side stream, against the same sequence in pieces that hand their state on."""
    p, _, _, _ = make("cuda", torch.float32, 1, 5000, 24, 16, False, False, True, True, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        y, h = call(p, None, True)
    torch.cuda.current_stream().wait_stream(side)
    st, ys = None, []
    with torch.no_grad():
        for lo in range(0, 5000, 1250):
            out, st = call({k: t[:, lo:lo + 1250] if k in ("u", "dt", "B", "C") else (st if k == "h0" else t) for k, t in p.items()}, None, True)
            ys.append(out)
    want = definition({k: t.double() if t is not None else None for k, t in p.items()}, None, True, torch.zeros_like(y).double(), None)
    within(y, *want["y"], "y")
    within(torch.cat(ys, 1), *want["y"], "y in pieces")
    within(h, *want["h"], "h")


@pytest.mark.gpu
def test_a_training_step_replays_from_a_graph():
    """Forward and backward of the whole layer in one captured graph: the bits of the eager step, on new inputs as well."""
    D, N = 40, 16
    w = layer_weights("cuda", D, N)
    x = torch.randn(2, 50, 2 * D + 2 * N + N // 2, device="cuda")
    n = torch.tensor([50, 21], device="cuda")
    dy = torch.randn(2, 50, D, device="cuda")

    def step():
        leaves = {k: t.detach().requires_grad_() for k, t in w.items()}
        xs = x.detach().requires_grad_()
        y, _ = layer(xs, leaves, n, (None, None, None))
        return [y.detach(), *torch.autograd.grad(y, [xs, *leaves.values()], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.mul_(0.5)
    n.clamp_(max=37)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("device", DEVICES)
def test_states_in_slices_of_one_buffer(device):
    """Old and new states interleaved in one buffer, which do not meet, are taken; shifted by a stream, they are refused."""
    B, D, N = 3, 8, 4
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g).to(device)                                               # noqa: E731
    row = dict(u=r(B, D), dt=r(B, D).abs(), A=-r(D, N).abs(), Bm=r(B, N), Cm=r(B, N))
    pair = r(B, 2, D, N)
    y, h = S.selective_scan_step(**row, h=pair[:, 0].clone())
    old = pair[:, 0].clone()
    y2, h2 = S.selective_scan_step(**row, h=pair[:, 0], out=pair[:, 1])
    assert torch.equal(y, y2) and torch.equal(h, pair[:, 1]) and torch.equal(old, pair[:, 0]) and h2.data_ptr() == pair[:, 1].data_ptr()
    both = r(2, B + 1, D, N)
    with pytest.raises(ValueError, match="overlaps"):
        S.selective_scan_step(**row, h=both[0, 1:], out=both[0, :B])
    x, w = r(B, D), r(D, 4)
    rows = r(B, 2, 3, D)
    _, new = MO.causal_conv_step(x, rows[:, 0].clone(), w)
    MO.causal_conv_step(x, rows[:, 0], w, out=rows[:, 1])
    assert torch.equal(new, rows[:, 1])


@pytest.mark.gpu
def test_states_that_overlap_other_inputs_are_refused():
    """A step reads its inputs while other threads already write states."""
    w, buf = torch.randn(8, 4, device="cuda"), torch.zeros(2, 4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps an input"):
        MO.causal_conv_step(buf[:, 3], torch.zeros(2, 3, 8, device="cuda"), w, out=buf[:, 1:])
    z = lambda *s: torch.zeros(*s, device="cuda")                                                        # noqa: E731
    pool = z(2, 8, 4)
    with pytest.raises(RuntimeError, match="overlaps an input"):
        S.selective_scan_step(z(2, 8), z(2, 8), z(8, 4), pool[0, :2], z(2, 4), z(2, 8, 4), out=pool)


def _calls(device):
    """{operator: (call of its tensors, those tensors)}, every one of which has a gradient."""
    g = torch.Generator().manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g).to(device)                                               # noqa: E731
    B, T, D, N = 2, 9, 8, 4
    return {
        "conv": (lambda x, w, b, st: MO.causal_conv(x, w, b, state=st), [r(B, T, D), r(D, 4), r(D), r(B, 3, D)]),
        "norm_rotate": (lambda q, k, qw, kw, qb, kb, an: NR.norm_rotate(q, k, qw, kw, qb, kb, angles=an),
                        [r(B, T, 3, D), r(B, T, 2, D), r(D), r(D), r(D), r(D), r(B, T, 3)]),
        "scan": (lambda u, dt, A, Bm, Cm, Dk, db, h0: S.selective_scan(u, dt, A, Bm, Cm, Dk, dt_bias=db, dt_softplus=True, h0=h0),
                 [r(B, T, D), r(B, T, D), -r(D, N).abs(), r(B, T, N), r(B, T, N), r(D), r(D), r(B, D, N)]),
    }


@pytest.mark.parametrize("name", ["conv", "norm_rotate", "scan"])
@pytest.mark.parametrize("device", DEVICES)
def test_each_gradient_alone_and_each_result_alone(device, name):
    """One input with a gradient at a time, and one result used at a time, give what all of them together give. A gradient
    is a sum of at most 144 terms, each off by at most 24 u: two ways to it differ by 2 (144 + 24) u = 2e-5 of the
    terms' magnitudes, which are at most 50 times the largest gradient here; a gradient of another input is off by all of it."""
    fn, tensors = _calls(device)[name]
    leaves = [t.clone().requires_grad_() for t in tensors]
    outs = fn(*leaves)
    seeds = [torch.randn(o.shape, generator=torch.Generator().manual_seed(2)).to(device) for o in outs]
    together = torch.autograd.grad(outs, leaves, seeds)
    parts = [torch.autograd.grad(fn(*leaves)[i], leaves, seeds[i], allow_unused=True) for i in range(2)]
    for i, want in enumerate(together):
        leaf = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(tensors)]
        used = [(o, s) for o, s in zip(fn(*leaf), seeds) if o.requires_grad]
        got, = torch.autograd.grad([o for o, _ in used], leaf[i], [s for _, s in used])
        both = sum(p[i] for p in parts if p[i] is not None)
        scale = want.abs().max() + sum(p[i].abs().max() for p in parts if p[i] is not None)
        assert (got - want).abs().max() <= 1e-3 * scale and (both - want).abs().max() <= 1e-3 * scale, i


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["conv", "norm_rotate", "scan"])
def test_a_second_derivative_is_refused(name):
    fn, tensors = _calls("cuda")[name]
    leaves = [t.clone().requires_grad_() for t in tensors]
    out = fn(*leaves)[0]
    seed = torch.ones_like(out).requires_grad_()
    first = torch.autograd.grad(out, leaves[0], seed, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative"):
        first.sum().backward()
    with pytest.raises(RuntimeError):                                        # no way from it to the input, which grad() refuses
        torch.autograd.grad(first.sum(), leaves[0])
    out = fn(*leaves)[0]
    plain, = torch.autograd.grad(out, leaves[0], seed.detach())
    assert torch.equal(first.detach(), plain)
