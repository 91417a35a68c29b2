"""Per-head RMS norm + rotation (`ops.norm_rotate`): the torch statement and the kernels against the definition in 64 bits.

Tolerances, from the arithmetic (u = 2^-24): the sum of Dh squares is off by at most Dh u of itself, the root of it by
half that plus 4 u, so v = x r w + b is off by (Dh / 2 + 8) u |v|-ish; sine and cosine of an angle rounded to 32 bits
(2 pi frac, |angle| < 6.3: 2^-22) are off by at most 2^-21. A rotated value is off by at most 2^-20 of the pair's
|v0| + |v1|, plus the norm's part. The gradients repeat the same operations on w dv, with one more sum over Dh; a sum over n rows in any
order is off by n u of the sum of magnitudes. E = 2^-19 + (Dh + 32) u covers each of them. A result of type t is rounded
once, by eps_t / 2 of its value."""
import math

import pytest
import torch

from burn_dragon_b200.ops import norm_rotate as NR
from burn_dragon_b200.ops import reference as R

U = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def definition(q, k, qw, kw, qb, kb, angle, n, eps):
    """float64, complex multiplication for the rotation; rows behind n are left out of every sum."""
    outs = []
    T = q.shape[1]
    keep = torch.ones(q.shape[:2], dtype=torch.bool, device=q.device) if n is None else torch.arange(T, device=q.device) < n[:, None]
    for x, w, b in ((q, qw, qb), (k, kw, kb)):
        if x is None:
            outs.append(None)
            continue
        x = torch.where(keep[..., None, None], x, 0.0)
        v = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        v = v * w if w is not None else v
        v = v + b if b is not None else v
        if angle is not None:
            P = angle.shape[-1]
            c = torch.view_as_complex(v[..., :2 * P].unflatten(-1, (P, 2)).contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, :, None]
            v = torch.cat((torch.view_as_real(c).flatten(-2), v[..., 2 * P:]), -1)
        outs.append(torch.where(keep[..., None, None], v, 0.0))
    return outs


def pairs(t):
    """|t_2i| + |t_2i+1| at both places of every pair"""
    a = t.abs().unflatten(-1, (-1, 2)).sum(-1, keepdim=True)
    return a.expand(*a.shape[:-1], 2).flatten(-2)


def within(got, want, bound, name):
    err = (got.double() - want).abs()
    lim = torch.finfo(got.dtype).eps / 2 * want.abs() + bound + (2.0 ** -25 if got.dtype == torch.float16 else 1e-30)
    assert got.shape == want.shape and bool((err <= lim).all()), (name, (err / lim).max().item())


# B, T, Hq, Hk, Dh, pairs, angles, weights per head, bias, lengths, view into wider rows
CASES = [
    (1, 1, 1, 0, 2, 1, "positions", False, False, False, False),
    (2, 7, 4, 2, 64, 32, "positions", False, False, False, True),
    (3, 33, 2, 2, 128, 64, "data", True, True, True, False),
    (2, 50, 5, 3, 80, 20, "positions", False, True, True, True),
    (2, 9, 3, 1, 34, 17, "data", True, False, True, True),          # rows that no 16-byte load fits
    (1, 300, 33, 11, 128, 64, "data", False, False, False, False),  # several slices of heads, several tokens a thread
    (2, 65, 3, 2, 256, 100, "positions", True, True, False, False),
    (1, 21, 2, 1, 512, 256, "data", False, True, True, False),
    (1, 12, 2, 2, 390, 3, "data", True, True, False, False),
    (5, 1, 8, 2, 64, 32, "positions", False, False, False, False),
    (2, 700, 1, 1, 16, 0, None, False, True, True, False),          # a norm alone, many tokens a block
]


def make(device, dtype, B, T, Hq, Hk, Dh, P, kind, heads, bias, ragged, view):
    g = torch.Generator().manual_seed(B + 10 * T + Hq + Dh + P)
    r = lambda *s: torch.randn(*s, generator=g)                                                          # noqa: E731
    wide = (r(B, T, Hq + Hk + 1, Dh) * 2).to(dtype).to(device)
    q = wide[:, :, 1:1 + Hq] if view else wide[:, :, 1:1 + Hq].contiguous()
    k = (wide[:, :, 1 + Hq:] if view else wide[:, :, 1 + Hq:].contiguous()) if Hk else None
    shape = lambda H: (H, Dh) if heads else (Dh,)                                                        # noqa: E731
    p = [1 + 0.3 * r(*shape(Hq)), 1 + 0.3 * r(*shape(Hk)) if Hk else None, r(*shape(Hq)) if bias else None, r(*shape(Hk)) if bias and Hk else None]
    qw, kw, qb, kb = (t.to(device) if t is not None else None for t in p)
    how = {}
    if kind == "data":
        how["angles"] = (3 * r(B, T, P)).to(device)
    elif kind == "positions":
        how["freqs"] = R.build_freqs(2 * P, 65536.0, "rope").to(device)
        how["positions"] = (torch.randint(0, 3_000_000, (B, 1), generator=g) + torch.arange(T)).to(device)
    n = torch.randint(0, T + 1, (B,), generator=g).to(device) if ragged else None
    if ragged:
        n[0] = 0 if B > 2 else T
    return (q, k, qw, kw, qb, kb), how, n


def exact_angle(how):
    if "angles" in how:
        return how["angles"].double().requires_grad_()
    if "freqs" in how:
        return 2 * math.pi * (how["positions"].double()[..., None] * how["freqs"][::2].double())
    return None


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_outputs_and_gradients(device, dtype, case):
    B, T, Hq, Hk, Dh, P, kind, heads, bias, ragged, view = case
    tensors, how, n = make(device, dtype, *case)
    leaves = [t.detach().requires_grad_() if t is not None else None for t in tensors]
    given = dict(how)
    if kind == "data":
        given["angles"] = how["angles"].detach().requires_grad_()
    got = NR.norm_rotate(*leaves, lengths=n, **given)
    exact = [t.detach().double().requires_grad_() if t is not None else None for t in tensors]
    angle = exact_angle(how)
    want = definition(*exact, angle, n, 1e-5)
    E = 2.0 ** -19 + (Dh + 32) * U
    keep = torch.ones(B, T, 1, 1, device=device, dtype=torch.float64) if n is None else \
        (torch.arange(T, device=device) < n[:, None])[..., None, None].double()
    norm = definition(*[t.detach() if t is not None else None for t in exact], None, n, 1e-5)           # v, before the rotation
    outs, dos = [], []
    for name, o, e, v in zip("qk", got, want, norm):
        if e is None:
            assert o is None
            continue
        assert o.dtype == dtype and o.is_contiguous()
        b = exact[4 if name == "q" else 5]
        slack = b.detach().abs().max() if b is not None else 0.0
        within(o.detach(), e.detach(), E * (pairs(v) + 2 * slack), name)
        outs.append((o, e))
        dos.append(torch.randn_like(o))
    names = ["q", "k", "q_weight", "k_weight", "q_bias", "k_bias"]
    have = [(m, t, x) for m, t, x in zip(names, leaves, exact) if t is not None]
    if kind == "data":
        have.append(("angles", given["angles"], angle))
    g = torch.autograd.grad([o for o, _ in outs], [t for _, t, _ in have], dos)
    w = torch.autograd.grad([e for _, e in outs], [x for _, _, x in have], [d.double() for d in dos])
    rows = B * T * (1 if heads else max(Hq, Hk)) + 64
    for (name, _, _), a, e in zip(have, g, w):
        if name == "angles":
            mag = sum((pairs(v)[..., :2 * P:2] * pairs(d.double())[..., :2 * P:2] * keep).sum(2) for v, d in zip([v for v in norm if v is not None], dos))
            slack = max(float(t.detach().abs().max()) for t in exact[4:] if t is not None) if bias else 0.0
            gm = sum((pairs(d.double())[..., :2 * P:2] * keep).sum(2) for d in dos)
            within(a, e, (4 * E + (Hq + Hk) * U) * (mag + 2 * slack * gm), name)
            continue
        i = 0 if name[0] == "q" else 1
        x, wt, d = exact[i].detach(), exact[2 + i].detach().abs(), dos[i].double()
        x = torch.where(keep > 0, x, 0.0)
        r = 1 / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt()
        hat, dv = (x * r).abs(), pairs(d) * keep
        if name in ("q", "k"):
            dhat = dv * wt.max()
            within(a, e, 4 * E * r * (dhat + hat * (dhat * hat).mean(-1, keepdim=True)), name)
        else:
            term = dv * hat if "weight" in name else dv
            total = term.sum((0, 1)) if heads else term.sum((0, 1, 2))
            within(a, e, (4 * E + rows * U) * total, name)


@pytest.mark.parametrize("device", DEVICES)
def test_matches_the_rotation_and_norm_that_the_models_use(device):
    """A plain rotation by position is `reference.rotate` (positions whose phases 32 bits hold), and the angle form is the
    pair rotation of the Mamba-3 block."""
    from burn_dragon_b200.models.mamba import Mamba3Block, rmsnorm
    x = torch.randn(2, 40, 3, 64, device=device)
    freqs = R.build_freqs(64, 10000.0, "rope").to(device)
    q, _ = NR.norm_rotate(x, freqs=freqs, positions=5)
    want = R.rotate(rmsnorm(x).transpose(1, 2), "rope", freqs, 5).transpose(1, 2)
    assert ((q - want).abs() <= 2.0 ** -17 * pairs(want)).all()            # 45 turns in 32 bits: 45 * 2 pi * 2^-24 of a radian
    ang = torch.randn(2, 40, 32, device=device)
    q, _ = NR.norm_rotate(x, angles=ang)
    assert ((q - Mamba3Block._rotate(rmsnorm(x), ang[:, :, None])).abs() <= 2.0 ** -18 * pairs(q)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_one_token_at_a_time_and_position_forms(device):
    q, k = torch.randn(3, 9, 4, 32, device=device), torch.randn(3, 9, 2, 32, device=device)
    freqs = R.build_freqs(32, 10000.0, "rope").to(device)
    far = 2 ** 33                                                           # a position that 32 bits do not hold
    whole = NR.norm_rotate(q, k, freqs=freqs, positions=far)
    pos = far + torch.arange(9, device=device)
    for other in (pos, pos.expand(3, 9), pos.repeat(3, 1)):
        assert all(torch.equal(a, b) for a, b in zip(whole, NR.norm_rotate(q, k, freqs=freqs, positions=other)))
    for t in range(9):
        a = NR.norm_rotate(q[:, t:t + 1], k[:, t:t + 1], freqs=freqs, positions=pos[t].expand(3, 1))
        assert torch.equal(a[0], whole[0][:, t:t + 1]) and torch.equal(a[1], whole[1][:, t:t + 1])
    small = torch.arange(4, 13, device=device)
    a, b = NR.norm_rotate(q, freqs=freqs, positions=small), NR.norm_rotate(q, freqs=freqs, positions=small.int())
    assert torch.equal(a[0], b[0]) and torch.equal(a[0], NR.norm_rotate(q, freqs=freqs, positions=4)[0])


@pytest.mark.parametrize("device", DEVICES)
def test_what_pads_a_batch_is_not_read_and_empty_calls(device):
    q, k = torch.randn(3, 20, 4, 32, device=device), torch.randn(3, 20, 2, 32, device=device)
    ang = torch.randn(3, 20, 16, device=device)
    w = torch.randn(32, device=device)
    n = torch.tensor([20, 0, 7], device=device)
    for t in (q, k, ang):
        t[1], t[2, 7:] = float("nan"), float("inf")
    leaves = [t.detach().requires_grad_() for t in (q, k, w, ang)]
    a, b = NR.norm_rotate(leaves[0], leaves[1], leaves[2], leaves[2], angles=leaves[3], lengths=n)
    assert torch.isfinite(a).all() and torch.isfinite(b).all() and (a[1] == 0).all() and (b[2, 7:] == 0).all()
    bad = torch.ones_like(a)
    bad[2, 7:] = float("nan")
    if device == "cuda":
        for g in torch.autograd.grad([a, b], leaves, [bad, torch.ones_like(b)]):
            assert torch.isfinite(g).all()
    for B, T in ((0, 4), (2, 0)):
        x = torch.zeros(B, T, 2, 8, device=device, requires_grad=True)
        wt = torch.ones(8, device=device, requires_grad=True)
        o, _ = NR.norm_rotate(x, q_weight=wt)
        gx, gw = torch.autograd.grad(o.sum(), (x, wt))
        assert o.shape == x.shape and gx.shape == x.shape and (gw == 0).all()
    z, _ = NR.norm_rotate(torch.zeros(1, 1, 1, 8, device=device))          # a row of zeros stays zero
    assert (z == 0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_one_output_without_gradient_and_large_values(device):
    q, k = torch.randn(2, 6, 2, 16, device=device, requires_grad=True), torch.randn(2, 6, 1, 16, device=device, requires_grad=True)
    a, b = NR.norm_rotate(q, k)
    gk, = torch.autograd.grad(b.square().sum(), k)
    assert torch.isfinite(gk).all()
    big, _ = NR.norm_rotate(torch.full((1, 1, 1, 16), 60000.0, device=device, dtype=torch.float16))
    assert (big.float() - 1).abs().max() <= 2.0 ** -11


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    q, k = torch.zeros(2, 3, 4, 16, device=device), torch.zeros(2, 3, 2, 16, device=device)
    f = torch.zeros(16, device=device)
    z = lambda *s: torch.zeros(*s, device=device)                                                        # noqa: E731
    bad = [
        (dict(q=q[0]), "q:"), (dict(q=q.long()), "q:"), (dict(q=z(2, 3, 4, 15)), "q:"), (dict(q=z(2, 3, 4, 514)), "q:"),
        (dict(k=k[:, :2]), "k:"), (dict(k=k.half()), "k:"), (dict(q_weight=z(15)), "q_weight"), (dict(q_weight=z(4, 16), k_weight=z(16)), "k_weight"),
        (dict(k=None, k_weight=z(16)), "come with k"), (dict(freqs=f, angles=z(2, 3, 8)), "one of the two"), (dict(angles=z(2, 3, 9)), "angles"),
        (dict(angles=z(2, 2, 8)), "angles"), (dict(freqs=z(18)), "freqs"), (dict(freqs=z(15)), "freqs"), (dict(freqs=f, positions=z(3)), "positions"),
        (dict(freqs=f, positions=z(2).long()), "positions"), (dict(positions=3), "positions"), (dict(lengths=z(3).long()), "lengths"),
        (dict(angles=z(2, 3, 8), positions=torch.zeros(3, dtype=torch.int64, device=device)), "positions"),
        (dict(q_bias=torch.zeros(16, device="meta")), "q_bias"),
    ]
    for change, message in bad:
        args = {**dict(q=q, k=k), **change}
        with pytest.raises(ValueError, match=message):
            NR.norm_rotate(args.pop("q"), args.pop("k"), **args)
    with pytest.raises(ValueError, match="no gradient"):
        NR.norm_rotate(q, freqs=f.requires_grad_())


@pytest.mark.gpu
def test_two_runs_give_the_same_bits_and_replay_from_a_graph():
    tensors, how, n = make("cuda", torch.bfloat16, 2, 333, 33, 11, 128, 64, "data", True, True, True, True)

    def grads():
        leaves = [t.detach().requires_grad_() for t in tensors] + [how["angles"].detach().requires_grad_()]
        o = NR.norm_rotate(*leaves[:6], angles=leaves[6], lengths=n)
        return [t.detach() for t in o] + list(torch.autograd.grad([t.float().square().sum() for t in o], leaves))

    assert all(torch.equal(p, q) for p, q in zip(grads(), grads()))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        a, b = NR.norm_rotate(*tensors, lengths=n, **how)
    tensors[0].mul_(0.5)
    how["angles"].add_(1)
    n.clamp_(max=50)
    graph.replay()
    with torch.no_grad():
        a2, b2 = NR.norm_rotate(*tensors, lengths=n, **how)
    assert torch.equal(a, a2) and torch.equal(b, b2)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_behind_a_length_without_eps(device):
    """eps = 0: the norm of a row behind a length, which reads as 0, must not reach a result (0 / 0 there). Against the
    sequences by themselves in float64. A term is off by about (16 + 8) u, a sum of 14 of them by 14 u more, together 3e-6 of
    the terms' magnitudes, and these are at most 14 times the largest: 1e-4 of the largest result holds them."""
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g).to(device)                                               # noqa: E731
    q, w, b, an, dy = r(2, 5, 2, 16), r(16), r(16), r(2, 5, 8), r(2, 5, 2, 16)
    n = torch.tensor([5, 2], device=device)
    leaves = [t.clone().requires_grad_() for t in (q, w, b, an)]
    out, _ = NR.norm_rotate(leaves[0], None, leaves[1], None, leaves[2], angles=leaves[3], lengths=n, eps=0.0)
    got = [out.detach(), *torch.autograd.grad(out, leaves, dy)]
    exact = [t.double().requires_grad_() for t in (q, w, b, an)]
    want = []
    for i, m in enumerate((5, 2)):
        o, _ = NR.norm_rotate(exact[0][i:i + 1, :m], None, exact[1], None, exact[2], angles=exact[3][i:i + 1, :m], eps=0.0)
        want.append(torch.cat((o, o.new_zeros(1, 5 - m, 2, 16)), 1))
    want = torch.cat(want)
    want = [want.detach(), *torch.autograd.grad(want, exact, dy.double())]
    for a, e in zip(got, want):
        assert (a.double() - e).abs().max() <= 1e-4 * e.abs().max()
    assert (got[0][1, 2:] == 0).all() and (got[1][1, 2:] == 0).all()
