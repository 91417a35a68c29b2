"""Calls of the state-space operators (`ops.mamba_ops.causal_conv`, `ops.norm_rotate`, `ops.selective_scan`) that are allowed but
unusual: states updated in place between a forward and its backward pass, other kinds of derivatives, infinities, growing
states, inputs that share a buffer. u = 2^-24 is half a unit in the last place of fp32."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from burn_dragon_b200.ops import mamba_ops as MO
from burn_dragon_b200.ops import norm_rotate as NR
from burn_dragon_b200.ops import selective_scan as S

U = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
NAMES = ["conv", "norm_rotate", "scan"]


def rand(device, seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g).to(device)


def calls(device):
    """{operator: (call of its tensors, those tensors)}; every tensor has a gradient."""
    r = rand(device, 9)
    B, T, D, N = 2, 9, 8, 4
    return {
        "conv": (lambda x, w, b, st: MO.causal_conv(x, w, b, state=st), [r(B, T, D), r(D, 4), r(D), r(B, 3, D)]),
        "norm_rotate": (lambda q, k, qw, kw, qb, kb, an: NR.norm_rotate(q, k, qw, kw, qb, kb, angles=an),
                        [r(B, T, 3, D), r(B, T, 2, D), r(D), r(D), r(D), r(D), r(B, T, 3)]),
        "scan": (lambda u, dt, A, Bm, Cm, Dk, db, h0: S.selective_scan(u, dt, A, Bm, Cm, Dk, dt_bias=db, dt_softplus=True, h0=h0),
                 [r(B, T, D), r(B, T, D), -r(D, N).abs(), r(B, T, N), r(B, T, N), r(D), r(D), r(B, D, N)]),
    }


def step_calls(device):
    """The same of the single-token forms, which take `out`."""
    r = rand(device, 10)
    B, D, N = 2, 8, 4
    return {
        "conv": (lambda x, st, w, b, out=None: MO.causal_conv_step(x, st, w, b, out=out), [r(B, D), r(B, 3, D), r(D, 4), r(D)], 1),
        "scan": (lambda u, dt, A, Bm, Cm, h, Dk, db, out=None: S.selective_scan_step(u, dt, A, Bm, Cm, h, Dk, dt_bias=db, dt_softplus=True, out=out),
                 [r(B, D), r(B, D), -r(D, N).abs(), r(B, N), r(B, N), r(B, D, N), r(D), r(D)], 5),
    }


@pytest.mark.parametrize("name", ["conv", "scan"])
@pytest.mark.parametrize("device", DEVICES)
def test_a_step_in_place_counts_as_a_change_of_its_state(device, name):
    fn, tensors, state = step_calls(device)[name]
    out = torch.empty_like(tensors[state])
    before, kept = out._version, tensors[state]._version
    fn(*tensors, out=out)
    assert out._version > before and tensors[state]._version == kept
    before = tensors[state]._version
    fn(*tensors, out=tensors[state])
    assert tensors[state]._version > before
    with torch.inference_mode():                                             # (tensors made there count no changes)
        inner = tensors[state].clone()
        fn(*tensors, out=inner)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["conv", "scan"])
def test_a_backward_pass_refuses_a_state_that_changed_since(name):
    fn, tensors = calls("cuda")[name]
    step, row, at = step_calls("cuda")[name]
    leaves = [t.clone().requires_grad_() for t in tensors[:-1]]
    state = tensors[-1].clone()
    y, _ = fn(*leaves, state)
    step(*row[:at], state, *row[at + 1:], out=torch.empty_like(state))       # the state itself stays: no objection
    want = torch.autograd.grad(y.sum(), leaves, retain_graph=True)
    step(*row[:at], state, *row[at + 1:], out=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), leaves)
    y, _ = fn(*leaves, tensors[-1])
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y.sum(), leaves)))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_tangents_are_carried_or_refused(device, name):
    """The torch statements carry a tangent; the kernels have no forward mode and say so, with and without a gradient."""
    fn, tensors = calls(device)[name]
    for i, t in enumerate(tensors):
        for grad in (False, True):
            with fwAD.dual_level():
                leaf = t.clone().requires_grad_(grad)
                args = [fwAD.make_dual(leaf, torch.ones_like(t)) if j == i else v for j, v in enumerate(tensors)]
                if device == "cuda":
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        fn(*args)
                else:
                    assert any(fwAD.unpack_dual(o).tangent is not None for o in fn(*args))
    if device == "cuda":
        fn(*tensors)


@pytest.mark.parametrize("name", ["conv", "scan"])
@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_tangents_of_single_tokens(device, name):
    fn, tensors, _ = step_calls(device)[name]
    for i, t in enumerate(tensors):
        with fwAD.dual_level():
            args = [fwAD.make_dual(v, torch.ones_like(v)) if j == i else v for j, v in enumerate(tensors)]
            if device == "cuda":
                with pytest.raises(RuntimeError, match="forward-mode"):
                    fn(*args)
            else:
                assert any(fwAD.unpack_dual(o).tangent is not None for o in fn(*args))


@pytest.mark.gpu
def test_forward_mode_tangents_of_frequencies():
    q, f = torch.randn(1, 2, 1, 8, device="cuda"), torch.rand(8, device="cuda")
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        NR.norm_rotate(q, freqs=fwAD.make_dual(f, torch.ones_like(f)))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("device", DEVICES)
def test_a_gradient_penalty_is_not_dropped(device, name):
    """The seed of the first derivative is a constant, the gradient depends on the inputs all the same: the torch statements
    differentiate it, the kernels refuse. Every input in turn, by backward() and by grad()."""
    fn, tensors = calls(device)[name]
    for i in range(len(tensors)):
        leaves = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(tensors)]
        for whole in (True, False):
            outs = fn(*leaves)
            used = [o for o in outs if o.requires_grad]
            first, = torch.autograd.grad(sum(o.sum() for o in used), leaves[i], create_graph=True)
            loss = sum(o.square().sum() for o in used) + first.square().sum()
            if device == "cuda":
                with pytest.raises(RuntimeError, match="no second derivative"):
                    loss.backward() if whole else torch.autograd.grad(loss, leaves[i])
            elif whole:
                loss.backward()
            else:
                torch.autograd.grad(loss, leaves[i])
    if device == "cuda":                              # asked for once, a gradient is what it was
        leaves = [t.clone().requires_grad_() for t in tensors]
        out = fn(*leaves)[0]
        once = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(once, torch.autograd.grad(out.sum(), leaves, create_graph=True)))


INF_STATES = [3, 5, 12, 16, 20, 33, 64]


@pytest.mark.parametrize("N", INF_STATES)
@pytest.mark.parametrize("T,D,ragged", [(20, 16, False), (300, 24, False), (20, 17, False), (37, 16, True)])
@pytest.mark.parametrize("device", DEVICES)
def test_an_infinite_input_reaches_its_own_results_only(device, N, T, D, ragged):
    """An infinite dt' u makes its own states infinite, and what is made of them: not the sums over the rows behind a
    sequence, where the state stays and everything is 0. B, C, dy > 0, so no infinity meets another; which results are
    infinite or NaN is the float64 statement's. A finite one is a sum of at most 64 T terms, each off by (24 + (24 + T) 2) u per
    step back, of which at most 50 matter (dt' A < -0.1: exp(-5) is left), and the sum by 64 T u more: 50 (24 + 648) u +
    19200 u = 3.2e-3 of the largest of its kind for T = 300."""
    g = torch.Generator().manual_seed(N + T)
    r = lambda *s: (torch.rand(*s, generator=g) + 0.1).to(device)                                        # noqa: E731
    p = dict(u=r(2, T, D), dt=r(2, T, D), A=-r(D, N) - 0.9, B=r(2, T, N), C=r(2, T, N), D=r(D), dt_bias=r(D), h0=r(2, D, N))
    p["u"][0, T // 2, 3] = float("inf")
    p["u"][1, 5, D - 1] = float("-inf")
    dy, dh = r(2, T, D), r(2, D, N)
    n = torch.tensor([T, 11], device=device) if ragged else None

    def both(q, dy, dh, fn):
        leaves = {k: t.detach().requires_grad_() for k, t in q.items()}
        y, h = fn(leaves["u"], leaves["dt"], leaves["A"], leaves["B"], leaves["C"], leaves["D"], dt_bias=leaves["dt_bias"], h0=leaves["h0"], lengths=n)
        return dict(y=y.detach(), h=h.detach(), **dict(zip(("d_" + k for k in leaves), torch.autograd.grad([y, h], list(leaves.values()), [dy, dh]))))

    got = both(p, dy, dh, S.selective_scan)
    want = both({k: t.double() for k, t in p.items()}, dy.double(), dh.double(), S.selective_scan_reference)
    if ragged:                                        # (the statement's own derivatives have 0 * inf at the rows behind a length)
        cut = {k: t[1:, :11] if k in ("u", "dt", "B", "C") else t[1:] if k == "h0" else t for k, t in p.items()}
        n = None
        one = both({k: t.double() for k, t in cut.items()}, dy[1:, :11].double(), dh[1:].double(), S.selective_scan_reference)
        first = {k: t[:1] if k in ("u", "dt", "B", "C", "h0") else t for k, t in p.items()}
        two = both({k: t.double() for k, t in first.items()}, dy[:1].double(), dh[:1].double(), S.selective_scan_reference)
        for k in want:
            if k in ("d_A", "d_D", "d_dt_bias"):
                want[k] = two[k] + one[k]
            elif k in ("h", "d_h0"):
                want[k] = torch.cat((two[k], one[k]))
            else:
                want[k] = torch.cat((two[k], torch.nn.functional.pad(one[k], (0, 0, 0, T - 11))))
    for k in got:
        if device == "cpu" and ragged and k not in ("y", "h"):
            continue
        a, e = got[k].double(), want[k]
        fine = torch.isfinite(e)
        assert torch.equal(torch.isfinite(a), fine) and torch.equal(torch.isnan(a), torch.isnan(e)), k
        assert torch.equal(a[~fine].nan_to_num(), e[~fine].nan_to_num()), k
        assert (a[fine] - e[fine]).abs().max() <= 3.2e-3 * e[fine].abs().max(), k


@pytest.mark.parametrize("N", [5, 12, 16])
@pytest.mark.parametrize("T", [20, 300])
@pytest.mark.parametrize("device", DEVICES)
def test_an_infinite_step_forgets_the_past(device, N, T):
    """dt' = inf: the decays are exp(-inf) = 0 and the states infinite; the other channels do not notice."""
    g = torch.Generator().manual_seed(N)
    r = lambda *s: (torch.rand(*s, generator=g) + 0.1).to(device)                                        # noqa: E731
    u, dt, A, Bm, Cm = r(1, T, 16), r(1, T, 16), -r(16, N) - 0.9, r(1, T, N), r(1, T, N)
    clean, _ = S.selective_scan(u, dt, A, Bm, Cm)
    dt[0, T // 2, 3] = float("inf")
    y, h = S.selective_scan(u, dt, A, Bm, Cm)
    assert torch.isinf(y[0, T // 2:, 3]).all() and torch.isinf(h[0, 3]).all()
    y[0, T // 2:, 3] = clean[0, T // 2:, 3]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("T", [1, 40, 300])
@pytest.mark.parametrize("device", DEVICES)
def test_without_a_skip_an_infinite_input_is_not_multiplied_by_zero(device, T):
    g = torch.Generator().manual_seed(T)
    r = lambda *s: (torch.rand(*s, generator=g) + 0.1).to(device)                                        # noqa: E731
    u, dt, A, Bm, Cm, h0 = r(2, T, 24), r(2, T, 24), -r(24, 16) - 0.9, r(2, T, 16), r(2, T, 16), r(2, 24, 16)
    u[1, T // 2, 5] = float("inf")
    with torch.no_grad():
        y, _ = S.selective_scan(u, dt, A, Bm, Cm, h0=h0)
        assert torch.isinf(y[1, T // 2:, 5]).all() and torch.isfinite(y[0]).all()
        if T == 1:
            y, h = S.selective_scan_step(u[:, 0], dt[:, 0], A, Bm[:, 0], Cm[:, 0], h0)
            assert torch.isinf(y[1, 5]) and torch.isinf(h[1, 5]).all() and torch.isfinite(y[0]).all()
    u[1, T // 2, 5] = 1
    leaf = u.clone().requires_grad_()
    dy = r(2, T, 24)
    dy[0, T // 2, 7] = float("inf")
    y, _ = S.selective_scan(leaf, dt, A, Bm, Cm, h0=h0)
    du, = torch.autograd.grad(y, leaf, dy)
    assert torch.isinf(du[0, :T // 2 + 1, 7]).all() and torch.isfinite(du[1]).all() and torch.isfinite(du[0, T // 2 + 1:]).all()


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("device", DEVICES)
def test_an_infinite_bias_does_not_reach_rows_behind_a_length(device, softplus):
    r = rand(device, 3)
    bias = torch.zeros(8, device=device)
    bias[2] = float("inf")
    h0 = r(2, 8, 4)
    y, h = S.selective_scan(r(2, 30, 8).abs(), r(2, 30, 8).abs(), -r(8, 4).abs() - 0.1, r(2, 30, 4).abs() + 0.1, r(2, 30, 4).abs() + 0.1, dt_bias=bias,
                            dt_softplus=softplus, h0=h0, lengths=torch.tensor([5, 30], device=device))
    assert torch.isfinite(h[0, :2]).all() and torch.isinf(y[0, 0, 2]) and (y[0, 5:] == 0).all() and not torch.isfinite(y[1, :, 2]).any()
    one, h1 = S.selective_scan(*(t[:, :1] for t in (r(1, 3, 8).abs(), r(1, 3, 8).abs())), -r(8, 4).abs() - 0.1, r(1, 1, 4).abs() + 0.1,
                               r(1, 1, 4).abs() + 0.1, dt_bias=bias, dt_softplus=softplus)
    assert torch.isinf(one[0, 0, 2]) and torch.isinf(h1[0, 2]).all() and torch.isfinite(h1[0, 3:]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_states_that_grow_while_they_are_zero(device):
    """A > 0 and inputs that start late: the growth over what came before is past 2^128, of a state of zero. Then the gradients
    where nothing of the outputs that are used reaches back over the growth. At most 20 steps of growth up to exp(3) hold
    something: a result is off by 20 (24 + 44 * 3) u and 2^4 u for its sums, 2e-4 of the largest of its kind."""
    T, D, N = 3000, 24, 16
    r = rand(device, 12)
    A = 0.4 + 0.1 * torch.rand(D, N, generator=torch.Generator().manual_seed(1)).to(device)
    u, dt, Bm, Cm, dy = r(1, T, D), torch.full((1, T, D), 6.0, device=device), r(1, T, N), r(1, T, N), r(1, T, D)
    u[:, :T - 10] = 0
    y, h = S.selective_scan(u, dt, A, Bm, Cm)
    y0, h0 = S.selective_scan_reference(*(t.double() for t in (u, dt, A, Bm, Cm)))
    for a, e in ((y, y0), (h, h0)):
        assert torch.isfinite(e).all() and (a.double() - e).abs().max() <= 2e-4 * e.abs().max()
    dy[:, 10:] = 0
    dt[:, :20], dt[:, T - 20:] = 0.01, 0.01
    leaves = [t.clone().requires_grad_() for t in (u, dt, A, Bm, Cm)]
    exact = [t.double().requires_grad_() for t in (u, dt, A, Bm, Cm)]
    got = torch.autograd.grad(S.selective_scan(*leaves)[0], leaves, dy)
    want = torch.autograd.grad(S.selective_scan_reference(*exact)[0], exact, dy.double())
    for a, e in zip(got, want):
        assert torch.isfinite(e).all() and (a.double() - e).abs().max() <= 2e-4 * e.abs().max()


@pytest.mark.parametrize("device", DEVICES)
def test_a_small_state_that_grows_within_a_few_steps(device):
    """h0 = 1e-30 and a growth of exp(115) = 9e49 in five steps: the result, 9e19, is a number of fp32, the growth is not. The
    sum of the steps' x = 115 is off by (24 + 5) u |x| = 2e-4."""
    T, D = 3000, 24
    z = lambda *s: torch.zeros(*s, device=device)                                                        # noqa: E731
    dt = z(1, T, D)
    dt[:, 1008:1013] = 23
    y, h = S.selective_scan(z(1, T, D), dt, torch.ones(D, 16, device=device), z(1, T, 16), z(1, T, 16), h0=torch.full((1, D, 16), 1e-30, device=device))
    assert (torch.log(h.double()) - (115 + math.log(1e-30))).abs().max() <= 2e-4 and (y == 0).all()
    dy, leaf = z(1, T, D), torch.full((1, D, 16), 1e-30, device=device).requires_grad_()
    _, h = S.selective_scan(z(1, T, D), dt, torch.ones(D, 16, device=device), z(1, T, 16), z(1, T, 16), h0=leaf)
    back, = torch.autograd.grad(h, leaf, torch.full_like(h, 1e-30))
    assert (torch.log(back.double()) - (115 + math.log(1e-30))).abs().max() <= 2e-4


@pytest.mark.parametrize("N", [12, 16])
@pytest.mark.parametrize("device", DEVICES)
def test_an_infinite_state_outlives_a_long_decay(device, N):
    """The decay over a segment of many steps is below the numbers of fp32; each step's is not, so that an infinite state (B, C, u > 0) or
    gradient (C, B, dy > 0) stays infinite as far as it reaches, and nothing else is touched."""
    T, D = 3000, 24
    g = torch.Generator().manual_seed(N)
    r = lambda *s: (torch.rand(*s, generator=g) + 0.5).to(device)                                        # noqa: E731
    u, dt, A, Bm, Cm, dy = r(1, T, D), r(1, T, D), -4 - r(D, N), r(1, T, N), r(1, T, N), r(1, T, D)
    clean, h0 = S.selective_scan(u, dt, A, Bm, Cm)
    bad = u.clone()
    bad[0, 100, 3] = float("inf")
    y, h = S.selective_scan(bad, dt, A, Bm, Cm)
    assert torch.isinf(y[0, 100:, 3]).all() and torch.isinf(h[0, 3]).all()
    rest = torch.ones(T, D, dtype=torch.bool, device=device)
    rest[100:, 3] = False
    assert torch.equal(y[0][rest], clean[0][rest]) and torch.equal(h[0, torch.arange(D) != 3], h0[0, torch.arange(D) != 3])
    dy[0, 2900, 3] = float("inf")
    leaf = u.clone().requires_grad_()
    du, = torch.autograd.grad(S.selective_scan(leaf, dt, A, Bm, Cm)[0], leaf, dy)
    assert torch.isinf(du[0, :2901, 3]).all() and torch.isfinite(du[0, 2901:]).all() and torch.isfinite(du[0, :, torch.arange(D) != 3]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_one_stream_in_place_under_another_batch_stride(device):
    """The batch stride of a single stream means nothing."""
    r = rand(device, 16)
    w, pool, x = r(8, 4), r(2, 5, 3, 8), r(1, 8)
    one, same = pool[:1, 2], pool[0, 2].unsqueeze(0)
    assert one.stride(0) != same.stride(0)
    y, new = MO.causal_conv_step(x, one.clone(), w)
    y2, _ = MO.causal_conv_step(x, one, w, out=same)
    assert torch.equal(y, y2) and torch.equal(one, new)


@pytest.mark.parametrize("device", DEVICES)
def test_states_and_rows_of_one_buffer_that_share_no_memory(device):
    """A stream's row beside its state in one buffer: no byte of one is a byte of the other."""
    r = rand(device, 14)
    B, D, N = 3, 8, 4
    w = r(D, 4)
    for lo, at in ((0, 3), (1, 0)):
        buf = r(B, 4, D)
        x, st = buf[:, at], buf[:, lo:lo + 3]
        y, new = MO.causal_conv_step(x.clone(), st.clone(), w)
        y2, _ = MO.causal_conv_step(x, st, w, out=st)
        assert torch.equal(y, y2) and torch.equal(st, new)
    buf = r(B, 2 * D + 2 * N + D * N)
    u, dt, Bm, Cm, h = buf.split([D, D, N, N, D * N], -1)
    h = h.unflatten(-1, (D, N))
    row = [u, dt, -r(D, N).abs(), Bm, Cm]
    y, new = S.selective_scan_step(*[t.clone() for t in row], h.clone())
    rest = buf[:, :-D * N].clone()
    y2, _ = S.selective_scan_step(*row, h, out=h)
    assert torch.equal(y, y2) and torch.equal(h, new) and torch.equal(buf[:, :-D * N], rest)


@pytest.mark.gpu
def test_states_that_overlap_a_parameter_are_refused():
    """Bias, skip and the marks of active streams are read while other threads write states."""
    z = lambda *s: torch.zeros(*s, device="cuda")                                                        # noqa: E731
    st = z(2, 3, 8)
    for more in (dict(bias=st[0, 0]), dict(active=st.view(torch.bool)[0, 0, :2])):
        with pytest.raises(RuntimeError, match="overlaps an input"):
            MO.causal_conv_step(z(2, 8), z(2, 3, 8), z(8, 4), out=st, **more)
    h = z(2, 8, 4)
    for more in (dict(D=h[0, :2].view(-1)), dict(dt_bias=h[1, 6:].view(-1)), dict(active=h.view(torch.bool)[0, 0, :2])):
        with pytest.raises(RuntimeError, match="overlaps an input"):
            S.selective_scan_step(z(2, 8), z(2, 8), z(8, 4), z(2, 4), z(2, 4), z(2, 8, 4), out=h, **more)


def test_states_that_overlap_through_another_storage_are_refused():
    """Two tensors made over the same memory have storages of their own."""
    memory = bytearray(4 * 72)
    old = torch.frombuffer(memory, dtype=torch.float32, count=48).view(2, 3, 8)
    new = torch.frombuffer(memory, dtype=torch.float32, count=48, offset=96).view(2, 3, 8)
    assert old.untyped_storage().data_ptr() != new.untyped_storage().data_ptr()
    with pytest.raises(ValueError, match="overlaps"):
        MO.causal_conv_step(torch.zeros(2, 8), old, torch.zeros(8, 4), out=new)
    again = torch.frombuffer(memory, dtype=torch.float32, count=48).view(2, 3, 8)
    MO.causal_conv_step(torch.zeros(2, 8), old, torch.zeros(8, 4), out=again)


@pytest.mark.parametrize("kind", ["far", "half"])
@pytest.mark.parametrize("device", DEVICES)
def test_angles_of_other_types(device, kind):
    """Angles keep the value they have in their own type: 10^7 radians in float64 (32 bits leave whole radians), bf16 angles
    whose sine is not one of bf16. A row's norm is off by (Dh / 2 + 8) u, its turn by 2^-21 |v|: 2^-19 of the pair holds them."""
    r = rand(device, 17)
    q, do = r(2, 5, 3, 16), r(2, 5, 3, 16)
    angle = 1e7 * r(2, 5, 8).double() if kind == "far" else (3 * r(2, 5, 8)).bfloat16()
    leaf = angle.clone().requires_grad_()
    out, _ = NR.norm_rotate(q, angles=leaf)
    da, = torch.autograd.grad(out, leaf, do)
    v = q.double() / (q.double().square().mean(-1, keepdim=True) + 1e-5).sqrt()
    turned = torch.view_as_complex(v.unflatten(-1, (8, 2))) * torch.polar(torch.ones(2, 5, 1, 8, device=device).double(), angle.double()[:, :, None])
    want = torch.view_as_real(turned).flatten(-2)
    size = turned.abs()[..., None].expand(*turned.shape, 2).flatten(-2)
    assert ((out.double() - want).abs() <= 2.0 ** -19 * size).all()
    cross = want[..., 0::2] * do.double()[..., 1::2] - want[..., 1::2] * do.double()[..., 0::2]
    scale = (turned.abs() * do.double().unflatten(-1, (8, 2)).abs().sum(-1)).sum(2)
    assert da.dtype == angle.dtype
    assert ((da.double() - cross.sum(2)).abs() <= 2.0 ** -18 * scale + torch.finfo(da.dtype).eps / 2 * cross.sum(2).abs()).all()


@pytest.mark.parametrize("form", ["int", "tensor"])
@pytest.mark.parametrize("device", DEVICES)
def test_frequencies_in_64_bits(device, form):
    """At position 3 10^9 a frequency rounded to 32 bits is off by 3 10^9 f 2^-25 turns, 90 f: in 64 bits nothing of that is left."""
    r = rand(device, 19)
    q, start = r(2, 5, 3, 16), 3_000_000_000
    freqs = (torch.rand(8, generator=torch.Generator().manual_seed(2), dtype=torch.float64) / 3).repeat_interleave(2).to(device)
    pos = start + torch.arange(5, device=device)
    out, _ = NR.norm_rotate(q, freqs=freqs, positions=start if form == "int" else pos)
    turns = pos.double()[:, None] * freqs[0::2]
    angle = 2 * math.pi * (turns - turns.floor())
    v = q.double() / (q.double().square().mean(-1, keepdim=True) + 1e-5).sqrt()
    turned = torch.view_as_complex(v.unflatten(-1, (8, 2))) * torch.polar(torch.ones_like(angle), angle)[None, :, None]
    size = turned.abs()[..., None].expand(*turned.shape, 2).flatten(-2)
    assert ((out.double() - torch.view_as_real(turned).flatten(-2)).abs() <= 2.0 ** -19 * size).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("device", DEVICES)
def test_rows_whose_squares_are_subnormal(device, dtype):
    """eps = 0 and elements of about 1e-20, whose squares (1e-40) are subnormal numbers of fp32, in steps of 1.4e-45: each is
    off by at most 7e-46, the mean by 1e-5 of itself with the elements drawn here, the result by half of that and its rounding."""
    r = rand(device, 18)
    x = (1e-20 * (1 + r(2, 3, 2, 16).abs())).to(dtype)
    leaf = x.clone().requires_grad_()
    out, _ = NR.norm_rotate(leaf, eps=0.0)
    dx, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    v = x.double().requires_grad_()
    want = v / v.square().mean(-1, keepdim=True).sqrt()
    dw, = torch.autograd.grad(want, v, torch.ones_like(want))
    half = torch.finfo(dtype).eps / 2
    assert ((out.double() - want).abs() <= (1e-5 + half) * want.abs()).all()
    if device == "cuda":                              # (torch's own derivative of the root takes its third power: inf)
        assert (dx.double() - dw).abs().max() <= (1e-4 + half) * (1 / x.double().square().mean(-1).sqrt()).max()


@pytest.mark.parametrize("device", DEVICES)
def test_the_state_behind_an_empty_prompt_is_its_own(device):
    """A prompt of no rows returns the state it was given, in memory of its own: a step in place on the one leaves the other."""
    z = lambda *s: torch.zeros(*s, device=device)                                                        # noqa: E731
    h0 = torch.randn(2, 8, 4, device=device)
    kept = h0.clone()
    _, h = S.selective_scan(z(2, 0, 8), z(2, 0, 8), z(8, 4), z(2, 0, 4), z(2, 0, 4), h0=h0)
    assert torch.equal(h, h0) and h.data_ptr() != h0.data_ptr()
    S.selective_scan_step(z(2, 8), z(2, 8) + 1, z(8, 4) - 1, z(2, 4), z(2, 4), h, out=h)
    assert torch.equal(h0, kept) and not torch.equal(h, h0)
    st = torch.randn(2, 3, 8, device=device)
    _, end = MO.causal_conv(z(2, 0, 8), z(8, 4), state=st)
    assert torch.equal(end, st) and end.data_ptr() != st.data_ptr()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,T,C,k,ragged", [
    (torch.bfloat16, 4, 20_000, 8, 4, False),         # 5000 tiles of 16 rows: a thread walks a second one
    (torch.float32, 3, 30_011, 6, 3, True),
    (torch.float16, 4, 20_000, 7, 2, True),           # element by element
    (torch.float32, 2, 2500, 4160, 4, False),         # tiles of 64 rows
    (torch.bfloat16, 2, 3000, 3968, 2, True),         # of 32
    (torch.bfloat16, 4, 20_100, 16, 5, True),         # a width known at run time
])
def test_convolutions_of_many_tiles(dtype, B, T, C, k, ragged):
    """Against the definition in 64 bits. A gradient row is a sum of k terms, each off by 16 u and the quick SiLU's 2^-19 (1 + m) for
    inputs of magnitude m; a parameter's is a sum of n = B T of them in an order whose longest chain is below n / 64 + 256 terms."""
    g = torch.Generator(device="cuda").manual_seed(C)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")                                           # noqa: E731
    x, dy, w, b, st = r(B, T, C).to(dtype), r(B, T, C).to(dtype), r(C, k) / k ** 0.5, 0.1 * r(C), r(B, k - 1, C).to(dtype)
    n = torch.randint(T // 2, T + 1, (B,), generator=g, device="cuda") if ragged else None
    leaves = [t.clone().requires_grad_() for t in (x, w, b, st)]
    y, _ = MO.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], lengths=n)
    dx, dw, db, dst = torch.autograd.grad(y, leaves, dy)
    keep = torch.ones(B, T, 1, device="cuda", dtype=torch.bool) if n is None else (torch.arange(T, device="cuda") < n[:, None])[..., None]
    eps = torch.finfo(dtype).eps / 2
    floor = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    for c in range(0, C, 1024):                       # channels are independent
        at = slice(c, c + 1024)
        seq = torch.cat((st[..., at].double(), torch.where(keep, x[..., at].double(), 0.0)), 1)
        pre = sum((seq[:, j:j + T] * w[at, j].double() for j in range(k)), b[at].double())
        mag = sum((seq[:, j:j + T].abs() * w[at, j].double().abs() for j in range(k)), b[at].double().abs())
        sig = torch.sigmoid(pre)
        off = 2.0 ** -19 * (1 + mag)
        want = torch.where(keep, pre * sig, 0.0)
        assert ((y[..., at].double() - want).abs() <= eps * want.abs() + off * mag + floor).all()
        gr = torch.where(keep, dy[..., at].double() * sig * (1 + pre * (1 - sig)), 0.0)
        bound = torch.where(keep, dy[..., at].double().abs() * off * (1 + mag), 0.0)
        ds, es = torch.zeros_like(seq), torch.zeros_like(seq)
        chain = (B * T / 64 + 256) * U
        for j in range(k):
            ds[:, j:j + T] += gr * w[at, j].double()
            es[:, j:j + T] += (bound + 16 * U * gr.abs()) * w[at, j].double().abs()
            want, lim = (gr * seq[:, j:j + T]).sum((0, 1)), ((bound + chain * gr.abs()) * seq[:, j:j + T].abs()).sum((0, 1))
            assert ((dw[at, j].double() - want).abs() <= lim + eps * want.abs()).all(), j
        assert ((db[at].double() - gr.sum((0, 1))).abs() <= (bound + chain * gr.abs()).sum((0, 1))).all()
        assert ((dx[..., at].double() - ds[:, k - 1:]).abs() <= eps * ds[:, k - 1:].abs() + es[:, k - 1:] + floor).all()
        assert ((dst[..., at].double() - ds[:, :k - 1]).abs() <= eps * ds[:, :k - 1].abs() + es[:, :k - 1] + floor).all()


@pytest.mark.parametrize("n", [8, 32, 128])
@pytest.mark.parametrize("form", ["sequence", "steps"])
@pytest.mark.parametrize("device", DEVICES)
def test_slow_states_do_not_drift(device, form, n):
    """A state that keeps its past for n steps adds up what its exponentials are off by on average, -1.5 to 0.6 10^-8 of themselves
    over the ranges of x here: with 1.6 10^-8 the mean over 1024 states is off by at most n times that. (A state's own
    roundings, up to 2^-24 to either side, leave at most 4 10^-8 of the mean.)"""
    D, N, T = 64, 16, 512
    g = torch.Generator().manual_seed(20)
    dt = ((torch.rand(1, T, D, generator=g) + 0.5) / n).to(device)
    A = (-1 - 0.01 * torch.rand(D, N, generator=g)).to(device)
    one = lambda *s: torch.ones(*s, device=device)                                                       # noqa: E731
    with torch.no_grad():
        if form == "sequence":
            _, h = S.selective_scan(one(1, T, D), dt, A, one(1, T, N), one(1, T, N))
        else:
            h = torch.zeros(1, D, N, device=device)
            for t in range(T):
                S.selective_scan_step(one(1, D), dt[:, t], A, one(1, N), one(1, N), h, out=h)
    want = torch.zeros(1, D, N, dtype=torch.float64, device=device)
    for t in range(T):
        want = torch.exp(dt[:, t, :, None].double() * A.double()) * want + dt[:, t, :, None].double()
    assert (h.double() / want - 1).mean().abs() <= n * 1.6e-8 + 4e-8


@pytest.mark.parametrize("device", DEVICES)
def test_lengths_in_32_bits(device):
    """The same bits whatever the type of the lengths, which may be a view; negative ones are 0, large ones all rows."""
    r = rand(device, 21)
    long = torch.tensor([[5, 0], [-1, 0], [40, 0], [17, 0]], device=device)[:, 0]
    x, w = r(4, 21, 16), r(16, 4)
    q, qw = r(4, 21, 2, 16), r(16)
    u, dt, A, Bm, Cm = r(4, 21, 16), r(4, 21, 16).abs(), -r(16, 8).abs(), r(4, 21, 8), r(4, 21, 8)
    for n in (long.int(), long.clamp(0, 21), long.clamp(0, 21).int()):
        assert all(torch.equal(a, b) for a, b in zip(MO.causal_conv(x, w, lengths=long), MO.causal_conv(x, w, lengths=n)))
        assert torch.equal(NR.norm_rotate(q, q_weight=qw, lengths=long)[0], NR.norm_rotate(q, q_weight=qw, lengths=n)[0])
        assert all(torch.equal(a, b) for a, b in zip(S.selective_scan(u, dt, A, Bm, Cm, lengths=long), S.selective_scan(u, dt, A, Bm, Cm, lengths=n)))


@pytest.mark.parametrize("device", DEVICES)
def test_a_convolution_of_one_tap(device):
    """Width 1 has a state of no rows: given or not, carried or stepped, it is act(bias + w x)."""
    r = rand(device, 22)
    x, w, b, st = r(3, 9, 24), r(24, 1), r(24), torch.zeros(3, 0, 24, device=device)
    n = torch.tensor([9, 0, 4], device=device)
    keep = (torch.arange(9, device=device) < n[:, None])[..., None]
    pre = x.double() * w[:, 0].double() + b.double()
    want = torch.where(keep, pre * torch.sigmoid(pre), 0.0)
    for state in (None, st):
        y, end = MO.causal_conv(x, w, b, state=state, lengths=n)
        assert end.shape == (3, 0, 24) and (y.double() - want).abs().max() <= 2.0 ** -19 * (1 + pre.abs().max()) * pre.abs().max()
    y1, end = MO.causal_conv_step(x[:, 0], st, w, b, active=n > 0)
    assert end.shape == (3, 0, 24) and (y1 - y[:, 0]).abs().max() <= 2.0 ** -20 * (1 + pre.abs().max()) * pre.abs().max()
    MO.causal_conv_step(x[:, 0], st, w, b, out=st)


@pytest.mark.gpu
def test_offsets_past_31_bits():
    """Views whose last sequence starts more than 2^31 elements in; only what is read of them exists in full."""
    B, T, step = 3, 20, 2 ** 30 + 64
    wide = torch.empty(B * step, device="cuda", dtype=torch.bfloat16)
    tail = wide.as_strided((B, 2 ** 14), (step, 1), step - 2 ** 14)
    tail.copy_(torch.randn(B, 2 ** 14, device="cuda"))
    view = lambda at, *s: wide.as_strided((B, T, *s), (step, 400, *torch.empty(*s).stride()), step - 2 ** 14 + at)   # noqa: E731
    u, dt, Bm, Cm, q = view(0, 64), view(64, 64), view(128, 16), view(144, 16), view(160, 3, 64)
    A = -torch.rand(64, 16, device="cuda")
    assert (B - 1) * step > 2 ** 31
    for fn, tensors in ((lambda *t: S.selective_scan(*t[:2], A, *t[2:], dt_softplus=True), [u, dt, Bm, Cm]), (lambda t: NR.norm_rotate(t, t[:, :, :2])[:2], [q])):
        leaves, dense = [t.detach().requires_grad_() for t in tensors], [t.detach().clone().requires_grad_() for t in tensors]
        got, want = fn(*leaves), fn(*dense)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        seeds = [torch.ones_like(o) for o in got]
        grads = [torch.autograd.grad(got, leaves, seeds), torch.autograd.grad(want, dense, seeds)]
        assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """The same inputs through forward and backward passes that run beside each other, each with scratch of its own."""
    fns = {k: v for k, v in calls("cuda").items()}
    streams = [torch.cuda.Stream() for _ in range(2)]
    big = {"conv": [torch.randn(4, 2000, 256, device="cuda"), torch.randn(256, 4, device="cuda"), torch.randn(256, device="cuda"),
                    torch.randn(4, 3, 256, device="cuda")],
           "norm_rotate": [torch.randn(4, 500, 8, 64, device="cuda"), torch.randn(4, 500, 2, 64, device="cuda")] +
                          [torch.randn(64, device="cuda") for _ in range(4)] + [torch.randn(4, 500, 32, device="cuda")],
           "scan": [torch.randn(2, 1500, 64, device="cuda"), torch.randn(2, 1500, 64, device="cuda"), -torch.rand(64, 16, device="cuda"),
                    torch.randn(2, 1500, 16, device="cuda"), torch.randn(2, 1500, 16, device="cuda"), torch.randn(64, device="cuda"),
                    torch.randn(64, device="cuda"), torch.randn(2, 64, 16, device="cuda")]}

    def run(name):
        leaves = [t.detach().requires_grad_() for t in big[name]]
        outs = fns[name][0](*leaves)
        return [*(o.detach() for o in outs), *torch.autograd.grad([o.square().sum() for o in outs], leaves)]

    want = {name: run(name) for name in NAMES}
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append({name: run(name) for name in NAMES})
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for name in NAMES for a, b in zip(want[name], g[name]))
