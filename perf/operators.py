"""The operators of a state-space layer between its two projections, as cases to be timed and compared.

  conv   causal depthwise convolution (+ SiLU) with a carried state       burn_dragon_b200.ops.mamba_ops
  qk     RMS norm of every query / key head and its rotation in one pass  burn_dragon_b200.ops.norm_rotate
  scan   selective scan, h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t         burn_dragon_b200.ops.selective_scan

Each has a `step` (one token for each stream of a batch), a `prompt` (forward) and a `train` case (forward and
every gradient). `run` computes the plain form in fp32 torch operations where `own` is false, and calls the
framework's operators where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases -------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 streams through the convolution of a 2048-wide model (expansion 2)
        dict(name="conv_step", op="conv", mode="step", dtype="bf16", B=64, T=1, C=4096, k=4, silu=True, ragged=False, carry=True),
        # segments of a prompt that carries its state on, at the widths of the Mamba-2 preset (512 + 2 * 128 channels)
        dict(name="conv_prompt_segment", op="conv", mode="prompt", dtype="fp32", B=4, T=1111, C=768, k=4, silu=True, ragged=True, carry=True),
        # a training batch of a 2048-wide model
        dict(name="conv_train", op="conv", mode="train", dtype="bf16", B=8, T=2048, C=4096, k=4, silu=True, ragged=False, carry=False),
        # decode: grouped queries and keys of 64 streams, each at a position of its own, far into a context
        dict(name="qk_step", op="qk", mode="prompt", dtype="bf16", B=64, T=1, Hq=32, Hk=8, Dh=128, rot=128, angles="positions", heads=False,
             bias=False, ragged=False),
        # training: the same heads over sequences of 4096 tokens
        dict(name="qk_train", op="qk", mode="train", dtype="bf16", B=4, T=4096, Hq=32, Hk=8, Dh=128, rot=128, angles="positions",
             heads=False, bias=False, ragged=False),
        # training: C and B of the Mamba-3 preset (state 128, rank 2) under angles that are learned from the data
        dict(name="qk_train_angles", op="qk", mode="train", dtype="fp32", B=8, T=1000, Hq=2, Hk=2, Dh=128, rot=128, angles="data",
             heads=True, bias=True, ragged=True),
        # one decode step of 64 streams, 4096 channels
        dict(name="scan_step", op="scan", mode="step", dtype="bf16", B=64, T=1, D=4096, N=16, ragged=False, carry=True),
        # a short prompt at the width of the presets (512 channels)
        dict(name="scan_prompt_short", op="scan", mode="prompt", dtype="fp32", B=1, T=257, D=512, N=16, ragged=False, carry=False),
        # a long prompt of one stream
        dict(name="scan_prompt_long", op="scan", mode="prompt", dtype="bf16", B=1, T=8192, D=4096, N=16, ragged=False, carry=False),
        # prompts of different lengths in one batch, a larger state, continued from a carried one
        dict(name="scan_prompt_ragged", op="scan", mode="prompt", dtype="fp16", B=6, T=777, D=1000, N=64, ragged=True, carry=True),
        # a training batch
        dict(name="scan_train", op="scan", mode="train", dtype="bf16", B=4, T=2048, D=2048, N=16, ragged=False, carry=False),
        # one segment of a long sequence whose state and its gradient are handed on, ragged, fp32
        dict(name="scan_train_segment", op="scan", mode="train", dtype="fp32", B=3, T=500, D=520, N=16, ragged=True, carry=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "qk", "scan", "scan"])
    mode = rng.choice(["prompt", "train", "step"] if op != "qk" else ["prompt", "train"])
    c = dict(op=op, mode=mode, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    ragged, carry = rng.random() < 0.4, rng.random() < 0.5
    if mode == "step":
        c.update(B=_log(rng, 1, 256), T=1)
        ragged, carry = False, True
    else:
        c.update(B=_log(rng, 1, 16), T=_log(rng, 1, 8192))
    rows = c["B"] * c["T"]
    if op == "conv":
        width = max(1, min(8192, 60_000_000 // rows))
        C = _log(rng, min(64, width), width)
        c.update(C=C - C % 8 if C > 64 and rng.random() < 0.7 else C, k=rng.choice([2, 3, 4, 4, 4, 5, 8]), silu=rng.random() < 0.8,
                 ragged=ragged, carry=carry)
    elif op == "qk":
        Dh = rng.choice([32, 64, 64, 80, 128, 128, 256, 2 * rng.randint(4, 128)])
        most = max(1, min(64, 75_000_000 // (rows * Dh) // 2))
        Hk = _log(rng, 1, min(16, most))
        c.update(Hq=Hk * rng.randint(1, max(1, most // Hk)), Hk=Hk, Dh=Dh, rot=rng.choice([Dh, Dh, max(2, Dh // 4 * 2)]),
                 angles=rng.choice(["positions", "positions", "data"]), heads=rng.random() < 0.4, bias=rng.random() < 0.4, ragged=ragged)
    else:
        N = rng.choice([16, 16, 16, 8, 32, 64, rng.randint(1, 64)])
        width = max(1, min(8192, 250_000_000 // (rows * N)))
        D = _log(rng, min(64, width), width)
        c.update(D=D - D % 8 if D > 64 and rng.random() < 0.7 else D, N=N, ragged=ragged, carry=carry)
    return c


# ---- inputs ------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    B, T = case["B"], case["T"]
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")                       # noqa: E731
    s = {"case": dict(case)}
    if case["ragged"]:
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device="cuda")
        s["lengths"][int(torch.randint(0, B, (1,), generator=g, device="cuda"))] = T
    else:
        s["lengths"] = None
    if case["op"] == "conv":
        C, k = case["C"], case["k"]
        s["x"] = randn(B, T, C).to(dt)
        s["w"] = randn(C, k) / math.sqrt(k)
        s["bias"] = 0.1 * randn(C)
        s["state"] = randn(B, k - 1, C).to(dt) if case["carry"] else None
        if case["mode"] == "train":
            s["dy"] = randn(B, T, C).to(dt)
    elif case["op"] == "qk":
        Hq, Hk, Dh, rot = case["Hq"], case["Hk"], case["Dh"], case["rot"]
        s["q"], s["k"] = randn(B, T, Hq, Dh).to(dt), randn(B, T, Hk, Dh).to(dt)
        for n, H in (("q", Hq), ("k", Hk)):
            shape = (H, Dh) if case["heads"] else (Dh,)
            s[n + "_weight"] = 1 + 0.1 * randn(*shape)
            s[n + "_bias"] = 0.1 * randn(*shape) if case["bias"] else None
        s["angles"] = s["freqs"] = s["positions"] = None
        if case["angles"] == "data":
            s["angles"] = torch.cumsum(0.1 * randn(B, T, rot // 2).abs(), dim=1)
        else:
            # cycles per position, the two channels of a pair alike; positions of streams that are far into their context
            pair = torch.arange(rot // 2, device="cuda", dtype=torch.float64).repeat_interleave(2)
            s["freqs"] = (65536.0 ** (-2.0 * pair / rot) / (2 * math.pi)).float()
            start = torch.randint(0, 200_000, (B, 1), generator=g, device="cuda")
            s["positions"] = start + torch.arange(T, device="cuda")
        if case["mode"] == "train":
            s["dq"], s["dk"] = randn(B, T, Hq, Dh).to(dt), randn(B, T, Hk, Dh).to(dt)
    else:
        D, N = case["D"], case["N"]
        s["u"] = torch.nn.functional.silu(randn(B, T, D)).to(dt)
        s["dt"] = (0.5 * randn(B, T, D)).to(dt)
        step = torch.exp(torch.rand(D, generator=g, device="cuda") * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))                             # softplus gives `step` back
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32).repeat(D, 1) * (1 + 0.05 * randn(D, N)).abs()
        s["B"], s["C"] = randn(B, T, N).to(dt), randn(B, T, N).to(dt)
        s["D"] = 1 + 0.1 * randn(D)
        s["h0"] = randn(B, D, N) if case["carry"] else None
        if case["mode"] == "train":
            s["dy"] = randn(B, T, D).to(dt)
            s["dhT"] = randn(B, D, N) if case["carry"] else None
    return s


# ---- the framework's operators -----------------------------------------------------------------------
def _leaf(t):
    return t.detach().requires_grad_() if t is not None else None


def _grads(outputs, douts, named):
    named = {n: t for n, t in named.items() if t is not None}
    pairs = [(o, d) for o, d in zip(outputs, douts) if d is not None]
    got = torch.autograd.grad([o for o, _ in pairs], list(named.values()), [d for _, d in pairs])
    return dict(zip(("d_" + n for n in named), got))


def _run_own(s):
    from burn_dragon_b200.ops import mamba_ops, norm_rotate, selective_scan
    c = s["case"]
    if c["op"] == "conv":
        act = "silu" if c["silu"] else None
        if c["mode"] == "step":
            y, st = mamba_ops.causal_conv_step(s["x"][:, 0], s["state"], s["w"], s["bias"], activation=act)
            return {"y": y, "state": st}
        if c["mode"] == "prompt":
            y, st = mamba_ops.causal_conv(s["x"], s["w"], s["bias"], state=s["state"], lengths=s["lengths"], activation=act)
            return {"y": y, "state": st}
        p = {n: _leaf(s[n]) for n in ("x", "w", "bias", "state")}
        y, st = mamba_ops.causal_conv(p["x"], p["w"], p["bias"], state=p["state"], lengths=s["lengths"], activation=act)
        return {"y": y.detach(), "state": st.detach(), **_grads([y], [s["dy"]], p)}
    if c["op"] == "qk":
        where = dict(freqs=s["freqs"], positions=s["positions"]) if s["freqs"] is not None else {}
        names = ("q", "k", "q_weight", "k_weight", "q_bias", "k_bias", "angles")
        p = {n: _leaf(s[n]) if c["mode"] == "train" else s[n] for n in names}
        q, k = norm_rotate.norm_rotate(p["q"], p["k"], p["q_weight"], p["k_weight"], p["q_bias"], p["k_bias"], angles=p["angles"],
                                       lengths=s["lengths"], **where)
        if c["mode"] != "train":
            return {"q": q, "k": k}
        return {"q": q.detach(), "k": k.detach(), **_grads([q, k], [s["dq"], s["dk"]], p)}
    if c["mode"] == "step":
        y, h = selective_scan.selective_scan_step(s["u"][:, 0], s["dt"][:, 0], s["A"], s["B"][:, 0], s["C"][:, 0], s["h0"], s["D"],
                                                  dt_bias=s["dt_bias"], dt_softplus=True)
        return {"y": y, "h": h}
    names = ("u", "dt", "A", "B", "C", "D", "dt_bias", "h0")
    p = {n: _leaf(s[n]) if c["mode"] == "train" else s[n] for n in names}
    y, h = selective_scan.selective_scan(p["u"], p["dt"], p["A"], p["B"], p["C"], p["D"], dt_bias=p["dt_bias"], dt_softplus=True,
                                         h0=p["h0"], lengths=s["lengths"])
    if c["mode"] != "train":
        return {"y": y, "h": h}
    return {"y": y.detach(), "h": h.detach(), **_grads([y, h], [s["dy"], s["dhT"]], p)}


# ---- the plain forms ---------------------------------------------------------------------------------
def _valid(s, B, T):
    """[B, T] truth values: the rows of each sequence, without what pads it."""
    t = torch.arange(T, device="cuda")
    return t < (s["lengths"][:, None] if s["lengths"] is not None else torch.full((B, 1), T, device="cuda"))


def _plain_conv(s):
    c = s["case"]
    B, T, C, k, dtype = c["B"], c["T"], c["C"], c["k"], s["x"].dtype
    keep = _valid(s, B, T)[..., None]
    x = torch.where(keep, s["x"].float(), 0.0)
    head = s["state"].float() if s["state"] is not None else x.new_zeros(B, k - 1, C)
    seq = torch.cat((head, x), 1)                                                        # [B, T + k - 1, C]
    taps = seq.unfold(1, k, 1)                                                           # [B, T, C, k]
    pre = (taps * s["w"]).sum(-1) + s["bias"]
    sig = torch.sigmoid(pre)
    y = torch.where(keep, pre * sig if c["silu"] else pre, 0.0)
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device="cuda")
    rows = n[:, None] + torch.arange(k - 1, device="cuda")
    out = {"y": y.to(dtype), "state": torch.gather(seq, 1, rows[..., None].expand(-1, -1, C)).to(dtype)}
    if c["mode"] != "train":
        return {"y": out["y"][:, 0], "state": out["state"]} if c["mode"] == "step" else out
    g = torch.where(keep, s["dy"].float(), 0.0)
    if c["silu"]:
        g = g * sig * (1 + pre * (1 - sig))
    padded = torch.nn.functional.pad(g, (0, 0, k - 1, k - 1))                            # [B, T + 2k - 2, C]
    dseq = (padded.unfold(1, k, 1) * s["w"].flip(1)).sum(-1)                             # [B, T + k - 1, C]
    out["d_x"] = dseq[:, k - 1:].to(dtype)
    out["d_w"] = (g[..., None] * taps).sum((0, 1))
    out["d_bias"] = g.sum((0, 1))
    if s["state"] is not None:
        out["d_state"] = dseq[:, :k - 1].to(dtype)
    return out


def _turn(v, cos, sin, rot):
    """Channel pairs (2i, 2i + 1) of the first `rot` channels of v [B, T, H, Dh], turned by the angle of pair i."""
    a, b = v[..., 0:rot:2], v[..., 1:rot:2]
    turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, v[..., rot:]), -1)


def _plain_qk_one(s, n, cos, sin, keep):
    """Output of one of q and k, and in training its gradients and what it adds to the angles' gradient."""
    c = s["case"]
    rot, train = c["rot"], c["mode"] == "train"
    x = torch.where(keep, s[n].float(), 0.0)
    w, b = s[n + "_weight"], s[n + "_bias"]
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
    hat = x * r
    v = hat * w + (b if b is not None else 0.0)
    got = {n: torch.where(keep, _turn(v, cos, sin, rot), 0.0).to(s[n].dtype)}
    if not train:
        return got, None
    dv = _turn(torch.where(keep, s["d" + n].float(), 0.0), cos, -sin, rot)
    dims = (0, 1) if c["heads"] else (0, 1, 2)
    dhat = dv * w
    got["d_" + n] = (r * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))).to(s[n].dtype)
    got["d_%s_weight" % n] = (dv * hat).sum(dims)
    if b is not None:
        got["d_%s_bias" % n] = dv.sum(dims)
    da = (v[..., 0:rot:2] * dv[..., 1:rot:2] - v[..., 1:rot:2] * dv[..., 0:rot:2]).sum(2)
    return got, da


def _plain_qk(s):
    c = s["case"]
    keep = _valid(s, c["B"], c["T"])[..., None, None]
    if s["angles"] is not None:
        angle = s["angles"]
        cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None]
    else:
        turns = s["positions"].double()[..., None] * s["freqs"][0::2].double()           # far positions: 64 bits
        angle = (turns - turns.floor()) * (2 * math.pi)
        cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    out, da_q = _plain_qk_one(s, "q", cos, sin, keep)
    more, da_k = _plain_qk_one(s, "k", cos, sin, keep)
    out.update(more)
    if c["mode"] == "train" and s["angles"] is not None:
        out["d_angles"] = da_q + da_k
    return out


def _recur(a, b):
    """x_t = a_t x_{t-1} + b_t along dimension 1, x_{-1} = 0, by doubling the reach of every element."""
    reach = 1
    while reach < a.shape[1]:
        b = torch.cat((b[:, :reach], b[:, reach:] + a[:, reach:] * b[:, :-reach]), 1)
        a = torch.cat((a[:, :reach], a[:, reach:] * a[:, :-reach]), 1)
        reach *= 2
    return b


def _plain_scan(s):
    c = s["case"]
    B, T, D, N, dtype = c["B"], c["T"], c["D"], c["N"], s["u"].dtype
    keep = _valid(s, B, T)[..., None]
    A, skip = s["A"], s["D"]
    pick = lambda n: torch.where(keep, s[n].float(), 0.0)                                # noqa: E731
    u, Bm, Cm = pick("u"), pick("B"), pick("C")
    raw = pick("dt") + s["dt_bias"]
    dt = torch.where(keep, torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20)))), 0.0)
    a = torch.exp(dt[..., None] * A)                                                     # [B, T, D, N]
    b = (dt * u)[..., None] * Bm[:, :, None]
    if s["h0"] is not None:
        b[:, 0] += a[:, 0] * s["h0"]
    h = _recur(a, b)
    del b
    y = (h * Cm[:, :, None]).sum(-1) + skip * u
    out = {"y": torch.where(keep, y, 0.0).to(dtype), "h": h[:, -1].clone()}
    if c["mode"] != "train":
        return {"y": out["y"][:, 0], "h": out["h"]} if c["mode"] == "step" else out
    dy = pick("dy")
    e = dy[..., None] * Cm[:, :, None]
    if s["dhT"] is not None:
        e[:, -1] += s["dhT"]
    g = _recur(torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), 1).flip(1), e.flip(1)).flip(1)
    del e
    gb = (g * Bm[:, :, None]).sum(-1)
    first = s["h0"][:, None] if s["h0"] is not None else torch.zeros_like(h[:, :1])
    q = g * a * torch.cat((first, h[:, :-1]), 1)
    draw_ = torch.where(keep, ((q * A).sum(-1) + u * gb) * torch.where(raw > 20, 1.0, torch.sigmoid(raw)), 0.0)
    out["d_u"] = torch.where(keep, dt * gb + skip * dy, 0.0).to(dtype)
    out["d_dt"] = draw_.to(dtype)
    out["d_A"] = (q * dt[..., None]).sum((0, 1))
    out["d_B"] = (g * (dt * u)[..., None]).sum(2).to(dtype)
    out["d_C"] = (h * dy[..., None]).sum(2).to(dtype)
    out["d_D"] = (dy * u).sum((0, 1))
    out["d_dt_bias"] = draw_.sum((0, 1))
    if s["h0"] is not None:
        out["d_h0"] = a[:, 0] * g[:, 0]
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"conv": _plain_conv, "qk": _plain_qk, "scan": _plain_scan}[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B, T, train = case["B"], case["T"], case["mode"] == "train"
    if case["op"] == "conv":
        n, edge = B * T * case["C"], B * (case["k"] - 1) * case["C"]
        tensors = 4 if train else 2
        params = case["C"] * (case["k"] + 1) * 4
        edges = edge * (1 + case["carry"] * (2 if train else 1))
        return {"bytes": tensors * n * size + edges * size + params * (2 if train else 1),
                "flops": n * (2 * case["k"] + 4) * (4 if train else 1)}
    if case["op"] == "qk":
        n = B * T * (case["Hq"] + case["Hk"]) * case["Dh"]
        at = B * T * (case["rot"] // 2 * 4 * (2 if train else 1) if case["angles"] == "data" else 8)
        params = (case["Hq"] + case["Hk"] if case["heads"] else 2) * case["Dh"] * 4 * (1 + case["bias"])
        return {"bytes": (4 if train else 2) * n * size + at + params * (2 if train else 1), "flops": n * (8 if not train else 26)}
    D, N = case["D"], case["N"]
    rows, h = B * T, B * D * N * 4
    tensors = (6 if train else 3) * rows * D * size + (4 if train else 2) * rows * N * size
    states = h * (1 + case["carry"]) * (2 if train and case["carry"] else 1)
    params = (D * N + 2 * D) * 4 * (2 if train else 1)
    return {"bytes": tensors + states + params, "flops": rows * D * (N * (6 if not train else 22) + 8)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def _exact_conv(c, s):
    B, T, C, k = c["B"], c["T"], c["C"], c["k"]
    lengths = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
    x, w, bias = (s[n].double().requires_grad_() for n in ("x", "w", "bias"))
    state = s["state"].double().requires_grad_() if s["state"] is not None else None
    ys, ends = [], []
    for b, n in enumerate(lengths):
        seq = torch.cat((state[b] if state is not None else x.new_zeros(k - 1, C), x[b, :n]))
        pre = bias + sum(seq[j:j + n] * w[:, j] for j in range(k))
        act = pre / (1 + torch.exp(-pre)) if c["silu"] else pre
        ys.append(torch.cat((act, x.new_zeros(T - n, C))))
        ends.append(seq[n:n + k - 1].detach())
    y, end = torch.stack(ys), torch.stack(ends)
    if c["mode"] != "train":
        return {"y": y.detach()[:, 0] if c["mode"] == "step" else y.detach(), "state": end}
    return {"y": y.detach(), "state": end, **_grads([y], [s["dy"].double()], {"x": x, "w": w, "bias": bias, "state": state})}


def _exact_qk(c, s):
    names = ("q", "k", "q_weight", "k_weight", "q_bias", "k_bias", "angles")
    p = {n: s[n].double().requires_grad_() if s[n] is not None else None for n in names}
    keep = torch.ones(c["B"], c["T"], 1, 1, device="cuda", dtype=torch.bool)
    if s["lengths"] is not None:
        keep = (torch.arange(c["T"], device="cuda")[None] < s["lengths"][:, None])[..., None, None]
    angle = p["angles"] if p["angles"] is not None else 2 * math.pi * (s["positions"].double()[..., None] * s["freqs"][::2].double())
    unit = torch.polar(torch.ones_like(angle), angle)[:, :, None]
    outs = []
    for n in ("q", "k"):
        x = p[n] * keep
        v = x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * p[n + "_weight"]
        if p[n + "_bias"] is not None:
            v = v + p[n + "_bias"]
        pairs = v[..., :c["rot"]].unflatten(-1, (-1, 2))
        turned = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * unit).flatten(-2)
        outs.append(torch.cat((turned, v[..., c["rot"]:]), -1) * keep)
    got = {"q": outs[0].detach(), "k": outs[1].detach()}
    if c["mode"] == "train":
        got.update(_grads(outs, [s["dq"].double(), s["dk"].double()], p))
    return got


def _exact_scan(c, s):
    B, T, D, N = c["B"], c["T"], c["D"], c["N"]
    train = c["mode"] == "train"
    if B * T * D * N * 8 * (2 if train else 0) > 60e9:
        return None
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device="cuda")
    u, raw, Bm, Cm = s["u"].double(), s["dt"].double() + s["dt_bias"].double(), s["B"].double(), s["C"].double()
    A, skip = s["A"].double(), s["D"].double()
    dt = torch.nn.functional.softplus(raw, threshold=40)
    h = s["h0"].double().clone() if s["h0"] is not None else u.new_zeros(B, D, N)
    y, past = torch.zeros_like(u), []
    for t in range(T):
        live = (t < lengths)[:, None, None]
        if train:
            past.append(h)
        new = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * u[:, t])[..., None] * Bm[:, t, None]
        h = torch.where(live, new, h)
        y[:, t] = ((h * Cm[:, t, None]).sum(-1) + skip * u[:, t]) * live[..., 0]
    got = {"y": y[:, 0] if c["mode"] == "step" else y, "h": h}
    if not train:
        return got
    dy = s["dy"].double()
    r = s["dhT"].double() if s["dhT"] is not None else torch.zeros_like(h)               # gradient of the state behind step t
    du, ddt, dB, dC = (torch.zeros_like(v) for v in (u, dt, Bm, Cm))
    dA, dD, dbias = torch.zeros_like(A), torch.zeros_like(skip), torch.zeros_like(skip)
    after = h
    for t in range(T - 1, -1, -1):
        live = (t < lengths)[:, None]
        a = torch.exp(dt[:, t, :, None] * A)
        dyt = dy[:, t] * live
        g = r + Cm[:, t, None] * dyt[..., None]
        gb = (g * Bm[:, t, None]).sum(-1)
        q = g * a * past[t]
        slope = torch.sigmoid(raw[:, t])
        du[:, t] = (dt[:, t] * gb + skip * dyt) * live
        ddt[:, t] = ((q * A).sum(-1) + u[:, t] * gb) * slope * live
        dA += (q * (dt[:, t] * live)[..., None]).sum(0)
        dB[:, t] = (g * (dt[:, t] * u[:, t])[..., None]).sum(1) * live
        dC[:, t] = (after * dyt[..., None]).sum(1)
        dD += (dyt * u[:, t]).sum(0)
        dbias += ddt[:, t].sum(0)
        r = torch.where(live[..., None], a * g, r)
        after = past[t]
    got.update(d_u=du, d_dt=ddt, d_A=dA, d_B=dB, d_C=dC, d_D=dD, d_dt_bias=dbias)
    if s["h0"] is not None:
        got["d_h0"] = r
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"conv": _exact_conv, "qk": _exact_qk, "scan": _exact_scan}[case["op"]](case, s)
