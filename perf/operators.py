"""Timed cases of the trainable policy's operators (g1.cu_amd/g1nn.py): what a gated residual policy runs when
it is trained on rollouts and when it acts.

* norm       root-mean-square norm of the residual stream after the addition of a block's output, forward and
             backward: (normed rows, new stream, gradients of the input, the stream and the weight)
* norm_q8    the same norm with its rows in 8 bits and a scale per row, as an acting policy uses it
* gated      both projections of the gated block, the activation and the product; with its gradients
             (train) or without (an acting policy)
* gated_q8   the gated block on 8-bit rows and 8-bit weights
* clip       the global norm of a policy's gradients, and the clipped gradients

Each operator has a plain form of elementary torch operations in 32 bits (own = False), the calls a user makes
of the framework (own = True), and a restatement in 64 bits (exact).
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "bf16": 2}
EPS = 1e-6
OBS, ACT = 100, 29


def _nn():
    at = os.path.join(ROOT, "g1.cu_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import g1nn
    return g1nn


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one robot acting: the residual stream's row on its way into an 8-bit block. The smallest call
        dict(name="norm_q8_1x1024", kind="norm_q8", M=1, K=1024, dtype="bf16", residual=True),
        # a ragged batch of evaluation worlds, a width that no vector divides
        dict(name="norm_q8_8191x1999", kind="norm_q8", M=8191, K=1999, dtype="fp32", residual=True),
        # the norm of one PPO minibatch (8192 worlds x 32 steps in four) at the policy's width
        dict(name="norm_65536x256", kind="norm", M=65536, K=256, dtype="fp32", residual=True),
        # the same minibatch in a wide mixed-precision policy: the largest norm
        dict(name="norm_bf16_65536x2048", kind="norm", M=65536, K=2048, dtype="bf16", residual=True),
        # one robot acting through the policy's width: latency alone
        dict(name="gated_1x256x512", kind="gated", M=1, K=256, F=512, dtype="fp32", act="silu", train=False),
        # a ragged batch of raw observations into an odd width, without gradients
        dict(name="gated_3001x100x389", kind="gated", M=3001, K=100, F=389, dtype="fp32", act="gelu", train=False),
        # one PPO minibatch through a gated block of the policy's width, with gradients
        dict(name="gated_train_65536x256x512", kind="gated", M=65536, K=256, F=512, dtype="fp32", act="silu",
             train=True),
        # the same minibatch through a wide mixed-precision block: the largest of all
        dict(name="gated_train_bf16_65536x512x2048", kind="gated", M=65536, K=512, F=2048, dtype="bf16", act="silu",
             train=True),
        # one robot acting through a wide 8-bit block of odd size
        dict(name="gated_q8_1x1024x2731", kind="gated_q8", M=1, K=1024, F=2731, dtype="bf16", act="silu"),
        # the training batch of worlds acting through an 8-bit block
        dict(name="gated_q8_8192x512x2048", kind="gated_q8", M=8192, K=512, F=2048, dtype="bf16", act="silu"),
        # the gradients of a small gated policy after one minibatch
        dict(name="clip_256x512x1", kind="clip", K=256, F=512, depth=1, dtype="fp32", norm=0.5),
        # those of a large mixed-precision policy: 16-bit gradients clipped into 32-bit ones
        dict(name="clip_bf16_2048x8192x5", kind="clip", K=2048, F=8192, depth=5, dtype="bf16", norm=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Seconds of a pass at moderate rates, to keep drawn cases below the largest listed one."""
    w = work(case)
    rate = {"fp32": 5e13, "bf16": 2e14}[case["dtype"]]
    return w["bytes"] / 2e12 + w["flops"] / rate


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["norm_q8", "norm", "gated", "gated", "gated_q8", "clip"])
        dtype = rng.choice(["fp32", "bf16"])
        act = rng.choice(["silu", "gelu"])
        M = _log_int(rng, 1, 65536)
        if kind == "clip":
            c = dict(kind=kind, K=_log_int(rng, 64, 2048), F=_log_int(rng, 64, 8192), depth=rng.randint(1, 5),
                     dtype=dtype, norm=rng.choice([0.5, 1.0, 20.0]))
        elif kind in ("norm", "norm_q8"):
            c = dict(kind=kind, M=M, K=_log_int(rng, 64, 4096), dtype=dtype, residual=rng.random() < 0.7)
        elif kind == "gated_q8":
            c = dict(kind=kind, M=M, K=_log_int(rng, 64, 1024), F=_log_int(rng, 64, 4096), dtype=dtype, act=act)
        else:
            c = dict(kind=kind, M=M, K=_log_int(rng, 64, 1024), F=_log_int(rng, 64, 2048), dtype=dtype, act=act,
                     train=rng.random() < 0.6)
        if _cost(c) <= most:
            return c


def _grad_shapes(case):
    """The parameter shapes of a gated residual policy: input layer, depth blocks, last norm, heads."""
    K, F = case["K"], case["F"]
    block = [(K,), (F, K), (F,), (F, K), (F,), (K, F), (K,)]
    return [(K, OBS), (K,)] + block * case["depth"] + [(K,), (ACT, K), (ACT,), (1, K), (1,), (ACT,)]


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dt = case["kind"], _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).add_(mean).to(dtype)

    s = dict(case=dict(case))
    if kind == "clip":
        # a step's gradients: heavier in some tensors than in others; scaled to a norm around 3
        shapes = _grad_shapes(case)
        n = sum(math.prod(x) for x in shapes)
        s["grads"] = [normal(*x, scale=3.0 / math.sqrt(n) * (0.5 + (i % 3))) for i, x in enumerate(shapes)]
        s["out"] = [torch.empty(x, device="cuda", dtype=torch.float32) for x in shapes]
        return s
    M, K = case["M"], case["K"]
    if kind in ("norm", "norm_q8"):
        # a block's output and a residual stream some layers deep: rows of different size
        rows = torch.exp(0.5 * torch.randn(M, 1, generator=gen, device="cuda"))
        s["x"] = (torch.randn(M, K, generator=gen, device="cuda") * rows).to(dt)
        s["r"] = (torch.randn(M, K, generator=gen, device="cuda") * (2 * rows)).to(dt) if case["residual"] else None
        s["w"] = normal(K, scale=0.1, mean=1.0)
        if kind == "norm":
            s["dy"] = normal(M, K, scale=1.0 / math.sqrt(M))
            s["dh"] = normal(M, K, scale=0.5 / math.sqrt(M)) if case["residual"] else None
            for k in ("x", "r", "w"):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    F = case["F"]
    if kind == "gated_q8":
        # what rms_norm_q8 writes of normed rows, and weights quantised once by rows
        def rows_q8(v):
            a = v.abs().amax(-1)
            return torch.round(v * (127.0 / a)[:, None]).to(torch.int8), a / 127.0
        s["q"], s["s"] = rows_q8(torch.randn(M, K, generator=gen, device="cuda"))
        s["qg"], s["sg"] = rows_q8(torch.randn(F, K, generator=gen, device="cuda") / math.sqrt(K))
        s["qu"], s["su"] = rows_q8(torch.randn(F, K, generator=gen, device="cuda") / math.sqrt(K))
        s["bg"] = normal(F, scale=0.1, dtype=torch.float32)
        s["bu"] = normal(F, scale=0.1, dtype=torch.float32)
        return s
    s["x"] = normal(M, K)
    s["wg"] = normal(F, K, scale=1.0 / math.sqrt(K))
    s["wu"] = normal(F, K, scale=1.0 / math.sqrt(K))
    s["bg"] = normal(F, scale=0.1)
    s["bu"] = normal(F, scale=0.1)
    if case["train"]:
        s["dy"] = normal(M, F, scale=1.0 / math.sqrt(M))
        for k in ("x", "wg", "wu", "bg", "bu"):
            s[k].requires_grad_()
    return s


# ------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    nn = _nn()
    c = s["case"]
    kind = c["kind"]
    if kind == "clip":
        norm = nn.clip_grad_norm(s["grads"], c["norm"], out=s["out"])
        return [norm] + s["out"]
    if kind == "norm":
        ins = [s["x"], s["w"]]
        if c["residual"]:
            ins.append(s["r"])
            y, h = nn.rms_norm(s["x"], s["w"], eps=EPS, residual=s["r"])
            grads = torch.autograd.grad([y, h], ins, [s["dy"], s["dh"]])
            return [y.detach(), h.detach(), *grads]
        y = nn.rms_norm(s["x"], s["w"], eps=EPS)
        return [y.detach(), *torch.autograd.grad(y, ins, s["dy"])]
    if kind == "norm_q8":
        # the 8-bit rows as the values they stand for
        if c["residual"]:
            q, scale, h = nn.rms_norm_q8(s["x"], s["w"], eps=EPS, residual=s["r"])
            return [q * scale[:, None], scale, h]
        q, scale = nn.rms_norm_q8(s["x"], s["w"], eps=EPS)
        return [q * scale[:, None], scale]
    if kind == "gated_q8":
        return nn.gated_linear_q8(s["q"], s["s"], s["qg"], s["sg"], s["qu"], s["su"], s["bg"], s["bu"],
                                  activation=c["act"], dtype=_TYPES[c["dtype"]])
    if not c["train"]:
        return nn.gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=c["act"])
    y = nn.gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=c["act"])
    ins = [s[k] for k in ("x", "wg", "wu", "bg", "bu")]
    return [y.detach(), *torch.autograd.grad(y, ins, s["dy"])]


# ------------------------------------------------------------------------------------ the plain forms
_GELU = math.sqrt(2.0 / math.pi)


def _act(g, name):
    """The activation and its derivative at g."""
    if name == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    t = torch.tanh(_GELU * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * _GELU * (1 + 3 * 0.044715 * g * g)


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    h = x + s["r"].float() if c["residual"] else x
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    xhat = h * rstd
    if c["kind"] == "norm_q8":
        u = h * w
        a = u.abs().amax(-1, keepdim=True)
        inv = torch.full_like(a, 127.0) / a
        q = torch.round(u * inv)
        scale = (a / 127.0) * rstd
        return [q * scale, scale[:, 0]] + ([h.to(dt)] if c["residual"] else [])
    dy = s["dy"].float()
    wdy = dy * w
    dx = rstd * (wdy - xhat * (wdy * xhat).mean(-1, keepdim=True))
    dw = (dy * xhat).sum(0)
    y = xhat * w
    if c["residual"]:
        dx = (dx + s["dh"].float()).to(dt)
        return [y.to(dt), h.to(dt), dx, dw.to(dt), dx]
    return [y.to(dt), dx.to(dt), dw.to(dt)]


def _plain_gated(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g = x @ wg.t() + s["bg"].float()
    u = x @ wu.t() + s["bu"].float()
    a, da = _act(g, c["act"])
    y = (a * u).to(dt)
    if not c["train"]:
        return y
    dy = s["dy"].float()
    dg = dy * u * da
    du = dy * a
    dx = dg @ wg + du @ wu
    return [y, dx.to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt), dg.sum(0).to(dt), du.sum(0).to(dt)]


def _plain_gated_q8(s):
    c = s["case"]
    # sums of products of whole numbers: in 32 bits, as everything else here
    q = s["q"].float()
    g = (q @ s["qg"].float().t()) * (s["s"][:, None] * s["sg"]) + s["bg"]
    u = (q @ s["qu"].float().t()) * (s["s"][:, None] * s["su"]) + s["bu"]
    return (_act(g, c["act"])[0] * u).to(_TYPES[c["dtype"]])


def _plain_clip(s):
    total = torch.sqrt(torch.stack([(g.float() * g.float()).sum() for g in s["grads"]]).sum())
    coef = torch.clamp(s["case"]["norm"] / (total + 1e-6), max=1.0)
    return [total] + [g.float() * coef for g in s["grads"]]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        kind = state["case"]["kind"]
        plain = {"clip": _plain_clip, "gated": _plain_gated, "gated_q8": _plain_gated_q8}.get(kind, _plain_norm)
        return plain(state)


# ------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b, kind = _BYTES[case["dtype"]], case["kind"]
    if kind == "clip":
        n = sum(math.prod(x) for x in _grad_shapes(case))
        return {"bytes": n * (b + 4), "flops": 3 * n}
    M, K = case["M"], case["K"]
    n, r = M * K, 1 if case.get("residual") else 0
    if kind == "norm_q8":
        return {"bytes": n * (b + 1 + 2 * r * b) + K * b + 4 * M, "flops": 6 * n}
    if kind == "norm":
        # x, r, w -> y, h; dy, dh -> dx (the stream's gradient is the same rows), dw
        return {"bytes": n * b * (4 + 3 * r) + 2 * K * b, "flops": 14 * n}
    F = case["F"]
    if kind == "gated_q8":
        return {"bytes": n + 4 * M + 2 * F * K + 16 * F + M * F * b, "flops": 4 * M * K * F}
    once = n * b + 2 * F * (K + 1) * b + M * F * b
    if not case["train"]:
        return {"bytes": once, "flops": 4 * M * K * F}
    return {"bytes": 2 * once, "flops": 12 * M * K * F}


# ------------------------------------------------------------------------------------ in 64 bits
def _wide(t):
    return None if t is None else t.detach().to(torch.float64)


def exact(case, seed):
    """The definitions in 64 bits. The 8-bit rows are rounded where 64-bit values round."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "clip":
        g = [_wide(x) for x in s["grads"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(x) for x in g]))
        factor = min(1.0, case["norm"] / (float(norm) + 1e-6))
        return [norm] + [x * factor for x in g]
    if kind in ("norm", "norm_q8"):
        h = _wide(s["x"]) if s["r"] is None else _wide(s["x"]) + _wide(s["r"])
        w, K = _wide(s["w"]), case["K"]
        size = torch.sqrt(torch.linalg.vector_norm(h, dim=1) ** 2 / K + EPS)
        if kind == "norm_q8":
            y = h * w / size[:, None]
            step = torch.amax(torch.abs(y), dim=1) / 127.0
            out = [torch.round(y / step[:, None]) * step[:, None], step]
            return out + ([h] if s["r"] is not None else [])
        y = h / size[:, None] * w
        # the Jacobian of h / size(h): (1 - h h^T / (K size^2)) / size
        v = _wide(s["dy"]) * w
        dx = (v - h * ((v * h).sum(1) / (K * size ** 2))[:, None]) / size[:, None]
        dw = torch.einsum("mk,mk->k", _wide(s["dy"]), h / size[:, None])
        if s["r"] is None:
            return [y, dx, dw]
        dx = dx + _wide(s["dh"])
        return [y, h, dx, dw, dx]
    if kind == "gated_q8":
        x, wg, wu = _wide(s["q"]), _wide(s["qg"]), _wide(s["qu"])
        x, wg, wu = x * _wide(s["s"])[:, None], wg * _wide(s["sg"])[:, None], wu * _wide(s["su"])[:, None]
    else:
        x, wg, wu = _wide(s["x"]), _wide(s["wg"]), _wide(s["wu"])
    gate = torch.addmm(_wide(s["bg"]), x, wg.t().contiguous())
    up = torch.addmm(_wide(s["bu"]), x, wu.t().contiguous())
    if case["act"] == "silu":
        e = torch.exp(-gate)
        a = gate / (1 + e)
        da = (1 + e + gate * e) / (1 + e) ** 2
    else:
        # 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z))
        z = math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
        p = 1 / (1 + torch.exp(-2 * z))
        a = gate * p
        da = p + gate * 2 * p * (1 - p) * math.sqrt(2 / math.pi) * (1 + 0.134145 * gate ** 2)
    if not case.get("train"):
        return a * up
    out = a * up
    dy = _wide(s["dy"])
    du = dy * a
    del a
    dg = dy * up * da
    del up, da, gate, dy
    dx = torch.mm(dg, wg) + torch.mm(du, wu)
    return [out, dx, torch.mm(dg.t().contiguous(), x), torch.mm(du.t().contiguous(), x), dg.sum(0), du.sum(0)]
