"""The policy operators (g1nn) against plain forms in 64 bits, with bounds that follow from the arithmetic: u is half
a unit in the last place of a 32-bit value, o of the output's type; a sum of n products is off by at most (n + 16) u
times the sum of their magnitudes (products, roundings and the few operations beside it included), whatever its
order."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6


@pytest.fixture(scope="module")
def nn():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import g1nn
    return g1nn


def _torch():
    import torch
    return torch


def _dtype(name):
    torch = _torch()
    return {"fp32": torch.float32, "bf16": torch.bfloat16}[name]


def _ulp(name):
    return U if name == "fp32" else 2.0 ** -8   # 24 and 8 significant bits


def _normal(gen, *shape, dtype, scale=1.0, mean=0.0):
    torch = _torch()
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale + mean).to(dtype)


def _gen(seed):
    return _torch().Generator().manual_seed(seed)


def _within(got, ref, bound, what):
    got, ref, bound = got.detach().double().cpu(), ref.double(), bound.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    far = (got - ref).abs() - bound
    assert bool((far <= 0).all()), (what, float(far.max()), int((far > 0).sum()))


# ------------------------------------------------------------------------------------ norm
def _norm_ref(x, w, r):
    h = x.double() if r is None else x.double() + r.double()
    s = 1 / (h.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    return h, s, h * s * w.double()


NORM_SHAPES = [(1, 1), (1, 1024), (3, 29), (5, 100), (257, 64), (130, 256), (2, 257), (64, 1000), (7, 1999), (9, 2048),
               (3, 4096), (4, 5001), (2, 9000), (2, 16384), (1, 32768), (1, 32767), (2100, 16), (0, 64)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K", NORM_SHAPES)
def test_norm(nn, M, K, residual, dtype):
    dt, g, o = _dtype(dtype), _gen(M * 7 + K), _ulp(dtype)
    x, w = _normal(g, M, K, dtype=dt), _normal(g, K, dtype=dt, scale=0.2, mean=1)
    r = _normal(g, M, K, dtype=dt, scale=2) if residual else None
    h, _, y = _norm_ref(x, w, r)
    got = nn.rms_norm(x.cuda(), w.cuda(), EPS, None if r is None else r.cuda())
    if residual:
        got, gh = got
        _within(gh, h, (U + o) * h.abs(), "h")
    _within(got, y, ((K + 16) * U + o) * y.abs(), "y")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K", NORM_SHAPES)
def test_norm_gradients(nn, M, K, residual, dtype):
    torch = _torch()
    dt, g, o = _dtype(dtype), _gen(M * 11 + K), _ulp(dtype)
    x, w = _normal(g, M, K, dtype=dt), _normal(g, K, dtype=dt, scale=0.2, mean=1)
    r = _normal(g, M, K, dtype=dt, scale=2) if residual else None
    dy, dh = _normal(g, M, K, dtype=dt), _normal(g, M, K, dtype=dt)
    h, s, _ = _norm_ref(x, w, r)
    xh, wdy = h * s, dy.double() * w.double()
    c = (wdy * xh).mean(-1, keepdim=True)
    dx, dw = s * (wdy - xh * c), (dy.double() * xh).sum(0)
    # the stream is read back in its own type: half an ulp of each of its values
    e = o if residual and dtype == "bf16" else 0
    mag = (wdy * xh).abs().mean(-1, keepdim=True)
    bound = s * (wdy.abs() + xh.abs() * mag) * (2 * K + 32) * U + s * xh.abs() * mag * 3 * e
    bw = (dy.double() * xh).abs().sum(0) * ((M + K + 32) * U + e)
    ins = [t.cuda().requires_grad_() for t in ([x, w, r] if residual else [x, w])]
    if residual:
        dx = dx + dh.double()
        bound = bound + 2 * U * dx.abs()
        out = nn.rms_norm(ins[0], ins[1], EPS, ins[2])
        got = torch.autograd.grad(out, ins, [dy.cuda(), dh.cuda()])
        assert torch.equal(got[0], got[2])
    else:
        got = torch.autograd.grad(nn.rms_norm(ins[0], ins[1], EPS), ins, dy.cuda())
    _within(got[0], dx, bound + o * dx.abs() * (1 + 1e-3), "dx")
    _within(got[1], dw, bw + o * dw.abs() * (1 + 1e-2), "dw")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M,K", NORM_SHAPES)
def test_norm_q8(nn, M, K, residual, dtype):
    torch = _torch()
    dt, g = _dtype(dtype), _gen(M * 13 + K)
    x, w = _normal(g, M, K, dtype=dt), _normal(g, K, dtype=dt, scale=0.2, mean=1)
    r = _normal(g, M, K, dtype=dt, scale=2) if residual else None
    h, _, y = _norm_ref(x, w, r)
    out = nn.rms_norm_q8(x.cuda(), w.cuda(), EPS, None if r is None else r.cuda())
    q, scale = out[0].cpu(), out[1].cpu()
    assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == x.shape[:-1]
    # the integers follow from 32-bit operations of single elements: they are those, exactly
    u32 = (x.float() + r.float() if residual else x.float()) * w.float()
    a32 = u32.abs().amax(-1, keepdim=True)
    assert torch.equal(q.float(), torch.round(u32 * (torch.full_like(a32, 127.0) / a32)))
    if M:
        assert int(q.abs().max()) == 127
    top = y.abs().amax(-1)
    _within(scale, top / 127, (K + 32) * U * top / 127, "scale")
    _within(q.double() * scale.double()[:, None], y, (top / 127 * 0.5)[:, None] + (K + 160) * U * top[:, None], "rows")
    if residual:
        _within(out[2], h, (U + _ulp(dtype)) * h.abs(), "h")


def test_norm_q8_rows_without_finite_size(nn):
    """Zero rows, rows below the smallest scale, and rows with an infinity or a NaN; their neighbours unchanged."""
    torch = _torch()
    x = _normal(_gen(1), 6, 96, dtype=torch.float32)
    x[1] = 0
    x[2] = 1e-40
    x[3, 95] = float("inf")
    x[4, 0] = float("nan")
    w = torch.ones(96)
    q, scale = (t.cpu() for t in nn.rms_norm_q8(x.cuda(), w.cuda()))
    assert not q[1:5].any()
    assert scale[1] == 0 and scale[2] == 0 and torch.isnan(scale[3]) and torch.isnan(scale[4])
    q1, s1 = nn.rms_norm_q8(x[[0, 5]].cuda(), w.cuda())
    assert torch.equal(q[[0, 5]], q1.cpu()) and torch.equal(scale[[0, 5]], s1.cpu())
    y = nn.rms_norm(x.cuda(), w.cuda()).cpu()
    assert not y[1].any() and torch.isnan(y[4]).all() and torch.isfinite(y[[0, 2, 5]]).all()


def test_norm_strides_and_broadcast_residual(nn):
    """Rows of a wider array, a residual that is one row for all, an address that 16 bytes do not divide."""
    torch = _torch()
    g = _gen(5)
    for K, pad, off in ((64, 16, 0), (64, 13, 3), (100, 4, 4), (33, 7, 1)):
        big = _normal(g, 40, K + pad + off, dtype=torch.float32).cuda()
        x = big[:, off:off + K].detach()
        r = _normal(g, 1, K, dtype=torch.float32).cuda().expand(40, K)
        w = _normal(g, K + 1, dtype=torch.float32).cuda()[1:]
        y, h = nn.rms_norm(x, w, EPS, r)
        y0, h0 = nn.rms_norm(x.contiguous(), w.clone(), EPS, r.contiguous())
        assert torch.equal(h, h0)
        torch.testing.assert_close(y, y0, rtol=(K + 16) * U, atol=0)
        # the gradient of a broadcast residual is the sum over the rows that shared it
        one = r[:1].detach().clone().requires_grad_()
        xs = x.detach().clone().requires_grad_()
        y, h = nn.rms_norm(xs, w, EPS, one.expand(40, K))
        dy = _normal(g, 40, K, dtype=torch.float32).cuda()
        gx, g1 = torch.autograd.grad([y, h], [xs, one], [dy, dy])
        torch.testing.assert_close(g1, gx.sum(0, keepdim=True), rtol=1e-5, atol=1e-4)
        # gradients that come as one value for all, and as every second row
        gs = torch.autograd.grad(nn.rms_norm(xs, w, EPS).sum(), xs)[0]
        ge = torch.autograd.grad(nn.rms_norm(xs, w, EPS), xs, torch.ones(40, K, device="cuda"))[0]
        assert torch.equal(gs, ge)
        dd = _normal(g, 80, K, dtype=torch.float32).cuda()
        ga = torch.autograd.grad(nn.rms_norm(xs, w, EPS), xs, dd[::2])[0]
        gb = torch.autograd.grad(nn.rms_norm(xs, w, EPS), xs, dd[::2].contiguous())[0]
        assert torch.equal(ga, gb)


def test_norm_only_the_stream_has_a_gradient(nn):
    torch = _torch()
    x, r, w = (torch.randn(4, 32, device="cuda", requires_grad=True), torch.randn(4, 32, device="cuda", requires_grad=True),
               torch.ones(32, device="cuda", requires_grad=True))
    _, h = nn.rms_norm(x, w, EPS, r)
    dh = torch.randn(4, 32, device="cuda")
    gx, gr = torch.autograd.grad(h, [x, r], dh)
    assert torch.equal(gx, dh) and torch.equal(gr, dh)


def test_norm_offsets_past_32_bits(nn):
    """More than 2^31 elements: the last rows."""
    torch = _torch()
    K, M = 4096, 2 ** 19 + 3
    x = torch.zeros(M, K, device="cuda", dtype=torch.bfloat16)
    tail = _normal(_gen(3), 3, K, dtype=torch.bfloat16).cuda()
    x[-3:] = tail
    w = torch.ones(K, device="cuda", dtype=torch.bfloat16)
    y = nn.rms_norm(x, w)
    assert torch.equal(y[-3:], nn.rms_norm(tail, w)) and not y[:-3:4099].any()
    del y
    q, s = nn.rms_norm_q8(x, w)
    q1, s1 = nn.rms_norm_q8(tail, w)
    assert torch.equal(q[-3:], q1) and torch.equal(s[-3:], s1)


# ------------------------------------------------------------------------------------ gated block
def _act_ref(g, name):
    torch = _torch()
    if name == "silu":
        p = torch.sigmoid(g)
        return g * p, p + g * p * (1 - p)
    if name == "sigmoid":
        p = torch.sigmoid(g)
        return p, p * (1 - p)
    if name == "elu":
        return torch.where(g > 0, g, torch.expm1(g)), torch.where(g > 0, torch.ones_like(g), torch.exp(g))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 0.134145 * g * g)


class _GatedRef:
    """Values in 64 bits and bounds of a gated block's outputs. The activations' first and second derivatives are
    below 1.2, and their 32-bit forms off by at most 16 u (1 + |g| + |g|^3)."""

    def __init__(self, x, wg, wu, bg, bu, act, dy, dtype):
        x, wg, wu, dy = (t.double() for t in (x, wg, wu, dy))
        K, F, M, o = x.shape[1], wg.shape[0], x.shape[0], _ulp(dtype)
        bg = bg.double() if bg is not None else x.new_zeros(F)
        bu = bu.double() if bu is not None else x.new_zeros(F)
        g, u = x @ wg.t() + bg, x @ wu.t() + bu
        eg = (K + 16) * U * (x.abs() @ wg.abs().t() + bg.abs())
        eu = (K + 16) * U * (x.abs() @ wu.abs().t() + bu.abs())
        a, d = _act_ref(g, act)
        ea = 1.2 * eg + 16 * U * (1 + g.abs() + g.abs() ** 3)
        self.y = a * u
        self.by = ea * u.abs() + a.abs() * eu + ea * eu + (4 * U + o) * self.y.abs()
        dg, du = dy * u * d, dy * a
        # what the products of the gradients read is held in the tensors' type
        edg = dy.abs() * (ea * u.abs() + eu * d.abs() + ea * eu) + (4 * U + o) * dg.abs() * (1 + 1e-3)
        edu = dy.abs() * ea + (4 * U + o) * du.abs() * (1 + 1e-3)

        def product(p, ep, q, n):
            v = p @ q
            return v, ep @ q.abs() + (n + 16) * U * (p.abs() + ep) @ q.abs()

        (x1, e1), (x2, e2) = product(dg, edg, wg, 2 * F), product(du, edu, wu, 2 * F)
        self.grads = [(x1 + x2, e1 + e2), product(dg.t(), edg.t(), x, M), product(du.t(), edu.t(), x, M),
                      (dg.sum(0), edg.sum(0) + (M + 16) * U * dg.abs().sum(0)),
                      (du.sum(0), edu.sum(0) + (M + 16) * U * du.abs().sum(0))]
        self.grads = [(v, e + o * (v.abs() + e)) for v, e in self.grads]


def _gated_inputs(M, K, F, dtype, seed, bias=True):
    dt, g = _dtype(dtype), _gen(seed)
    x = _normal(g, M, K, dtype=dt)
    wg, wu = (_normal(g, F, K, dtype=dt, scale=K ** -0.5) for _ in range(2))
    bg, bu = (_normal(g, F, dtype=dt, scale=0.3) if bias else None for _ in range(2))
    return x, wg, wu, bg, bu, _normal(g, M, F, dtype=dt)


def _cuda(ts):
    return [None if t is None else t.cuda() for t in ts]


GATED_SHAPES = [(1, 1, 1), (1, 256, 512), (1, 100, 389), (2, 64, 64), (5, 33, 17), (8, 1024, 96), (9, 40, 129),
                (16, 512, 72), (31, 65, 64), (64, 256, 200), (100, 29, 100), (129, 128, 130), (300, 72, 33),
                (257, 511, 65), (1000, 16, 8), (0, 32, 16)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,K,F", GATED_SHAPES)
def test_gated(nn, M, K, F, dtype):
    for act in nn.ACTIVATIONS:
        ins = _gated_inputs(M, K, F, dtype, M + K + F, bias=act != "elu")
        ref = _GatedRef(*ins[:5], act, ins[5], dtype)
        y = nn.gated_linear(*_cuda(ins[:5]), activation=act)
        _within(y, ref.y, ref.by, (act, "y"))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,K,F", GATED_SHAPES + [(5000, 24, 40)])
def test_gated_gradients(nn, M, K, F, dtype):
    torch = _torch()
    for act in ("silu", "gelu") if M > 20 else nn.ACTIVATIONS:
        ins = _gated_inputs(M, K, F, dtype, M + K + F + 1)
        ref = _GatedRef(*ins[:5], act, ins[5], dtype)
        dev = [t.cuda().requires_grad_() for t in ins[:5]]
        y = nn.gated_linear(*dev, activation=act)
        _within(y, ref.y, ref.by, (act, "y"))
        got = torch.autograd.grad(y, dev, ins[5].cuda())
        for v, (r, b), name in zip(got, ref.grads, ("dx", "dwg", "dwu", "dbg", "dbu")):
            _within(v, r, b, (act, name))


def test_gated_gradients_wanted_singly(nn):
    """Each gradient alone is the one that comes with all the others; without biases too."""
    torch = _torch()
    ins = _gated_inputs(70, 48, 36, "fp32", 3)
    dev = [t.cuda() for t in ins[:5]]
    dy = ins[5].cuda()
    every = [t.clone().requires_grad_() for t in dev]
    whole = torch.autograd.grad(nn.gated_linear(*every), every, dy)
    for i in range(5):
        args = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(dev)]
        assert torch.equal(torch.autograd.grad(nn.gated_linear(*args), args[i], dy)[0], whole[i]), i
    some = [t.clone().requires_grad_() for t in dev[:3]]
    ref = _GatedRef(*ins[:3], None, None, "silu", ins[5], "fp32")
    got = torch.autograd.grad(nn.gated_linear(*some), some, dy)
    for v, (r, b) in zip(got, ref.grads):
        _within(v, r, b, "no bias")


def test_gradients_against_differences(nn):
    """A loss of the norm, the gated block and a stream of two blocks, against central differences along random
    directions. The step is 1e-2 of the inputs' size: the difference is off by about 1e-4 of the loss's third
    derivative, and its 32-bit noise by 1e-7 / 1e-2 of the loss's terms; 1 % holds both."""
    torch = _torch()
    g = _gen(9)
    M, K, F = 12, 40, 24
    x, r = _normal(g, M, K, dtype=torch.float32), _normal(g, M, K, dtype=torch.float32)
    w = _normal(g, K, dtype=torch.float32, scale=0.2, mean=1)
    wg, wu = (_normal(g, F, K, dtype=torch.float32, scale=K ** -0.5) for _ in range(2))
    bg, bu = (_normal(g, F, dtype=torch.float32, scale=0.3) for _ in range(2))
    ins = [t.cuda() for t in (x, r, w, wg, wu, bg, bu)]
    cy, ch = _normal(g, M, F, dtype=torch.float32).cuda(), _normal(g, M, K, dtype=torch.float32).cuda()

    def loss(x, r, w, wg, wu, bg, bu, act):
        y, h = nn.rms_norm(x, w, EPS, r)
        z = nn.gated_linear(y, wg, wu, bg, bu, activation=act)
        return (z * cy).double().sum() + (h * ch).double().sum()

    for act in nn.ACTIVATIONS:
        leaves = [t.clone().requires_grad_() for t in ins]
        grads = torch.autograd.grad(loss(*leaves, act), leaves)
        for i, t in enumerate(ins):
            d = _normal(g, *t.shape, dtype=torch.float32).cuda()
            d = d / d.norm() * t.norm()
            step = [1e-2 * d if j == i else 0 for j in range(len(ins))]
            up = loss(*[a + s for a, s in zip(ins, step)], act)
            down = loss(*[a - s for a, s in zip(ins, step)], act)
            slope = float((grads[i] * d).double().sum())
            size = float(grads[i].double().norm() * d.double().norm()) / math.sqrt(t.numel())
            assert abs(float(up - down) / 2e-2 - slope) <= 1e-2 * max(abs(slope), size), (act, i)


def test_gated_strides(nn):
    """Rows of a wider array, weights that are the halves of one matrix, an odd address, and dy of any layout."""
    torch = _torch()
    g = _gen(21)
    for dtype in ("fp32", "bf16"):
        dt = _dtype(dtype)
        for M, K, F, pad, off in ((50, 64, 48, 8, 0), (3, 64, 48, 8, 8), (50, 100, 33, 5, 1), (1, 33, 20, 3, 2)):
            x = _normal(g, M, K + pad + off, dtype=dt).cuda()[:, off:off + K]
            both = _normal(g, F, 2 * K, dtype=dt, scale=K ** -0.5).cuda()
            wg, wu = both[:, :K], both[:, K:]
            bias = _normal(g, 2 * F + 1, dtype=dt).cuda()
            bg, bu = bias[1:F + 1], bias[F + 1:]
            dy = _normal(g, M, 2 * F, dtype=dt).cuda()[:, F:]
            ref = _GatedRef(*[t.cpu() for t in (x, wg, wu, bg, bu)], "gelu", dy.cpu(), dtype)
            ins = [t.detach().requires_grad_() for t in (x, wg, wu, bg, bu)]
            y = nn.gated_linear(*ins, activation="gelu")
            _within(y, ref.y, ref.by, "y")
            for v, (r, b) in zip(torch.autograd.grad(y, ins, dy), ref.grads):
                _within(v, r, b, (dtype, M, K, F))
            one = torch.autograd.grad(nn.gated_linear(*ins).sum(), ins)
            two = torch.autograd.grad(nn.gated_linear(*ins), ins, torch.ones(M, F, dtype=dt, device="cuda"))
            assert all(torch.equal(p, q) for p, q in zip(one, two))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_gated_values_without_size(nn, M, dtype):
    """An infinity or a NaN stays in the row it is in, and is there what the formula gives; values near the type's
    largest too."""
    torch = _torch()
    x, wg, wu, bg, bu, _ = _gated_inputs(M, 40, 24, dtype, 4)
    bad = [0, M // 2, M - 1]
    for value in (float("inf"), -float("inf"), float("nan"), 3.3e38):
        for row in bad:
            z = x.clone()
            z[row, 7] = value
            wz = wu.clone()
            wz[3] = 0      # 0 times an infinity
            g, u = z.double() @ wg.double().t() + bg.double(), z.double() @ wz.double().t() + bu.double()
            y = _act_ref(g, "sigmoid")[0] * u
            got = nn.gated_linear(*_cuda((z, wg, wz, bg, bu)), activation="sigmoid").double().cpu()
            others = [i for i in range(M) if i != row]
            assert torch.isfinite(got[others]).all()
            plain = nn.gated_linear(*_cuda((x, wg, wz, bg, bu)), activation="sigmoid").double().cpu()
            assert torch.equal(got[others], plain[others])
            if math.isfinite(value):
                ok = y[row].abs() < 1e38
                assert torch.isfinite(got[row][ok]).all()
                torch.testing.assert_close(got[row][ok], y[row][ok], rtol=2 ** -7, atol=1e33)
            else:
                assert torch.equal(torch.isnan(got[row]), torch.isnan(y[row])), (value, row)
                m = ~torch.isnan(y[row]) & torch.isinf(y[row])
                assert torch.equal(got[row][m], y[row][m])


def test_gated_offsets_past_32_bits(nn):
    torch = _torch()
    M, K, F = 2 ** 21 + 5, 8, 1040
    x = torch.zeros(M, K, device="cuda", dtype=torch.bfloat16)
    _, wg, wu, bg, bu, _ = _cuda(_gated_inputs(1, K, F, "bf16", 8))
    tail = _normal(_gen(3), 5, K, dtype=torch.bfloat16).cuda()
    x[-5:] = tail
    y = nn.gated_linear(x, wg, wu, bg, bu)
    _within(y[-5:], *(lambda r: (r.y, r.by))(_GatedRef(*[t.cpu() for t in (tail, wg, wu, bg, bu)], "silu",
                                                       torch.zeros(5, F), "bf16")), "tail")


# ------------------------------------------------------------------------------------ gated block in 8 bits
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,K,F", GATED_SHAPES + [(1, 1024, 2731), (40, 1500, 40)])
def test_gated_q8(nn, M, K, F, dtype):
    torch = _torch()
    rng = np.random.default_rng(M + K + F)
    q, qg, qu = (torch.from_numpy(rng.integers(-127, 128, s).astype(np.int8)) for s in ((M, K), (F, K), (F, K)))
    s = torch.from_numpy(rng.uniform(0.5, 2, M).astype(np.float32)) / 127
    sg, su = (torch.from_numpy(rng.uniform(0.5, 2, F).astype(np.float32)) / (127 * math.sqrt(K)) for _ in range(2))
    bg, bu = (torch.from_numpy(rng.normal(0, 0.3, F).astype(np.float32)) for _ in range(2))
    dt, o = _dtype(dtype), _ulp(dtype)
    for act, b in (("silu", True), ("gelu", False), ("sigmoid", True), ("elu", True)):
        bias = (bg, bu) if b else (torch.zeros(F), torch.zeros(F))
        gi = (q.double() @ qg.double().t()) * s.double()[:, None] * sg.double()
        ui = (q.double() @ qu.double().t()) * s.double()[:, None] * su.double()
        g, u = gi + bias[0].double(), ui + bias[1].double()
        eg, eu = 4 * U * (gi.abs() + g.abs()), 4 * U * (ui.abs() + u.abs())
        a, _ = _act_ref(g, act)
        ea = 1.2 * eg + 16 * U * (1 + g.abs() + g.abs() ** 3)
        y = nn.gated_linear_q8(*_cuda((q, s, qg, sg, qu, su)), *(_cuda(bias) if b else ()), activation=act, dtype=dt)
        _within(y, a * u, ea * u.abs() + a.abs() * eu + ea * eu + (4 * U + o) * (a * u).abs(), act)


def test_gated_q8_strides_and_extremes(nn):
    """8-bit rows of a wider array at odd addresses; sums at their largest."""
    torch = _torch()
    rng = np.random.default_rng(2)
    for M, K, F, off in ((1, 48, 20, 0), (33, 48, 20, 5), (33, 64, 70, 16)):
        big = torch.from_numpy(rng.integers(-128, 128, (M, 2 * K + off)).astype(np.int8)).cuda()
        q = big[:, off:off + K]
        qg, qu = (torch.from_numpy(rng.integers(-127, 128, (F, K)).astype(np.int8)).cuda() for _ in range(2))
        s, sg = torch.rand(M, device="cuda") / 127, torch.rand(F, device="cuda") / 127
        a = nn.gated_linear_q8(q, s, qg, sg, qu, sg)
        b = nn.gated_linear_q8(q.contiguous(), s, qg, sg, qu, sg)
        assert torch.equal(a, b)
    K = 131072
    q = torch.full((2, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((3, K), -127, dtype=torch.int8, device="cuda")
    one = torch.ones(3, device="cuda")
    y = nn.gated_linear_q8(q, one[:2], w, one, w, one, activation="sigmoid")
    assert bool((y == 128.0 * 127 * K).all())


# ------------------------------------------------------------------------------------ clipping
def _clip_ref(grads, max_norm):
    torch = _torch()
    norm = torch.sqrt(sum(g.double().pow(2).sum() for g in grads))
    return norm, float(min(1.0, max_norm / (float(norm) + 1e-6)))


CLIP_SETS = [[(1,)], [(29,), (0,), (29, 256), (256, 100)], [(3, 5)] * 7, [(17,)] * 150, [(300000,), (16384,), (16385,), (1,)],
             [(4000, 1111)], [()]]


@pytest.mark.parametrize("types", ["fp32", "bf16", "mixed", "wide"])
@pytest.mark.parametrize("shapes", CLIP_SETS, ids=range(len(CLIP_SETS)))
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_clip(nn, shapes, types, max_norm):
    """In place and into other tensors: "wide" is 16-bit gradients into 32-bit ones."""
    torch = _torch()
    g = _gen(len(shapes))
    kinds = {"fp32": ["fp32"], "bf16": ["bf16"], "mixed": ["fp32", "bf16"], "wide": ["bf16"]}[types]
    grads = [_normal(g, *s, dtype=_dtype(kinds[i % len(kinds)])) for i, s in enumerate(shapes)]
    norm, f = _clip_ref(grads, max_norm)
    dev = [t.cuda() for t in grads]
    outs = [torch.full(t.shape, 7.0, dtype=torch.float32 if types == "wide" else t.dtype, device="cuda") for t in dev]
    got = nn.clip_grad_norm(dev, max_norm, out=outs)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - float(norm)) <= 2 * U * float(norm)
    for a, b, o in zip(dev, grads, outs):
        assert torch.equal(a.cpu(), b)
        ref = b.double() * f
        _within(o, ref, ref.abs() * (6 * U + (2.0 ** -8 if o.dtype == torch.bfloat16 else 0)), "out")
    again = nn.clip_grad_norm(dev, max_norm)
    assert torch.equal(again, got)
    for a, o in zip(dev, outs):
        assert torch.equal(a.float(), o.to(a.dtype).float())


def test_clip_sizes_beyond_32_bits_of_range(nn):
    """Squares that 32 bits cannot hold, gradients too small for them, and norms that are infinite or NaN."""
    torch = _torch()
    for size in (1e30, 1e-30):
        g = torch.full((1000,), size, device="cuda")
        norm = nn.clip_grad_norm([g], 1.0)
        assert abs(float(norm) / (size * math.sqrt(1000)) - 1) <= 2 * U
        assert abs(float(g[3]) / min(size, 1 / math.sqrt(1000)) - 1) <= 6 * U
    for value in (float("inf"), float("nan")):
        g, h = torch.ones(5000, device="cuda"), torch.ones(7, device="cuda")
        g[4321] = value
        norm = nn.clip_grad_norm([g, h], 1.0)
        if math.isnan(value):
            assert math.isnan(float(norm)) and bool(torch.isnan(g).all()) and bool(torch.isnan(h).all())
        else:
            assert float(norm) == value and not h.any() and bool(torch.isnan(g[4321])) and float(g.nansum()) == 0


def test_clip_unaligned_and_parameters(nn):
    """Tensors at odd addresses; parameters with and without a gradient."""
    torch = _torch()
    base = _normal(_gen(2), 5003, dtype=torch.float32).cuda()
    parts = [base[1:1000], base[1000:1003], base[1003:]]
    norm, f = _clip_ref([p.cpu() for p in parts], 1.0)
    before = base.clone()
    got = nn.clip_grad_norm(parts, 1.0)
    assert abs(float(got) - float(norm)) <= 2 * U * float(norm)
    assert base[0] == before[0]
    torch.testing.assert_close(base[1:], before[1:] * f, rtol=8 * U, atol=0)
    ps = [torch.nn.Parameter(torch.zeros(10, device="cuda")) for _ in range(3)]
    ps[0].grad, ps[2].grad = torch.full((10,), 3.0, device="cuda"), torch.full((10,), 4.0, device="cuda")
    assert abs(float(nn.clip_grad_norm_(ps, 1.0)) - 5 * math.sqrt(10)) < 1e-5
    assert abs(float(ps[0].grad[0]) - 3 / (5 * math.sqrt(10))) < 1e-6 and ps[1].grad is None
    assert float(nn.clip_grad_norm_(ps[1:2], 1.0)) == 0


def test_twice_differentiated_is_refused(nn):
    """A graph of the gradients is refused, not answered with zeros."""
    torch = _torch()
    x, w = torch.randn(3, 8, device="cuda", requires_grad=True), torch.ones(8, device="cuda")
    for y in (nn.rms_norm(x, w), nn.gated_linear(x, torch.randn(4, 8, device="cuda"), torch.randn(4, 8, device="cuda"))):
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_clipping_in_place_is_seen_by_autograd(nn):
    """A tensor that a graph has saved is not silently changed under it."""
    torch = _torch()
    a, g = torch.ones(4, device="cuda", requires_grad=True), torch.full((4,), 5.0, device="cuda")
    y = (a * g).sum()
    nn.clip_grad_norm([g], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals_on_the_gpu(nn):
    """Types, shapes, layouts and places that the kernels do not take."""
    torch = _torch()
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    wg = torch.randn(6, 8, device="cuda")
    q, s = nn.rms_norm_q8(x, w)
    qg, sg = nn.quantize_rows(wg)
    bad = [
        lambda: nn.rms_norm(x.double(), w.double()), lambda: nn.rms_norm(x, w.bfloat16()), lambda: nn.rms_norm(x, w[:7]),
        lambda: nn.rms_norm(x, w.cpu()), lambda: nn.rms_norm(x, None), lambda: nn.rms_norm(x, w, residual=x[:2]),
        lambda: nn.rms_norm(x, w, residual=x.bfloat16()), lambda: nn.rms_norm(x.t(), torch.ones(4, device="cuda")),
        lambda: nn.rms_norm(torch.zeros(1, 32769, device="cuda"), torch.ones(32769, device="cuda")),
        lambda: nn.rms_norm(torch.zeros(2, 0, device="cuda"), torch.ones(0, device="cuda")),
        lambda: nn.rms_norm(x[:, ::2], torch.ones(4, device="cuda")),
        lambda: nn.gated_linear(x, wg, wg[:5]), lambda: nn.gated_linear(x, wg[:, :7], wg[:, :7]),
        lambda: nn.gated_linear(x, wg, wg, torch.ones(5, device="cuda")), lambda: nn.gated_linear(x, wg, wg, activation="relu"),
        lambda: nn.gated_linear(x, wg.t(), wg.t()), lambda: nn.gated_linear(x, wg, wg.bfloat16()),
        lambda: nn.gated_linear_q8(x, s, qg, sg, qg, sg), lambda: nn.gated_linear_q8(q, s[:3], qg, sg, qg, sg),
        lambda: nn.gated_linear_q8(q, s, qg, sg, qg[:5], sg), lambda: nn.gated_linear_q8(q, s, qg, sg.double(), qg, sg),
        lambda: nn.gated_linear_q8(q, s, qg, None, qg, sg), lambda: nn.gated_linear_q8(q, s, qg, sg, qg, sg, dtype=torch.half),
        lambda: nn.clip_grad_norm([x, x.cpu()], 1.0), lambda: nn.clip_grad_norm([x.half()], 1.0),
        lambda: nn.clip_grad_norm([x.t()], 1.0), lambda: nn.clip_grad_norm([x], 1.0, out=[]),
        lambda: nn.clip_grad_norm([x], 1.0, out=[x[:2]]), lambda: nn.clip_grad_norm([x], -1.0),
        lambda: nn.clip_grad_norm([x], float("nan")), lambda: nn.clip_grad_norm([x], 1.0, out=[x.cpu()]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(i)


# ------------------------------------------------------------------------------------ large tiles
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "q8"])
@pytest.mark.parametrize("M,K,F", [(4200, 72, 1032), (8200, 40, 2056), (16500, 512, 24), (4100, 1030, 520)])
def test_gated_in_large_tiles(nn, M, K, F, dtype):
    """Products with enough tiles for the large and the huge ones (128 x 128 from 256 on, 256 x 128 from 1024 on, for the
    gradients' products too), their edges and lengths odd. The 64-bit values are computed on the GPU."""
    torch = _torch()
    if dtype == "q8":
        rng = np.random.default_rng(K)
        q, qg, qu = (torch.from_numpy(rng.integers(-127, 128, s).astype(np.int8)).cuda() for s in ((M, K), (F, K), (F, K)))
        s, sg = torch.rand(M, device="cuda") / 127, torch.rand(F, device="cuda") / (127 * math.sqrt(K))
        g = (q.double() @ qg.double().t().contiguous()) * s.double()[:, None] * sg.double()
        u = (q.double() @ qu.double().t().contiguous()) * s.double()[:, None] * sg.double()
        a, _ = _act_ref(g, "silu")
        ea = 1.2 * 8 * U * g.abs() + 16 * U * (1 + g.abs() + g.abs() ** 3)
        bound = ea * u.abs() + a.abs() * 8 * U * u.abs() + 4 * U * (a * u).abs()
        for dt, o in ((torch.float32, 0), (torch.bfloat16, 2.0 ** -8)):
            y = nn.gated_linear_q8(q, s, qg, sg, qu, sg, dtype=dt)
            assert bool(((y.double() - a * u).abs() <= bound + o * (a * u).abs()).all()), dt
        return
    ins = [t.cuda() for t in _gated_inputs(M, K, F, dtype, K + F)]
    ref = _GatedRef(*ins[:5], "silu", ins[5], dtype)
    dev = [t.requires_grad_() for t in ins[:5]]
    y = nn.gated_linear(*dev)
    got = [y, *torch.autograd.grad(y, dev, ins[5])]
    for v, (r, b), name in zip(got, [(ref.y, ref.by), *ref.grads], ("y", "dx", "dwg", "dwu", "dbg", "dbu")):
        far = (v.detach().double() - r).abs() - b
        assert bool((far <= 0).all()), (name, float(far.max()))


def test_gated_values_without_size_in_large_tiles(nn):
    torch = _torch()
    x, wg, wu, bg, bu, _ = _cuda(_gated_inputs(4200, 72, 1032, "fp32", 5))
    plain = nn.gated_linear(x, wg, wu, bg, bu, activation="sigmoid")
    z = x.clone()
    z[130, 70], z[4199, 0] = float("inf"), float("nan")
    g, u = z[[130, 4199]].double() @ wg.double().t().contiguous() + bg, z[[130, 4199]].double() @ wu.double().t().contiguous() + bu
    ref = _act_ref(g, "sigmoid")[0] * u
    got = nn.gated_linear(z, wg, wu, bg, bu, activation="sigmoid")
    rest = torch.ones(4200, dtype=torch.bool, device="cuda")
    rest[[130, 4199]] = False
    assert torch.equal(got[rest], plain[rest])
    assert torch.equal(torch.isnan(got[[130, 4199]]), torch.isnan(ref))
    m = torch.isinf(ref)
    assert bool(m.any()) and torch.equal(got[[130, 4199]][m].double(), ref[m])


def test_gated_gradients_past_32_bits(nn):
    """A workspace of more than 2^31 elements: the gradients of the last rows, and of weights that only those rows move."""
    torch = _torch()
    M, K, F, n = 2 ** 20 + 5, 8, 1040, 5
    tail, wg, wu, bg, bu, dtail = _cuda(_gated_inputs(n, K, F, "bf16", 8))
    x, dy = torch.zeros(M, K, device="cuda", dtype=torch.bfloat16), torch.zeros(M, F, device="cuda", dtype=torch.bfloat16)
    x[-n:], dy[-n:] = tail, dtail
    ins = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    got = torch.autograd.grad(nn.gated_linear(*ins), ins, dy)
    assert not got[0][:-n:997].any()
    ref = _GatedRef(*[t.detach().cpu() for t in (tail, wg, wu, bg, bu)], "silu", dtail.cpu(), "bf16")
    for v, (r, b) in zip([got[0][-n:], *got[1:]], ref.grads):
        _within(v, r, b, "tail")


def test_rows_of_one_and_three_dimensions(nn):
    torch = _torch()
    g = _gen(7)
    x, r = (_normal(g, 2, 3, 40, dtype=torch.float32).cuda() for _ in range(2))
    w = _normal(g, 40, dtype=torch.float32, mean=1).cuda()
    wg, wu = (_normal(g, 24, 40, dtype=torch.float32).cuda() for _ in range(2))
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    y, h = nn.rms_norm(x, w, EPS, r)
    y2, h2 = nn.rms_norm(flat(x), w, EPS, flat(r))
    assert y.shape == x.shape and torch.equal(flat(y), y2) and torch.equal(flat(h), h2)
    q, s, _ = nn.rms_norm_q8(x, w, EPS, r)
    assert s.shape == (2, 3)
    (qg, sg), (qu, su) = nn.quantize_rows(wg), nn.quantize_rows(wu)
    z = nn.gated_linear_q8(q, s, qg, sg, qu, su)
    assert z.shape == (2, 3, 24) and torch.equal(flat(z), nn.gated_linear_q8(flat(q), s.reshape(-1), qg, sg, qu, su))
    ins = [t.clone().requires_grad_() for t in (x, wg, wu)]
    z = nn.gated_linear(*ins)
    dz = torch.randn_like(z)
    gx, gg, gu = torch.autograd.grad(z, ins, dz)
    flats = [t.detach().clone().requires_grad_() for t in (flat(x), wg, wu)]
    for a, b in zip((flat(gx), gg, gu), torch.autograd.grad(nn.gated_linear(*flats), flats, flat(dz))):
        assert torch.equal(a, b)
    one = nn.gated_linear(x[0, 0], wg, wu)
    assert one.shape == (24,) and torch.equal(one, nn.gated_linear(x[0, :1], wg, wu)[0])
    q1, s1 = nn.rms_norm_q8(x[0, 0], w)
    assert s1.shape == () and q1.shape == (40,)
    with pytest.raises(ValueError):
        nn.rms_norm(x.transpose(0, 1), w)


@pytest.mark.parametrize("M,K,F", [(40, 256, 512), (100, 65, 700), (33, 30, 31), (1000, 72, 100), (9, 40, 64), (32, 128, 40),
                                   (5, 100, 40), (17, 33, 20)])
def test_gated_at_the_changes_of_form(nn, M, K, F):
    """Rows on both sides of the forms' limits (a wave per output, tiny, small tiles), with gradients, whose column
    sums are counted by form."""
    torch = _torch()
    for dtype in ("fp32", "bf16"):
        ins = _gated_inputs(M, K, F, dtype, 2 * M + K)
        ref = _GatedRef(*ins[:5], "gelu", ins[5], dtype)
        dev = [t.cuda().requires_grad_() for t in ins[:5]]
        y = nn.gated_linear(*dev, activation="gelu")
        _within(y, ref.y, ref.by, (dtype, "y"))
        for v, (r, b), name in zip(torch.autograd.grad(y, dev, ins[5].cuda()), ref.grads, ("dx", "dwg", "dwu", "dbg", "dbu")):
            _within(v, r, b, (dtype, name))
