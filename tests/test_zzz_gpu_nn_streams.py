"""The policy operators on other streams than the default one, and in a captured graph.

In a file that runs after all others: work on a second stream makes blocks of the null stream's launches start on
another XCD than the first from then on, and environments created in such a process hand their work items over
with fences, which the environment's tests do not expect."""
import pytest

from test_gpu_nn import EPS, _gated_inputs, _gen, _normal, _torch, nn  # noqa: F401

pytestmark = pytest.mark.gpu


def _everything(nn, t):
    """One pass through every operator: the outputs."""
    torch = _torch()
    y, h = nn.rms_norm(t["x"], t["w"], EPS, t["r"])
    z = nn.gated_linear(y, t["wg"], t["wu"], t["bg"], t["bu"])
    ins = [t["x"], t["w"], t["r"], t["wg"], t["wu"], t["bg"], t["bu"]]
    grads = torch.autograd.grad([z, h], ins, [t["dz"], t["dh"]])
    norm = nn.clip_grad_norm([g for g in grads], 0.5, out=t["out"])
    q, s, h8 = nn.rms_norm_q8(t["x"], t["w"], EPS, t["r"])
    z8 = nn.gated_linear_q8(q, s, t["qg"], t["sg"], t["qu"], t["su"])
    return [y, h, z, *grads, norm, *t["out"], q, s, h8, z8]


def _everything_inputs(nn, seed, M=333, K=96, F=80):
    torch = _torch()
    x, wg, wu, bg, bu, dz = _gated_inputs(M, K, F, "fp32", seed)
    g = _gen(seed + 1)
    r, dh = _normal(g, M, K, dtype=torch.float32), _normal(g, M, K, dtype=torch.float32)
    t = dict(x=x, r=r, w=_normal(g, K, dtype=torch.float32, mean=1, scale=0.2), wg=wg, wu=wu, bg=bg, bu=bu, dz=dz, dh=dh)
    t = {k: v.cuda() for k, v in t.items()}
    (t["qg"], t["sg"]), (t["qu"], t["su"]) = nn.quantize_rows(t["wg"]), nn.quantize_rows(t["wu"])
    for k in ("x", "r", "w", "wg", "wu", "bg", "bu"):
        t[k].requires_grad_()
    t["out"] = [torch.empty_like(t[k].detach()) for k in ("x", "w", "r", "wg", "wu", "bg", "bu")]
    return t


def test_same_results_every_time_and_on_other_streams(nn):
    torch = _torch()
    t = _everything_inputs(nn, 1)
    first = [v.detach().clone() for v in _everything(nn, t)]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _everything(nn, t)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        # inputs that this stream writes just before, behind enough work that an unordered launch would miss them
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(8):
            busy = busy @ busy * 1e-2
        u = {k: v if k == "out" else v.detach().clone().requires_grad_(v.requires_grad) for k, v in t.items()}
        got = [v.detach().clone() for v in _everything(nn, u)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_graph_capture(nn):
    """A captured pass, replayed on new inputs several times with eager work between: each replay as the eager pass."""
    torch = _torch()
    t = _everything_inputs(nn, 2)
    static = ("x", "r", "wg", "wu", "dz", "dh")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _everything(nn, t)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _everything(nn, t)
    for seed in (3, 4, 5):
        new = _everything_inputs(nn, seed)
        with torch.no_grad():
            for k in static:
                t[k].copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        got = [v.detach().clone() for v in held]
        eager = {k: v if k == "out" else v.detach().clone().requires_grad_(v.requires_grad) for k, v in t.items()}
        eager["out"] = [torch.empty_like(o) for o in t["out"]]
        assert all(torch.equal(a, b) for a, b in zip(got, _everything(nn, eager))), seed
