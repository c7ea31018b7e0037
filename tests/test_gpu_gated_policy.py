"""The gated policy of ppo_train on g1nn's operators: its outputs and gradients against the same network written out in
64 bits on the CPU, its 8-bit acting form against the values its 8-bit tensors stand for, and a short training run.

Bounds: an output that is a few sums of at most 512 32-bit products deep is off by less than 512 * 2^-24 = 3e-5 of the
magnitudes in it, per layer; five layers, and magnitudes up to a few times the outputs' norm: 1e-3 of the norm."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pt():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import ppo_train
    return ppo_train


def _norm(x, w):
    return x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w


def _plain(policy, z, gated=None):
    """The network in 64 bits; `gated`(block, n) replaces the product of a block's projections."""
    import torch
    lin = lambda l, v: v @ l.weight.t() + l.bias  # noqa: E731
    h = lin(policy.inp, z)
    for b in policy.blocks:
        n = _norm(h, b.norm)
        y = torch.nn.functional.silu(lin(b.gate, n)) * lin(b.up, n) if gated is None else gated(b, n)
        h = h + lin(b.down, y)
    n = _norm(h, policy.norm)
    return lin(policy.mu_head, n), lin(policy.v_head, n).squeeze(-1)


def _near(got, ref, what):
    d = (got.detach().cpu().double() - ref.detach()).norm() / ref.detach().norm()
    assert float(d) <= 1e-3, (what, float(d))


@pytest.mark.parametrize("rows", [1, 7, 300])
def test_policy_and_its_gradients(pt, rows):
    import copy

    import torch
    torch.manual_seed(rows)
    policy = pt.GatedPolicy(width=96, hidden=136, depth=2)
    wide = copy.deepcopy(policy).double()
    policy = policy.cuda()
    z = torch.randn(rows, 100, dtype=torch.float64)
    mu, log_std, v = policy(z.float().cuda())
    rmu, rv = _plain(wide, z.float().double())
    _near(mu, rmu, "mu")
    _near(v, rv, "v")
    cm, cv = torch.randn(rows, 29, dtype=torch.float64), torch.randn(rows, dtype=torch.float64)
    ((mu * cm.float().cuda()).sum() + (v * cv.float().cuda()).sum() + log_std.sum()).backward()
    ((rmu * cm.float().double()).sum() + (rv * cv.float().double()).sum() + wide.log_std.sum()).backward()
    for (name, p), q in zip(policy.named_parameters(), wide.parameters()):
        _near(p.grad, q.grad, name)


def test_acting_in_8_bits(pt):
    import copy

    import torch
    torch.manual_seed(3)
    policy = pt.GatedPolicy(width=128, hidden=200, depth=2).cuda()
    acting = pt.ActingPolicy(policy)
    z = torch.randn(65, 100, device="cuda")
    mu, _, v = acting(z)
    wide = copy.deepcopy(policy).cpu().double()
    held = {id(b): [t.cpu().double() for t in w] for b, w in zip(wide.blocks, acting.q8)}

    def gated(b, n):
        qg, sg, qu, su = held[id(b)]
        step = n.abs().amax(-1, keepdim=True) / 127
        q = torch.round(n / step) * step
        g = q @ (qg * sg[:, None]).t() + b.gate.bias
        u = q @ (qu * su[:, None]).t() + b.up.bias
        return torch.nn.functional.silu(g) * u

    rmu, rv = _plain(wide, z.cpu().double(), gated)
    # a value that 32 and 64 bits round to different whole numbers moves its row by a step of 1/127 of its largest: about
    # one value in 10^4, each a 128th part of a row
    _near(mu, rmu, "mu")
    _near(v, rv, "v")
    full, _, _ = policy(z)
    # 8 bits against 32: a step is 0.8 % of a row's largest value, the rounding of both factors a few parts in a thousand
    assert float((mu - full).norm() / full.norm()) <= 0.03
    assert not mu.requires_grad


def test_short_training_run(pt):
    import torch
    lines = []
    rows = pt.train(2, 64, 4, seed=5, eval_every=1, eval_steps=3, log=lines.append, gated=(64, 96, 2), act_q8=True)
    assert len(rows) == 2 and all(torch.isfinite(torch.tensor([r["loss"], r["reward_per_step"], r["forward_m"]])).all()
                                  for r in rows)
    again = pt.train(2, 64, 4, seed=5, eval_every=1, eval_steps=3, log=lines.append, gated=(64, 96, 2), act_q8=True)
    assert [r["reward_per_step"] for r in again] == [r["reward_per_step"] for r in rows]


def test_update_moves_the_policy_and_clips(pt):
    """One update: the parameters change, and the last gradients have the clipped norm."""
    import g1env
    import g1nn
    import torch
    torch.manual_seed(2)
    H, N = 8, 64
    policy = pt.GatedPolicy(width=64, hidden=96, depth=1).cuda()
    before = [p.detach().clone() for p in policy.parameters()]
    opt = torch.optim.Adam(policy.parameters(), lr=3e-4)
    stats = pt.ObsStats(pt.OBS, "cuda")
    traj = g1env.Trajectory(H, N)
    cfg = pt.PPOSettings(max_grad_norm=1e-3)
    with g1env.Env(N, substeps=2, pgs_iters=8, seed=1) as env:
        obs = torch.from_numpy(env.reset()).cuda()
        nobs, obs = pt.collect_steps(env, policy, stats, traj, obs)
        assert env.check() == 0
    assert torch.equal(traj.O[1:].isfinite().all(), torch.tensor(True, device="cuda")) and bool((traj.D <= 1).all())
    pt.ppo_update(policy, opt, nobs, traj, cfg, g1nn.clip_grad_norm_)
    assert all(not torch.equal(p, b) for p, b in zip(policy.parameters(), before))
    norm = torch.sqrt(sum(p.grad.double().pow(2).sum() for p in policy.parameters()))
    assert abs(float(norm) / 1e-3 - 1) < 1e-5
