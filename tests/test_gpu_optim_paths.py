"""GPU: forms of the optimiser-step operators that long and large lists reach -- several launches of an update beyond the cache, sums
beyond it before an update, scaling beyond it after sums from it -- against the formulas in float64 on the device.

Bounds are those of the roundings, in half steps u of the arithmetic (float32; float64 for float64 tensors), as update_bounds() counts
them.  For float64 tensors the expected values are rounded as often themselves: twice the bound."""
import math
import random
import types

import numpy as np
import pytest

from test_gpu_optim import HALF, TINY, _t, make, norm_tol

pytestmark = pytest.mark.gpu

MIB = 1 << 20
SIZE = {"float64": 8, "float32": 4, "bfloat16": 2, "float16": 2}


def wide_of(dtype):
    return "float64" if dtype == "float64" else "float32"


def values_for(dtype, mib, state):
    """Values whose gradients (state: whose four tensors) take a little more than so many MiB; an odd number."""
    per = 2 * SIZE[dtype] + 2 * SIZE[wide_of(dtype)] if state else SIZE[dtype]
    return int(mib * MIB / per * 1.01) | 1


def update_bounds(X, G, M, V, t, lr, b1, b2, eps, wd, decoupled, c, c_err, u):
    """One step and the largest errors of x, m and v.  Rounded once each: factor and product of clipping, b1, 1 - b1, b2, 1 - b2, wd,
    every product that is not in a fused sum, every fused sum, the root, its scale, eps, the quotient, size and keep."""
    w = 2.0 ** -53
    G1 = c * G
    eg = (2 * u + c_err) * G1.abs()
    if wd and not decoupled:
        eg = eg + 2 * u * (wd * X).abs()
        G1 = G1 + wd * X
        eg = eg + u * G1.abs()
    M1 = b1 * M + (1 - b1) * G1
    em = 2 * u * (b1 * M).abs() + (1 - b1) * (eg + 2 * u * G1.abs()) + u * M1.abs()
    V1 = b2 * V + (1 - b2) * G1 * G1
    ev = 2 * u * b2 * V + (1 - b2) * (2 * G1.abs() * eg + eg * eg + 4 * u * G1 * G1) + u * V1
    s = V1.sqrt()
    es = (ev / (2 * s)).nan_to_num(posinf=0.0).where(V1 > 0, ev.sqrt()) + u * s
    root = 1 / math.sqrt(-math.expm1(t * math.log1p(b2 - 1)))
    d = s * root + eps
    ed = es * root + (2 * u + 6 * w) * s * root + u * eps + u * d
    size = lr / -math.expm1(t * math.log1p(b1 - 1)) if b1 else lr
    q = M1 / d
    eq = em / d + q.abs() * ed / d + u * q.abs()
    keep = 1 - lr * wd if decoupled else 1.0
    X1 = X * keep - size * q
    ex = size * eq + (2 * u + 6 * w) * size * q.abs() + (3 * u * (X * keep).abs() if decoupled else 0) + u * X1.abs()
    return (X1, 1.02 * ex), (M1, 1.02 * em), (V1, 1.02 * ev)


def cuts(n, parts, seed):
    """Sizes of so many tensors that add up to n, short, long and empty ones."""
    rng = random.Random(seed)
    if parts == 1:
        return [n]
    weights = [rng.choice([0.0, rng.random() * 1e-4, rng.random(), rng.random()]) for _ in range(parts - 1)] + [1.0]
    sizes = [int(n * w / sum(weights)) for w in weights]
    return sizes[:-1] + [n - sum(sizes[:-1])]


def check_update(dtype, n, parts, most=None, p=2.0, wd=0.0, decoupled=False, betas=(0.9, 0.99), eps=1e-6):
    torch, optim = _t()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n + parts)
    kind, wide = getattr(torch, dtype), getattr(torch, wide_of(dtype))
    new = lambda k: torch.randn(n, dtype=torch.float32, device="cuda", generator=gen).to(k)      # noqa: E731
    x, g, m, v = new(kind), new(kind), new(wide).mul_(0.3), new(wide).square_()
    sizes = cuts(n, parts, parts)
    lrs, counts = [1e-3 * (1 + i % 70) for i in range(parts)], [float(1 + i % 9) for i in range(parts)]
    steps = [torch.full((), c, device="cuda") for c in counts]
    want, limit = None, None
    if most is not None:
        # in pieces: the float64 copy of all of it would be large
        pieces = [q.double().abs() for q in g.split(1 << 24)]
        want = float(max(q.max() for q in pieces)) if p == math.inf else float(sum(q.pow_(p).sum() for q in pieces)) ** (1 / p)
        del pieces
        limit = most * want
    keep = g.clone()
    q, a, b = x.clone(), m.clone(), v.clone()
    norm = optim.adam_step(list(q.split(sizes)), list(g.split(sizes)), list(a.split(sizes)), list(b.split(sizes)), steps, lrs, betas, eps,
                           wd, decoupled, limit, p)
    assert [float(s) for s in steps] == [c + 1 for c in counts] and torch.equal(g, keep)
    c = 1.0
    if most is not None:
        assert abs(float(norm) - want) <= (n + 8) * 2.0 ** -53 * want
        c = min(1.0, limit / (want + 1e-6))
    u = HALF[wide_of(dtype)]
    own = HALF[dtype] if dtype != wide_of(dtype) else 0.0
    twice, at = 2 if dtype == "float64" else 1, 0
    for i, k in enumerate(sizes):
        for lo in range(at, at + k, 1 << 24):
            hi = min(lo + (1 << 24), at + k)
            X, G, M, V = (z[lo:hi].double() for z in (x, g, m, v))
            for what, got, (ref, err) in zip("xmv", (q, a, b), update_bounds(X, G, M, V, counts[i] + 1, lrs[i], *betas, eps, wd, decoupled, c,
                                                                             (n + 8) * 2.0 ** -53 if most is not None else 0.0, u)):
                slack = twice * err + (own * (ref.abs() + err) if what == "x" else 0) + TINY[dtype if what == "x" else wide_of(dtype)]
                over = (got[lo:hi].double() - ref).abs() - slack
                assert bool((over <= 0).all()), (what, i, k, float(over.max()))
        at += k


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("most", [None, 0.3])
@pytest.mark.parametrize("parts", [1, 3, 16, 17, 98, 99, 109, 110, 219, 430])
def test_updates_beyond_the_cache_in_one_launch_and_in_several(dtype, most, parts):
    """A rate and a count of its own for every tensor, so that a launch that takes another's shows."""
    check_update(dtype, values_for(dtype, 64, True), parts, most)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("wd,decoupled", [(0.1, False), (0.1, True)])
@pytest.mark.parametrize("parts", [3, 230])
def test_decay_beyond_the_cache(dtype, wd, decoupled, parts):
    check_update(dtype, values_for(dtype, 64, True), parts, 0.5, wd=wd, decoupled=decoupled)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("parts", [2, 98, 99, 300])
def test_gradients_beyond_the_cache_before_an_update(dtype, p, parts):
    """More than 256 MiB of them: the sums read past the cache, in the launch that counts the steps or in their own."""
    check_update(dtype, values_for(dtype, 256, False), parts, 0.4, p)


@pytest.mark.parametrize("dtype", ["float64", "float16"])
def test_gradients_of_other_types_beyond_the_cache_before_an_update(dtype):
    check_update(dtype, values_for(dtype, 256, False), 5, 0.4)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("mib", [63, 65, 96, 127, 129])
@pytest.mark.parametrize("parts", [2, 300])
def test_clipping_around_the_borders_of_the_cache(dtype, mib, parts):
    """Scaling goes past the cache from 64 MiB on, the sums from 128 MiB on."""
    torch, optim = _t()
    n = values_for(dtype, mib / 1.01, False)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(mib)
    whole = torch.randn(n + 3, dtype=torch.float32, device="cuda", generator=gen).to(getattr(torch, dtype))[3:]
    sizes = cuts(n, parts, 7)
    ts = list(whole.split(sizes))
    if parts > 2:
        ts = ts[::2] + ts[1::2]             # not in the order of their addresses, so that few are neighbours
    keep = whole.clone()
    for p in (2.0, 1.0, math.inf):
        X = keep.double()
        want = float(X.abs().max()) if p == math.inf else float(X.abs().pow(p).sum()) ** (1 / p)
        whole.copy_(keep)
        assert abs(float(optim.clip_grad_norm_(ts, 2 * want, p)) - want) <= (n + 8) * 2.0 ** -53 * want
        assert torch.equal(whole, keep)
        norm = float(optim.clip_grad_norm_(ts, 0.3 * want, p))
        assert abs(norm - want) <= (n + 8) * 2.0 ** -53 * want
        c = 0.3 * want / (norm + 1e-6)
        rel = HALF[dtype] + 4 * 2.0 ** -53 + {"float64": 0.0, "float32": 2.0 ** -24}.get(dtype, 2.0 ** -23)
        E = X.mul_(c)
        assert bool(((whole.double() - E).abs() <= 1.001 * rel * E.abs() + TINY[dtype]).all())


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 1e-40, 1e-38, 1e-8, 1e20, 1e38, 2.0 ** 127])
def test_extreme_moments_and_eps_beyond_the_cache(eps):
    """In half steps: root, its scale, eps and their sum 1 each, quotient, size and product 1 each: 7; a step among subnormal ones."""
    torch, optim = _t()
    n = 9 * 500_000
    m0 = [0.0, 1e-30, -1e-22, 1e-3, 1e2, 0.0, 1e-3, 1e-3, 1e2]
    v0 = [3e-42, 1e-45, 1e-38, 1e-30, 1e-12, 1.0, 1.0, 1e30, 3e38]
    if eps:
        v0[:2] = [0.0, 0.0]
    m, v = (torch.tensor(a, device="cuda").repeat(n // 9) for a in (m0, v0))
    x, g, t = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.full((), 9.0, device="cuda")
    optim.adam_step([x], [g], [m], [v], [t], 0.5, (0.9, 0.99), eps)
    d = v.double().sqrt() / math.sqrt(1 - 0.99 ** 10) + eps
    want = -0.5 / (1 - 0.9 ** 10) * m.double() / d
    got = x.double()
    big = want.abs() > 3.5e38
    assert bool((got[big].isinf() & (got[big].sign() == want[big].sign())).all())
    err = (got[~big] - want[~big]).abs() - (7.01 * 2.0 ** -24 * want[~big].abs() + 2.0 ** -126)
    assert bool((err <= 0).all()), (got[:9].tolist(), want[:9].tolist())


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("sizes", [[(30000,), (1,), (64, 64)], [(1 + 997 * i % 4000,) for i in range(300)], [(3_000_001,), (70001,)]])
def test_the_norms_of_the_three_operators(dtype, sizes):
    """The same but for the order of their sums: within the error of two of them."""
    torch, optim = _t()
    wide = getattr(torch, wide_of(dtype))
    for p in (1.0, 2.0, math.inf):
        ts = make(sizes, [dtype], 41)
        norm = float(optim.grad_norm(ts, p))
        adam = float(optim.adam_step([t.clone() for t in ts], ts, *[[torch.zeros(t.shape, dtype=wide, device="cuda") for t in ts] for _ in range(2)],
                                     [torch.zeros((), device="cuda") for _ in ts], 1e-3, max_norm=1.0, norm_type=p))
        clip = float(optim.clip_grad_norm_(ts, 1.0, p))
        tol = 0.0 if p == math.inf else 2 * norm_tol([np.empty(t.numel()) for t in ts]) * norm
        assert abs(adam - norm) <= tol and abs(clip - norm) <= tol


def _policy(**solver):
    torch, optim = _t()
    from mbrl_amd.strategies import VariationalOptimization
    from test_strategy_host import cfg_vo, fake_agent
    cfg = cfg_vo()
    for k, value in solver.items():
        cfg.SOLVER[k] = value
    agent = fake_agent()
    agent.engine = types.SimpleNamespace(device=torch.device("cuda"))
    return VariationalOptimization(cfg, agent)


@pytest.mark.parametrize("fused", [False, True])
def test_the_strategys_norm_is_of_the_gradients_before_the_step(fused):
    torch, optim = _t()
    pol = _policy(FUSED=fused, CLIP_GRAD_NORM=0.25)
    assert type(pol.optimizer) is (optim.FusedAdam if fused else torch.optim.Adam)
    seen = []
    for k in range(3):
        stats = pol.optimize((pol.mean.sum() * (3.0 + k)).expand(4, 5) + 0 * pol.sd.sum(),
                             grad_sync=lambda grads: seen.append((float(optim.grad_norm(grads)), sum(g.numel() for g in grads))))
        norm, n = seen[-1]
        assert abs(stats["grad_norm"] - norm) <= 2 * (n + 4) * 2.0 ** -53 * norm and norm > 0.25
    assert float(pol.optimizer.state[pol.mean]["step"]) == 3.0


def test_the_trainer_heeds_the_bound(tmp_path):
    """A bound that every gradient exceeds leads elsewhere than none, with torch's Adam and with the fused update."""
    torch, optim = _t()
    from test_gpu_trainer import _cfg, _train
    base = dict(SOLVER__BASE_LR=0.02, MODEL__POLICY__NETWORK=False)
    for fused in (False, True):
        res = []
        for tag, bound in (("none", 0.0), ("clipped", 1e-3)):
            agent, _, _ = _train(_cfg("InvertedDoublePendulumEnv", **base, SOLVER__FUSED=fused, SOLVER__CLIP_GRAD_NORM=bound), tmp_path, "%s%d" % (tag, fused))
            res.append({k: v.cpu().double() for k, v in agent.policy_net.state_dict().items()})
        assert any(not torch.allclose(res[0][k], res[1][k], rtol=1e-6, atol=1e-9) for k in res[0])
