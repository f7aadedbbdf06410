"""GPU: results of the optimiser-step operators that are known to the last bit, or by a few roundings, in each of their forms: one
block, several launches, and lists beyond the cache.  Companions fill a list up to each form without touching what is compared."""
import math

import numpy as np
import pytest

from test_gpu_optim import HALF, TINY, _t, make

pytestmark = pytest.mark.gpu

# values of a float32 companion: none, 2.4 MB of the four tensors (several launches), 96 MB (past the cache: from 64 MB on)
COMPANIONS = {"one block": 0, "several launches": 150001, "beyond the cache": 6_000_003}


def companion(n, count=4):
    torch, _ = _t()
    return [[torch.zeros(n, device="cuda")] if n else [] for _ in range(count)]


def adam(x, g, m, v, steps, more, **kw):
    torch, optim = _t()
    extra = companion(more)
    steps = steps + [torch.zeros((), device="cuda") for _ in extra[0]]
    return optim.adam_step(x + extra[0], g + extra[1], m + extra[2], v + extra[3], steps, kw.pop("lr"), **kw)


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 1e-40, 1e-8, 2.0 ** 70])
@pytest.mark.parametrize("more", list(COMPANIONS.values()), ids=list(COMPANIONS))
def test_root_and_quotient_are_correctly_rounded(more, eps):
    """Betas of 1/2 after 10 000 steps and no gradient: m and v are halved, 1 - b^t is 1, and x = -(m / (sqrt(v) + eps)) / 2 has
    three roundings, the root's, the sum's and the quotient's, which numpy makes the same way."""
    torch, _ = _t()
    rng = np.random.default_rng(5)
    m0 = rng.standard_normal(9001).astype(np.float32)
    v0 = (10.0 ** rng.uniform(-37, 37, 9001)).astype(np.float32)
    v0[:64] = (10.0 ** rng.uniform(-44, -38, 64)).astype(np.float32)          # subnormal ones
    m, v = torch.from_numpy(m0).cuda(), torch.from_numpy(v0).cuda()
    x, g, t = torch.zeros(9001, device="cuda"), torch.zeros(9001, device="cuda"), torch.full((), 1e4, device="cuda")
    adam([x], [g], [m], [v], [t], more, lr=0.5, betas=(0.5, 0.5), eps=eps)
    half = np.float32(0.5)
    assert np.array_equal(m.cpu().numpy(), half * m0) and np.array_equal(v.cpu().numpy(), half * v0)
    want = -half * ((half * m0) / (np.sqrt(half * v0) + np.float32(eps)))
    assert np.array_equal(x.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("wd,decoupled", [(0.0, False), (0.1, False), (0.1, True)])
def test_an_update_does_not_hang_on_the_rest_of_the_list(dtype, wd, decoupled):
    """The same bits alone, beside a middle list and beside one beyond the cache."""
    torch, _ = _t()
    wide = torch.float64 if dtype == "float64" else torch.float32
    results = []
    for more in COMPANIONS.values():
        sizes = [(4001,), (63, 5)]
        x, g = make(sizes, [dtype], 3, scale=1e-3), make(sizes, [dtype], 4)
        m, v = ([t.to(wide).mul_(0.1) for t in make(sizes, [dtype], s)] for s in (5, 6))
        v = [t.square_() for t in v]
        steps = [torch.full((), 3.0 + i, device="cuda") for i in range(2)]
        adam(x, g, m, v, steps, more, lr=0.01, weight_decay=wd, decoupled=decoupled)
        results.append(x + m + v)
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))


@pytest.mark.parametrize("dtype", ["float64", "float32", "bfloat16", "float16"])
@pytest.mark.parametrize("more", list(COMPANIONS.values()), ids=list(COMPANIONS))
@pytest.mark.parametrize("most", [1e-19, 1e-20, 1e-25, 1e-37, 1e-44, 1e-60, 1e-200])
def test_clipping_by_tiny_factors(dtype, more, most):
    """Gradients near a type's largest value and a bound far below 1: factors of 1e-57 and less, whose product with them is a normal
    float32 value.  Factor and product are rounded once each (2 u), to a 16-bit type once more; the last of the steps among
    subnormal values."""
    torch, optim = _t()
    top = {"float64": 1e100, "float16": 6e4}.get(dtype, 3e38)
    a = torch.tensor([top, -top / 3, top / 1e5, 1.0, 0.0, -2e-4], dtype=torch.float64).to(getattr(torch, dtype)).repeat(700)
    x = a.cuda()
    big = torch.full((1,), 1e38, device="cuda")            # the norm is far from 1 whatever the type
    extra = companion(more, 1)[0]
    norm = float(optim.clip_grad_norm_([x, big] + extra, most))
    ref = a.double().numpy()
    want = math.sqrt(np.sum(ref.astype(np.longdouble) ** 2) + np.longdouble(float(np.float32(1e38))) ** 2)
    assert abs(norm - want) <= (ref.size + 5) * 2.0 ** -53 * want
    c = np.longdouble(most) / (np.longdouble(want) + np.longdouble(1e-6))
    rel = HALF[dtype] + (ref.size + 9) * 2.0 ** -53 + {"float64": 0.0, "float32": 2.0 ** -24}.get(dtype, 2.0 ** -23)
    err = np.abs(x.double().cpu().numpy() - ref * c) - (1.001 * rel * np.abs(ref * c) + TINY[dtype])
    assert np.all(err <= 0), (x[:6].tolist(), [float(r) for r in (ref * c)[:6]])


@pytest.mark.parametrize("most", [1e-20, 1e-25, 1e-37, 1e-44])
def test_adam_clips_by_tiny_factors(most):
    """b1 = 0: the first moment is the clipped gradient, factor and product rounded once each."""
    torch, optim = _t()
    g = torch.tensor([3e38, -1e38, 1e33, 1.0], device="cuda")
    x, m, v, t = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros((), device="cuda")
    norm = float(optim.adam_step([x], [g], [m], [v], [t], 0.0, betas=(0.0, 0.9), max_norm=most))
    ref = g.double().cpu().numpy()
    want = math.sqrt(np.sum(ref ** 2))
    assert norm == pytest.approx(want, rel=8 * 2.0 ** -53)
    c = most / (want + 1e-6)
    got = m.double().cpu().numpy()
    assert np.all(np.abs(got - ref * c) <= (2.01 * 2.0 ** -24) * np.abs(ref * c) + 2.0 ** -149), (got, ref * c)


@pytest.mark.parametrize("more", list(COMPANIONS.values()), ids=list(COMPANIONS))
@pytest.mark.parametrize("p", [1, 2, math.inf])
def test_an_infinite_bound_clips_nothing(more, p):
    """Any norm that is a number is within it, an infinite one too; a NaN norm still makes every value NaN."""
    torch, optim = _t()
    for bad in (1.0, math.inf, math.nan):
        x = make([(300,)], ["float32"], 9)[0]
        x[7] = bad
        keep = x.clone()
        norm = float(optim.clip_grad_norm_([x] + companion(more, 1)[0], math.inf, p))
        assert math.isnan(norm) if math.isnan(bad) else norm == float(optim.grad_norm([keep], p))
        assert bool(x.isnan().all()) if math.isnan(bad) else torch.equal(x, keep)
    states = []
    for limit in (None, math.inf):
        g = make([(300,)], ["float32"], 9)[0]
        g[7] = -math.inf
        x, m, v, t = torch.ones(300, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros((), device="cuda")
        norm = adam([x], [g], [m], [v], [t], more, lr=0.1, max_norm=limit, norm_type=p)
        assert limit is None or float(norm) == math.inf
        states.append((x, m, v))
    for a, b in zip(*states):
        assert torch.allclose(a, b, rtol=0, atol=0, equal_nan=True) and bool(a[:7].isfinite().all())
