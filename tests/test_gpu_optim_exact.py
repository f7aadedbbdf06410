"""GPU: results of the optimiser-step operators that are known to the last bit, or by a few roundings, in each of their forms: one
block, several launches, and lists beyond the cache.  Companions fill a list up to each form without touching what is compared."""
import numpy as np
import pytest

from test_gpu_optim import HALF, _t, make

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
