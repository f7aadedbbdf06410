"""GPU: the optimiser-step operators (optim.py over csrc/optim.hip) against their formulas in 64 bits on the host.

Tolerances.  u = half a step of a type: 2^-53, 2^-24, 2^-8 (bfloat16), 2^-11 (float16), relative.  A sum of n positive
terms in float64, in any order, is off by at most n 2^-53 relative (each addition rounds once; a square or its conversion adds
one more); a square root halves it and rounds once: (n + 4) 2^-53 bounds every norm here, the host's own included twice.
A clipped value is a product rounded once to its type, of a factor that is off by the norm's error and three roundings;
all but float64 values are multiplied in float32 (the factor's rounding: 2^-24 more, and the product's before it is
rounded to 16 bits: 2^-24 more there).  adam_bounds() counts the update's roundings."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float64": 5e-324, "float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}     # a step among subnormals
TYPES = list(HALF)


def _t():
    import torch
    import mbrl_amd  # noqa: F401
    from mbrl_amd import optim
    return torch, optim


def make(sizes, dtypes, seed=0, scale=1.0, misaligned=False, positive=False):
    """Tensors of these sizes on the GPU, types dealt out in turn; misaligned: slices of one buffer a type, so that they
    start anywhere."""
    torch, _ = _t()
    rng = np.random.default_rng(seed)
    out, offset = [], {}
    need = {d: sum(int(np.prod(s)) + 1 for s in sizes) + 7 for d in dtypes}
    buf = {d: torch.zeros(need[d], dtype=getattr(torch, d), device="cuda") for d in dtypes} if misaligned else {}
    for i, s in enumerate(sizes):
        d = dtypes[i % len(dtypes)]
        x = rng.standard_normal(s) * scale * 10.0 ** rng.uniform(-2, 1)
        x = torch.from_numpy(np.asarray(np.abs(x) if positive else x)).to(getattr(torch, d)).cuda()
        if misaligned:
            o = offset.get(d, 1)
            view = buf[d][o:o + x.numel()].view(x.shape)
            view.copy_(x)
            offset[d] = o + x.numel() + i % 2
            x = view
        out.append(x)
    return out


def host(ts):
    return [t.detach().double().cpu().numpy().astype(np.float64) for t in ts]


def ref_norm(arrays, p):
    flat = np.concatenate([a.reshape(-1) for a in arrays] + [np.zeros(0)]).astype(np.longdouble)
    if not flat.size:
        return 0.0
    if p == math.inf:
        return float(np.max(np.abs(flat)))
    return float(np.sum(np.abs(flat) ** int(p)) ** (np.longdouble(1) / int(p)))


def norm_tol(arrays):
    return (sum(a.size for a in arrays) + 4) * 2.0 ** -53


ODD = [(0,), (1,), (3,), (7, 5), (64,), (257,), (511,), (512,), (513,), (3, 0, 2), (1025,), (63, 65)]


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("misaligned", [False, True])
def test_norm(p, dtypes, misaligned):
    _, optim = _t()
    ts = make(ODD, dtypes, misaligned=misaligned)
    arrays = host(ts)
    got = optim.grad_norm(ts, p)
    assert got.shape == () and str(got.dtype) == "torch.float64"
    want = ref_norm(arrays, p)
    assert abs(float(got) - want) <= (0.0 if p == math.inf else norm_tol(arrays) * want)


@pytest.mark.parametrize("n", [1, 4095, 4096, 4097, 70001, 300007])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_and_clip_of_one_tensor(n, dtype):
    check_clip([(n,)], [dtype], 0.3)


def check_clip(sizes, dtypes, fraction, p=2.0, misaligned=False, seed=1):
    _, optim = _t()
    ts = make(sizes, dtypes, seed=seed, misaligned=misaligned)
    arrays = host(ts)
    want = ref_norm(arrays, p)
    most = fraction * want
    norm = optim.clip_grad_norm_(ts, most, p)
    assert abs(float(norm) - want) <= norm_tol(arrays) * want
    c = min(1.0, most / (want + 1e-6))
    for t, a in zip(ts, arrays):
        name = str(t.dtype)[6:]
        rel = HALF[name] + norm_tol(arrays) + 4 * 2.0 ** -53 + {"float64": 0.0, "float32": 2.0 ** -24}.get(name, 2 * 2.0 ** -24)
        got = t.double().cpu().numpy()
        if fraction > 1.0:
            assert np.array_equal(got, a)
        else:
            assert np.all(np.abs(got - a * c) <= 1.001 * rel * np.abs(a * c) + TINY[name]), name
    return ts


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("fraction", [0.3, 0.0, 3.0])
def test_clip(p, dtypes, fraction):
    check_clip(ODD, dtypes, fraction, p)
    check_clip(ODD, dtypes, fraction, p, misaligned=True)


@pytest.mark.parametrize("count", [64, 65, 191, 192, 193, 400, 1000])
def test_many_tensors(count):
    """Around the borders of what one launch takes, and of one wave's search for a unit's tensor."""
    rng = np.random.default_rng(count)
    sizes = [(int(rng.integers(0, 700)),) for _ in range(count)]
    check_clip(sizes, TYPES, 0.4, misaligned=True)
    check_adam(sizes, ["float32", "bfloat16"], most=0.5, misaligned=True)


@pytest.mark.parametrize("count", [16, 17, 58, 59, 98, 99, 109, 110, 128, 129, 160, 161, 246, 247, 492, 493])
def test_list_borders(count):
    """Around the sizes of lists and the numbers of tensors that one block takes on: lists of short tensors, and of one long one
    among them, which need not be short."""
    rng = np.random.default_rng(count)
    sizes = [(int(rng.integers(1, 60)),) for _ in range(count)]
    check_clip(sizes, TYPES, 0.4, misaligned=True)
    check_adam(sizes, TYPES, most=0.5, misaligned=True, steps=1)
    sizes[count // 2] = (70001,)
    check_clip(sizes, ["float32", "float16"], 0.4)
    check_adam(sizes, ["float32", "float16"], steps=1)
    check_adam(sizes, ["bfloat16", "float64"], most=0.5, steps=1)


def test_empty_lists_and_zeros():
    torch, optim = _t()
    for ts in ([], [torch.zeros(0, device="cuda")], [torch.zeros((0, 4), device="cuda", dtype=torch.float16)] * 3):
        assert float(optim.grad_norm(ts)) == 0.0 and float(optim.clip_grad_norm_(ts, 1.0)) == 0.0
    for count in (1, 53, 81, 200):
        ts, steps = [torch.zeros(0, device="cuda") for _ in range(count)], [torch.zeros((), device="cuda") for _ in range(count)]
        assert float(optim.grad_norm(ts)) == 0.0 and float(optim.clip_grad_norm_(ts, 1.0)) == 0.0
        assert float(optim.adam_step(ts, ts, ts, ts, steps, 1e-3, max_norm=1.0)) == 0.0 and all(float(s) == 1.0 for s in steps)
    ts = [torch.zeros(100, device="cuda"), -torch.zeros(3, device="cuda", dtype=torch.float64)]
    for p in (1, 2, math.inf):
        assert float(optim.grad_norm(ts, p)) == 0.0
    assert float(optim.clip_grad_norm_(ts, 1.0)) == 0.0 and all(not bool(t.any()) for t in ts)
    assert optim.adam_step([], [], [], [], [], 1e-3) is None
    assert float(optim.adam_step([], [], [], [], [], 1e-3, max_norm=1.0)) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_nan_and_infinity(dtype, p):
    torch, optim = _t()
    for bad, n in ((math.nan, 5), (math.inf, 5000), (-math.inf, 700)):
        ts = make([(33,), (n,)], [dtype], seed=3)
        ts[1][n - 1] = bad
        norm = float(optim.grad_norm(ts, p))
        assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
        with pytest.raises(RuntimeError, match="norm of the gradients"):
            optim.clip_grad_norm_(ts, 1.0, p, error_if_nonfinite=True)
        keep = host(ts)
        optim.clip_grad_norm_(ts, 1.0, p)
        got = host(ts)
        if math.isnan(bad):
            assert all(np.isnan(a).all() for a in got)
        else:
            assert not got[0].any() and not got[1][:-1].any() and np.isnan(got[1][-1]) and np.isfinite(keep[0]).all()
    # both: a NaN wins over an infinity wherever they are
    ts = make([(3,), (900,)], [dtype], seed=4)
    ts[0][1], ts[1][890] = math.inf, math.nan
    assert math.isnan(float(optim.grad_norm(ts, p)))
    ts[0][1], ts[1][890] = math.nan, math.inf
    assert math.isnan(float(optim.grad_norm(ts, p)))


def test_largest_and_smallest_values():
    torch, optim = _t()
    x = torch.full((1000,), 3e38, device="cuda")
    assert float(optim.grad_norm([x])) == pytest.approx(float(np.float32(3e38)) * math.sqrt(1000), rel=1e-12)
    assert float(optim.grad_norm([x.bfloat16()])) == pytest.approx(float(x.bfloat16()[0]) * math.sqrt(1000), rel=1e-12)
    optim.clip_grad_norm_([x], 1.0)
    assert np.allclose(x.cpu().numpy(), 1 / math.sqrt(1000), rtol=2.0 ** -23, atol=0)
    s = torch.full((77,), 1e-45, device="cuda")                     # a subnormal: not flushed
    assert float(optim.grad_norm([s])) == pytest.approx(float(s[0]) * math.sqrt(77), rel=1e-12) and float(s[0]) > 0
    d = torch.tensor([1e300, 1.0], dtype=torch.float64, device="cuda")
    assert float(optim.grad_norm([d])) == math.inf and float(optim.grad_norm([d], math.inf)) == 1e300


def test_any_dense_order_of_values():
    torch, optim = _t()
    base = make([(6, 10, 4)], ["float32"], seed=8)[0]
    for x in (base.permute(2, 0, 1).contiguous().permute(1, 2, 0), base.clone().t() if base.dim() == 2 else base.clone().transpose(0, 2)):
        a = x.cpu().numpy().astype(np.float64)
        norm = optim.clip_grad_norm_([x], 0.5 * ref_norm([a], 2))
        c = 0.5 * ref_norm([a], 2) / (float(norm) + 1e-6)
        assert np.all(np.abs(x.double().cpu().numpy() - c * a) <= 2.02 * 2.0 ** -24 * np.abs(c * a))
    rows = base.view(6, 40)[2]                                       # a row of a matrix: the rest stays as it was
    keep = base.clone()
    optim.clip_grad_norm_([rows], 0.0)
    assert not bool(base.view(6, 40)[2].any()) and torch.equal(base.view(6, 40)[3:], keep.view(6, 40)[3:])
    assert torch.equal(base.view(6, 40)[:2], keep.view(6, 40)[:2])


def test_same_bits_every_time_and_shared_memory_is_refused():
    torch, optim = _t()
    ts = make([(100003,), (999,), (40, 6)], TYPES, seed=5)
    norms = {float(optim.grad_norm(ts, p)) for _ in range(20) for p in (2,)}
    assert len(norms) == 1
    x = torch.ones(100, device="cuda")
    # counted twice where it is only read: sqrt(200) from two exact sums of 100, one rounding
    assert float(optim.grad_norm([x, x])) == math.sqrt(200.0)
    for pair in ([x, x], [x[:60], x[50:]], [x, x[3:4]]):
        with pytest.raises(ValueError, match="share memory"):
            optim.clip_grad_norm_(pair, 1.0)
    assert bool((x == 1).all())
    optim.clip_grad_norm_([x[:50], x[50:]], 1.0)
    step = torch.zeros((), device="cuda")
    y = [torch.ones(100, device="cuda") for _ in range(6)]
    with pytest.raises(ValueError, match="shares memory"):
        optim.adam_step(y[:2], y[2:4], y[4:5] * 2, [y[5], torch.ones(100, device="cuda")], [step, step.clone()], 1e-3)
    with pytest.raises(ValueError, match="shares memory"):       # one counter for two parameters
        optim.adam_step(y[:2], y[2:4], y[4:], [torch.ones(100, device="cuda") for _ in range(2)], [step, step], 1e-3)


# ---- Adam ----
def adam_bounds(x, g, m, v, t, lr, b1, b2, eps, wd, decoupled, c, u, c_err):
    """One step in extended precision (so that float64 results can be held to their own roundings) and the largest errors, with
    u the half step of the arithmetic.
    g1 = c g: factor rounded, product: 2u (and the factor's own error).  L2: wd rounded, one fused product: 2u |wd x| + u |g1|.
    m': a1 = 1 - b1 rounded, a1 g1 rounded, b1 rounded, one fused sum.
    v': a2 rounded, two products, g1 squared (twice its error); b2 rounded; one fused sum.
    d = sqrt(v') root + eps: half of v's error, sqrt, root and eps rounded, one fused sum.  A float32 root may be the hardware's
    own, within a step (2 u) instead of half a one, of an argument that may have been scaled by a power of 2.
    x' = x keep - size (m' / d): quotient, size, keep, product, one fused sum.  A float32 quotient may be the product with the
    hardware's reciprocal: a step (2 u) and the product's rounding (u) instead of u.
    size and root come from 1 - b^t = -expm1(t log1p(b - 1)) in float64: log1p and expm1 within a step (2 w with w = 2^-53), the
    product w, and expm1 of a negative number passes on at most its argument's relative error: 5 w, a division (and a root)
    more: 6 w.  keep = 1 - lr wd: two roundings."""
    own = 2 if u == 2.0 ** -24 else 0        # u more in a float32 quotient, half of that in a root
    x, g, m, v = (a.astype(np.longdouble) for a in (x, g, m, v))
    b1, b2, one, w = np.longdouble(b1), np.longdouble(b2), np.longdouble(1), 2.0 ** -53
    g1 = np.longdouble(c) * g
    eg = (2 * u + c_err) * np.abs(g1)
    if not decoupled and wd:
        g1 = g1 + np.longdouble(wd) * x
        eg = eg + 2 * u * np.abs(wd * x) + u * np.abs(g1)
    m1 = b1 * m + (1 - b1) * g1
    em = 2 * u * np.abs(b1 * m) + (1 - b1) * (eg + 2 * u * np.abs(g1)) + u * np.abs(m1)
    v1 = b2 * v + (1 - b2) * g1 * g1
    ev = 2 * u * b2 * v + (1 - b2) * (2 * np.abs(g1) * eg + eg * eg + 4 * u * g1 * g1) + u * v1
    root = one / np.sqrt(one - b2 ** t)
    s = np.sqrt(v1)
    es = np.where(v1 > 0, ev / (2 * np.where(v1 > 0, s, 1)), np.sqrt(ev)) + (1 + own / 2) * u * s
    d = s * root + eps
    ed = es * root + (3 * u + 6 * w) * s * root + u * eps + u * d
    size = lr / (one - b1 ** t)
    q = m1 / d
    eq = em / d + np.abs(q) * ed / d + (1 + own) * u * np.abs(q)
    keep = one - np.longdouble(lr) * np.longdouble(wd) if decoupled else one
    x1 = x * keep - size * q
    ex = size * eq + (2 * u + 6 * w) * size * np.abs(q) + 3 * u * np.abs(x * keep) * (1 if decoupled else 0) + u * np.abs(x1)
    return (x1, 1.02 * ex), (m1, 1.02 * em), (v1, 1.02 * ev)


def check_adam(sizes, dtypes, most=None, p=2.0, wd=0.0, decoupled=False, misaligned=False, steps=2, seed=11, lrs=(1e-3, 1e-2)):
    torch, optim = _t()
    wide = lambda d: "float64" if d == "float64" else "float32"      # noqa: E731
    xs = make(sizes, dtypes, seed, misaligned=misaligned)
    ms = [t.to(getattr(torch, wide(str(x.dtype)[6:]))).mul_(0.1) for t, x in zip(make(sizes, dtypes, seed + 1), xs)]
    vs = [t.to(getattr(torch, wide(str(x.dtype)[6:]))).square_().mul_(0.1) for t, x in zip(make(sizes, dtypes, seed + 2), xs)]
    counts = [torch.tensor(float(i % 5), device="cuda") for i in range(len(sizes))]
    lr = [lrs[i % len(lrs)] for i in range(len(sizes))]
    b1, b2, eps = 0.9, 0.99, 1e-6
    for k in range(steps):
        gs = make(sizes, dtypes, seed + 10 + k, misaligned=misaligned)
        ax, ag, am, av = host(xs), host(gs), host(ms), host(vs)
        limit = None if most is None else most * ref_norm(ag, p)
        versions = [x._version for x in xs]
        norm = optim.adam_step(xs, gs, ms, vs, counts, lr, (b1, b2), eps, wd, decoupled, limit, p)
        c, c_err = 1.0, 0.0
        if most is None:
            assert norm is None
        else:
            want = ref_norm(ag, p)
            assert abs(float(norm) - want) <= norm_tol(ag) * want
            c, c_err = min(1.0, limit / (want + 1e-6)), norm_tol(ag) + 4 * 2.0 ** -53
        for i, (x, g, m, v) in enumerate(zip(xs, gs, ms, vs)):
            name, t = str(x.dtype)[6:], i % 5 + k + 1
            assert float(counts[i]) == t and x._version > versions[i]     # views of one buffer count together
            assert np.array_equal(g.double().cpu().numpy(), ag[i])                    # gradients are only read
            bounds = adam_bounds(ax[i], ag[i], am[i], av[i], t, lr[i], b1, b2, eps, wd, decoupled, c, HALF[wide(name)], c_err)
            for what, got, (ref, err), extra in (("x", x, bounds[0], HALF[name] if name != wide(name) else 0.0), ("m", m, bounds[1], 0.0),
                                                 ("v", v, bounds[2], 0.0)):
                got = got.double().cpu().numpy().astype(np.longdouble)
                slack = err + extra * (np.abs(ref) + err) + TINY[name if what == "x" else wide(name)]
                assert np.all(np.abs(got - ref) <= slack), (what, name, sizes[i], float(np.max(np.abs(got - ref) / slack)))


@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("wd,decoupled", [(0.0, False), (0.1, False), (0.1, True)])
@pytest.mark.parametrize("most", [None, 0.3, 3.0])
def test_adam(dtypes, wd, decoupled, most):
    check_adam(ODD, dtypes, most, wd=wd, decoupled=decoupled)


@pytest.mark.parametrize("p", [1.0, math.inf])
def test_adam_clips_by_other_norms(p):
    check_adam(ODD, TYPES, 0.3, p, misaligned=True)


@pytest.mark.parametrize("count", [79, 80, 81, 159, 160, 161])
def test_adam_list_borders(count):
    check_adam([(1 + 37 * i % 90,) for i in range(count)], TYPES, misaligned=True)


@pytest.mark.parametrize("n", [4095, 8193, 70001, 1 << 20])
@pytest.mark.parametrize("dtype", TYPES)
def test_adam_of_one_tensor(n, dtype):
    check_adam([(n,)], [dtype], 0.5)


@pytest.mark.parametrize("count,rates", [(99, 1), (99, 99), (130, 64), (130, 65), (416, 3), (417, 3), (600, 200)])
def test_adam_rates_of_long_lists(count, rates):
    """Learning rates of their own, more than a launch that counts the steps holds, and as many tensors."""
    check_adam([(1 + 37 * i % 50,) for i in range(count)], ["float32"], wd=0.1, lrs=[1e-3 * (k + 1) / rates for k in range(rates)])


def test_adam_of_the_smallest_and_largest_moments():
    """Second moments from nothing and subnormal values to the largest, with and without eps, against float64.  m, v, root, scale,
    sum, quotient, size and product: 12 half steps at most."""
    torch, optim = _t()
    v = torch.tensor([0.0, 1e-45, 3e-42, 1e-38, 2e-30, 1e-12, 1.0, 1e20, 3e38], device="cuda")
    for eps in (0.0, 1e-8):
        for n in (9, 300001):
            vs = v.repeat(n // 9 + 1)[:n].contiguous()
            m = torch.full((n,), 1e-3, device="cuda")
            x, g, t = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.full((), 9.0, device="cuda")
            want_v = vs.double().cpu().numpy() * float(np.float32(0.99))
            want_v = want_v.astype(np.float32).astype(np.float64)          # one rounding, of subnormal values too
            optim.adam_step([x], [g], [m], [vs], [t], 0.5, (0.9, 0.99), eps)
            assert np.array_equal(vs.double().cpu().numpy(), want_v)
            m1 = m.double().cpu().numpy()
            d = np.sqrt(want_v) / math.sqrt(1 - 0.99 ** 10) + eps
            with np.errstate(divide="ignore"):
                want = -0.5 / (1 - 0.9 ** 10) * m1 / d
            got = x.double().cpu().numpy()
            big = np.abs(want) > 3e38
            assert np.all(np.isinf(got[big]) & (got[big] < 0)) and np.all(np.abs(got[~big] - want[~big]) <= 12 * 2.0 ** -24 * np.abs(want[~big]) + 1e-37)


@pytest.mark.parametrize("eps", [2.0 ** -149, 1e-40, 1e-38, 2e-38, 1e20, 1e38, 2.0 ** 127])
def test_adam_with_an_eps_at_the_ends_of_float32(eps):
    """An eps whose reciprocal is subnormal or infinite, or that is subnormal itself, over second moments that leave it alone in
    the denominator or not.  Roundings as in adam_bounds(): root 2 (in half steps), its scale, eps and the sum 1 each,
    quotient 3, size and product 1 each: 10."""
    torch, optim = _t()
    m0 = [0.0, 1e-30, -1e-22, 1e-3, 1e2, 0.0, 1e-3, 1e-3, 1e2]
    v0 = [0.0, 0.0, 0.0, 1e-30, 1e-12, 1.0, 1.0, 1e30, 3e38]
    for n in (9, 9 * 40000):
        m, v = (torch.tensor(a, device="cuda").repeat(n // 9) for a in (m0, v0))
        x, g, t = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.full((), 9.0, device="cuda")
        optim.adam_step([x], [g], [m], [v], [t], 0.5, (0.9, 0.99), eps)
        d = np.sqrt(v.double().cpu().numpy()) / math.sqrt(1 - 0.99 ** 10) + eps
        want = -0.5 / (1 - 0.9 ** 10) * m.double().cpu().numpy() / d
        got = x.double().cpu().numpy()
        big = np.abs(want) > 3.5e38
        assert np.all(np.isinf(got[big]) & (np.sign(got[big]) == np.sign(want[big])))
        err = np.abs(got[~big] - want[~big]) - (10 * 2.0 ** -24 * np.abs(want[~big]) + 2.0 ** -126)
        assert np.all(err <= 0), (eps, n, got[:9], want[:9])


def test_adam_keeps_infinite_parameters_apart_from_their_moments():
    torch, optim = _t()
    x, g = torch.full((5,), math.inf, device="cuda"), torch.ones(5, device="cuda")
    m, v, t = torch.zeros(5, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros((), device="cuda")
    optim.adam_step([x], [g], [m], [v], [t], 1e-3)
    assert bool(torch.isinf(x).all()) and np.allclose(m.cpu(), 0.1) and np.allclose(v.cpu(), 1e-3)
    # a first step of size lr whatever the gradient's scale; nothing where there has never been a gradient
    x, g = torch.zeros(4, device="cuda"), torch.tensor([1e-3, -1e3, 0.0, 1.0], device="cuda")
    m, v, t = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros((), device="cuda")
    optim.adam_step([x], [g], [m], [v], [t], 0.5)
    assert np.allclose(x.cpu(), [-0.5, 0.5, 0.0, -0.5], rtol=2e-5)


def test_fused_adam_follows_torchs_adam():
    """Same rule, other rounding: float64 parameters agree to 1e-12 relative over 25 steps (about 30 roundings of 2^-53 a
    step on values of order 1, no cancellation beyond the update's own size); parameters without a gradient rest."""
    torch, optim = _t()
    for wd, decoupled in ((0.0, False), (0.02, False), (0.02, True)):
        a = [t.clone().requires_grad_() for t in make([(6, 40), (6, 40), (17,), (4, 3, 2)], ["float64"], 21)]
        b = [t.detach().clone().requires_grad_() for t in a]
        kw = dict(betas=(0.85, 0.97), eps=1e-7, weight_decay=wd, decoupled_weight_decay=decoupled)
        mine = optim.FusedAdam([{"params": a[:2], "lr": 0.01}, {"params": a[2:], "lr": 0.003}], **kw)
        ref = torch.optim.Adam([{"params": b[:2], "lr": 0.01}, {"params": b[2:], "lr": 0.003}], **kw)
        for k in range(25):
            gs = make([tuple(t.shape) for t in a], ["float64"], 100 + k)
            for i, (x, y, g) in enumerate(zip(a, b, gs)):
                x.grad, y.grad = (None, None) if i == 2 and k % 3 else (g, g.clone())
            mine.step()
            ref.step()
            if k == 12:                       # each goes on from the other's state
                s, r = mine.state_dict(), ref.state_dict()
                mine.load_state_dict(r)
                ref.load_state_dict(s)
        for x, y in zip(a, b):
            assert torch.allclose(x, y, rtol=1e-12, atol=1e-12)
            assert float(mine.state[x]["step"]) == float(ref.state[y]["step"])


def test_captured_and_replayed():
    """Both calls in one graph, replayed with eager work and a second graph between the replays: the counters go on, and each
    replay gives the bits of the eager calls."""
    torch, optim = _t()
    sizes = [(300, 7), (513,), (100001,), (0,)]

    def state():
        xs, gs = make(sizes, ["float32", "float64"], 31), make(sizes, ["float32", "float64"], 32)
        return xs, gs, [torch.zeros_like(x) for x in xs], [torch.zeros_like(x) for x in xs], [torch.zeros((), device="cuda") for _ in xs]

    def one(s):
        n = optim.clip_grad_norm_(s[1], 5.0)
        return n, optim.adam_step(*s, 0.01, max_norm=2.0, norm_type=1)
    eager, graphs, norms = state(), [], []
    states = [state(), state()]
    for s in states:
        warm = [[t.clone() for t in l] for l in s]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one(warm)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(one(s))
        graphs.append(g)
    for k in range(5):
        fresh = make(sizes, ["float32", "float64"], 50 + k)
        for l in (eager, *states):
            for a, b in zip(l[1], fresh):
                a.copy_(b)
        want = one(eager)
        for g in graphs:
            g.replay()
        one([[t.clone() for t in l] for l in eager])           # eager work of the same kind between
        torch.cuda.synchronize()
        for s, n in zip(states, norms):
            assert float(n[0]) == float(want[0]) and float(n[1]) == float(want[1])
            for la, lb in zip(s, eager):
                for a, b in zip(la, lb):
                    assert torch.equal(a, b), k
        assert float(eager[4][0]) == k + 1
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(ValueError, match="captured"):
            optim.clip_grad_norm_(eager[1], 1.0, error_if_nonfinite=True)
        optim.grad_norm(eager[1])


@pytest.mark.parametrize("sizes", [[(40,), (6, 7)], [(1 + 37 * i % 90,) for i in range(450)], [(17_000_001,), (33,)]])
def test_captured_and_replayed_lists_of_all_lengths(sizes):
    """One block's work, several launches of counts, sums and updates, and lists beyond the cache: every replay gives the bits of
    the eager calls."""
    torch, optim = _t()
    types = ["float32", "bfloat16"]

    def state():
        xs, gs = make(sizes, types, 35), make(sizes, types, 36)
        ms, vs = ([torch.zeros(x.shape, device="cuda") for x in xs] for _ in range(2))
        return xs, gs, ms, vs, [torch.zeros((), device="cuda") for _ in xs]

    def one(s):
        n = optim.clip_grad_norm_(s[1], 5.0)
        return n, optim.adam_step(*s, [1e-3 * (1 + i % 70) for i in range(len(sizes))], max_norm=2.0)
    eager, graphed, graph = state(), state(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norms = one(graphed)
    for k in range(3):
        for l in (eager, graphed):
            for a, b in zip(l[1], make(sizes, types, 60 + k)):
                a.copy_(b)
        want = one(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert [float(a) for a in norms] == [float(a) for a in want]
        for la, lb in zip(graphed, eager):
            assert all(torch.equal(a, b) for a, b in zip(la, lb)), k
        assert all(float(c) == k + 1 for c in graphed[4][:2])


def test_streams_beside_each_other():
    torch, optim = _t()
    lists = [make([(200003,), (77,)], ["float32"], 60 + i) for i in range(4)]
    want = [host(l) for l in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    torch.cuda.synchronize()
    norms = []
    for l, s in zip(lists, streams):
        with torch.cuda.stream(s):
            norms.append([optim.clip_grad_norm_(l, 1.0) for _ in range(3)])
    torch.cuda.synchronize()
    for l, a, n in zip(lists, want, norms):
        assert abs(float(n[0]) - ref_norm(a, 2)) <= norm_tol(a) * ref_norm(a, 2)
        # clipped once: under the bound from then on, but for the rounding of 2e5 values
        assert abs(float(n[1]) - 1.0) < 2e-6 and float(n[2]) <= 1.0 + 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_does_not_hang_on_addresses(dtype):
    """The same values in tensors of their own, one behind another, at odd places and in any dense order: the same bits, so that
    all ranks of a sharded run clip by the same factor."""
    torch, optim = _t()
    for sizes in ([(700,), (3, 5), (0,), (4097,), (512,), (64, 64)], [(1 + 997 * i % 4000,) for i in range(300)], [(1 << 20,), (70001,), (1,)]):
        apart = make(sizes, [dtype], seed=75)
        n = sum(t.numel() for t in apart)
        results = []
        for lead in (0, 1, 7):
            buf = torch.zeros(n + lead, dtype=apart[0].dtype, device="cuda")[lead:]
            views = [v.view(t.shape) for v, t in zip(buf.split([t.numel() for t in apart]), apart)]
            results.append([v.copy_(t) for v, t in zip(views, apart)])
        for p in (1, 2):
            want = float(optim.grad_norm(apart, p))
            assert all(float(optim.grad_norm(v, p)) == want for v in results)
        want = float(optim.clip_grad_norm_([t.clone() for t in apart], 1.0))
        adam = lambda ts: float(optim.adam_step([t.clone() for t in ts], ts, *[[torch.zeros(t.shape, dtype=torch.float64 if dtype == "float64"    # noqa: E731
                                 else torch.float32, device="cuda") for t in ts] for _ in range(2)],
                                [torch.zeros((), device="cuda") for _ in ts], 0.0, max_norm=1.0))
        first = adam(apart)
        for v in results:
            assert adam(v) == first and float(optim.clip_grad_norm_(v, 1.0)) == want
        for v in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(v, results[0]))


@pytest.mark.parametrize("dtype", TYPES)
def test_neighbours_in_one_buffer(dtype):
    """Tensors that follow each other in memory, empty ones and another type between them, and a gap: every value once."""
    torch, optim = _t()
    sizes = [700, 1, 0, 0, 63, 4097, 512, 0, 9, 30000]
    whole = make([(sum(sizes) + 5,)], [dtype], seed=71)[0]
    parts = list(whole[:sum(sizes)].split(sizes))
    other = make([(333,)], ["float32" if dtype != "float32" else "float64"], seed=72)[0]
    ts = parts[:4] + [other] + parts[4:8] + parts[9:]           # parts[8] is left out
    for p in (2.0, math.inf):
        arrays = host(ts)
        assert abs(float(optim.grad_norm(ts, p)) - ref_norm(arrays, p)) <= norm_tol(arrays) * ref_norm(arrays, p)
        assert float(optim.grad_norm(ts[::-1], p)) == pytest.approx(ref_norm(arrays, p), rel=1e-12)
    keep = whole.clone()
    optim.clip_grad_norm_(ts, 0.0)
    at = sum(sizes[:8])
    assert torch.equal(whole[at:at + 9], keep[at:at + 9]) and torch.equal(whole[sum(sizes):], keep[sum(sizes):])
    assert not any(bool(t.any()) for t in ts)


@pytest.mark.parametrize("dtype,n", [("float32", 69_000_001), ("bfloat16", 138_000_003), ("float16", 138_000_003), ("float64", 35_000_001)])
def test_lists_beyond_the_cache(dtype, n):
    """More than 256 MB, where the accesses and the walk are others; expected values in float64 on the device."""
    torch, optim = _t()
    kind = getattr(torch, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    # two tensors of one odd buffer (one run to the norm) and a small one apart
    whole = torch.randn(n + 1, dtype=torch.float32, device="cuda", generator=g).to(kind)[1:]
    ts = [whole[:n // 3], whole[n // 3:], torch.randn(77, dtype=torch.float32, device="cuda", generator=g).to(kind)]
    total = sum(float(t.double().square().sum()) for t in ts)
    want = math.sqrt(total)
    tol = (n + 81) * 2.0 ** -53
    assert abs(float(optim.grad_norm(ts)) - want) <= tol * want
    assert float(optim.grad_norm(ts, math.inf)) == max(float(t.abs().max()) for t in ts)
    keep = [t.clone() for t in ts]
    norm = optim.clip_grad_norm_(ts, 2 * want)
    assert all(torch.equal(a, b) for a, b in zip(ts, keep))
    norm = optim.clip_grad_norm_(ts, 0.3 * want)
    c = 0.3 * want / (float(norm) + 1e-6)
    rel = HALF[dtype] + 4 * 2.0 ** -53 + {"float64": 0.0, "float32": 2.0 ** -24}.get(dtype, 2 * 2.0 ** -24)
    for t, k in zip(ts, keep):
        e = k.double() * c
        assert bool(((t.double() - e).abs() <= 1.001 * rel * e.abs() + TINY[dtype]).all())


@pytest.mark.parametrize("dtype,n", [("float32", 17_000_001), ("bfloat16", 23_000_003), ("float64", 9_000_001)])
@pytest.mark.parametrize("most", [None, 0.3])
@pytest.mark.parametrize("parts", [3, 90])
def test_adam_beyond_the_cache(dtype, n, most, parts):
    """The same of the update, for 3 tensors and for more than one launch takes."""
    torch, optim = _t()
    kind, wide = getattr(torch, dtype), torch.float64 if dtype == "float64" else torch.float32
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    new = lambda k: torch.randn(n, dtype=torch.float32, device="cuda", generator=g).to(k)      # noqa: E731
    p, x, m, v = new(kind), new(kind), new(wide), new(wide).square_()
    cut = lambda t: list(t.tensor_split(parts))       # noqa: E731
    q, a, b = p.clone(), m.clone(), v.clone()
    norm = optim.adam_step(cut(q), cut(x), cut(a), cut(b), [torch.ones((), device="cuda") for _ in range(parts)], 0.01, weight_decay=0.1,
                           max_norm=None if most is None else most * math.sqrt(n))
    c = 1.0
    if most is not None:
        want = float(x.double().square().sum()) ** 0.5
        assert abs(float(norm) - want) <= (n + 4) * 2.0 ** -53 * want
        c = most * math.sqrt(n) / (float(norm) + 1e-6)
    u, w = HALF["float64" if dtype == "float64" else "float32"], 2.0 ** -53
    for s in torch.arange(n, device="cuda").tensor_split(8):
        lo, hi = int(s[0]), int(s[-1]) + 1
        X, G, M, V = (t[lo:hi].double() for t in (p, x, m, v))
        G = c * G + 0.1 * X
        M1, V1 = 0.9 * M + 0.1 * G, 0.999 * V + 0.001 * G * G
        d = V1.sqrt() / math.sqrt(1 - 0.999 ** 2) + 1e-8
        X1 = X - 0.01 / (1 - 0.9 ** 2) * M1 / d
        # adam_bounds(), its terms rounded up: 8 u of each summand of m', 12 u of v', 24 u of the update's parts; the factor
        # 1 - 0.999^2 written as here is off by 2^-53 / 0.002 = 500 w
        em = 8 * u * (0.9 * M.abs() + 0.1 * (c * x[lo:hi].double().abs() + 0.2 * X.abs()))
        ev = 12 * u * (V1 + 0.002 * (c * x[lo:hi].double().abs() + 0.1 * X.abs()).square())
        ex = 0.0527 * (em + (24 * u + 600 * w) * M1.abs() + M1.abs() * ev / V1) / d + 2 * u * X1.abs() + (HALF[dtype] if kind != wide else 0.0) * X1.abs() * 1.01
        for got, ref, e in ((q, X1, ex), (a, M1, em), (b, V1, ev)):
            assert bool(((got[lo:hi].double() - ref).abs() <= e + 1e-37).all())


def test_more_values_than_32_bits_count():
    """One float16 tensor of 2^31 + 4099 values (4 GiB): the last ones count, and are reached."""
    torch, optim = _t()
    n = (1 << 31) + 4099
    x = torch.zeros(n, dtype=torch.float16, device="cuda")
    at = [0, (1 << 31) - 1, 1 << 31, (1 << 31) + 4096, n - 1]
    x[at] = 3.0
    assert float(optim.grad_norm([x])) == math.sqrt(45.0)
    optim.clip_grad_norm_([x], 0.5 * (math.sqrt(45.0) + 1e-6))
    assert x[at].tolist() == [1.5] * 5 and int(torch.count_nonzero(x)) == 5


@pytest.mark.parametrize("others", [0, 16, 300])
def test_more_values_than_fit_32_bits(others):
    """2^32 + 4099 float16 values (8 GiB), alone and among short tensors: the last ones count, and are reached."""
    torch, optim = _t()
    n = (1 << 32) + 4099
    x = torch.zeros(n, dtype=torch.float16, device="cuda")
    x[0], x[-1], x[-4099] = 3.0, 4.0, 12.0
    ts = [torch.zeros(5, device="cuda") for _ in range(others)]
    ts.insert(others // 2, x)
    assert float(optim.grad_norm(ts)) == 13.0 and float(optim.grad_norm(ts, math.inf)) == 12.0
    assert float(optim.clip_grad_norm_(ts, 6.5)) == 13.0
    assert [float(x[i]) for i in (0, -1, -4099)] == [1.5, 2.0, 6.0] and int((x != 0).sum(dtype=torch.int64)) == 3


def test_a_run_of_them_together():
    """What a training loop does with them: gradients by autograd, their norm, clipping, update -- against the same in float64
    on the host, which starts every step from the same weights."""
    torch, optim = _t()
    torch.manual_seed(0)
    from mbrl_amd.strategies import FeedForward
    net = FeedForward(18, [64, 64, 32, 8], 6).cuda()
    ref = FeedForward(18, [64, 64, 32, 8], 6).double()
    ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
    opt, oref = optim.FusedAdam(net.parameters(), 1e-3, max_norm=0.25), torch.optim.Adam(ref.parameters(), 1e-3, foreach=False)
    data = torch.randn(5, 64, 18)
    for k in range(5):
        ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
        for model, o, x in ((net, opt, data[k].cuda()), (ref, oref, data[k].double())):
            o.zero_grad()
            (model(x) ** 2).sum().backward()
        before = optim.grad_norm([p.grad for p in net.parameters()])
        opt.step()
        want = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.25)
        oref.step()
        assert float(opt.grad_norm) == float(before)
        assert float(before) == pytest.approx(float(want), rel=1e-3)        # float32 network against float64
        first = optim.clip_grad_norm_([p.grad for p in net.parameters()], 0.25)
        assert float(first) == float(before)
        assert float(optim.grad_norm([p.grad for p in net.parameters()])) <= 0.25 * (1 + 2.0 ** -22)
        # an entry of Adam's step is at most lr (1 - b1) / sqrt(1 - b2) = 3.2 lr: where a gradient's sign is rounding, the two differ by twice that
        off = torch.cat([(p.detach().double().cpu() - q.detach()).abs().reshape(-1) for p, q in zip(net.parameters(), ref.parameters())])
        assert float(off.max()) <= 2 * 3.2e-3 and float(off.median()) <= 1e-5


def test_fused_adam_captured():
    """A captured step() counts its steps on the device: replays follow eager steps bit for bit, with other gradients each time."""
    torch, optim = _t()
    sizes = [(40, 30), (30,), (6, 40)]
    eager, graphed = ([t.clone().requires_grad_() for t in make(sizes, ["float32", "float32", "float64"], 81)] for _ in range(2))
    opts = [optim.FusedAdam(l, 0.01, weight_decay=0.01, max_norm=1.5) for l in (eager, graphed)]
    for l in (eager, graphed):
        for p in l:
            p.grad = torch.zeros_like(p)
    opts[1].step()                        # makes the state outside the capture
    opts[0].step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[1].step()
    norm = opts[1].grad_norm
    for k in range(4):
        for p, q, g in zip(eager, graphed, make(sizes, ["float32", "float32", "float64"], 90 + k)):
            p.grad.copy_(g)
            q.grad.copy_(g)
        opts[0].step()
        graph.replay()
        float(optim.grad_norm([p.grad for p in eager]))
        assert float(norm) == float(opts[0].grad_norm)
        for p, q in zip(eager, graphed):
            assert torch.equal(p, q) and torch.equal(opts[0].state[p]["exp_avg_sq"], opts[1].state[q]["exp_avg_sq"])
            assert float(opts[1].state[q]["step"]) == k + 2


def test_fused_adam_refuses_a_first_step_under_capture():
    """Its state would be zeroed by every replay."""
    torch, optim = _t()
    x = torch.ones(5, device="cuda", requires_grad=True)
    x.grad = torch.ones_like(x)
    opt = optim.FusedAdam([x], 0.01)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.zeros(1, device="cuda")
        with pytest.raises(RuntimeError, match="before it is captured"):
            opt.step()
    assert bool((x == 1).all()) and not opt.state[x]
    opt.step()
    assert float(opt.state[x]["step"]) == 1.0


def test_fused_adam_saves_and_goes_on():
    """16-bit parameters with their float32 moments, many of them: saved, loaded into a new optimiser, the same bits from there on.
    A closure, a scheduler, and a parameter of permuted dimensions on the way."""
    torch, optim = _t()
    sizes = [(11, 7, 5)] + [(3 * i % 50,) for i in range(120)]

    def params():
        ps = [t.clone().requires_grad_() for t in make(sizes, ["bfloat16", "float16", "float32"], 101)]
        ps[0] = ps[0].detach().permute(2, 0, 1).contiguous().permute(1, 2, 0).requires_grad_()
        return ps

    def run(ps, opt, sched, ks):
        for k in ks:
            gs = make(sizes, ["bfloat16", "float16", "float32"], 200 + k)

            def closure():
                for p, g in zip(ps, gs):
                    p.grad = torch.empty_like(p).copy_(g)       # laid out like its parameter, as autograd leaves it
                return k
            assert opt.step(closure) == k
            sched.step()
    a, b = params(), params()
    one = optim.FusedAdam(a, 0.05, max_norm=3.0, norm_type=1, weight_decay=0.1, decoupled_weight_decay=True)
    sa = torch.optim.lr_scheduler.StepLR(one, 1, 0.5)
    run(a, one, sa, range(6))
    first = optim.FusedAdam(b, 0.05, max_norm=3.0, norm_type=1, weight_decay=0.1, decoupled_weight_decay=True)
    sb = torch.optim.lr_scheduler.StepLR(first, 1, 0.5)
    run(b, first, sb, range(3))
    second = optim.FusedAdam(b, 1.0, max_norm=3.0, norm_type=1)
    sc = torch.optim.lr_scheduler.StepLR(second, 1, 0.5)
    second.load_state_dict(first.state_dict())
    sc.load_state_dict(sb.state_dict())
    run(b, second, sc, range(3, 6))
    assert one.param_groups[0]["lr"] == second.param_groups[0]["lr"] == pytest.approx(0.05 / 64)
    for p, q in zip(a, b):
        assert torch.equal(p, q) and torch.equal(one.state[p]["exp_avg"], second.state[q]["exp_avg"])
    assert one.state[a[0]]["exp_avg"].stride() == a[0].stride() and one.state[a[0]]["exp_avg"].dtype == torch.float32
    with pytest.raises(ValueError, match="another order"):
        a[0].grad = torch.zeros((11, 7, 5), dtype=a[0].dtype, device="cuda")
        one.step()


def test_threads_and_inference_tensors():
    torch, optim = _t()
    import threading
    lists = [make([(30011,), (5,), (700,)], ["float32", "float64"], 300 + i) for i in range(4)]
    want = [host(l) for l in lists]
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got[i] = float(optim.grad_norm(lists[i]))
                with pytest.raises(ValueError, match="norm_type"):
                    optim.grad_norm(lists[i], 5)
        except Exception as e:          # noqa: BLE001
            errors.append(e)
    torch.cuda.synchronize()
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not errors
    for g, a in zip(got, want):
        assert abs(g - ref_norm(a, 2)) <= norm_tol(a) * ref_norm(a, 2)
    with torch.inference_mode():
        x = torch.full((64,), 2.0, device="cuda")
        assert float(optim.clip_grad_norm_([x], 8.0)) == 16.0
    assert float(x[3]) == pytest.approx(1.0)


@pytest.mark.parametrize("fused", [False, True])
def test_trainer_clips(fused, tmp_path):
    """do_training with SOLVER.CLIP_GRAD_NORM: the same parameters whether torch's Adam follows the clipping or the fused
    update clips on its way, and every step's norm within the bound changes nothing against no clipping at all."""
    torch, optim = _t()
    from test_gpu_trainer import _cfg, _train
    base = dict(SOLVER__BASE_LR=0.02, MODEL__POLICY__NETWORK=False)
    res = {}
    for tag, over in (("torch", dict(SOLVER__CLIP_GRAD_NORM=1e-3)), ("fused", dict(SOLVER__CLIP_GRAD_NORM=1e-3, SOLVER__FUSED=True)),
                      ("idle", dict(SOLVER__CLIP_GRAD_NORM=1e12, SOLVER__FUSED=fused)), ("none", dict(SOLVER__FUSED=fused))):
        agent, rows, d = _train(_cfg("InvertedDoublePendulumEnv", **base, **over), tmp_path, tag)
        res[tag] = {k: v.cpu().double() for k, v in agent.policy_net.state_dict().items()}
        assert type(agent.policy_net.optimizer) is (optim.FusedAdam if over.get("SOLVER__FUSED") else torch.optim.Adam)
    for k in res["torch"]:
        assert torch.allclose(res["torch"][k], res["fused"][k], rtol=1e-6, atol=1e-9), k
        assert torch.equal(res["idle"][k], res["none"][k]), k
        assert torch.isfinite(res["fused"][k]).all()
