"""CPU: what the optimiser-step operators (optim.py, include/mbrl.h) refuse -- all of it is decided on the host, before any
launch -- and how the strategy and its optimiser reach them."""
import copy
import ctypes as C
import math

import pytest
import torch

import mbrl_amd  # noqa: F401
from mbrl_amd import lib, optim
from mbrl_amd.strategies import VariationalOptimization, build_optimizer
from test_strategy_host import cfg_vo, fake_agent

Z = torch.zeros


def test_no_cpu_path():
    for call in (lambda: optim.grad_norm([Z(3)]), lambda: optim.clip_grad_norm_([Z(3)], 1.0),
                 lambda: optim.adam_step([Z(3)], [Z(3)], [Z(3)], [Z(3)], [Z(())], 1e-3)):
        with pytest.raises(lib.MbrlError, match="no CPU path"):
            call()
    if not torch.cuda.is_available():
        with pytest.raises(lib.MbrlError, match="no GPU"):
            optim.grad_norm([])


@pytest.mark.parametrize("call,error,text", [
    (lambda: optim.grad_norm(Z(3)), TypeError, "a list"),
    (lambda: optim.grad_norm(7), TypeError, "iterable"),
    (lambda: optim.grad_norm([Z(3), None]), TypeError, "element 1 is not a tensor"),
    (lambda: optim.grad_norm([Z(3)], 3.0), ValueError, "norm_type"),
    (lambda: optim.grad_norm([Z(3)], -math.inf), ValueError, "norm_type"),
    (lambda: optim.grad_norm([Z(3)], math.nan), ValueError, "norm_type"),
    (lambda: optim.grad_norm([Z(3)], "x"), TypeError, "real number"),
    (lambda: optim.grad_norm([Z(3, dtype=torch.int32)]), ValueError, "float64, float32"),
    (lambda: optim.grad_norm([Z(3, dtype=torch.complex64)]), ValueError, "float64, float32"),
    (lambda: optim.grad_norm([Z(3).to_sparse()]), ValueError, "strided"),
    (lambda: optim.grad_norm([Z(4, 6)[:, :3]]), ValueError, "gaps"),
    (lambda: optim.grad_norm([Z(1).expand(5)]), ValueError, "repeated"),
    (lambda: optim.grad_norm([torch._neg_view(Z(3))]), ValueError, "negated"),
    (lambda: optim.clip_grad_norm_(Z(3), 1.0, error_if_nonfinite=True), TypeError, "a list"),
    (lambda: optim.clip_grad_norm_([Z(3)], -1.0), ValueError, "max_norm"),
    (lambda: optim.clip_grad_norm_([Z(3)], math.nan), ValueError, "max_norm"),
    (lambda: optim.clip_grad_norm_([Z(8)[::2]], 1.0), ValueError, "gaps"),
])
def test_refused_lists(call, error, text):
    with pytest.raises(error, match=text):
        call()


def _adam(**over):
    a = dict(params=[Z(4, 6)], grads=[Z(4, 6)], exp_avgs=[Z(4, 6)], exp_avg_sqs=[Z(4, 6)], steps=[Z(())], lr=1e-3)
    a.update(over)
    return optim.adam_step(**a)


@pytest.mark.parametrize("over,error,text", [
    (dict(grads=[]), ValueError, "grads: not as many"),
    (dict(steps=[Z(()), Z(())]), ValueError, "steps: not as many"),
    (dict(grads=[Z(6, 4)]), ValueError, "grads: element 0 has another shape"),
    (dict(grads=[Z(6, 4).t()]), ValueError, "another order"),
    (dict(grads=[Z(4, 6, dtype=torch.bfloat16)]), ValueError, "another type"),
    (dict(exp_avgs=[Z(4, 6, dtype=torch.float64)]), ValueError, "exp_avgs: element 0 is not float32"),
    (dict(params=[Z(4, 6).half()], grads=[Z(4, 6).half()], exp_avg_sqs=[Z(4, 6).half()]), ValueError, "exp_avg_sqs: element 0 is not float32"),
    (dict(steps=[Z((), dtype=torch.int64)]), ValueError, "one float32 value"),
    (dict(steps=[Z(2)]), ValueError, "one float32 value"),
    (dict(lr=-1.0), ValueError, "lr must be finite"),
    (dict(lr=math.inf), ValueError, "lr must be finite"),
    (dict(lr=[1e-3, 1e-3]), ValueError, "lr: one number"),
    (dict(weight_decay=[]), ValueError, "weight_decay: one number"),
    (dict(weight_decay=math.nan), ValueError, "weight_decay must be finite"),
    (dict(max_norm=-0.5), ValueError, "max_norm"),
    (dict(max_norm=1.0, norm_type=0.5), ValueError, "norm_type"),
    (dict(exp_avgs=[Z(8, 6)[::2]]), ValueError, "gaps"),
])
def test_refused_adam_steps(over, error, text):
    with pytest.raises(error, match=text):
        _adam(**over)


def test_a_list_of_rates_that_changes_while_it_is_read():
    class Shrinks:
        def __float__(self):
            rates.clear()
            return 1e-3
    rates = [Shrinks()] + [1e-3] * 63
    n = len(rates)
    with pytest.raises(lib.MbrlError, match="no CPU path"):
        optim.adam_step(*([Z(2) for _ in range(n)] for _ in range(4)), [Z(()) for _ in range(n)], rates)


def _arrays(ptrs, numel, dtype):
    n = len(ptrs)
    return n, (C.c_void_p * n)(*ptrs), (C.c_int64 * n)(*numel), (C.c_int * n)(*dtype)


def test_abi_refusals():
    """Addresses here are numbers that nothing follows: every call is refused before a launch."""
    L = lib.load()
    ws, norm = C.c_void_p(0x1000), C.c_void_p(0x8000)
    need = lambda op, l: L.mbrl_optim_workspace_bytes(op, l[0], l[2], l[3])      # noqa: E731
    long = _arrays([0x1000000 * (i + 1) for i in range(3)], [100000] * 3, [1] * 3)
    big = need(2, long)
    assert big > 0 and need(0, _arrays([], [], [])) == 0 and need(0, _arrays([1], [16], [1])) == 0
    assert need(2, _arrays([0] * 500, [1 << 20] * 500, [2] * 500)) > big
    assert need(3, long) == -7 and L.mbrl_optim_workspace_bytes(0, -1, None, None) == -6 and L.mbrl_optim_workspace_bytes(0, 2, None, None) == -1
    clip = lambda l, most=1.0, kind=2, w=ws, b=big, out=norm: L.mbrl_clip_grad_norm(*l, kind, most, w, b, out, None)   # noqa: E731
    good = _arrays([0x10000, 0x20000], [16, 16], [1, 1])
    assert clip(good, kind=3) == -7 and b"norm type" in L.mbrl_last_error()
    assert clip(good, most=-1.0) == -7 and clip(good, most=math.nan) == -7
    assert clip(long, b=need(1, long) - 1) == -8 and b"workspace" in L.mbrl_last_error()
    assert clip(long, w=None) == -1 and clip(good, out=None) == -1
    assert clip(_arrays([0x10000, None], [16, 16], [1, 1])) == -1
    assert clip(_arrays([0x10000], [-1], [1])) == -6 and clip(_arrays([0x10000], [1 << 41], [1])) == -6
    assert clip(_arrays([0x10000], [16], [4])) == -7 and clip(_arrays([0x10000], [16], [-1])) == -7
    # shared memory: the same tensor twice, an overlap of one value, one tensor inside another
    for ptrs, numel in (([0x10000, 0x10000], [16, 16]), ([0x10000, 0x1003c], [16, 16]), ([0x10000, 0x10010], [16, 1])):
        assert clip(_arrays(ptrs, numel, [1, 1])) == -7 and b"share memory" in L.mbrl_last_error()
        assert clip(_arrays(ptrs[::-1], numel[::-1], [1, 1])) == -7
    one, f64 = (C.c_int64 * 1)(16), (C.c_double * 1)(0.0)
    p = lambda a: (C.c_void_p * 1)(a)      # noqa: E731

    def adam(params=0x10000, grads=0x20000, avgs=0x30000, sqs=0x40000, steps=0x50000, b1=0.9, b2=0.999, eps=1e-8, bytes_=big):
        return L.mbrl_adam_step(1, p(params), p(grads), p(avgs), p(sqs), p(steps), one, (C.c_int * 1)(1), f64, f64, b1, b2, eps, 0, 2,
                                1.0, ws, bytes_, None, None)
    assert adam(b1=1.0) == -7 and adam(b2=-0.1) == -7 and adam(b1=math.nan) == -7 and adam(eps=-1.0) == -7
    assert adam(steps=None) == -1 and adam(grads=None) == -1
    for over in (dict(avgs=0x10000), dict(sqs=0x30000), dict(grads=0x10020), dict(steps=0x40004)):
        assert adam(**over) == -7 and b"shares memory" in L.mbrl_last_error(), over
    # also in a list too long for the short sort: 70 000 tensors, one pair shared
    n = 70000
    many = _arrays([0x100000 + 64 * ((i * 7919) % n) for i in range(n)], [16] * n, [1] * n)
    many[1][n - 1] = many[1][0]
    assert clip(many, b=need(1, many)) == -7 and b"share memory" in L.mbrl_last_error()
    # gradients are only read: two parameters may have the same one, and the norm may count a tensor twice
    assert L.mbrl_grad_norm(*good, 5, ws, big, norm, None) == -7


def test_abi_refuses_what_is_no_device_address():
    L = lib.load()
    ws, norm, at = C.c_void_p(0x1000), C.c_void_p(0x8000), 1 << 48
    l = _arrays([0x10000, at], [16, 16], [1, 1])
    assert L.mbrl_grad_norm(*l, 2, ws, 1 << 20, norm, None) == -1 and b"address" in L.mbrl_last_error()
    assert L.mbrl_clip_grad_norm(*l, 2, 1.0, ws, 1 << 20, norm, None) == -1
    good = [0x10000, 0x20000, 0x30000, 0x40000]
    f64, step = (C.c_double * 1)(0.0), (C.c_void_p * 1)(0x50000)
    for i in range(4):
        ptrs = [(C.c_void_p * 1)(at if k == i else p) for k, p in enumerate(good)]
        assert L.mbrl_adam_step(1, *ptrs, step, (C.c_int64 * 1)(16), (C.c_int * 1)(1), f64, f64, 0.9, 0.999, 1e-8, 0, 2, 1.0, ws, 1 << 20,
                                None, None) == -1 and b"address" in L.mbrl_last_error()


def test_fused_adam_construction_and_state_dict():
    p = [torch.nn.Parameter(Z(3)), torch.nn.Parameter(Z(2, 2, dtype=torch.bfloat16))]
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(max_norm=-1.0), dict(norm_type=3)):
        with pytest.raises(ValueError):
            optim.FusedAdam(p, **bad)
    opt = optim.FusedAdam([{"params": [p[0]], "lr": 0.1}, {"params": [p[1]], "betas": (0.5, 0.9)}])
    with pytest.raises(ValueError, match="betas has to be the same"):
        opt.step()
    opt = optim.FusedAdam(p, 0.1)
    opt.step()                                   # no gradients: nothing to do, as torch's optimisers
    assert not opt.state and opt.grad_norm is None
    p[0].grad = Z(3)
    with pytest.raises(lib.MbrlError, match="no CPU path"):
        opt.step()
    # torch's Adam writes its state; float32 moments of a bfloat16 parameter survive loading
    state = {i: {"step": torch.tensor(7.0), "exp_avg": torch.full_like(q, 1 / 3, dtype=torch.float32),
                 "exp_avg_sq": torch.full_like(q, 1 / 7, dtype=torch.float32)} for i, q in enumerate(p)}
    ref = torch.optim.Adam(p, 0.25, betas=(0.8, 0.95))
    opt.load_state_dict({"state": state, "param_groups": ref.state_dict()["param_groups"]})
    assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["betas"] == (0.8, 0.95)
    for q in p:
        assert opt.state[q]["exp_avg"].dtype == torch.float32 and float(opt.state[q]["step"]) == 7.0
        assert torch.equal(opt.state[q]["exp_avg_sq"], torch.full_like(q, 1 / 7, dtype=torch.float32))
    again = optim.FusedAdam(p, 0.1)
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state[p[1]]["exp_avg"], opt.state[p[1]]["exp_avg"])
    ref.load_state_dict(opt.state_dict())        # and back
    assert float(ref.state[p[0]]["step"]) == 7.0
    twin = copy.deepcopy(optim.FusedAdam(p, 0.1, max_norm=3.0, norm_type=1))
    assert (twin.max_norm, twin.norm_type, twin.grad_norm) == (3.0, 1, None)
    opt.state[p[0]].clear()
    opt.state[p[0]]["mine"] = 1                  # another's entry does not pass for the state
    with pytest.raises(lib.MbrlError, match="no CPU path"):
        opt.step()
    assert float(opt.state[p[0]]["step"]) == 0.0 and opt.state[p[0]]["mine"] == 1
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(torch.optim.Adam(p, amsgrad=True).state_dict())


def test_build_optimizer_and_default_keys():
    cfg = cfg_vo()
    assert cfg.SOLVER.CLIP_GRAD_NORM == 0.0 and cfg.SOLVER.FUSED is False
    named = [("mean", torch.nn.Parameter(Z(2))), ("sd", torch.nn.Parameter(Z(2)))]
    assert type(build_optimizer(cfg, named)) is torch.optim.Adam
    cfg.merge_from_list(["SOLVER.FUSED", "True", "SOLVER.CLIP_GRAD_NORM", "2.5", "SOLVER.STD_LR_FACTOR", "0.5"])
    opt = build_optimizer(cfg, named)
    assert type(opt) is optim.FusedAdam and opt.max_norm == 2.5
    assert [g["lr"] for g in opt.param_groups] == [cfg.SOLVER.BASE_LR, 0.5 * cfg.SOLVER.BASE_LR]
    cfg.SOLVER.OPTIMIZER = "sgd"
    with pytest.raises(ValueError, match="FUSED"):
        build_optimizer(cfg, named)


@pytest.mark.parametrize("solver", ["adam", "sgd"])
def test_strategy_clips_the_summed_gradient_before_the_step(solver, monkeypatch):
    """Order of one optimisation step: backward, sum over ranks, clip by the global norm, update."""
    calls = []

    def clip(grads, max_norm):
        calls.append("clip")
        norm = torch.sqrt(sum(g.double().square().sum() for g in grads))
        for g in grads:
            g.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))
        return norm
    monkeypatch.setattr(optim, "clip_grad_norm_", clip)
    cfg = cfg_vo()
    cfg.SOLVER.OPTIMIZER, cfg.SOLVER.CLIP_GRAD_NORM, cfg.SOLVER.BASE_LR = solver, 0.25, 0.5
    pol = VariationalOptimization(cfg, fake_agent())
    before = [p.detach().clone() for p in pol.parameters()]
    loss = (pol.mean.sum() * 3.0).expand(4, 5) + 0 * pol.sd.sum()

    def sync(grads):
        calls.append("sync")
        assert float(grads[0].abs().max()) > 1.0           # not clipped yet
    stats = pol.optimize(loss, grad_sync=sync)
    assert calls == ["sync", "clip"]
    g = 3.0 * 5                                            # of every entry of the mean: 5 steps, batch mean
    assert stats["grad_norm"] == pytest.approx(g * math.sqrt(5))
    if solver == "sgd":
        want = before[0] - 0.5 * 0.25 * torch.ones_like(before[0]) / math.sqrt(5)
        assert torch.allclose(pol.mean.detach(), want, rtol=0, atol=1e-6)
    calls.clear()
    monkeypatch.undo()
    cfg.SOLVER.CLIP_GRAD_NORM = -1.0
    with pytest.raises(ValueError, match="max_norm"):
        pol.optimize((pol.mean.sum() * 3.0).expand(4, 5) + 0 * pol.sd.sum())
    cfg.SOLVER.CLIP_GRAD_NORM = 0.0
    assert "grad_norm" not in pol.optimize((pol.mean.sum() * 3.0).expand(4, 5) + 0 * pol.sd.sum()) and not calls
