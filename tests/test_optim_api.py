"""CPU: what the optimiser-step operators refuse of autograd's, and FusedAdam beside torch's optimisers where no kernel is needed."""
import pytest
import torch

import mbrl_amd  # noqa: F401
from mbrl_amd import lib, optim

Z = torch.zeros


def test_the_norm_refuses_what_autograd_would_record():
    """A loss with the norm of gradients in it would lose that term without a word."""
    w = torch.ones(3, requires_grad=True)
    g, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    for x in (w, g, w[1:], w.view(1, 3)):
        with pytest.raises(ValueError, match="grads: element 1 requires grad"):
            optim.grad_norm([Z(2), x])
        for call in (lambda: optim.grad_norm([x.detach()]), lambda: _no_grad(lambda: optim.grad_norm([x])),
                     # changed in place, outside autograd, as torch's own clipping
                     lambda: optim.clip_grad_norm_([x], 1.0), lambda: optim.clip_grad_norm_([x], 1.0, error_if_nonfinite=True)):
            with pytest.raises(lib.MbrlError, match="no CPU path"):        # as far as a CPU tensor gets
                call()


def _no_grad(f):
    with torch.no_grad():
        return f()


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        x = fwd.make_dual(torch.ones(4), torch.ones(4))
        for dual in (x, 2 * x, x[1:], x.view(2, 2)):
            same = lambda: Z(dual.shape)      # noqa: E731
            for call in (lambda: optim.grad_norm([dual]), lambda: optim.clip_grad_norm_([dual], 1.0),
                         lambda: optim.adam_step([same()], [dual], [same()], [same()], [Z(())], 1e-3),
                         lambda: optim.adam_step([dual], [same()], [same()], [same()], [Z(())], 1e-3)):
                with pytest.raises(ValueError, match="forward-mode tangent"):
                    call()
    with pytest.raises(lib.MbrlError, match="no CPU path"):
        optim.grad_norm([torch.ones(4)])


def test_the_norm_of_a_step_without_gradients(monkeypatch):
    """Not the norm of an earlier step."""
    p = torch.nn.Parameter(Z(3))
    monkeypatch.setattr(optim, "adam_step", lambda *a: None if a[10] is None else torch.tensor(5.0, dtype=torch.float64))
    opt = optim.FusedAdam([p], 0.1, max_norm=1.0)
    opt.step()
    assert float(opt.grad_norm) == 0.0 and opt.grad_norm.dtype == torch.float64 and opt.grad_norm.shape == ()
    p.grad = torch.ones(3)
    opt.step()
    assert float(opt.grad_norm) == 5.0
    opt.zero_grad()
    opt.step()
    assert float(opt.grad_norm) == 0.0
    p.grad, opt.max_norm = torch.ones(3), None
    opt.step()
    assert opt.grad_norm is None
    opt.grad_norm = torch.tensor(5.0)
    opt.zero_grad()
    opt.step()
    assert opt.grad_norm is None


def _state(p, value):
    return {"step": torch.tensor(7.0), "exp_avg": torch.full_like(p, value, dtype=torch.float32),
            "exp_avg_sq": torch.full_like(p, value * value, dtype=torch.float32)}


def test_hooks_of_loading_count():
    """What a hook makes of the dict is what is loaded, and a hook behind sees, and may change, what stays."""
    p = torch.nn.Parameter(Z(4, dtype=torch.bfloat16))
    opt = optim.FusedAdam([p], 0.1)
    saved = {"state": {0: _state(p, 0.1)}, "param_groups": opt.state_dict()["param_groups"]}

    def other_moments(_, sd):
        return dict(sd, state={0: _state(p, 0.3)})
    seen = []

    def behind(o):
        seen.append(o.state[p]["exp_avg"].clone())
        o.state[p]["exp_avg_sq"].fill_(2.0)
    handles = [opt.register_load_state_dict_pre_hook(other_moments), opt.register_load_state_dict_post_hook(behind)]
    for _ in range(2):
        opt.load_state_dict(saved)
        want = torch.full((4,), 0.3)
        assert seen[-1].dtype == torch.float32 and torch.equal(seen[-1], want) and torch.equal(opt.state[p]["exp_avg"], want)
        assert bool((opt.state[p]["exp_avg_sq"] == 2.0).all())
    for h in handles:
        h.remove()
    opt.load_state_dict(saved)
    assert torch.equal(opt.state[p]["exp_avg"], torch.full((4,), 0.1)) and len(seen) == 2

    def plain(_, sd):        # a hook may take out what is not offered
        return dict(sd, param_groups=[dict(g, amsgrad=False) for g in sd["param_groups"]])
    ams = dict(saved, param_groups=[dict(g, amsgrad=True) for g in saved["param_groups"]])
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(ams)
    opt.register_load_state_dict_pre_hook(plain)
    opt.load_state_dict(ams)


def test_moments_of_another_shape_are_refused():
    p = torch.nn.Parameter(Z(4, 6))
    opt = optim.FusedAdam([p], 0.1)
    opt.load_state_dict({"state": {0: _state(p, 0.1)}, "param_groups": opt.state_dict()["param_groups"]})
    for shape in ((6,), (1,), (4, 1), (24,), (1, 4, 6)):
        wrong = {"state": {0: _state(Z(shape), 0.2)}, "param_groups": opt.state_dict()["param_groups"]}
        wrong["param_groups"][0]["lr"] = 9.0
        with pytest.raises(ValueError, match="another shape"):
            opt.load_state_dict(wrong)
        assert opt.param_groups[0]["lr"] == 0.1 and torch.equal(opt.state[p]["exp_avg"], torch.full((4, 6), 0.1))
    with pytest.raises(ValueError):                    # as the base class: another number of parameters
        opt.load_state_dict({"state": {}, "param_groups": [dict(opt.state_dict()["param_groups"][0], params=[0, 1])]})


@pytest.mark.parametrize("key,value", [("maximize", True), ("amsgrad", True), ("max_norm", 1.0), ("norm_type", 1)])
def test_groups_with_options_that_would_not_be_followed(key, value):
    """A group that asks to maximise must not be minimised."""
    p, q = torch.nn.Parameter(Z(2)), torch.nn.Parameter(Z(2))
    with pytest.raises(ValueError, match=key):
        optim.FusedAdam([{"params": [p], key: value}], 0.1)
    opt = optim.FusedAdam([p], 0.1)
    with pytest.raises(ValueError, match=key):
        opt.add_param_group({"params": [q], key: value})
    with pytest.raises(TypeError):
        opt.add_param_group([q])                       # as the base class
    opt.add_param_group({"params": [q], "amsgrad": False, "maximize": False, "name": "second"})
    assert len(opt.param_groups) == 2


def test_the_strategy_clips_by_the_bound_of_the_moment(monkeypatch):
    """SOLVER.CLIP_GRAD_NORM is read at every step, whichever optimiser follows it."""
    from mbrl_amd.strategies import VariationalOptimization
    from test_strategy_host import cfg_vo, fake_agent
    bounds = []

    def adam_step(*a):
        bounds.append(a[10])
        return None if a[10] is None else torch.sqrt(sum(g.double().square().sum() for g in a[1]))
    monkeypatch.setattr(optim, "adam_step", adam_step)
    cfg = cfg_vo()
    cfg.SOLVER.FUSED = True
    pol = VariationalOptimization(cfg, fake_agent())
    loss = lambda: (pol.mean.sum() * 3.0).expand(4, 5) + 0 * pol.sd.sum()      # noqa: E731
    for bound in (0.0, 2.5, 0.5, 0.0):
        cfg.SOLVER.CLIP_GRAD_NORM = bound
        stats = pol.optimize(loss())
        assert bounds[-1] == (bound or None)
        if bound:        # of every entry of the mean 3 over 5 steps, 5 entries
            assert stats["grad_norm"] == pytest.approx(15.0 * 5 ** 0.5)
        else:
            assert "grad_norm" not in stats
