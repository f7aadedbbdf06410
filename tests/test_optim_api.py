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
