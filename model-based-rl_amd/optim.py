"""Optimiser-step operators over lists of tensors on the HIP device: the global gradient norm, clipping by it, and the Adam
update that takes the clipped gradient (C ABI: include/mbrl.h; kernels: csrc/optim.hip).

The reference bounds gradients value by value and steps torch's Adam over its parameters
(model/blocks/policy/strategies.py:311-364, solver/build.py:4-25).  Gradients that come through finite differences of contact
dynamics can grow with every step of the horizon, and bounding their global norm keeps a direction that bounding values
does not.  `strategies.VariationalOptimization.optimize` calls these under SOLVER.CLIP_GRAD_NORM and SOLVER.FUSED.

All functions take lists of float64 / float32 / bfloat16 / float16 tensors of one GPU (types may be mixed), launch on the
current stream, never wait for the device (but for error_if_nonfinite) and can be captured into a graph.  Tensors have to be
dense -- any order of dimensions, any alignment, no gaps or repeats.  There is no CPU path.  Autograd records none of them:
what is changed in place is changed as under torch.no_grad(), and forward-mode tangents are refused.
"""
import ctypes as C
import importlib.util
import math
import os

import torch

from . import lib

_bind = None


def bind():
    """The host module that turns lists of tensors into the arguments of the C ABI (csrc/optim_bind.so)."""
    global _bind
    if _bind is None:
        path = os.path.join(lib.HERE, "csrc", "optim_bind.so")
        if not os.path.exists(path):
            raise lib.MbrlError("host module not built: %s is missing (run __graft_entry__.build())" % path)
        L = lib.load()
        spec = importlib.util.spec_from_file_location("optim_bind", path)
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        m.connect(lib.MbrlError, *(C.cast(getattr(L, n), C.c_void_p).value for n in
                                   ("mbrl_optim_workspace_bytes", "mbrl_grad_norm", "mbrl_clip_grad_norm", "mbrl_adam_step",
                                    "mbrl_last_error")))
        _bind = m
    return _bind


def grad_norm(grads, norm_type=2.0):
    """Norm over all values of all tensors in `grads` as a 0-d float64 tensor, summed in float64.  norm_type 1, 2 or inf.
    0 for an empty list, NaN if any value is NaN.  The result carries no gradient: tensors that require grad are refused unless
    under torch.no_grad().  The same values in tensors of the same sizes give the same bits wherever they lie, so ranks that
    hold the same gradients find the same norm; the other operators order the sum in their own way, and their norms may
    differ from this one in the last bits."""
    return (_bind or bind()).grad_norm(grads, norm_type)


def clip_grad_norm_(grads, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Multiplies every value of every tensor in `grads` by min(1, max_norm / (norm + 1e-6)), in place, and returns the norm
    as it was (0-d float64).  A factor of 1 (norm + 1e-6 <= max_norm) leaves the values untouched, bit for bit, and
    so does max_norm=inf for every norm that is a number.  A NaN norm makes every value NaN, an infinite one makes finite
    values 0; error_if_nonfinite=True raises RuntimeError before anything is changed instead (it takes the norm once more and
    waits for the device, so not under graph capture).  Tensors that share memory are refused."""
    b = _bind or bind()
    if error_if_nonfinite:
        grads = grads if isinstance(grads, torch.Tensor) else tuple(grads)        # an iterator would be empty the second time
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise ValueError("clip_grad_norm_: error_if_nonfinite waits for the device and cannot be captured into a graph")
        with torch.no_grad():
            norm = float(b.grad_norm(grads, norm_type))
        if not math.isfinite(norm):
            raise RuntimeError("clip_grad_norm_: the norm of the gradients is %r" % norm)
    return b.clip_grad_norm_(grads, max_norm, norm_type)


def adam_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled=False,
              max_norm=None, norm_type=2.0):
    """One Adam step (torch.optim.Adam's arithmetic) of all `params`, in place, in as few launches as the list allows.

    exp_avgs / exp_avg_sqs: float64 for float64 parameters, float32 for all others, shaped and laid out like their
    parameter; steps: one float32 value in device memory each, counted up here; lr, weight_decay: one number or one for
    each tensor; decoupled: weight decay on the parameter (AdamW) instead of on the gradient.  max_norm: the gradients enter
    multiplied as by clip_grad_norm_, but are not written, and 16-bit ones not rounded in between; returns their norm
    (0-d float64) then, else None.
    Memory that is written must not be shared between tensors."""
    return (_bind or bind()).adam_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr, betas[0], betas[1], eps, weight_decay,
                                       decoupled, max_norm, norm_type)


class FusedAdam(torch.optim.Optimizer):
    """torch.optim.Adam's rule as one adam_step over all parameters that have a gradient, with the gradients clipped by their
    global norm on the way (max_norm; None: not).  `grad_norm` holds the norm of the last step (0-d float64; 0 of a step without
    gradients) then, else None.

    lr and weight_decay go by parameter group; betas, eps and decoupled_weight_decay are the same for all groups.  State is
    named and shaped as torch.optim.Adam's (float32 moments for 16-bit parameters), so a state_dict of either loads
    into the other.  The step counts live on the device: a captured step() counts on with every replay (with the learning
    rates of its capture).  The first step of a parameter makes its state and cannot be captured."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, decoupled_weight_decay=False,
                 max_norm=None, norm_type=2.0):
        if not 0.0 <= lr < math.inf:
            raise ValueError("FusedAdam: lr must be finite and not negative, got %r" % (lr,))
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("FusedAdam: betas must be in [0, 1), got %r" % (betas,))
        if not eps >= 0.0:
            raise ValueError("FusedAdam: eps must not be negative, got %r" % (eps,))
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError("FusedAdam: max_norm must not be negative, got %r" % (max_norm,))
        if norm_type not in (1, 2, math.inf):
            raise ValueError("FusedAdam: norm_type has to be 1, 2 or inf, got %r" % (norm_type,))
        self.max_norm, self.norm_type, self.grad_norm = max_norm, norm_type, None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      decoupled_weight_decay=bool(decoupled_weight_decay)))

    def add_param_group(self, param_group):
        keys = param_group if isinstance(param_group, dict) else {}        # the base class refuses what is no dict
        for k in ("amsgrad", "maximize"):
            if keys.get(k):
                raise ValueError("FusedAdam: %s is not offered" % k)
        for k in ("max_norm", "norm_type"):
            if k in keys:
                raise ValueError("FusedAdam: %s is the optimiser's, not a parameter group's" % k)
        super().add_param_group(param_group)

    def _common(self):
        first = self.param_groups[0]
        for g in self.param_groups:
            for k in ("betas", "eps", "decoupled_weight_decay"):
                if g[k] is not first[k] and g[k] != first[k]:
                    raise ValueError("FusedAdam: %s has to be the same in all parameter groups" % k)
        return first

    def _new_state(self, p):
        s = self.state[p]
        wide = torch.float64 if p.dtype == torch.float64 else torch.float32
        s["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
        for k in ("exp_avg", "exp_avg_sq"):
            s[k] = torch.zeros_like(p, dtype=wide, memory_format=torch.preserve_format)
        return s

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        first, state = self._common(), self.state
        params, grads, avgs, sqs, steps, lr, wd = [], [], [], [], [], [], []
        for group in self.param_groups:
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                s = state[p]
                if "exp_avg" not in s:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("FusedAdam: take a first step before it is captured into a graph (a replay would zero "
                                           "the state that it makes)")
                    self._new_state(p)
                params.append(p)
                grads.append(g)
                avgs.append(s["exp_avg"])
                sqs.append(s["exp_avg_sq"])
                steps.append(s["step"])
                lr.append(group["lr"])
                wd.append(group["weight_decay"])
        if params:
            self.grad_norm = adam_step(params, grads, avgs, sqs, steps, lr, first["betas"], first["eps"], wd,
                                       first["decoupled_weight_decay"], self.max_norm, self.norm_type)
        elif self.max_norm is None:
            self.grad_norm = None
        else:        # of no gradients, as clip_grad_norm_([])
            device = next((p.device for group in self.param_groups for p in group["params"]), None)
            self.grad_norm = torch.zeros((), dtype=torch.float64, device=device)
        return loss

    def __getstate__(self):        # for copies and pickles; the base class keeps its own three attributes only
        return dict(super().__getstate__(), max_norm=self.max_norm, norm_type=self.norm_type, grad_norm=None)

    def load_state_dict(self, state_dict):
        """As Optimizer.load_state_dict, its hooks too, but moments keep their float32 (or float64) values: the base class
        rounds them to their parameter's type.  Moments of another shape than their parameter are refused before
        anything is changed."""
        ids, loaded = [], {}

        def before(_, state_dict):        # last of its kind: sees what the other hooks made of the dict
            if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]) or \
                    any("max_exp_avg_sq" in s for s in state_dict["state"].values()):
                raise ValueError("FusedAdam: amsgrad and maximize are not offered")
            ids.extend(i for g in state_dict["param_groups"] for i in g["params"])
            for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
                saved = state_dict["state"].get(i)
                if not saved or "exp_avg" not in saved:
                    continue
                for k in ("exp_avg", "exp_avg_sq"):
                    if saved[k].shape != p.shape:
                        raise ValueError("FusedAdam: %s of parameter %r has another shape than it" % (k, i))
                loaded[i] = saved

        def after(_):                     # first of its kind: the others see the moments as they stay
            for g in self.param_groups:
                g.setdefault("decoupled_weight_decay", self.defaults["decoupled_weight_decay"])
            for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
                if i not in loaded:
                    continue
                s = self._new_state(p)
                s["step"].copy_(torch.as_tensor(loaded[i]["step"], dtype=torch.float32))
                for k in ("exp_avg", "exp_avg_sq"):
                    s[k].copy_(loaded[i][k])

        hooks = [self.register_load_state_dict_pre_hook(before), self.register_load_state_dict_post_hook(after, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()
