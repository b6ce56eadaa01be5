"""tf.keras.optimizers.legacy.Adam, AdamW and ExponentialDecay, as one launch over a model's flat buffers.

Reference: ``build_optimizer`` run_model.py:77-89, run_unet.py:48-66, run_context_encoder.py:144-162.
The update is the Keras (legacy / ResourceApplyAdam) form, not torch's: epsilon 1e-7 sits outside the
square root and the bias correction is folded into the step size,
``alpha = lr * sqrt(1 - b2^t) / (1 - b1^t)``, ``theta -= alpha * m / (sqrt(v) + eps)``.
The update counter and the decayed learning rate live on the device, so a HIP graph that contains the
step replays the schedule by itself.
"""
from __future__ import annotations

import math
from typing import Dict, Iterable, Optional, Tuple

import torch

from . import ops


class ExponentialDecay:
    """tf.keras.optimizers.schedules.ExponentialDecay."""

    def __init__(self, initial_learning_rate, decay_steps, decay_rate, staircase=False):
        if decay_steps <= 0:
            raise ValueError("decay_steps must be positive")
        self.initial_learning_rate = float(initial_learning_rate)
        self.decay_steps = int(decay_steps)
        self.decay_rate = float(decay_rate)
        self.staircase = bool(staircase)

    def __call__(self, step: int) -> float:
        p = step / self.decay_steps
        if self.staircase:
            p = math.floor(p)
        return self.initial_learning_rate * self.decay_rate ** p


class Adam:
    takes_slabs = True  # apply_model can sum kernel gradients that are still slabs of partial sums

    def __init__(self, learning_rate=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-7):
        if isinstance(learning_rate, ExponentialDecay):
            self.schedule: Optional[ExponentialDecay] = learning_rate
            self.lr0 = learning_rate.initial_learning_rate
        else:
            self.schedule = None
            self.lr0 = float(learning_rate)
        self.beta_1, self.beta_2, self.epsilon = float(beta_1), float(beta_2), float(epsilon)
        self._state: Optional[torch.Tensor] = None  # int64[3] on the device: update count, {alpha, lr}, arrival counter
        self._slots: Dict[int, Tuple[torch.Tensor, torch.Tensor]] = {}
        self._slots_of: Dict[int, torch.Tensor] = {}  # the parameters that the slots belong to

    # ---- device state
    def _ensure_state(self, device):
        if self._state is None:
            self._state = torch.zeros(3, dtype=torch.int64, device=device)
        return self._state

    def _slots_for(self, model):
        key = id(model)
        if key not in self._slots or self._slots_of[key] is not model._params:  # an id is given out again once its model is gone
            self._slots[key], self._slots_of[key] = self._zero_slots(model), model._params
        return self._slots[key]

    def _zero_slots(self, model):
        return torch.zeros_like(model._params), torch.zeros_like(model._params)

    @property
    def iterations(self) -> int:
        return 0 if self._state is None else int(self._state[0].item())

    def current_lr(self) -> float:
        it = self.iterations
        return self.schedule(it) if self.schedule is not None else self.lr0

    def _prepare(self, device):
        st = self._ensure_state(device)
        sc = self.schedule
        ops.adam_prepare(st, self.lr0, self.beta_1, self.beta_2, sc.decay_steps if sc else 0,
                         sc.decay_rate if sc else 1.0, sc.staircase if sc else False)
        return st

    def prepare(self, device):
        """Advance the update counter and refresh the step size on the current stream; the matching
        ``apply_model(..., prepared=True)`` then only runs the parameter update."""
        self._prepare(device)

    # ---- the fused path: one launch over the model's whole flat parameter buffer
    def apply_model(self, model, grad_scale: float = 1.0, prepared: bool = False, zero_grads: bool = False, fold=None,
                    slabs=None):
        """``zero_grads``: the launch also clears the model's gradient buffer (training loops whose next backward
        accumulates into it), which saves the separate fill of the next step.  ``fold``: a pending scalar fold
        ``(partials, n, scale, out, running, running_weight)`` (the loss of a forward launch that left per-workgroup
        sums) carried by the same launch.  ``slabs``: kernel / bias gradients still lying as slabs of partial sums
        (``ops.conv2d_wgrad_batch_slabs``); the one-launch form sums them on the way in."""
        m, v = self._slots_for(model)
        st = self._ensure_state(model._params.device)
        if slabs is not None and prepared:
            raise ValueError("apply_model: gradient slabs need the one-launch form (prepared=False)")
        if prepared:
            if fold is not None:
                ops.fold_scalar(fold[0], fold[1], fold[2], fold[3], False, fold[4], fold[5])
            ops.adam_apply(model._params, model._grads, m, v, st, self.beta_1, self.beta_2, self.epsilon, grad_scale,
                           zero_grads)
            if model._params_lp is not None:
                model._refresh_lp()  # the convs of a bf16 model read this copy
        else:  # schedule, update and (bf16 models) the refresh of the filter copy in one launch
            sc = self.schedule
            ops.adam_step(model._params, model._grads, m, v, st, self.lr0, self.beta_1, self.beta_2, self.epsilon,
                          sc.decay_steps if sc else 0, sc.decay_rate if sc else 1.0, sc.staircase if sc else False,
                          grad_scale, zero_grads, model._params_lp, fold, slabs)
            model._lp_dirty = False
        model._grads_clean = bool(zero_grads)

    # ---- keras surface: optimizer.apply_gradients(zip(grads, variables))
    def apply_gradients(self, grads_and_vars: Iterable):
        pairs = [(g, v) for g, v in grads_and_vars if g is not None]
        if not pairs:
            return
        owners = {id(v.owner) for _, v in pairs}
        model = pairs[0][1].owner
        if len(owners) == 1 and model is not None:
            tv = model.trainable_variables
            whole = len(pairs) == len(tv) and all(
                v is t and isinstance(g, torch.Tensor) and g.data_ptr() == t.grad.data_ptr() for (g, v), t in zip(pairs, tv))
            if whole:
                self.apply_model(model)
                return
        # general path: one launch per variable, moments sliced out of the owner's flat slot buffers
        st = self._prepare(pairs[0][1].data.device)
        for g, var in pairs:
            m, v = self._slots_for(var.owner)
            sl = slice(var.offset, var.offset + var.size)
            g = g.as_subclass(torch.Tensor).to(dtype=torch.float32).contiguous().view(-1)
            ops.adam_apply(var.data.view(-1), g, m[sl], v[sl], st, self.beta_1, self.beta_2, self.epsilon, 1.0)
            if var.owner is not None:
                var.owner._lp_dirty = True

    # ---- checkpointing (not a reference feature; used by the fixed-seed trajectory tests)
    def state_dict(self) -> dict:
        return {"state": None if self._state is None else self._state.cpu(),
                "slots": {k: (m.cpu(), v.cpu()) for k, (m, v) in self._slots.items()}}


def _apart(grads, written):
    """The gradients, each that shares memory with another one or with a tensor of ``written`` as a copy of its own."""
    spans = [(t.data_ptr(), 0, -1, t) for t in written] + [(g.data_ptr(), 1, i, g) for i, g in enumerate(grads)]
    spans = sorted((s for s in spans if s[3].numel() > 0), key=lambda s: s[:3])
    grads, end, last = list(grads), 0, -1
    for begin, is_grad, i, t in spans:
        if begin < end and is_grad:
            grads[i] = t.clone()
            continue
        if begin < end and last >= 0:  # what is kept so far lies apart: the last one alone can reach this far
            grads[last] = grads[last].clone()
        end, last = max(end, begin + t.numel() * t.element_size()), i
    return grads


class AdamW(Adam):
    """tf.keras.optimizers.AdamW: ``Adam`` with decoupled weight decay, ``theta -= lr * weight_decay * theta`` ahead of the
    update, and optionally the gradients clipped by their global norm.  All variables of a model are one launch
    (``ops.adamw_step``), two with ``global_clipnorm``.

    ``state_bits=8``: both moments are held in 8 bits, in blocks of 256 elements with an exponent byte each (2.01 instead of
    8 bytes per weight), rounded by random bits of a generator seeded with ``seed``; ``moments`` gives their values."""

    takes_slabs = False

    def __init__(self, learning_rate=1e-3, weight_decay=4e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-7, global_clipnorm=None,
                 state_bits=32, seed=1833):
        super().__init__(learning_rate, beta_1, beta_2, epsilon)
        if weight_decay < 0:
            raise ValueError("weight_decay must not be negative")
        if epsilon < 1e-12:
            raise ValueError("epsilon must be at least 1e-12")
        if global_clipnorm is not None and global_clipnorm <= 0:
            raise ValueError("global_clipnorm must be positive")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits!r}")
        self.weight_decay = float(weight_decay)
        self.global_clipnorm = None if global_clipnorm is None else float(global_clipnorm)
        self.state_bits, self.seed = int(state_bits), int(seed)
        self._excluded, self._excluded_names = (), ()
        self._plans: Dict[int, tuple] = {}  # id(model) -> (model, plan)

    def exclude_from_weight_decay(self, var_list=None, var_names=None):
        """Variables (or all whose name contains one of ``var_names``) that are updated without weight decay.  To be called
        before the first step."""
        if self._plans:
            raise ValueError("exclude_from_weight_decay must be called before the first step")
        self._excluded = tuple(var_list or ())
        self._excluded_names = tuple(var_names or ())

    def _decay_of(self, var) -> float:
        out = any(var is v for v in self._excluded) or any(n in var.name for n in self._excluded_names)
        return 0.0 if out else self.weight_decay

    # ---- moments: flat over a model's variables; in 8 bits every variable starts on a block of its own
    def _zero_slots(self, model):
        if self.state_bits == 32:
            return super()._zero_slots(model)
        blocks = sum(-(-v.size // ops.ADAMW_BLOCK) for v in model.trainable_variables)
        zeros = lambda n: torch.zeros(n, dtype=torch.uint8, device=model._params.device)  # noqa: E731
        return zeros(blocks * ops.ADAMW_BLOCK), zeros(blocks * ops.ADAMW_BLOCK), zeros(blocks), zeros(blocks)

    def _moments_of(self, var):
        """(m, v, m_exp, v_exp) of one variable; the exponents are None with 32-bit moments."""
        s = self._slots_for(var.owner)
        if self.state_bits == 32:
            sl = slice(var.offset, var.offset + var.size)
            return s[0][sl], s[1][sl], None, None
        block = 0
        for v in var.owner.trainable_variables:
            if v is var:
                break
            block += -(-v.size // ops.ADAMW_BLOCK)
        sl = slice(block * ops.ADAMW_BLOCK, block * ops.ADAMW_BLOCK + var.size)
        be = slice(block, block - (-var.size // ops.ADAMW_BLOCK))
        return s[0][sl], s[1][sl], s[2][be], s[3][be]

    def moments(self, var):
        """float32 copies of a variable's two moments."""
        m, v, m_exp, v_exp = self._moments_of(var)
        if m_exp is None:
            return m.view(var.shape).clone(), v.view(var.shape).clone()
        out = [torch.empty(var.shape, dtype=torch.float32, device=m.device) for _ in range(2)]
        ops.adamw_decode(m, m_exp, out[0], False)
        ops.adamw_decode(v, v_exp, out[1], True)
        return out[0], out[1]

    def _plan(self, variables, grads, copies: bool):
        mom = [self._moments_of(v) for v in variables]
        eight = self.state_bits == 8
        return ops.AdamWPlan([v.data.view(-1) for v in variables], grads, [s[0] for s in mom], [s[1] for s in mom],
                             [self._decay_of(v) for v in variables], m_exp=[s[2] for s in mom] if eight else None,
                             v_exp=[s[3] for s in mom] if eight else None,
                             params_lp=[v.data_lp.view(-1) for v in variables] if copies else None)

    def _step(self, plan, device, grad_scale, zero_grads=False):
        sc = self.schedule
        ops.adamw_step(plan, self._ensure_state(device), self.lr0, self.beta_1, self.beta_2, self.epsilon,
                       sc.decay_steps if sc else 0, sc.decay_rate if sc else 1.0, sc.staircase if sc else False, grad_scale,
                       self.global_clipnorm or 0.0, self.seed, zero_grads)

    def prepare(self, device):
        """Nothing to do ahead: the update launch advances the count and derives the step size itself."""
        self._ensure_state(device)

    def apply_model(self, model, grad_scale: float = 1.0, prepared: bool = False, zero_grads: bool = False, fold=None,
                    slabs=None):
        """``Adam.apply_model``, except that gradient slabs are refused (``takes_slabs``)."""
        if slabs is not None:
            raise ValueError("apply_model: AdamW takes summed gradients, not slabs")
        entry = self._plans.get(id(model))
        if entry is None:
            tv = model.trainable_variables
            entry = self._plans[id(model)] = (model, self._plan(tv, [v.grad.view(-1) for v in tv], model._params_lp is not None))
        if fold is not None:
            ops.fold_scalar(fold[0], fold[1], fold[2], fold[3], False, fold[4], fold[5])
        self._step(entry[1], model._params.device, grad_scale, zero_grads)
        model._lp_dirty = False
        model._grads_clean = bool(zero_grads)

    def apply_gradients(self, grads_and_vars: Iterable):
        pairs = [(g, v) for g, v in grads_and_vars if g is not None]
        if not pairs:
            return
        if len({id(v) for _, v in pairs}) != len(pairs):
            raise ValueError("apply_gradients: a variable appears twice")
        tv = pairs[0][1].owner.trainable_variables
        if len(pairs) == len(tv) and all(v is t and isinstance(g, torch.Tensor) and g.data_ptr() == t.grad.data_ptr()
                                         for (g, v), t in zip(pairs, tv)):
            self.apply_model(pairs[0][1].owner)
            return
        # some variables, or gradients of the caller's, which are only read and may share memory: a plan for this call
        grads = []
        for g, v in pairs:
            g = g.as_subclass(torch.Tensor).to(device=v.data.device, dtype=torch.float32).contiguous().view(-1)
            if g.numel() != v.size:
                raise ValueError(f"apply_gradients: gradient of {v.name} has {g.numel()} elements, not {v.size}")
            grads.append(g)
        variables = [v for _, v in pairs]
        owners = {id(v.owner): v.owner for v in variables}.values()
        grads = _apart(grads, [t for m in owners for t in (m._params, *self._slots_for(m))])
        self._step(self._plan(variables, grads, False), variables[0].data.device, 1.0)
        for v in variables:
            v.owner._lp_dirty = True

    def state_dict(self) -> dict:
        return {"state": None if self._state is None else self._state.cpu(),
                "slots": {k: tuple(t.cpu() for t in s) for k, s in self._slots.items()}}


def legacy_adam(learning_rate=1e-3, beta_1=0.9, beta_2=0.999, epsilon=1e-7) -> Adam:
    return Adam(learning_rate, beta_1, beta_2, epsilon)
