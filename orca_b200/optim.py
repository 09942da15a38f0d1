"""AdamW over all parameters at once, moments in 32 or in 8 bits, gradients cut to a norm over all of them: the optimiser of a training step on
trained rows (the reference trains with PyTorch's Adam, train.py, which is AdamW without weight decay)."""
from __future__ import annotations

import copy

import torch

from . import _lib

BLOCK = 256      # elements of a tensor that share the exponents of their moments in 8 bits


class AdamW(torch.optim.Optimizer):
    """AdamW (I. Loshchilov, F. Hutter, 2019) for dense parameters in fp32, bf16 or fp16 on one CUDA device, in one launch for those of a type; an
    optimiser as PyTorch's are, with groups, schedulers and state dicts.

    params, lr, betas, eps, weight_decay   of all or of a group; lr may be one fp32 value on the device, which a captured step reads at every
              replay; with an eps of 0 an element that has had no gradient, or one whose square is nothing in fp32, does not stay finite
    max_norm  gradients are scaled to a norm over all parameters of at most this (inf: the norm is taken, nothing is scaled); ``grad_norm``
              has the norm of the last step then, on the device.  A step whose norm is not finite changes nothing.
    bits      32: moments in fp32, eight bytes an element.  8: a byte each, and two for 256 elements (include/orca_b200.h has the format); what a
              moment loses to 8 bits is rounded up or down by chance that follows from step and place, so that it is right on average.  A block
              of 256 whose moment is not finite is NaN altogether.

    A parameter without a gradient is left as it is, its step too.  State is there from the beginning, so a first step can be captured; ``state[p]``
    holds ``step`` (int32 on the device), ``exp_avg``, ``exp_avg_sq`` and with 8 bits ``exponents``, which may be exchanged for others of
    the same kind.  Steps enqueue on the current stream; a second step of the same optimiser is ordered behind the first by the caller."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, bits=32):
        if bits not in (8, 32):
            raise ValueError(f"moments in 8 or 32 bits, not {bits}")
        max_norm = None if max_norm is None else float(max_norm)
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"max_norm {max_norm}")
        self.bits, self.max_norm = bits, max_norm
        self._work, self._norm, self.device = None, None, None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    @property
    def grad_norm(self):
        """The norm over all gradients of the last step (fp32 on the device, overwritten by the next), None without max_norm."""
        return None if self.max_norm is None else self._norm

    def add_param_group(self, param_group):
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("state would be zero again at every replay: make an optimiser before its steps are captured")
        before = len(self.param_groups)
        super().add_param_group(param_group)
        try:
            group = self.param_groups[before]
            self._check(group)
            self._make_states(group["params"])
            if self.device is not None:
                _lib.settle(self.device)      # (its steps may be on any stream)
        except BaseException:
            for p in self.param_groups[before]["params"]:
                self.state.pop(p, None)
            del self.param_groups[before:]
            raise

    def _check(self, group):
        lr, betas = group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor) and lr.is_cuda:
            if lr.dtype is not torch.float32 or lr.numel() != 1:
                raise ValueError("lr on the device is one fp32 value")
        elif not 0 <= float(lr):
            raise ValueError(f"lr {float(lr)}")
        if len(betas) != 2 or not all(0 <= float(b) < 1 for b in betas):
            raise ValueError(f"betas are two values from 0 to below 1, not {betas}")
        if not (float(group["eps"]) == 0 or 1.2e-38 <= float(group["eps"]) <= 3.4e38) or not 0 <= float(group["weight_decay"]):
            raise ValueError(f"eps {group['eps']}, weight_decay {group['weight_decay']}")
        if group.get("maximize") or group.get("amsgrad") or (group.get("decoupled_weight_decay") is False and group["weight_decay"] != 0):
            raise ValueError("no maximize, no amsgrad, and weight decay apart from the gradients")
        for p in group["params"]:
            if p.dtype not in _lib.TYPES or p.layout is not torch.strided:
                raise TypeError(f"dense parameters in fp32, bf16 or fp16, not {p.dtype}, {p.layout}")
            device = _lib.require_cuda(p.device)
            if self.device is None:
                self.device = device
                self._work = torch.zeros(_lib.lib().orca_adamw_work_bytes(), dtype=torch.uint8, device=device)
                self._norm = torch.zeros((), dtype=torch.float32, device=device)
            if device != self.device:
                raise ValueError(f"parameters on {self.device} and on {device}")
            if not torch.empty_like(p, device="meta").stride() == p.stride():
                raise ValueError(f"a parameter's elements lie side by side in memory, not with strides {p.stride()} for {tuple(p.shape)}")
        ends = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for g in self.param_groups for p in g["params"] if p.numel())
        if any(b < e for (_, e), (b, _) in zip(ends, ends[1:])):
            raise ValueError("two parameters share memory")

    def _make_states(self, params):
        if not params:
            return
        steps = torch.zeros(len(params), dtype=torch.int32, device=self.device).split(1)
        made = []
        for p, step in zip(params, steps):
            state = self.state[p]
            state["step"] = step
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.empty_like(p, dtype=torch.uint8 if self.bits == 8 else torch.float32, requires_grad=False)
                made.append(state[name])
            if self.bits == 8:
                state["exponents"] = torch.empty(-(-p.numel() // BLOCK), 2, dtype=torch.uint8, device=p.device)
                made.append(state["exponents"])
        torch._foreach_zero_(made)

    def step(self, closure=None):
        """One step with the gradients that the parameters have.  Returns what ``closure`` does, which is called before."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._work is not None:      # (there are parameters)
            _lib.rows().adamw(self.param_groups, self.state, self.bits, -1.0 if self.max_norm is None else self.max_norm, self._norm, self._work)
        return loss

    def moments(self):
        """The values of all parameters' ``exp_avg`` and ``exp_avg_sq``, two lists in the order of the groups: with 8 bits new tensors in bf16, which holds
        each value exactly (all of them in one buffer, which lives as long as any), with 32 the state's own."""
        if self.bits == 8 and self._work is not None:
            return _lib.rows().moments(self.param_groups, self.state, self._work)
        return tuple([self.state[p][name] for g in self.param_groups for p in g["params"]] for name in ("exp_avg", "exp_avg_sq"))

    def _in_order(self, p, theirs, mine):
        """Whether moments of a checkpoint can be laid beside p's elements: they have its sizes (with 8 bits, whose blocks are those of memory, its order, too), or
        are one behind the other, in memory's order or that of a p that lies so.  (And whether those that are there lie beside them.)"""
        whole = p.is_contiguous()
        if not (whole or mine.dim() == 1 if mine.is_contiguous() else (mine.shape, mine.stride()) == (p.shape, p.stride())):
            return False
        if theirs.shape != p.shape:
            return theirs.dim() == 1 or (whole and theirs.is_contiguous())
        return self.bits == 32 or theirs.stride() == p.stride() or (whole and theirs.is_contiguous())

    @staticmethod
    def _flat(t):
        return t.as_strided((t.numel(),), (1,))

    def load_state_dict(self, state_dict):
        """Takes over groups' settings and copies state (and a rate, where that is on the device) into the tensors that are there.  With 32 bits also that of PyTorch's
        own AdamW, or Adam without weight decay; a parameter without state starts at zero.  What does not fit, or is another optimiser's (maximize, amsgrad, Adam's
        weight decay), is refused before anything is changed.  Hooks that are registered for it are called, as PyTorch's own does."""
        state_dict = dict(state_dict)
        for hook in list(self._optimizer_load_state_dict_pre_hooks.values()):
            other = hook(self, state_dict)
            state_dict = state_dict if other is None else other
        groups, states = state_dict["param_groups"], state_dict["state"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("groups of other numbers of parameters")
        names = ("exp_avg", "exp_avg_sq") + (("exponents",) if self.bits == 8 else ())
        pairs = []
        params = [p for g in self.param_groups for p in g["params"]]
        self._make_states([p for p in params if not self.state.get(p)])      # (that were taken out)
        for index, p in zip((i for g in groups for i in g["params"]), params):
            mine, theirs = self.state[p], states.get(index)
            for name in names:
                if theirs and (name not in theirs or theirs[name].numel() != mine[name].numel() or (theirs[name].dtype is torch.uint8) != (self.bits == 8)
                               or (name != "exponents" and not self._in_order(p, theirs[name], mine[name]))):
                    raise ValueError(f"parameter {index} has no '{name}' of {mine[name].numel()} for moments in {self.bits} bits, in the order of its elements")
            step = 0
            if theirs:
                try:
                    step = float(theirs["step"])
                except (KeyError, TypeError, ValueError, RuntimeError):
                    step = -1.0
                if not (0 <= step < 2 ** 31 and step == int(step)):
                    raise ValueError(f"parameter {index} has no 'step' that is a whole number from 0 to below 2^31")
            pairs.append((p, mine, theirs, int(step)))
        settings = []
        for group, theirs in zip(self.param_groups, groups):
            new = copy.deepcopy({k: v for k, v in theirs.items() if k != "params" and (k in ("lr", "betas", "eps", "weight_decay") or k not in group)})
            if isinstance(new.get("lr"), torch.Tensor):
                new["lr"] = float(new["lr"])
            self._check({**group, **new})
            settings.append(new)
        for p, mine, theirs, step in pairs:
            mine["step"].fill_(step)
            for name in names:
                if not theirs:
                    mine[name].zero_()
                elif theirs[name].shape != p.shape or name == "exponents":      # (one behind the other, as they lie in memory)
                    self._flat(mine[name]).copy_(theirs[name].reshape(-1))
                else:
                    mine[name].as_strided(p.shape, p.stride()).copy_(theirs[name])
        for group, new in zip(self.param_groups, settings):
            if isinstance(group["lr"], torch.Tensor):      # (a captured step reads it)
                group["lr"].fill_(new.pop("lr", group["lr"]))
            group.update(new)
        for hook in list(self._optimizer_load_state_dict_post_hooks.values()):
            hook(self)

    def __getstate__(self):
        return dict(super().__getstate__(), bits=self.bits, max_norm=self.max_norm, device=self.device, _work=self._work, _norm=self._norm)
