"""FusedAdamW: ``torch.optim.AdamW`` semantics, one kernel launch per step.

The whole parameter set is updated by a single multi-tensor kernel
(``csrc/kernels/adamw.cu``) that streams (p, g, m, v) once: 28 bytes per fp32
parameter, the HBM floor of the update.  State is kept in the standard
``state[p] = {"step", "exp_avg", "exp_avg_sq"}`` layout, so ``state_dict()`` is
interchangeable with ``torch.optim.AdamW`` (checkpoints load either way).
``grad_scale`` lets a caller fold a deferred gradient scaling (for example the
1/world of a summed allreduce) into the update instead of a separate pass.

``state_bits=8`` keeps the moments in 8 bits (``mccl_b200.optim.moments``): ``exp_avg`` and ``exp_avg_sq`` are then padded float8
tensors with ``exp_avg_scale`` and ``exp_avg_sq_scale`` beside them, 2.03 bytes a parameter instead of 8, and a step streams 16 bytes
instead of 28.  ``bfloat16`` parameters are the upper half of an fp32 value that the update is made on; the lower half is their
state ``low`` (int16), so that no update is too small for them.  Checkpoints of either kind, and ``torch.optim.AdamW``'s, load
into the other; :meth:`FusedAdamW.moments` gives a parameter's moments as fp32 numbers.  The step's number, which counts for what is
rounded up, is the host's: a step of either kind is not captured into a graph.
"""
from __future__ import annotations

from typing import Iterable

import torch

from .. import require_native
from .moments import GROUP, pack_moment, padded, unpack_moment

_TYPES = (torch.float32, torch.bfloat16)
_EXTRAS = ("exp_avg_scale", "exp_avg_sq_scale", "low")
_REFUSED = "FusedAdamW handles contiguous float32 or bfloat16 CUDA parameters"


def _handled(p: torch.Tensor) -> bool:
    return p.is_cuda and p.dtype in _TYPES and p.is_contiguous()


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params: Iterable, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, got {state_bits!r}")
        if lr < 0 or eps < 0 or weight_decay < 0 or not (0 <= betas[0] < 1) or not (0 <= betas[1] < 1):
            raise ValueError("invalid AdamW hyper-parameters")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits = state_bits
        self._plans = {}
        # DDP hands back bucket parameters as tensors that may be fresh Python objects: find ours by address
        self._by_ptr = {}
        self._index_params()
        self._bw_cache = {}
        self._bw_touched = []
        self._bw_step = 0
        self._bw_done = set()
        self._native_hook = None   # BucketOptimizerState when the native DDP hook is installed

    def _index_params(self) -> None:
        self._by_ptr = {p.data_ptr(): (p, gi) for gi, g in enumerate(self.param_groups) for p in g["params"]}

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        if hasattr(self, "_by_ptr"):  # the base constructor calls this before our fields exist
            self._index_params()
            self._bw_cache.clear()

    def _state_of(self, p):
        st = self.state[p]
        if "exp_avg" not in st:
            st["step"] = torch.tensor(0.0)
            if self.state_bits == 8:
                n = padded(p.numel())
                for name, kind in (("exp_avg", torch.float8_e4m3fn), ("exp_avg_sq", torch.float8_e5m2)):
                    st[name] = torch.zeros(n, dtype=torch.uint8, device=p.device).view(kind)
                    st[name + "_scale"] = torch.zeros(n // GROUP, device=p.device)
            else:
                st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format, dtype=torch.float32)
                st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format, dtype=torch.float32)
        if p.dtype is torch.bfloat16 and "low" not in st:
            st["low"] = torch.zeros_like(p, dtype=torch.int16)
        return st

    @staticmethod
    def _extra_of(st):
        """What the kernel for several kinds is given beside the moments; None where fp32 is all there is."""
        extra = tuple(st.get(name) for name in _EXTRAS)
        return None if all(e is None for e in extra) else extra

    def moments(self, p: torch.Tensor):
        """``(exp_avg, exp_avg_sq)`` of a parameter as float32 numbers of its shape, whatever they are kept as."""
        st = self._state_of(p)
        return tuple(unpack_moment(st[name], st[name + "_scale"], p.shape) if name + "_scale" in st else st[name].clone()
                     for name in ("exp_avg", "exp_avg_sq"))

    def _by_step(self, params):
        """``{step number of the coming update: its parameters}``; one entry unless some parameter missed a step."""
        counters = [self._state_of(p)["step"] for p in params]
        if all(isinstance(c, torch.Tensor) and c.is_cuda for c in counters):
            # (torch's own fused AdamW keeps them on the device: one copy for all instead of one for each)
            counters = torch.stack([c.reshape(()) for c in counters]).tolist()
        out = {}
        for p, c in zip(params, counters):
            out.setdefault(int(c) + 1, []).append(p)
        return out

    def _plan_for(self, gi, params):
        key = (gi, tuple(p.data_ptr() for p in params))
        plan = self._plans.get(gi)
        if plan is None or plan[0] != key:
            native = require_native()
            ms, vs, extra = [], [], []
            for p in params:
                st = self._state_of(p)
                ms.append(st["exp_avg"])
                vs.append(st["exp_avg_sq"])
                extra.append(self._extra_of(st))
            extra = [e or (None, None, None) for e in extra] if any(extra) else []
            plan = (key, native.AdamWPlan([p.data for p in params], ms, vs, extra))
            self._plans[gi] = plan
        return plan[1]

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: float = 1.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._native_hook is not None:  # parameters the native bucket hook updated during backward
            used_step, ptrs = self._native_hook.take_stepped()
            if ptrs:
                self._bw_step = used_step
                self._bw_touched.append([self._by_ptr[a][0] for a in ptrs if a in self._by_ptr])
        for own in self._bw_touched:  # updated inside backward: only their step counters are left to refresh
            for p in own:
                self.state[p]["step"].fill_(float(self._bw_step))
                self._bw_done.add(id(p))
        self._bw_touched = []
        for gi, group in enumerate(self.param_groups):
            # the ordinary step, all of the group's parameters on the plan of the last one: one native call does the
            # checks, the launch and the counters (a Python pass over the parameters took 4 us for each)
            plan = self._plans.get(gi)
            if plan is not None and not self._bw_done and len(plan[0][1]) == len(group["params"]):
                entries = [self.state.get(p) for p in group["params"]]
                steps = [e.get("step") if e is not None else None for e in entries]
                b1, b2 = group["betas"]
                if plan[1].step_group(group["params"], steps, group["lr"], b1, b2, group["eps"], group["weight_decay"],
                                      grad_scale):
                    continue
            # parameters already updated inside backward are skipped
            params = [p for p in group["params"] if p.grad is not None and id(p) not in self._bw_done]
            if not params:
                continue
            if not all(_handled(p) for p in params):
                raise RuntimeError(_REFUSED + " (see mccl_b200.params.ensure_contiguous_parameters)")
            b1, b2 = group["betas"]
            # the bias corrections are those of a parameter's own counter: one launch for each value among them
            for part, (step, own) in enumerate(self._by_step(params).items()):
                plan = self._plan_for(gi if part == 0 else (gi, part), own)
                grads = [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in own]
                plan.step(grads, group["lr"], b1, b2, group["eps"], group["weight_decay"], step, grad_scale)
                for p in own:
                    s = self.state[p]["step"]
                    if isinstance(s, torch.Tensor):
                        s.fill_(float(step))  # host tensor, as torch.optim.AdamW keeps it by default
                    else:
                        self.state[p]["step"] = step
        self._bw_done = set()
        return loss

    # ---- per-bucket stepping (optimizer inside backward) -----------------------
    # One step number, that of the first trainable parameter, serves all that is updated inside backward.  Parameters
    # whose counters differ from it (as a checkpoint can hold them) are left to `step()`, which knows each one's own.
    def _next_step(self) -> int:
        trainable = (p for g in self.param_groups for p in g["params"] if p.requires_grad)
        st = self.state[next(trainable, self.param_groups[0]["params"][0])]
        return int(st["step"]) + 1 if "step" in st else 1

    def _on_shared_step(self, params) -> set:
        return {id(p) for p in self._by_step(params).get(self._next_step(), ())}

    def begin_step_in_backward(self) -> int:
        """Advances the shared step counter once per iteration; returns the new step."""
        self._bw_step = self._next_step()
        self._bw_done = set()
        self._bw_touched = []
        return self._bw_step

    def bucket_plans(self, key, params):
        """Launch plans of one DDP bucket: a list of ``(plan, group, own_params, positions)``, without the parameters
        that ``step()`` will update.

        A bucket may hold parameters of several param groups (for example weights with weight decay
        and biases without); each group gets its own plan so that every parameter is updated with its
        own group's hyper-parameters.  ``positions`` are the indices of the group's parameters inside
        ``params`` (and inside ``bucket.gradients()``).  The cache entry is keyed by the addresses of
        all the bucket's parameters, so a rebuilt bucket is noticed even if its first parameter stays.
        """
        sig = tuple(p.data_ptr() for p in params)
        ent = self._bw_cache.get(key)
        if ent is None or ent[0] != sig:
            by_group = {}
            try:
                found = [self._by_ptr[p.data_ptr()] for p in params]
            except KeyError:
                raise KeyError("a DDP bucket holds a parameter this optimizer was not given") from None
            here = self._on_shared_step([own for own, _ in found])
            for pos, (own, gi) in enumerate(found):
                if id(own) not in here:
                    continue
                by_group.setdefault(gi, ([], []))
                by_group[gi][0].append(own)
                by_group[gi][1].append(pos)
            plans = []
            for gi in sorted(by_group):
                own, pos = by_group[gi]
                plans.append((self._plan_for(("bucket", key, gi), own), self.param_groups[gi], own, pos))
            ent = (sig, plans)
            self._bw_cache[key] = ent
        return ent[1]

    # ---- native hook support ------------------------------------------------------
    def ensure_state(self) -> None:
        """Creates the AdamW state of every parameter (so that a native hook can be given the tensors)."""
        for group in self.param_groups:
            for p in group["params"]:
                self._state_of(p)

    def attach_native_hook(self, hook_state) -> None:
        """Hands parameters, state tensors and group indices to a ``BucketOptimizerState``."""
        self.ensure_state()
        here = self._on_shared_step([p for g in self.param_groups for p in g["params"]])
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                if not _handled(p):
                    raise RuntimeError(_REFUSED)
                st = self.state[p]
                hook_state.add_param(p.data, st["exp_avg"], st["exp_avg_sq"], gi if id(p) in here else -1, self._extra_of(st))
        self._native_hook = hook_state
        self.sync_native_hook()

    def sync_native_hook(self) -> None:
        """Pushes the groups' current hyper-parameters and the next step number to the native hook.

        Called before every forward: whatever a learning-rate scheduler did since the last step is
        what the bucket updates of the coming backward use.
        """
        if self._native_hook is None:
            return
        for gi, group in enumerate(self.param_groups):
            b1, b2 = group["betas"]
            self._native_hook.set_hyper(gi, group["lr"], b1, b2, group["eps"], group["weight_decay"])
        self._native_hook.set_step(self._next_step())

    def mark_bucket_stepped(self, own) -> None:
        self._bw_touched.append(own)

    def load_state_dict(self, state_dict):
        loaded = []
        last = self.register_load_state_dict_pre_hook(lambda _, d: loaded.append(d))  # what the program's own hooks make of it
        try:
            super().load_state_dict(state_dict)
        finally:
            last.remove()
        saved, own = ([i for g in groups for i in g["params"]] for groups in (loaded[0]["param_groups"], self.param_groups))
        for i, p in zip(saved, own):
            if i in loaded[0]["state"]:
                self._adopt(p, loaded[0]["state"][i])
        self._plans.clear()  # state tensors were replaced
        self._bw_cache.clear()
        if self._native_hook is not None:
            self.attach_native_hook(self._native_hook)

    def _adopt(self, p, saved) -> None:
        """A parameter's saved state as this optimizer keeps it; the base class has cast every tensor to the parameter's type."""
        if "exp_avg" not in saved or "exp_avg_sq" not in saved:
            return
        st = self.state[p]
        st.pop("low", None)  # a bf16 parameter's, for one that may be of another type now
        if self.state_bits == 32 and p.dtype is torch.float32 and "exp_avg_scale" not in saved:
            return  # as it came
        for name, kind in (("exp_avg", torch.float8_e4m3fn), ("exp_avg_sq", torch.float8_e5m2)):
            moment, scale = saved[name].to(p.device), saved.get(name + "_scale")
            scale = scale if scale is None else scale.to(p.device)
            if (scale is not None) == (self.state_bits == 8):
                st[name] = moment if scale is not None else moment.float()
                if scale is not None:
                    st[name + "_scale"] = scale
            elif scale is None:
                st[name], st[name + "_scale"] = pack_moment(moment, kind)
            else:
                st[name] = unpack_moment(moment, scale, p.shape)
                st.pop(name + "_scale", None)
        if p.dtype is torch.bfloat16 and "low" in saved:
            st["low"] = saved["low"].to(p.device)
