"""``AdamW``: decoupled weight decay, the averages in 32 or in 8 bits (functional/adamw.py has the formulas and the 8-bit format).

The reference leaves optimizers to torch; this is torch's ``AdamW`` for the package's layers, with the same arguments and
``state_dict`` keys."""
from __future__ import annotations

import torch

from ..functional.adamw import adamw_empty_state, adamw_state_values, adamw_step
from ..functional.clip import grad_norm
from ..functional.tracing import refused_under_trace


class AdamW(torch.optim.Optimizer):
    """``state_bits``: 32, or 8 (a quarter of the memory and less than that to read and write; a state of a parameter is then
    ``exp_avg`` and ``exp_avg_sq`` codes, laid out like it, with ``exp_avg_scale`` and ``exp_avg_sq_scale``).

    ``lr`` may be a float32 tensor on the GPU, which a captured graph reads at every replay.  ``step`` of a parameter's state is an int64
    on the GPU, shared by the parameters that have been updated the same number of times; parameters without a gradient are left out
    of a step, as torch's optimizers leave them out.  A step can be captured into a graph once one with the same gradients has been
    taken.  Parameters must be on the GPU, float16, bfloat16 or float32, and fill their memory.

    ``max_norm``: gradients are clipped to that joint norm (of all groups) as the step reads them; ``p.grad`` stays as it is, and ``grad_norm`` is
    the norm that the last step found, a float32 on the GPU (of a captured step: of its last replay).  It belongs to the optimizer, not to its
    state, and may be changed between steps.  The gradients must be on one GPU then; without it parameters may be on several."""

    max_norm: float | None = None
    grad_norm: torch.Tensor | None = None

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits: int = 32,
                 max_norm: float | None = None) -> None:
        if not isinstance(lr, torch.Tensor) and not lr >= 0:
            raise ValueError(f"lr must not be negative (got {lr})")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError(f"betas must be in [0, 1) (got {betas})")
        if not (eps == 0 or 2.0 ** -126 <= eps <= 2.0 ** 120) or not weight_decay >= 0:
            raise ValueError(f"eps must be 0 or from 2^-126 to 2^120 and weight_decay not negative (got {eps}, {weight_decay})")
        if state_bits not in (8, 32):
            raise ValueError(f"averages are held in 8 or in 32 bits (got {state_bits})")
        if max_norm is not None and not max_norm >= 0:
            raise ValueError(f"max_norm must not be negative (got {max_norm})")
        self.max_norm = max_norm
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "grad_norm": self.grad_norm}

    def _init_state(self, p: torch.Tensor, bits: int, step: torch.Tensor) -> None:
        if bits not in (8, 32):
            raise ValueError(f"averages are held in 8 or in 32 bits (got {bits})")
        state = self.state[p]
        state["step"] = step
        if bits == 8:
            state["exp_avg"], state["exp_avg_scale"] = adamw_empty_state(p)
            state["exp_avg_sq"], state["exp_avg_sq_scale"] = adamw_empty_state(p)
        else:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)

    @staticmethod
    def _not_captured(p: torch.Tensor, what: str) -> None:
        # (a replay would do it again: averages back to zero, a count back to what it was)
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} cannot be captured into a graph: take a step with the same gradients before the capture")

    @staticmethod
    def _averages(states, key):
        return [(s[key], s[key + "_scale"]) if key + "_scale" in s else s[key] for s in states]

    @refused_under_trace
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        factor = None
        if self.max_norm is not None:
            grads = [p.grad for group in self.param_groups for p in group["params"] if p.grad is not None]
            if grads:
                self.grad_norm, factor = grad_norm(grads, max_norm=self.max_norm)
        for group in self.param_groups:
            fresh: dict[torch.device, torch.Tensor] = {}
            together: dict[int, list[torch.Tensor]] = {}  # by the step tensor that the parameters share
            members: dict[int, int] = {}
            for p in group["params"]:
                state = self.state.get(p)
                if state:
                    members[id(state["step"])] = members.get(id(state["step"]), 0) + 1
                if p.grad is None:
                    continue
                if not state:
                    self._not_captured(p, "a parameter's first step")
                    if p.device not in fresh:
                        fresh[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
                    self._init_state(p, group["state_bits"], fresh[p.device])
                    state = self.state[p]
                    members[id(state["step"])] = members.get(id(state["step"]), 0) + 1
                together.setdefault(id(state["step"]), []).append(p)
            for key, params in together.items():
                states = [self.state[p] for p in params]
                step = states[0]["step"]
                if len(params) < members[key]:  # the others stay behind, with a count of their own
                    self._not_captured(params[0], "the first step without some of the parameters")
                    step = step.clone()
                    for s in states:
                        s["step"] = step
                adamw_step(params, [p.grad for p in params], self._averages(states, "exp_avg"), self._averages(states, "exp_avg_sq"), step,
                           lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                           grad_scale=factor)
        return loss

    def state_values(self, p: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Both averages of a parameter as float32 tensors of its shape."""
        s = self.state[p]
        if "exp_avg_scale" not in s:
            return s["exp_avg"], s["exp_avg_sq"]
        (m,), (v,) = adamw_state_values(self._averages([s], "exp_avg"), self._averages([s], "exp_avg_sq"))
        return m, v

    @staticmethod
    def _codes_like(p: torch.Tensor, codes: torch.Tensor) -> torch.Tensor:
        """Saved codes of an average of ``p`` with its strides.  They and their scales go by the order of the parameter's memory, so they fit
        no other layout (codes without a shape are of a contiguous parameter)."""
        kept = codes.view(p.shape) if codes.dim() == 1 and codes.numel() == p.numel() else codes
        if kept.shape != p.shape or any(n > 1 and a != b for n, a, b in zip(p.shape, kept.stride(), p.stride())):
            raise ValueError(f"averages in 8 bits of a parameter laid out as {tuple(codes.shape)}, strides {codes.stride()}, "
                             f"fit none of {tuple(p.shape)}, strides {p.stride()}")
        return torch.as_strided(kept, p.shape, p.stride())

    def _saved(self, state_dict):
        """(parameter, its saved state) pairs of a state dict with this optimizer's groups."""
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for number, p in zip(saved["params"], group["params"]):
                if state_dict["state"].get(number):
                    yield group, p, state_dict["state"][number]

    def load_state_dict(self, state_dict) -> None:
        """torch's, which casts states to their parameters' dtypes; the averages and counts are then put back as they were saved, before hooks
        behind it run.  Averages in 32 bits are laid out like their parameters; those in 8 are refused where the layouts differ.  A state of
        torch's own AdamW is taken too, but for its ``amsgrad`` and ``maximize``, which are refused."""
        taken = []

        def before(_, given):  # (behind other hooks, which may have replaced what is loaded)
            for group in given["param_groups"]:
                for key in ("amsgrad", "maximize"):
                    if group.get(key):
                        raise ValueError(f"{key} is not built")
            for _, p, saved in self._saved(given):
                for key in ("exp_avg", "exp_avg_sq"):
                    if key + "_scale" in saved:
                        self._codes_like(p, saved[key])
            taken.append(given)

        def after(_):
            for group in self.param_groups:
                for key, value in self.defaults.items():
                    group.setdefault(key, value)
            self._put_back(taken[0])

        hooks = self.register_load_state_dict_pre_hook(before), self.register_load_state_dict_post_hook(after, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _put_back(self, state_dict) -> None:
        shared: dict[tuple, torch.Tensor] = {}
        for group, p, saved in self._saved(state_dict):
            state = self.state[p]
            for key, value in saved.items():
                if not isinstance(value, torch.Tensor):
                    state[key] = value
                    continue
                kept = value.detach().to(p.device, copy=True)
                if key + "_scale" in saved:
                    kept = self._codes_like(p, kept)
                elif key in ("exp_avg", "exp_avg_sq") and kept.shape == p.shape:
                    kept = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(kept)
                state[key] = kept
            count = int(state["step"])
            state["step"] = shared.setdefault((id(group), p.device, count), torch.full((), count, dtype=torch.int64, device=p.device))
