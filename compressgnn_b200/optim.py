"""The optimiser of a training step on the package's own kernel (``runtime.adamw_step``): one launch for all tensors of a type,
the moments in 32 or in 8 bits, the gradients clipped by their norm without a pass that writes them."""
import torch

from . import runtime as _native


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay; ``weight_decay=0`` is Adam), as ``torch.optim.AdamW`` computes it.

    ``max_norm``: the gradients of all groups are clipped by their common 2-norm, which ``step`` leaves in ``grad_norm``
    (a float32 tensor on the device); the gradients themselves are not changed.
    ``state_bits=8``: moments of tensors with ``least_8bit`` elements or more are held in 8 bits, 6 bytes a float32
    parameter less to keep and 12 less to move a step; smaller ones, and float64, keep theirs in full.  ``seed`` is the key
    of their stochastic rounding.

    The groups hold ``max_norm`` and ``seed`` as they hold the rest, so a schedule may set them and a loaded state brings its own; but
    there is one of each, and groups that differ in them are refused.

    Parameters are contiguous.  ``lr`` may be a CUDA tensor of one float32.  The steps taken are counted on the device, so a step can be captured into
    a CUDA graph once the state exists (after one step outside of the capture)."""

    grad_norm = None
    _COMMON = ("max_norm", "seed")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, state_bits=32,
                 least_8bit=4096, seed=0):
        if not torch.is_tensor(lr) and not lr >= 0.0:
            raise ValueError("lr must not be negative")
        if not all(0.0 <= beta < 1.0 for beta in betas):
            raise ValueError("the betas must lie in [0, 1)")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("eps and weight_decay must not be negative")
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError("max_norm must not be negative")
        if state_bits not in (8, 32):
            raise ValueError("Supported state_bits: 8, 32")
        # (all of it in the defaults: they are what a copy of an optimiser takes along)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, max_norm=max_norm,
                                      state_bits=state_bits, least_8bit=least_8bit, seed=seed))

    def _begin(self, params):
        """State for parameters that have none yet: ``(group, parameter)`` pairs."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take one step outside of the capture first, the state is made there")
        steps = torch.zeros(len(params), dtype=torch.int64, device=params[0][1].device)
        for (group, p), step in zip(params, steps.unbind()):
            state = self.state[p]
            state["step"] = step
            wide = torch.float64 if p.dtype == torch.float64 else torch.float32
            if group["state_bits"] == 8 and p.numel() >= group["least_8bit"] and wide == torch.float32:
                blocks = (p.numel() + 255) // 256
                for name in ("exp_avg", "exp_avg_sq"):  # (the second holds the root)
                    state[name] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                    state[name + "_scale"] = torch.ones(blocks, device=p.device)
            else:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros(p.shape, dtype=wide, device=p.device)

    def add_param_group(self, group):
        for name in self._COMMON if isinstance(group, dict) else ():  # (the base class refuses others)
            common = self.param_groups[0][name] if self.param_groups else self.defaults[name]
            if group.setdefault(name, common) != common:
                raise ValueError(f"AdamW: {name} is common to all groups")
        super().add_param_group(group)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        max_norm, seed = (self.param_groups[0][name] for name in self._COMMON)
        if any((group["max_norm"], group["seed"]) != (max_norm, seed) for group in self.param_groups):
            raise RuntimeError("AdamW: max_norm and seed are common to all groups, set them in each")
        if max_norm is not None:
            self.grad_norm = None  # (of a step without a gradient)
        calls, fresh = {}, []
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_cuda:
                    raise RuntimeError("compressgnn_b200 runs on CUDA tensors only (no CPU optimiser path)")
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                if not self.state[p]:
                    fresh.append((group, p))
                calls.setdefault((p.device, tuple(group["betas"]), group["eps"]), []).append((group, p))
        if max_norm is not None and len(calls) > 1:
            raise RuntimeError("AdamW: with max_norm all parameters lie on one device and share betas and eps")
        for device in {p.device for _, p in fresh}:
            self._begin([(group, p) for group, p in fresh if p.device == device])
        for number, ((_, betas, eps), members) in enumerate(calls.items()):
            states = [self.state[p] for _, p in members]
            norm = _native.adamw_step(
                [p for _, p in members], [p.grad.contiguous() for _, p in members], [s["exp_avg"] for s in states],
                [s["exp_avg_sq"] for s in states], [s["step"] for s in states], [group["lr"] for group, _ in members], betas, eps,
                [group["weight_decay"] for group, _ in members], max_norm, [s.get("exp_avg_scale") for s in states],
                [s.get("exp_avg_sq_scale") for s in states], int(seed) + (number << 32))
            if max_norm is not None:
                self.grad_norm = norm
        return loss

    def load_state_dict(self, state_dict):
        """(The base class casts a parameter's state to its type: the moments keep theirs, and the count stays whole.)  A state of another
        optimiser, ``torch.optim.AdamW`` among them, is refused: its groups lack settings, its counts are fractions on the host."""
        ours = all(set(self.defaults) <= set(group) for group in state_dict["param_groups"])
        for state in filter(None, state_dict["state"].values()):
            step = state.get("step")
            ours = ours and "exp_avg" in state and "exp_avg_sq" in state and torch.is_tensor(step) and step.dtype == torch.int64
        if not ours:
            raise ValueError("AdamW: this is the state of another optimiser")
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        ours = [p for group in self.param_groups for p in group["params"]]
        for number, p in zip(saved, ours):
            if number in state_dict["state"]:
                self.state[p] = {name: value.to(p.device, copy=True) if torch.is_tensor(value) else value
                                 for name, value in state_dict["state"][number].items()}
