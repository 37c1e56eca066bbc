"""AdamW over many tensors at once, with moments in 32 or 8 bits.

The reference trains with torch.optim.Adam (self_benchmark/a64fx/model/utils.py:24), a loop of element-wise passes
over every parameter.  Here one kernel launch updates up to 480 tensors: `adamw_step` is the plain call on lists of
tensors, `AdamW` the torch.optim.Optimizer around it.

8-bit moments (`state_bits=8`) take 2.03 bytes a parameter instead of 8: e4m3 codes of the first moment and of the
second moment's square root, in blocks of 256 elements with an fp32 scale each.
"""
import weakref

import torch

from . import _lib

STATE_BLOCK = 256
FP8 = torch.float8_e4m3fn


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, scales=None, masters=None, device_scalars: torch.Tensor = None) -> None:
    """One AdamW step over lists of tensors, in place:

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    params, grads: one type (float32, bfloat16 or float16), contiguous, on one device.  exp_avgs, exp_avg_sqs:
    float32, or float8_e4m3fn codes of m and of sqrt(v) with `scales`, (ceil(n / 256), 2) float32 per tensor.
    masters: for 16-bit parameters, float32 copies (None where there is none) that are updated and that the
    parameters are rounded from.  step: t, from 1.  device_scalars: what `AdamW(capturable=True)` keeps on the device
    instead of step and lr.  No two tensors may overlap."""
    _lib.ops().adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales, masters, device_scalars, step, lr, *betas, eps,
                          weight_decay)


def _zero_moment(bits: int, like: torch.Tensor) -> torch.Tensor:
    dtype = torch.float32 if bits == 32 else torch.uint8
    t = torch.zeros_like(like, dtype=dtype, memory_format=torch.contiguous_format)
    return t if bits == 32 else t.view(FP8)


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) whose step is one launch for all parameters of one type in a group.

    state_bits: 32, or 8 for block-quantised moments.  master_weights: keep a float32 copy of 16-bit parameters and
    round the parameter from it at every step.  capturable: the step count lives on the device, so that `step()` can
    be captured into a CUDA graph and replayed; `lr` may then be a 0-dim float32 CUDA tensor that the caller changes
    between replays.  Parameters that have always stepped together share a count, and part when one of them has no
    gradient in a step; a capture, and every step after it, takes all parameters of a count or none.  Parameters are
    dense float32, bfloat16 or float16 CUDA tensors, and contiguous."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, master_weights: bool = False, capturable: bool = False):
        if not isinstance(lr, torch.Tensor) and lr < 0.0:
            raise ValueError(f"AdamW: negative learning rate {lr}")
        if isinstance(lr, torch.Tensor) and not (capturable and lr.is_cuda and lr.dim() == 0 and lr.dtype == torch.float32):
            raise ValueError("AdamW: a tensor lr must be a 0-dim float32 CUDA tensor and needs capturable=True")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), not {betas}")
        if eps < 0.0 or weight_decay < 0.0:
            raise ValueError("AdamW: eps and weight_decay must not be negative")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, not {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, capturable=capturable))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        if len({id(p) for p in params}) != len(params):  # two updates of one tensor in one launch would race
            self.param_groups.pop()
            raise ValueError("AdamW: a parameter is listed twice in a group")

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but the moments keep the types they were saved in (torch would cast them to the parameter's)."""
        for group in state_dict["param_groups"]:
            if not {"state_bits", "master_weights", "capturable"} <= group.keys():
                raise ValueError("AdamW: the state dict is another optimiser's")
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        for mine, theirs in zip(self.param_groups, state_dict["param_groups"]):
            shared = {}  # one count on the device for all parameters that agree on it
            for p, key in zip(mine["params"], theirs["params"]):
                if key not in saved:
                    continue
                state = {k: v.detach().to(p.device, copy=True) if isinstance(v, torch.Tensor) else v
                         for k, v in saved[key].items()}
                step = int(state["step"])
                if mine["capturable"]:
                    step = shared.setdefault((p.device, step), torch.tensor(step, dtype=torch.int64, device=p.device))
                state["step"] = step
                self.state[p] = state

    def _new_state(self, p, group, fresh) -> dict:
        n, bits = p.numel(), group["state_bits"]
        state = {"step": 0, "exp_avg": _zero_moment(bits, p), "exp_avg_sq": _zero_moment(bits, p)}
        if group["capturable"]:  # parameters that begin together share a count
            if p.device not in fresh:
                fresh[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
            state["step"] = fresh[p.device]
        if bits == 8:
            state["scales"] = torch.zeros(((n + STATE_BLOCK - 1) // STATE_BLOCK, 2), dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32, memory_format=torch.contiguous_format)
        self.state[p] = state
        return state

    def _own_counts(self, members, capturing) -> None:
        """Device counts for the parameters that step together: one that is also held by a parameter that does not step
        now stays with that one, and the others go on with a copy.  A count of a captured step is advanced by every
        replay, so it stays with all of its parameters."""
        stepping = {id(p) for p, _ in members}
        idle = {id(s["step"]) for p, s in self.state.items() if s and id(p) not in stepping}
        known = self.__dict__.setdefault("_captured", {})  # id -> weak reference: counts of captured steps
        counts = {id(s["step"]): s["step"] for _, s in members}
        shared = {k: c for k, c in counts.items() if k in idle}
        if shared and capturing:
            raise RuntimeError("AdamW: take a step with the gradients of these parameters alone before capturing (they share "
                               "their step count with parameters that have no gradient)")
        if any(k in known and known[k]() is c for k, c in shared.items()):
            raise RuntimeError("AdamW: a captured step updates parameters that have no gradient now together with others that "
                               "have one: their step count is shared (once the graph is not replayed any more, "
                               "load_state_dict(state_dict()) gives them other counts)")
        if capturing:
            known.update((k, weakref.ref(c)) for k, c in counts.items())
        copies = {k: c.clone() for k, c in shared.items()}
        for _, state in members:
            state["step"] = copies.get(id(state["step"]), state["step"])

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        for group in self.param_groups:
            if capturing and not group["capturable"]:
                raise RuntimeError("AdamW: a step that is captured into a graph needs capturable=True")
            fresh, members, calls = {}, [], {}  # calls: (device, count) -> type -> members
            for p in group["params"]:
                if p.grad is None:
                    continue
                _lib.require_cuda(p, p.grad)
                if p.grad.is_sparse or not p.is_contiguous():
                    raise RuntimeError("AdamW: parameters must be contiguous, gradients dense")
                state = self.state[p]
                if not state:
                    if capturing:
                        raise RuntimeError("AdamW: take one step before capturing (it creates the moments)")
                    state = self._new_state(p, group, fresh)
                members.append((p, state))
            if group["capturable"]:
                self._own_counts(members, capturing)
            for p, state in members:
                if group["capturable"]:
                    key = (p.device, id(state["step"]))
                else:
                    state["step"] += 1
                    key = (p.device, state["step"])
                calls.setdefault(key, {}).setdefault(p.dtype, []).append((p, state))
            for (device, count), by_type in calls.items():
                scalars = None
                if group["capturable"]:
                    scalars = self._tick(group, device, next(iter(by_type.values()))[0][1]["step"])
                for members in by_type.values():
                    self._update(group, members, 0 if group["capturable"] else count, scalars)
        return loss

    @staticmethod
    def _tick(group, device, step):
        """Counts a step on the device and returns its scalars."""
        lib, lr, (b1, b2) = _lib.lib(), group["lr"], group["betas"]
        if isinstance(lr, torch.Tensor) and lr.device != device:
            raise RuntimeError(f"AdamW: lr is on {lr.device}, parameters on {device}")
        lr_ptr, host_lr = (lr.data_ptr(), 0.0) if isinstance(lr, torch.Tensor) else (0, float(lr))
        scalars = torch.empty(lib.gnnagg_adamw_scalars_bytes(), dtype=torch.uint8, device=device)
        with _lib.device_of(scalars):
            rc = lib.gnnagg_adamw_tick(step.data_ptr(), lr_ptr, host_lr, b1, b2, group["eps"], group["weight_decay"],
                                       scalars.data_ptr(), _lib.stream_ptr(device))
        _lib.check(rc, "adamw_tick")
        return scalars

    @staticmethod
    def _update(group, members, step, scalars):
        states = [s for _, s in members]
        adamw_step([p for p, _ in members],
                   [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p, _ in members],
                   [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], step=step,
                   lr=0.0 if scalars is not None else group["lr"], betas=group["betas"], eps=group["eps"],
                   weight_decay=group["weight_decay"],
                   scales=[s["scales"] for s in states] if group["state_bits"] == 8 else None,
                   masters=[s.get("master") for s in states] if group["master_weights"] else None,
                   device_scalars=scalars)
