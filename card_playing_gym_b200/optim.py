"""AdamW over many tensors in two launches, with 32-bit or 8-bit moments and the global-norm clip inside the step.

The reference clips the actor's and the critic's gradients to one global norm and then runs torch's fused Adam
(rl/trainer.py:175-183, 392-401, 474-485), skipping the step where a gradient is not finite. ``AdamW`` does all of it
on the device (csrc/adamw.cu): the norm, the clip, the skip, decoupled weight decay and the update, with no host read.
With ``weight_decay=0`` it is Adam. It is a ``torch.optim.Optimizer`` (parameter groups, learning-rate schedulers,
``state_dict``).
"""

from __future__ import annotations

from array import array
from operator import attrgetter

import torch

from . import _native as nat

_dtype_of, _layout_of, _bytes_of = attrgetter("dtype"), attrgetter("layout"), attrgetter("nbytes")

BLOCK = 256  # entries of one scale of the 8-bit moments; every parameter's state starts on a multiple of it


class AdamW(torch.optim.Optimizer):
    """AdamW(params, lr, betas, eps, weight_decay, state_bits=32 | 8, max_norm=None).

    Parameters are contiguous CUDA tensors of one dtype (float32, float16 or bfloat16) on one device. 16-bit
    parameters keep float32 master copies in the state, which the step updates and rounds once into the parameter. Where a
    parameter has been written to since (a checkpoint loaded into the model, an in-place edit), the next step takes
    its values over into the master copy; it sees writes that count the parameter's version up or give it another
    address, which writes through ``.data`` do not.

    ``state_bits=8`` holds m and sqrt(v) as e4m3 codes scaled by the largest magnitude of each block of 256
    entries. ``max_norm`` clips the gradients' global norm, coefficient min(1, max_norm / (norm + 1e-6)); where the
    norm is not finite the step changes nothing and does not count. Without ``max_norm`` a gradient that is not
    finite reaches its parameter, and with 8-bit moments the rest of its block.

    The state is flat: ``flat[name]`` holds every parameter's entries in order, each parameter starting on a multiple
    of 256 (``exp_avg``, ``exp_avg_sq``; with 8 bits ``exp_avg``, ``exp_avg_sq_root`` and their ``_scale`` per
    block; ``master``), and ``state[p]`` has views of it. ``steps`` (int64) counts the steps on the device, one
    count for all parameters; ``grad_norm`` (float32) is the last step's norm before clipping, where ``max_norm`` is
    set. A parameter whose ``grad`` is None is left as it is.

    Learning rates and the other hyperparameters are read on the host at every ``step``: a captured CUDA graph
    replays those of its capture.
    """

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, max_norm: float | None = None) -> None:
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm must be positive (or None for no clip)")
        self.state_bits = state_bits
        self.max_norm = max_norm
        self._built = False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self._build()

    def add_param_group(self, param_group: dict) -> None:
        if self._built:
            raise ValueError("the state is laid out once: pass every parameter group to the constructor")
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        beta1, beta2 = group["betas"]
        if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
            raise ValueError("betas must lie in [0, 1)")
        if group["lr"] < 0 or group["eps"] < 0 or group["weight_decay"] < 0:
            raise ValueError("lr, eps and weight_decay must not be negative")

    # -- the state ----------------------------------------------------------------------------------------------------
    def _build(self) -> None:
        self._parameters = [p for group in self.param_groups for p in group["params"]]
        first = self._parameters[0]
        if first.dtype not in nat.DTYPE_CODES:
            raise ValueError(f"parameters must be float32, float16 or bfloat16, not {first.dtype}")
        for p in self._parameters:
            if not p.is_cuda:
                raise ValueError("card_playing_gym_b200 kernels take CUDA tensors only (there is no CPU path)")
            if p.dtype != first.dtype or p.device != first.device:
                raise ValueError("parameters must share one dtype and one device")
            if not p.is_contiguous():
                raise ValueError("parameters must be contiguous")
        device = first.device
        starts, total = [], 0
        for p in self._parameters:
            starts.append(total)
            total += -(-p.numel() // BLOCK) * BLOCK
        total = max(total, BLOCK)
        flat: dict[str, torch.Tensor] = {}
        if self.state_bits == 32:
            flat["exp_avg"] = torch.zeros(total, device=device)
            flat["exp_avg_sq"] = torch.zeros(total, device=device)
        else:
            for name in ("exp_avg", "exp_avg_sq_root"):
                flat[name] = torch.zeros(total, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
                flat[name + "_scale"] = torch.zeros(total // BLOCK, device=device)
        if first.dtype != torch.float32:
            flat["master"] = torch.zeros(total, device=device)
        self.flat = flat
        self.steps = torch.zeros((), dtype=torch.int64, device=device)
        self.grad_norm = torch.zeros((), device=device)
        self._control = torch.zeros(nat.query("cg_adamw_control_bytes", len(self.param_groups)), dtype=torch.uint8,
                                    device=device)
        for p, start in zip(self._parameters, starts):
            size = p.numel()
            views = {}
            for name, value in flat.items():
                if name.endswith("_scale"):
                    views[name] = value[start // BLOCK:start // BLOCK + -(-size // BLOCK)]
                else:
                    views[name] = value[start:start + size].view(p.shape)
            if "master" in views:
                views["master"].copy_(p.detach())
            self.state[p] = views
        # What the master copies were last known to follow.
        self._versions = [p._version for p in self._parameters]
        self._addresses = array("Q", map(torch.Tensor.data_ptr, self._parameters))
        # The host's side of the step: extents and groups are fixed, addresses are gathered at every step.
        self._table = (nat.AdamWTensor * len(self._parameters))()
        self._dtype = first.dtype
        self._bytes = [p.nbytes for p in self._parameters]
        need = nat.query("cg_adamw_workspace_bytes", len(self._table)) if self.max_norm else 0
        self._workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        index = 0
        for number, group in enumerate(self.param_groups):
            for _ in group["params"]:
                self._table[index].numel = self._parameters[index].numel()
                self._table[index].state = starts[index]
                self._table[index].group = number
                index += 1
        self._groups = (nat.AdamWGroup * len(self.param_groups))()
        self._built = True

    def state_dict(self) -> dict:
        """torch's layout, with the step count beside it."""

        return {**super().state_dict(), "steps": self.steps.clone(), "state_bits": self.state_bits}

    def load_state_dict(self, state_dict: dict) -> None:
        """Copies a ``state_dict`` of an optimizer over the same parameters, in order, into the flat state."""

        if state_dict.get("state_bits") != self.state_bits:
            raise ValueError(f"a state of {state_dict.get('state_bits')} bits does not load into {self.state_bits}")
        saved = state_dict["param_groups"]
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the saved parameter groups have other sizes")
        order = [i for group in saved for i in group["params"]]
        for index, p in zip(order, self._parameters):
            entry = state_dict["state"][index]
            if {k: v.shape for k, v in entry.items()} != {k: v.shape for k, v in self.state[p].items()}:
                raise ValueError("the saved state has other names or shapes")
        for index, p in zip(order, self._parameters):
            for name, value in state_dict["state"][index].items():
                self.state[p][name].copy_(value)
        for group, entry in zip(self.param_groups, saved):
            group.update({k: v for k, v in entry.items() if k != "params"})
        self.steps.copy_(state_dict["steps"])

    # -- the step -----------------------------------------------------------------------------------------------------
    def _check(self, params: list, grads: list) -> None:
        """That the table still describes the parameters and gradients: one pass per property, for the host's sake.

        torch holds a gradient to its parameter's shape, dtype and device when it is set; its size in bytes is checked
        here again, since the parameter may have changed between."""

        sizes, given = self._bytes, [g for g in grads if g is not None]
        if len(given) != len(grads):
            sizes = [n for g, n in zip(grads, sizes) if g is not None]
            grads = given
        if (list(map(_bytes_of, params)) != self._bytes or set(map(_dtype_of, params)) != {self._dtype}
                or set(map(torch.Tensor.get_device, params)) != {self.steps.get_device()}
                or not all(map(torch.Tensor.is_contiguous, params))):
            raise ValueError("a parameter has changed its size, dtype, device or layout since the optimizer was built")
        if set(map(_layout_of, grads)) - {torch.strided} or not all(map(torch.Tensor.is_contiguous, grads)):
            raise ValueError("a gradient is not dense and contiguous")
        if list(map(_bytes_of, grads)) != sizes:
            raise ValueError("a gradient has not its parameter's size")

    def _follow(self, params: list, addresses: array) -> None:
        """Takes parameters that something else has written to into their master copies. An entry that is its master
        rounded keeps the master's low bits, so that a checkpoint's parameters and masters load in either order."""

        moved = addresses != self._addresses
        for p, known in zip(params, self._versions):
            if moved or p._version != known:
                master, value = self.state[p]["master"], p.detach()
                master.copy_(torch.where(master.to(value.dtype) == value, master, value.float()))
        self._addresses = addresses

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        flat, device = self.flat, self.steps.device
        params = self._parameters
        grads = [p.grad for p in params]
        self._check(params, grads)
        table = self._table
        from_params = array("Q", map(torch.Tensor.data_ptr, params))
        from_grads = array("Q", [0 if g is None else g.data_ptr() for g in grads])
        if "master" in flat and ([p._version for p in params] != self._versions or from_params != self._addresses):
            self._follow(params, from_params)
        for entry, group in zip(self._groups, self.param_groups):
            entry.lr, entry.eps, entry.weight_decay = group["lr"], group["eps"], group["weight_decay"]
            entry.beta1, entry.beta2 = group["betas"]
        second = flat["exp_avg_sq" if self.state_bits == 32 else "exp_avg_sq_root"]
        workspace = self._workspace
        with nat.on_device(device):
            nat.call("cg_adamw_step", table, from_params.buffer_info()[0], from_grads.buffer_info()[0], len(table),
                     nat.DTYPE_CODES[self._dtype], self._groups, len(self._groups), self.state_bits,
                     nat.ptr(flat["exp_avg"]), nat.ptr(flat.get("exp_avg_scale")), nat.ptr(second),
                     nat.ptr(flat.get("exp_avg_sq_root_scale")), nat.ptr(flat.get("master")), nat.ptr(self.steps),
                     float(self.max_norm or 0.0), nat.ptr(self.grad_norm), nat.ptr(self._control),
                     nat.ptr(workspace), 0 if workspace is None else workspace.numel(), nat.stream_handle(device))
        # The kernel writes through addresses: autograd learns here that a graph's saved weights have changed.
        torch.autograd.graph.increment_version([p for p, g in zip(params, from_grads) if g] if 0 in from_grads else params)
        if "master" in flat:
            self._versions = [p._version for p in params]
        return loss
