"""Fused Adam over one flat parameter buffer per optimizer.

The reference builds two ``torch.optim.Adam`` objects (<arch>/main.py:34-44: G = encoder+decoder,
lr 1e-4; D = discriminator, lr/2; betas (0.5, 0.999), eps 1e-8, no weight decay).  Here every
parameter of an optimizer becomes a view into ONE contiguous f32 buffer and so does its gradient:
the update is a single bandwidth-bound HIP kernel (28 B/param) and the data-parallel gradient
exchange is an all-reduce over contiguous slices of that buffer with no packing copies.
"""
from __future__ import annotations

from typing import Callable, Iterable, List, Optional

import torch

from . import lib as L
from . import ops


class FlatAdam:
    ALIGN = 4           # every tensor starts at a multiple of this many elements (16 bytes)

    def __init__(self, params: Iterable[torch.nn.Parameter], lr=1e-3, betas=(0.9, 0.999), eps=1e-8):
        self.params: List[torch.nn.Parameter] = [p for p in params if p.requires_grad]
        if not self.params:
            raise ValueError("FlatAdam got an empty parameter list")
        dev = self.params[0].device
        if dev.type != "cuda":
            raise RuntimeError("FlatAdam needs parameters on the GPU (move the model first); no CPU fallback")
        self.lr, self.betas, self.eps = float(lr), (float(betas[0]), float(betas[1])), float(eps)
        self.step_count = 0
        self.offsets = []
        off = 0
        for p in self.params:
            self.offsets.append(off)
            off += (p.numel() + self.ALIGN - 1) // self.ALIGN * self.ALIGN
        self.numel = off
        self.flat_p = torch.zeros(off, dtype=torch.float32, device=dev)
        self.flat_g = torch.zeros(off, dtype=torch.float32, device=dev)
        self._alloc_state(off, dev)
        for p, o in zip(self.params, self.offsets):
            n = p.numel()
            self.flat_p[o:o + n].copy_(p.data.reshape(-1))
            p.data = self.flat_p[o:o + n].view(p.shape)
            p.grad = self.flat_g[o:o + n].view(p.shape)
        # packed-weight caches (ops.PackedWeights) of these parameters are keyed on this cell: bumped by step()
        self._epoch = ops.EpochCell(ops.PARAM_EPOCH[0] + 1)
        for p in self.params:
            p._vg_epoch = self._epoch
        ops.PARAM_EPOCH[0] += 1

    def _alloc_state(self, n: int, dev):
        self.exp_avg = torch.zeros(n, dtype=torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(n, dtype=torch.float32, device=dev)

    # torch.optim surface used by the training loop
    def zero_grad(self, set_to_none: bool = False):
        self.flat_g.zero_()
        base_p, base_g = self.flat_p.data_ptr(), self.flat_g.data_ptr()
        for p, o in zip(self.params, self.offsets):
            if p.data_ptr() != base_p + 4 * o:
                # someone rebound p.data (model.to(), .float(), a manual assignment): the forward would read that
                # storage while step() updates flat_p.  Take the new values and alias again.
                if p.device != self.flat_p.device or p.dtype != torch.float32:
                    raise RuntimeError("FlatAdam: a parameter left the optimizer's device/dtype; rebuild the optimizers")
                self.flat_p[o:o + p.numel()].copy_(p.data.reshape(-1))
                p.data = self.flat_p[o:o + p.numel()].view(p.shape)
                self._epoch[0] += 1
            if p.grad is None or p.grad.data_ptr() != base_g + 4 * o:   # re-attach if someone set .grad = None
                p.grad = self.flat_g[o:o + p.numel()].view(p.shape)

    def step(self, grad_scale: float = 1.0):
        self.step_count += 1
        self._update(grad_scale)
        self._epoch[0] += 1
        ops.repack_all(self._epoch)         # every packed weight image of these parameters, one launch

    def _update(self, grad_scale: float):
        L.check(L.load().vg_adam_step(self.flat_p.data_ptr(), self.flat_g.data_ptr(), self.exp_avg.data_ptr(),
                                      self.exp_avg_sq.data_ptr(), self.numel, self.lr, self.betas[0], self.betas[1],
                                      self.eps, self.step_count, grad_scale, L.stream()), "adam_step")

    @property
    def param_groups(self):
        return [{"params": self.params, "lr": self.lr, "betas": self.betas, "eps": self.eps}]

    def set_lr(self, lr: float):
        self.lr = float(lr)

    def state_dict(self):
        """torch.optim.Adam-compatible layout ({'state': {i: {step, exp_avg, exp_avg_sq}}, 'param_groups': [...]})."""
        state = {}
        for i, (p, o) in enumerate(zip(self.params, self.offsets)):
            n = p.numel()
            state[i] = {"step": torch.tensor(float(self.step_count)),
                        "exp_avg": self.exp_avg[o:o + n].view(p.shape).clone(),
                        "exp_avg_sq": self.exp_avg_sq[o:o + n].view(p.shape).clone()}
        return {"state": state, "param_groups": [{"lr": self.lr, "betas": self.betas, "eps": self.eps, "weight_decay": 0,
                                                  "amsgrad": False, "params": list(range(len(self.params)))}]}

    def load_state_dict(self, sd):
        for i, (p, o) in enumerate(zip(self.params, self.offsets)):
            st = sd["state"].get(i)
            if st is None:
                continue
            n = p.numel()
            self.exp_avg[o:o + n].copy_(st["exp_avg"].reshape(-1))
            self.exp_avg_sq[o:o + n].copy_(st["exp_avg_sq"].reshape(-1))
            self.step_count = int(st["step"])
        g = sd["param_groups"][0]
        self.lr, self.betas, self.eps = float(g["lr"]), tuple(g["betas"]), float(g["eps"])


class FlatAdamW(FlatAdam):
    """AdamW (decoupled weight decay) over all tensors of an optimizer in one launch, states in 32 or in 8 bits.

    ``p = p (1 - lr wd) - lr m^ / (sqrt(v^) + eps)``; ``decay_filter(parameter)`` says which parameters are decayed (default:
    all, as in torch.optim.AdamW).  Hyperparameters may change between steps.

    ``state_bits=8``: the moments take 2 bytes a parameter instead of 8.  Every 256 elements of a tensor share one f32 scale for
    ``exp_avg`` and one for ``root_sq`` (the root of the second moment; half the dynamic range of the moment itself), kept as
    e4m3 values (``exp_avg * exp_avg_scale``).  A step uses this step's moments before they are rounded.  An element whose
    gradient is not finite keeps NaN moments, as it would in 32 bits; the rest of its 256 is not touched.

    ``rounding`` (8 bits): 'nearest' leaves a moment where it is when a step changes it by less than half a code, 3 to 6 %, and
    with ``betas[1] = 0.999`` nearly all do: only the largest of its 256 is followed, through the scale.  Where gradients inside a
    block change against each other, second moments are wrong by that ratio for good (half of a block's gradients grow three
    times: the other half's root is 2.3 times too large 1000 steps later), and with them those elements' step sizes.
    'stochastic' rounds up with the probability of what is cut off: moments follow on average, each with a noise of some 20 %.
    Its chance comes from an element's place, its gradient and the step's number, so a run repeats bit for bit; a step takes a
    tenth to a fifth longer (2.8 M parameters: 12.2 us, 10.2 to nearest; 169 M: 515, 470).  It is what a long run should take, and
    what ``config.optimizer = 'adamw8bit'`` does.

    ``load_state_dict`` takes the hyperparameters of the file, as torch does: a ``FlatAdam`` file (32 bits) brings a weight
    decay of 0.  8- and 32-bit states are not converted into each other (ValueError).  A step captured into a graph repeats its
    learning rate and bias correction on every replay."""

    ALIGN = 256         # elements that share a scale (csrc/adamw.hip)

    def __init__(self, params: Iterable[torch.nn.Parameter], lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 decay_filter: Optional[Callable[[torch.nn.Parameter], bool]] = None, state_bits: int = 32, rounding: str = "nearest"):
        if state_bits not in (8, 32):
            raise ValueError(f"FlatAdamW: state_bits must be 8 or 32, got {state_bits}")
        if rounding not in ("nearest", "stochastic") or (rounding == "stochastic" and state_bits != 8):
            raise ValueError(f"FlatAdamW: rounding must be 'nearest' or, with state_bits=8, 'stochastic', got {rounding!r} with {state_bits} bits")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError(f"FlatAdamW: lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
        self.state_bits, self.rounding, self.weight_decay = state_bits, rounding, float(weight_decay)
        params = list(params)
        if any(p.dtype != torch.float32 or p.device != params[0].device for p in params if p.requires_grad):
            raise RuntimeError("FlatAdamW needs float32 parameters on one GPU")
        super().__init__(params, lr, betas, eps)
        self.decays = [decay_filter is None or bool(decay_filter(p)) for p in self.params]
        ends = self.offsets[1:] + [self.numel]
        blocks = torch.tensor([(hi - lo) // self.ALIGN for lo, hi in zip(self.offsets, ends)])
        self._decay = None if all(self.decays) else torch.tensor(self.decays).to(torch.uint8).repeat_interleave(blocks).to(self.flat_p.device)

    def _alloc_state(self, n: int, dev):
        if self.state_bits == 32:
            return super()._alloc_state(n, dev)
        self.exp_avg = torch.zeros(n, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.root_sq = torch.zeros(n, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
        self.exp_avg_scale = torch.zeros(n // self.ALIGN, dtype=torch.float32, device=dev)
        self.root_sq_scale = torch.zeros(n // self.ALIGN, dtype=torch.float32, device=dev)

    def step(self, grad_scale: float = 1.0):
        with ops._on_device("adamw_step", self.flat_p):      # the update and the re-packed weight images
            super().step(grad_scale)

    def _update(self, grad_scale: float):
        lib = L.load()
        tail = (L.ptr(self._decay), self.numel, self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay, self.step_count,
                grad_scale)
        if self.state_bits == 32:
            L.check(lib.vg_adamw_step(self.flat_p.data_ptr(), self.flat_g.data_ptr(), self.exp_avg.data_ptr(),
                                      self.exp_avg_sq.data_ptr(), *tail, L.stream()), "adamw_step")
        else:
            step8 = lib.vg_adamw8_step if self.rounding == "nearest" else lib.vg_adamw8_dithered_step
            L.check(step8(self.flat_p.data_ptr(), self.flat_g.data_ptr(), self.exp_avg.data_ptr(), self.exp_avg_scale.data_ptr(),
                          self.root_sq.data_ptr(), self.root_sq_scale.data_ptr(), *tail, L.stream()), "adamw8_step")

    @property
    def param_groups(self):
        return [{"params": self.params, "lr": self.lr, "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay}]

    def state_dict(self):
        """32 bits: torch.optim.AdamW's layout.  8 bits: the e4m3 codes as uint8 and their scales, per parameter."""
        if self.state_bits == 32:
            sd = super().state_dict()
        else:
            state = {}
            for i, (p, o) in enumerate(zip(self.params, self.offsets)):
                n, b, e = p.numel(), o // self.ALIGN, (o + p.numel() + self.ALIGN - 1) // self.ALIGN
                state[i] = {"step": torch.tensor(float(self.step_count)),
                            "exp_avg_codes": self.exp_avg[o:o + n].view(torch.uint8).view(p.shape).clone(),
                            "exp_avg_scale": self.exp_avg_scale[b:e].clone(),
                            "root_sq_codes": self.root_sq[o:o + n].view(torch.uint8).view(p.shape).clone(),
                            "root_sq_scale": self.root_sq_scale[b:e].clone()}
            sd = {"state": state, "param_groups": [{"lr": self.lr, "betas": self.betas, "eps": self.eps, "amsgrad": False,
                                                    "params": list(range(len(self.params)))}]}
        sd["param_groups"][0]["weight_decay"] = self.weight_decay
        return sd

    def load_state_dict(self, sd):
        eight = [i for i, st in sd["state"].items() if "exp_avg_codes" in st]
        if (self.state_bits == 8) != bool(eight) and sd["state"]:
            raise ValueError(f"FlatAdamW: the file holds {'8' if eight else '32'}-bit states, the optimizer keeps {self.state_bits} bits")
        if self.state_bits == 32:
            super().load_state_dict(sd)
        else:
            for i, (p, o) in enumerate(zip(self.params, self.offsets)):
                st = sd["state"].get(i)
                if st is None:
                    continue
                n, b, e = p.numel(), o // self.ALIGN, (o + p.numel() + self.ALIGN - 1) // self.ALIGN
                self.exp_avg.view(torch.uint8)[o:o + n].copy_(st["exp_avg_codes"].reshape(-1))
                self.root_sq.view(torch.uint8)[o:o + n].copy_(st["root_sq_codes"].reshape(-1))
                self.exp_avg_scale[b:e].copy_(st["exp_avg_scale"])
                self.root_sq_scale[b:e].copy_(st["root_sq_scale"])
                self.step_count = int(st["step"])
            g = sd["param_groups"][0]
            self.lr, self.betas, self.eps = float(g["lr"]), tuple(g["betas"]), float(g["eps"])
        self.weight_decay = float(sd["param_groups"][0].get("weight_decay", self.weight_decay))


class StepLR:
    """torch.optim.lr_scheduler.StepLR(step_size=30, gamma=0.5) as used by <arch>/main.py:46-48."""

    def __init__(self, optimizer: FlatAdam, step_size: int, gamma: float = 0.1):
        self.opt, self.step_size, self.gamma = optimizer, step_size, gamma
        self.base_lr, self.last_epoch = optimizer.lr, 0

    def step(self):
        self.last_epoch += 1
        self.opt.set_lr(self.base_lr * self.gamma ** (self.last_epoch // self.step_size))

    def state_dict(self):
        return {"step_size": self.step_size, "gamma": self.gamma, "base_lrs": [self.base_lr], "last_epoch": self.last_epoch}

    def load_state_dict(self, sd):
        self.last_epoch = sd["last_epoch"]
        self.base_lr = sd["base_lrs"][0]
        self.opt.set_lr(self.base_lr * self.gamma ** (self.last_epoch // self.step_size))
