"""AdamW over many tensors in one launch, with its two moments in 8 bits or in 32.

The parameters may lie anywhere (they need no common buffer) and be fp32 or bf16.  The moments of all of them live in flat
buffers, every tensor's on a multiple of 256 values.  With 8 bits the first moment and the ROOT of the second are e4m3
codes with one power-of-two scale for every 256 values: 2.008 bytes a parameter instead of 8.  Checkpoints hold the
moments as fp32 ``exp_avg`` and ``exp_avg_sq``, the names and shapes that ``FusedAdamW`` and ``torch.optim.AdamW`` write, so
a run may change between them; encoding what was decoded gives the same values, so saving and loading changes nothing.
Update rule and defaults: torch.optim.AdamW, as configured in maester/config.py:147-154.
"""
from __future__ import annotations

import math

import numpy as np
import torch
from torch.optim import Optimizer

from maester_b200.ops import reference as ref

_TYPES = (torch.float32, torch.bfloat16)


class AdamWMulti(Optimizer):
    """``state_bits``: 8 or 32.  All parameters on one device, contiguous, fp32 or bf16, with gradients of their own type; a
    parameter without a gradient is left alone and its step number stays.  bf16 parameters are read, updated in fp32 and
    rounded once (to nearest).  ``step()`` cannot be captured into a CUDA graph: the learning rate and the step number are
    launch arguments.  Parameters cannot be added later, and the optimizer cannot be copied or pickled as an object (use
    ``state_dict``)."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 8, fused=None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits has to be 8 or 32, got {state_bits!r}")
        self._sealed = False
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        for g in self.param_groups:
            b1, b2 = g["betas"]
            if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and g["eps"] >= 0.0 and g["weight_decay"] >= 0.0 and g["lr"] >= 0.0):
                raise ValueError(f"lr, eps and weight decay have to be at least 0, betas in [0, 1): got lr={g['lr']}, "
                                 f"betas={g['betas']}, eps={g['eps']}, weight_decay={g['weight_decay']}")
        self.state_bits = state_bits
        every = [p for g in self.param_groups for p in g["params"]]
        self.device = every[0].device
        self._off: dict[torch.Tensor, tuple[int, int]] = {}   # parameter -> (state offset, elements)
        total = 0
        for p in every:
            if p.device != self.device:
                raise ValueError(f"parameters on {self.device} and on {p.device}: one optimizer drives one device")
            if p.dtype not in _TYPES:
                raise TypeError(f"fp32 or bf16 parameters are wanted, got {p.dtype}")
            if not p.is_contiguous():
                raise ValueError(f"a parameter of shape {tuple(p.shape)} is not contiguous (strides {p.stride()})")
            self._off[p] = (total, p.numel())
            total += -(-p.numel() // ref.STATE_BLOCK) * ref.STATE_BLOCK
        if state_bits == 8:
            blocks = total // ref.STATE_BLOCK
            code = lambda: torch.zeros(total, device=self.device, dtype=torch.float8_e4m3fn)
            exps = lambda k: torch.full((blocks,), k + 127, device=self.device, dtype=torch.uint8)
            self._buffers = {"exp_avg": code(), "exp_avg_exp": exps(ref.STATE_MIN_EXP),
                             "exp_avg_root": code(), "exp_avg_root_exp": exps(ref.ROOT_MIN_EXP)}
        else:
            self._buffers = {k: torch.zeros(total, device=self.device) for k in ("exp_avg", "exp_avg_sq")}
        self._steps: dict[torch.Tensor, int] = {p: 0 for p in every}
        self._copies: dict[torch.Tensor, torch.Tensor] = {}
        self.writes_lowp = False    # the sharding runtime's 16-bit parameters are written by step()
        self._sealed = True

    def add_param_group(self, group) -> None:
        if self._sealed:
            raise RuntimeError("the state buffers are laid out once: give every parameter to the constructor")
        super().add_param_group(group)

    def state_buffers(self) -> dict[str, torch.Tensor]:
        """The flat state buffers themselves: ``exp_avg``, ``exp_avg_root`` (codes) with ``exp_avg_exp``,
        ``exp_avg_root_exp`` (one biased exponent for 256 values), or fp32 ``exp_avg``, ``exp_avg_sq``.  A parameter's part
        starts where the parts before it, each rounded up to 256 values, end."""
        return dict(self._buffers)

    def attach_copies(self, copies: dict) -> None:
        """{fp32 parameter: bf16 tensor of as many elements}: ``step()`` also writes the updated value there, rounded."""
        for p, c in copies.items():
            if p not in self._off or p.dtype != torch.float32:
                raise ValueError("a 16-bit copy belongs to an fp32 parameter of this optimizer")
            if c.dtype != torch.bfloat16 or c.numel() != p.numel() or not c.is_contiguous() or c.device != self.device:
                raise ValueError(f"the copy of a parameter of {p.numel()} elements has to be a contiguous bf16 tensor of as "
                                 f"many on {self.device}")
        self._copies.update(copies)

    def attach_sharding(self, sharded) -> None:
        """Write the sharding runtime's 16-bit shard with the update (called by the optimizer builder)."""
        lp = getattr(sharded, "shard_lp", None)
        if lp is None or lp.dtype != torch.bfloat16 or not lp.is_cuda or lp.device != self.device or sharded.fused \
                or sharded.cpu_offload:
            return
        seg = sharded.flat_segments()
        self.attach_copies({p: lp[seg[p][0]:seg[p][0] + n] for p, (_, n) in self._off.items() if n})
        self.writes_lowp = True

    # ---- stepping
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamWMulti.step() cannot be captured: learning rate and step number are launch arguments")
        work: dict[tuple, list] = {}
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.layout is not torch.strided or g.dtype != p.dtype or g.device != p.device:
                    raise RuntimeError(f"the gradient of a {p.dtype} parameter on {p.device} has to be a dense tensor of its "
                                       f"type there, got {g.dtype} on {g.device} ({g.layout})")
                if p.dtype not in _TYPES or p.device != self.device or p.numel() != self._off[p][1] or not p.is_contiguous():
                    raise RuntimeError("a parameter was replaced by one of another type, device or layout")
                work.setdefault((gi, p.dtype, self._steps[p] + 1), []).append((p, g if g.is_contiguous() else g.contiguous()))
        for (gi, dtype, t), pairs in work.items():
            group = self.param_groups[gi]
            b1, b2 = group["betas"]
            lr = float(group["lr"])
            hyper = dict(b1=b1, b2=b2, decay=1 - lr * group["weight_decay"], step_size=lr / (1 - b1 ** t),
                         inv_root=1 / math.sqrt(1 - b2 ** t), eps=group["eps"])
            (self._launch if self.device.type == "cuda" else self._plain)(pairs, dtype, hyper)
            for p, _ in pairs:
                self._steps[p] = t
        return loss

    def _launch(self, pairs, dtype, h) -> None:
        from maester_b200.ops import cuda as C
        off, copies = self._off, self._copies
        rows = [(p.data_ptr(), g.data_ptr(), copies[p].data_ptr() if p in copies else 0, off[p][1], off[p][0], 0)
                for p, g in pairs]
        f = self._buffers
        m, r = f["exp_avg"], f["exp_avg_root" if self.state_bits == 8 else "exp_avg_sq"]
        C.adamw_multi(np.array(rows, dtype=np.int64), dtype == torch.bfloat16, self.state_bits, m, f.get("exp_avg_exp"), r,
                      f.get("exp_avg_root_exp"),
                      (h["b1"], 1 - h["b1"], h["b2"], 1 - h["b2"], h["decay"], h["step_size"], h["inv_root"], h["eps"]))

    def _plain(self, pairs, dtype, h) -> None:
        for p, g in pairs:
            m, v = self._moments(p)
            new, m, root, v = ref.adamw_multi_step(p.data.float().view(-1), g.float().view(-1), m, v, **h)
            p.copy_(new.view(p.shape))
            if p in self._copies:
                self._copies[p].view(-1).copy_(p.view(-1))
            self._store(p, m, root, v)

    # ---- states
    def _moments(self, p) -> tuple[torch.Tensor, torch.Tensor]:
        """fp32 (exp_avg, exp_avg_sq) of one parameter, flat."""
        off, n = self._off[p]
        f = self._buffers
        if self.state_bits == 32:
            return f["exp_avg"][off:off + n], f["exp_avg_sq"][off:off + n]
        end = off + -(-n // ref.STATE_BLOCK) * ref.STATE_BLOCK
        blk = slice(off // ref.STATE_BLOCK, end // ref.STATE_BLOCK)
        m, r = (ref.state_decode(f[k][off:end], f[k + "_exp"][blk])[:n] for k in ("exp_avg", "exp_avg_root"))
        return m, r * r

    def _store(self, p, m=None, root=None, v=None) -> None:
        off, n = self._off[p]
        f = self._buffers
        if n == 0:
            return
        if self.state_bits == 32:
            if m is not None:
                f["exp_avg"][off:off + n].copy_(m)
            if v is not None:
                f["exp_avg_sq"][off:off + n].copy_(v)
            return
        end = off + -(-n // ref.STATE_BLOCK) * ref.STATE_BLOCK
        blk = slice(off // ref.STATE_BLOCK, end // ref.STATE_BLOCK)
        if root is None and v is not None:
            root = v.sqrt()
        for k, x, is_root in (("exp_avg", m, False), ("exp_avg_root", root, True)):
            if x is not None:
                codes, exps = ref.state_encode(torch.nn.functional.pad(x, (0, end - off - n)), is_root)
                f[k][off:end].copy_(codes)
                f[k + "_exp"][blk].copy_(exps)

    def param_state(self, p) -> dict[str, torch.Tensor]:
        """What a checkpoint holds of one parameter: ``step``, and fp32 ``exp_avg`` and ``exp_avg_sq`` of its shape."""
        m, v = self._moments(p)
        return {"step": torch.tensor(float(self._steps[p])), "exp_avg": m.clone().view(p.shape),
                "exp_avg_sq": v.clone().view(p.shape)}

    @torch.no_grad()
    def load_param_state(self, p, state: dict) -> None:
        """Take over any of ``step``, ``exp_avg``, ``exp_avg_sq`` of one parameter."""
        n = p.numel()
        flat = {}
        for k in ("exp_avg", "exp_avg_sq"):
            if k in state:
                x = state[k]
                if x.numel() != n:
                    raise ValueError(f"{k} of {x.numel()} elements for a parameter of {n}")
                flat[k] = x.detach().to(device=self.device, dtype=torch.float32).reshape(-1)
        self._store(p, m=flat.get("exp_avg"), v=flat.get("exp_avg_sq"))
        if "step" in state:
            self._steps[p] = int(state["step"])

    def state_dict(self) -> dict:
        sd = super().state_dict()
        sd["state"] = {i: self.param_state(p) for i, p in enumerate(p for g in self.param_groups for p in g["params"])}
        return sd

    def load_state_dict(self, state_dict: dict) -> None:
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        for i, p in enumerate(p for g in self.param_groups for p in g["params"]):
            if i in state_dict["state"]:
                self.load_param_state(p, state_dict["state"][i])
