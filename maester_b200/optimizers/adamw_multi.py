"""AdamW over many tensors in one launch, with its two moments in 8 bits or in 32.

The parameters may lie anywhere (they need no common buffer) and be fp32 or bf16.  The moments of all of them live in flat
buffers, every tensor's on a multiple of 256 values.  With 8 bits the first moment and the ROOT of the second are e4m3
codes with one power-of-two scale for every 256 values: 2.008 bytes a parameter instead of 8.  An average that moves by
less than half a code a step would stand still if it were rounded to nearest, so from a parameter's second step on a value
becomes one of its two neighbouring codes at random, with itself (for the root, its square) as the expectation; the random
numbers are a hash of the step number and the place, so a run repeats, also one that was saved and loaded.  Checkpoints hold the
moments as fp32 ``exp_avg`` and ``exp_avg_sq``, the names and shapes that ``FusedAdamW`` and ``torch.optim.AdamW`` write, so
a run may change between them; encoding what was decoded gives the same values, so saving and loading changes nothing.
Update rule and defaults: torch.optim.AdamW, as configured in maester/config.py:147-154.
"""
from __future__ import annotations

import math
import operator

import numpy as np
import torch
from torch.autograd.graph import increment_version
from torch.optim import Optimizer

from maester_b200.ops import reference as ref

_TYPES = (torch.float32, torch.bfloat16)
NOISE_FROM = 2      # step number of a parameter from which its 8-bit codes are rounded stochastically
# a step looks at every tensor: mapped over the lists, which takes half the time of a loop
_grad, _dtype = map(operator.attrgetter, ("grad", "dtype"))
_device, _numel, _contiguous, _address = (torch.Tensor.get_device, torch.Tensor.numel, torch.Tensor.is_contiguous,
                                          torch.Tensor.data_ptr)
_held_at, _held_bytes = torch.UntypedStorage.data_ptr, torch.UntypedStorage.nbytes


def _missing(x: torch.Tensor) -> int:
    """Bytes that a tensor's storage is short of what the tensor spans (a storage may have been resized under it)."""
    return (x.storage_offset() + x.numel()) * x.element_size() - x.untyped_storage().nbytes() if x.numel() else 0


def _overlap(tensors) -> bool:
    """Do two of these contiguous tensors share memory?  (One whose storage has been freed has none.)"""
    spans = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size()) for x in tensors
                   if x.numel() and x.untyped_storage().nbytes())
    return any(a[1] > b[0] > 0 for a, b in zip(spans, spans[1:]))


class _Slot:
    """A parameter, its row in the batch's table, where its states lie, and how many steps it has taken."""

    __slots__ = ("param", "row", "offset", "numel", "step", "copy")

    def __init__(self, param, row: int, offset: int, numel: int):
        self.param, self.row, self.offset, self.numel, self.step, self.copy = param, row, offset, numel, 0, None


class _Batch:
    __slots__ = ("group", "dtype", "slots", "params", "sizes", "memory", "storages", "bytes", "addresses", "table")

    def __init__(self, group: int, dtype: torch.dtype):
        self.group, self.dtype, self.slots = group, dtype, []


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
        # (the rest is what torch.optim.AdamW keeps in its groups: a checkpoint's reader asks for every key that it has itself)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, amsgrad=False, maximize=False,
                                      foreach=None, capturable=False, differentiable=False, fused=True,
                                      decoupled_weight_decay=True))
        for g in self.param_groups:
            b1, b2 = g["betas"]
            if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and g["eps"] >= 0.0 and g["weight_decay"] >= 0.0 and g["lr"] >= 0.0):
                raise ValueError(f"lr, eps and weight decay have to be at least 0, betas in [0, 1): got lr={g['lr']}, "
                                 f"betas={g['betas']}, eps={g['eps']}, weight_decay={g['weight_decay']}")
        self.state_bits = state_bits
        every = [p for g in self.param_groups for p in g["params"]]
        self.device = every[0].device
        self._slots: dict[torch.Tensor, _Slot] = {}
        self._batches: list[_Batch] = []                      # parameters of one group and type: one table, one launch
        total = 0
        of = {id(p): gi for gi, g in enumerate(self.param_groups) for p in g["params"]}
        for p in every:
            if p.device != self.device:
                raise ValueError(f"parameters on {self.device} and on {p.device}: one optimizer drives one device")
            if p.dtype not in _TYPES:
                raise TypeError(f"fp32 or bf16 parameters are wanted, got {p.dtype}")
            if not p.is_contiguous():
                raise ValueError(f"a parameter of shape {tuple(p.shape)} is not contiguous (strides {p.stride()})")
            batch = next((b for b in self._batches if b.group == of[id(p)] and b.dtype == p.dtype), None)
            if batch is None:
                batch = _Batch(of[id(p)], p.dtype)
                self._batches.append(batch)
            self._slots[p] = slot = _Slot(p, len(batch.slots), total, p.numel())
            batch.slots.append(slot)
            total += -(-p.numel() // ref.STATE_BLOCK) * ref.STATE_BLOCK
        if _overlap(every):
            raise ValueError("two parameters share memory, or one is given twice: a step would update it twice at a time")
        if state_bits == 8:
            blocks = total // ref.STATE_BLOCK
            code = lambda: torch.zeros(total, device=self.device, dtype=torch.float8_e4m3fn)
            exps = lambda k: torch.full((blocks,), k + 127, device=self.device, dtype=torch.uint8)
            self._buffers = {"exp_avg": code(), "exp_avg_exp": exps(ref.STATE_MIN_EXP),
                             "exp_avg_root": code(), "exp_avg_root_exp": exps(ref.ROOT_MIN_EXP)}
        else:
            self._buffers = {k: torch.zeros(total, device=self.device) for k in ("exp_avg", "exp_avg_sq")}
        for b in self._batches:
            b.params, b.sizes = [s.param for s in b.slots], [s.numel for s in b.slots]
            b.table = np.array([(0, 0, 0, s.numel, s.offset, 0) for s in b.slots], dtype=np.int64)
            self._take_memory(b)
        self._copy_storages, self._copy_memory = [], []       # of the 16-bit copies: theirs once each, and where they were
        self._mark()
        self.writes_lowp = False    # the sharding runtime's 16-bit parameters are written by step()
        self._sealed = True

    def _mark(self) -> None:
        """Entries in ``state``: torch's checkpoint helpers let an optimizer without any step with zeros first."""
        for p in self._slots:
            self.state[p] = {}

    def add_param_group(self, group) -> None:
        if self._sealed:
            raise RuntimeError("the state buffers are laid out once: give every parameter to the constructor")
        super().add_param_group(group)

    def __getstate__(self):
        raise TypeError("AdamWMulti cannot be copied or pickled as an object: use state_dict()")

    def state_buffers(self) -> dict[str, torch.Tensor]:
        """The flat state buffers themselves: ``exp_avg``, ``exp_avg_root`` (codes) with ``exp_avg_exp``,
        ``exp_avg_root_exp`` (one biased exponent for 256 values), or fp32 ``exp_avg``, ``exp_avg_sq``.  A parameter's part
        starts where the parts before it, each rounded up to 256 values, end."""
        return dict(self._buffers)

    def attach_copies(self, copies: dict) -> None:
        """{fp32 parameter: bf16 tensor of as many elements}: ``step()`` also writes the updated value there, rounded.  A
        copy whose memory has been freed (its storage resized to nothing) when ``step()`` is called is left out."""
        for p, c in copies.items():
            if p not in self._slots or p.dtype != torch.float32:
                raise ValueError("a 16-bit copy belongs to an fp32 parameter of this optimizer")
            if c.dtype != torch.bfloat16 or c.numel() != p.numel() or not c.is_contiguous() or c.device != self.device:
                raise ValueError(f"the copy of a parameter of {p.numel()} elements has to be a contiguous bf16 tensor of as "
                                 f"many on {self.device}")
        after = {p: x.copy for p, x in self._slots.items() if x.copy is not None} | copies
        if _overlap([*self._slots, *after.values()]):
            raise ValueError("16-bit copies share memory, with one another or with a parameter")
        for p, c in copies.items():
            self._slots[p].copy = c.detach()   # (of its own: the caller's tensor may change its shape or take another storage)
        held = [x.copy.untyped_storage() for x in self._slots.values() if x.copy is not None]
        self._copy_storages, self._copy_memory = list({s._cdata: s for s in held}.values()), None
        self._find_copies()

    def _find_copies(self) -> None:
        """Note where the copies are.  Holding a tensor does not keep its storage from being resized: looked at in every step."""
        now = list(map(_held_at, self._copy_storages)) + list(map(_held_bytes, self._copy_storages))
        if now == self._copy_memory:
            return
        for b in self._batches:
            at = []
            for x in b.slots:
                gone = x.copy is None or x.copy.untyped_storage().nbytes() == 0
                if not gone and _missing(x.copy) > 0:
                    raise RuntimeError(f"the storage of a 16-bit copy of {x.numel} elements has been resized to "
                                       f"{x.copy.untyped_storage().nbytes()} bytes")
                at.append(0 if gone else x.copy.data_ptr())
            b.table[:, 2] = at
        self._copy_memory = now

    def attach_sharding(self, sharded) -> None:
        """Write the sharding runtime's 16-bit shard with the update (called by the optimizer builder)."""
        lp = getattr(sharded, "shard_lp", None)
        if lp is None or lp.dtype != torch.bfloat16 or not lp.is_cuda or lp.device != self.device or sharded.fused \
                or sharded.cpu_offload:
            return
        seg = sharded.flat_segments()
        self.attach_copies({p: lp[seg[p][0]:seg[p][0] + s.numel] for p, s in self._slots.items() if s.numel})
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
        for key in ("amsgrad", "maximize"):         # (another optimizer's settings may have been loaded)
            if any(g.get(key) for g in self.param_groups):
                raise RuntimeError(f"AdamWMulti has no {key}")
        self._find_parameters()
        self._find_copies()
        work = []                                   # (everything is looked at before anything runs)
        for batch in self._batches:
            slots, sizes, grads = batch.slots, batch.sizes, list(map(_grad, batch.params))
            if any(g is None for g in grads):
                live = [i for i, g in enumerate(grads) if g is not None]
                if not live:
                    continue
                slots, sizes, grads = ([x[i] for i in live] for x in (slots, sizes, grads))
            if not self._check(batch.dtype, sizes, grads):
                grads = [g.contiguous() for g in grads]
            work.append((batch, slots, grads))
        for batch, slots, grads in work:
            group = self.param_groups[batch.group]
            b1, b2 = group["betas"]
            lr = float(group["lr"])
            steps = {x.step for x in slots}     # one number, unless some had no gradient before
            for t in sorted(steps, reverse=True):                 # (downwards: a slot that has moved on is not met again)
                some = (slots, grads) if len(steps) == 1 else tuple(
                    [y for x, y in zip(slots, z) if x.step == t] for z in (slots, grads))
                t += 1
                hyper = dict(b1=b1, b2=b2, decay=1 - lr * group["weight_decay"], step_size=lr / (1 - b1 ** t),
                             inv_root=1 / math.sqrt(1 - b2 ** t), eps=group["eps"])
                (self._launch if self.device.type == "cuda" else self._plain)(batch, *some, hyper)
                for x in some[0]:
                    x.step = t
        return loss

    def _find_parameters(self) -> None:
        """Parameters of the size and type they had, in the memory they were in, are what they were: that memory is held, so
        nothing else can have its addresses."""
        if all(list(map(_address, b.params)) == b.addresses and list(map(_numel, b.params)) == b.sizes
               and all(map(_contiguous, b.params)) and set(map(_dtype, b.params)) == {b.dtype}
               and list(map(_held_bytes, b.storages)) == b.bytes for b in self._batches):
            return
        for b in self._batches:
            self._take_memory(b)
        if _overlap([*self._slots, *(x.copy for x in self._slots.values() if x.copy is not None)]):
            for b in self._batches:
                b.addresses = None                  # (looked at again in the next step)
            raise RuntimeError("two parameters, or a parameter and a copy, share memory: a step would update it twice at a time")

    def _take_memory(self, batch) -> None:
        """Note where the parameters are and hold that memory."""
        batch.addresses = None
        for p, n in zip(batch.params, batch.sizes):
            if p.dtype is not batch.dtype or p.device != self.device or p.numel() != n or not p.is_contiguous() or (
                    n and not p.data_ptr()) or _missing(p) > 0:
                raise RuntimeError("a parameter was replaced by one of another type, size, device or layout, or has no memory")
        batch.memory = [p.detach() for p in batch.params]
        batch.storages = list({s._cdata: s for s in (m.untyped_storage() for m in batch.memory)}.values())
        batch.bytes = list(map(_held_bytes, batch.storages))
        batch.addresses = list(map(_address, batch.memory))
        batch.table[:, 0] = batch.addresses

    def _check(self, dtype, sizes, grads) -> bool:
        """Gradients are what the table says (a kernel gets nothing but their addresses).  Are they contiguous?"""
        device = self.device.index if self.device.type == "cuda" else -1
        contiguous = all(map(_contiguous, grads))       # (no sparse gradient is)
        if not ((contiguous or all(g.layout is torch.strided for g in grads)) and set(map(_dtype, grads)) == {dtype}
                and set(map(_device, grads)) == {device} and list(map(_numel, grads)) == sizes):
            g = next(g for g, n in zip(grads, sizes) if g.dtype is not dtype or g.layout is not torch.strided
                     or g.get_device() != device or g.numel() != n)
            raise RuntimeError(f"the gradient of a {dtype} parameter on {self.device} has to be a dense tensor of its type and "
                               f"size there, got {g.dtype} {tuple(g.shape)} on {g.device} ({g.layout})")
        return contiguous

    def _launch(self, batch, slots, grads, h) -> None:
        from maester_b200.ops import cuda as C
        table = batch.table if len(slots) == len(batch.slots) else batch.table[[s.row for s in slots]]
        table[:, 1] = list(map(_address, grads))
        f, step = self._buffers, slots[0].step + 1
        key = ref.state_noise_key(step) if self.state_bits == 8 and step >= NOISE_FROM else -1
        C.adamw_multi(table, batch.dtype is torch.bfloat16, self.state_bits, f["exp_avg"], f.get("exp_avg_exp"),
                      f["exp_avg_root" if self.state_bits == 8 else "exp_avg_sq"], f.get("exp_avg_root_exp"),
                      (h["b1"], 1 - h["b1"], h["b2"], 1 - h["b2"], h["decay"], h["step_size"], h["inv_root"], h["eps"]), key)
        # (a backward pass through a graph of before this step is an error, as after torch's own optimizers)
        increment_version([x.param for x in slots])
        if self._copy_storages:
            increment_version([x.copy for x in slots if x.copy is not None])

    def _plain(self, batch, slots, grads, h) -> None:
        for s, g in zip(slots, grads):
            p = s.param
            m, v = self._moments(p)
            new, m, root, v = ref.adamw_multi_step(p.data.float().view(-1), g.float().reshape(-1), m, v, **h)
            p.copy_(new.view(p.shape))
            if batch.table[s.row, 2]:
                s.copy.view(-1).copy_(p.view(-1))
            self._store(p, m, root, v, s.step + 1)

    # ---- states
    def _moments(self, p) -> tuple[torch.Tensor, torch.Tensor]:
        """fp32 (exp_avg, exp_avg_sq) of one parameter, flat."""
        off, n = self._slots[p].offset, self._slots[p].numel
        f = self._buffers
        if self.state_bits == 32:
            return f["exp_avg"][off:off + n], f["exp_avg_sq"][off:off + n]
        end = off + -(-n // ref.STATE_BLOCK) * ref.STATE_BLOCK
        blk = slice(off // ref.STATE_BLOCK, end // ref.STATE_BLOCK)
        m, r = (ref.state_decode(f[k][off:end], f[k + "_exp"][blk])[:n] for k in ("exp_avg", "exp_avg_root"))
        return m, r * r

    def _store(self, p, m=None, root=None, v=None, step: int = 1) -> None:
        """Take over moments: as they are, or as codes, rounded as in step number ``step``."""
        off, n = self._slots[p].offset, self._slots[p].numel
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
        noise = None if step < NOISE_FROM else ref.state_noise(step, off, end - off, self.device)
        for k, x, is_root in (("exp_avg", m, False), ("exp_avg_root", root, True)):
            if x is not None:
                codes, exps = ref.state_encode(torch.nn.functional.pad(x, (0, end - off - n)), is_root, noise)
                f[k][off:end].copy_(codes)
                f[k + "_exp"][blk].copy_(exps)

    def param_state(self, p) -> dict[str, torch.Tensor]:
        """What a checkpoint holds of one parameter: ``step``, and fp32 ``exp_avg`` and ``exp_avg_sq`` of its shape, on the
        host (on the device those of all parameters would take four times the memory of 8-bit states)."""
        m, v = (x.to("cpu", copy=True).view(p.shape) for x in self._moments(p))
        return {"step": torch.tensor(float(self._slots[p].step)), "exp_avg": m, "exp_avg_sq": v}

    @staticmethod
    def _fits(p, state: dict) -> None:
        for k in ("exp_avg", "exp_avg_sq"):
            if k in state and state[k].numel() != p.numel():
                raise ValueError(f"{k} of {state[k].numel()} elements for a parameter of {p.numel()}")

    @torch.no_grad()
    def load_param_state(self, p, state: dict) -> None:
        """Take over any of ``step``, ``exp_avg``, ``exp_avg_sq`` of one parameter."""
        self._fits(p, state)
        flat = {k: state[k].detach().to(device=self.device, dtype=torch.float32).reshape(-1)
                for k in ("exp_avg", "exp_avg_sq") if k in state}
        self._store(p, m=flat.get("exp_avg"), v=flat.get("exp_avg_sq"))
        if "step" in state:
            self._slots[p].step = int(state["step"])

    def state_dict(self) -> dict:
        sd = super().state_dict()
        sd["state"] = {i: self.param_state(p) for i, p in enumerate(p for g in self.param_groups for p in g["params"])}
        return sd

    def load_state_dict(self, state_dict: dict) -> None:
        """Moments and step numbers become those of ``state_dict``; a parameter, or a part of its state, that is not in it
        starts afresh."""
        every = [p for g in self.param_groups for p in g["params"]]
        states = [state_dict["state"].get(i, {}) for g in state_dict["param_groups"] for i in g["params"]]
        for p, state in zip(every, states):     # (as many as there are, or the next call says so)
            self._fits(p, state)
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        self._mark()
        for k, x in self._buffers.items():
            x.view(torch.uint8).fill_(0 if not k.endswith("_exp") else
                                      127 + (ref.ROOT_MIN_EXP if "root" in k else ref.STATE_MIN_EXP))
        for p, state in zip(every, states):
            self._slots[p].step = 0
            self.load_param_state(p, state)
