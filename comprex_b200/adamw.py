"""AdamW over all tensors of a model in one kernel launch, with states in 32 bits or in 8.

The optimizer for gradients that are ready to be applied: those of one GPU, or those that DistributedDataParallel has
averaged through :func:`comprex_b200.ddp_hook.comprex_hook`.  (:class:`~comprex_b200.optim.ComprexOptimizer` exchanges
the gradients itself and keeps one setting for the whole model.)

    opt = cx.AdamW(model.parameters(), lr=3e-4, weight_decay=0.1, state_bits=8)

Decoupled weight decay and bias corrections as in ``torch.optim.AdamW``:

    m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2
    p = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

Tensors of 16 bits have 32-bit weights behind them, which take the step; the tensor is their rounded copy.  Every
parameter group has its own settings and every tensor its own step count: a tensor without a gradient is left alone.

States live in flat buffers in which tensor ``i`` starts at a multiple of 256 elements, in the order of the
parameters (:meth:`AdamW.flat_state`).  A tensor that is frozen has none; with its first gradient the buffers are laid
out anew.  With ``state_bits=8`` each block of 256 elements keeps ``exp_avg`` and ``exp_avg_rms``, the square root of
the second moment, as ``float8_e4m3fn`` times a power of two: 2.03 bytes an element instead of 8.  They are rounded at
random (up as often as what is cut off is part of a step), because a moving average with a beta near one would never
leave its value under rounding to nearest; the random bits are a hash of the element's place, the number of the
optimizer's step and ``seed``, so a run can be repeated bit for bit and does not depend on the launch.  A gradient that
is no number spoils its own element, and the 8-bit states of its block.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import _lib
from ._lib import ComprexError
from .optim import _dense_layout

_BLOCK = 256
_ONE_STEP = np.array([[0], [1]])


class AdamW(torch.optim.Optimizer):
    """``params``: tensors of one type (float32, bfloat16, float16) on one device, each without gaps in memory."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self._check_settings(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))
        self.state_bits, self.seed = int(state_bits), int(seed)
        chosen = [p for g in self.param_groups for p in g["params"] if p.requires_grad]
        if not chosen:
            raise ValueError("optimizer got an empty parameter list")
        self._take(chosen)

    def _take(self, chosen) -> None:
        """Lay out the flat states for these tensors, in the order of the parameters; the others rest until they get a gradient."""
        first = chosen[0]
        self._dtype, self._device = first.dtype, first.device
        self._code, self._dev = _lib.dtype_code(first.dtype), _lib.dev_code(first)
        if first.device.type not in ("cuda", "cpu"):
            raise ComprexError(f"parameters on {first.device} are not supported")
        ids = {id(p) for p in chosen}
        every = [(i, group, p) for i, (group, p) in enumerate((j, p) for j, g in enumerate(self.param_groups) for p in g["params"])]
        mine = [e for e in every if id(e[2]) in ids]
        for _, _, p in mine:
            if p.dtype != self._dtype or p.device != self._device:
                raise ComprexError("all parameters must share one dtype and live on one device")
            if p.layout != torch.strided or not _dense_layout(p):
                raise ComprexError("a parameter has gaps in memory")
        kept = dict(self.__dict__)
        try:
            self._index, group, self._params = (list(x) for x in zip(*mine))
            self._group, self._frozen = np.array(group), [p for _, _, p in every if id(p) not in ids]
            self._lay_out()
        except BaseException:
            self.__dict__.clear()
            self.__dict__.update(kept)
            raise

    @torch.no_grad()
    def _take_too(self, more) -> None:
        """Lay the flat states out anew with tensors that had none; what is there is copied into its new place."""
        self._place()
        kept = dict(self.__dict__)
        try:
            self._take(self._params + more)
            at = {id(p): i for i, p in enumerate(self._params)}
            for i, (p, first) in enumerate(zip(kept["_params"], kept["_first"])):
                j = at[id(p)]
                blocks, to = int(kept["_first"][i + 1] - first), int(self._first[j])
                for name, old in kept["_flat"].items():
                    per = 1 if name.endswith("_scale") else _BLOCK
                    self._flat[name][to * per:(to + blocks) * per].copy_(old[int(first) * per:(int(first) + blocks) * per])
                self._steps[j] = kept["_steps"][i]
            self._turns = kept["_turns"]
        except BaseException:
            self.__dict__.clear()
            self.__dict__.update(kept)
            raise

    @staticmethod
    def _check_settings(group):
        b1, b2 = group["betas"]
        if not (group["lr"] >= 0 and group["eps"] >= 0 and group["weight_decay"] >= 0 and 0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError("lr, eps and weight_decay must not be negative, betas lie in [0, 1)")

    def add_param_group(self, param_group):
        if hasattr(self, "_lay"):
            raise ComprexError("the flat states are laid out at construction: give all parameter groups there")
        super().add_param_group(param_group)

    def _lay_out(self) -> None:
        self._layout = _lib.host().layout(self._params)
        if self._layout is None:
            raise ComprexError("a parameter has no memory of its own (a fake or wrapped tensor, a sign that is only noted)")
        dev = self._device
        numel = np.array([p.numel() for p in self._params], dtype=np.int64)
        blocks = -(-numel // _BLOCK)
        first = np.concatenate(([0], np.cumsum(blocks)))
        self._first, self._numel = first, numel
        k, nblk = len(numel), int(first[-1])
        n = nblk * _BLOCK
        put = lambda a, dt: torch.from_numpy(a.astype(dt)).to(dev)  # noqa: E731
        self._lay = {
            "blk_seg": put(np.repeat(np.arange(k), blocks), np.int32), "seg_blk": put(first[:-1], np.int64),
            "seg_len": put(numel, np.int64), "seg_class": torch.zeros(k, dtype=torch.int32, device=dev),
            "seg_param": torch.zeros(k, dtype=torch.int64, device=dev), "seg_grad": torch.zeros(k, dtype=torch.int64, device=dev),
        }
        state = {}
        if self._dtype != torch.float32:
            state["master"] = torch.zeros(n, dtype=torch.float32, device=dev)
        if self.state_bits == 32:
            state |= {s: torch.zeros(n, dtype=torch.float32, device=dev) for s in ("exp_avg", "exp_avg_sq")}
        else:
            for s in ("exp_avg", "exp_avg_rms"):
                state[s] = torch.zeros(n, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
                state[s + "_scale"] = torch.zeros(nblk, dtype=torch.float32, device=dev)
        self._flat = state
        self._steps = np.zeros(k, dtype=np.int64)
        self._turns = 0                       # steps that moved any tensor: what the random bits go by
        a = self._args = _lib.AdamW()
        for name, t in self._lay.items():
            setattr(a, name, t.data_ptr())
        a.blocks, a.segs, a.dtype, a.bits = nblk, k, self._code, self.state_bits
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("exp_avg", "exp_avg_rms")
        a.m, a.v = (state[s].data_ptr() for s in names)
        if self.state_bits == 8:
            a.m_scale, a.v_scale = (state[s + "_scale"].data_ptr() for s in names)
        if "master" in state:
            a.master = state["master"].data_ptr()
            self._take_master()
        # host copies of what the device holds, and pinned buffers to bring it there
        self._now = {"seg_param": torch.zeros(k, dtype=torch.int64), "seg_grad": torch.zeros(k, dtype=torch.int64),
                     "seg_class": torch.zeros(k, dtype=torch.int32)}
        self._collect, self._scalar_type = _lib.host().collect, _lib.host().scalar_type(self._params[0])
        self._ring = {}
        self._classes, self._same = None, False
        self._place()

    def _place(self) -> None:
        """The table of the tensors' addresses.  A tensor may be another one than at construction, but not another kind: the
        flat states have its length and its memory order."""
        changed = _lib.host().addresses(self._params, self._layout, self._now["seg_param"].data_ptr())
        if changed < 0:
            raise ComprexError(f"parameter {-1 - changed} is not as it was when the optimizer was made (shape, type, device or memory "
                               "order): convert or move a model before its optimizer is made")
        if changed:
            self._upload("seg_param")

    def _upload(self, name) -> None:
        """Table ``name`` to the device, in stream order and without waiting for it."""
        try:
            self._send(name)
        except BaseException:
            self._now[name].fill_(-1)         # not what the device holds: the next step sends it
            raise

    def _send(self, name) -> None:
        src = self._now[name]
        if self._device.type != "cuda":
            self._lay[name].copy_(src)
            return
        ring = self._ring.setdefault(name, [])
        stream = torch.cuda.current_stream(self._device)
        slot = next((r for r in ring if r[1].query()), None)     # a buffer whose last copy has finished
        if slot is None and len(ring) < 4:
            slot = (torch.empty_like(src).pin_memory(), torch.cuda.Event())
            ring.append(slot)
        if slot is None:
            slot = ring.pop(0)
            slot[1].synchronize()
            ring.append(slot)
        slot[0].copy_(src)
        self._lay[name].copy_(slot[0], non_blocking=True)
        slot[1].record(stream)

    def _grads(self) -> bool:
        """Bring the table of gradient addresses up to date (0: none); whether it has changed."""
        now = self._now["seg_grad"]
        changed = self._collect(self._params, self._scalar_type, 0, now.data_ptr())
        if changed == 2:                      # rare: another type or memory order than the tensor's
            now.fill_(-1)
            for p in self._params:
                g = p.grad
                if g is None:
                    continue
                if g.layout != torch.strided or g.size() != p.size() or g.device != p.device:
                    raise ComprexError("a gradient is sparse, on another device or does not have its parameter's shape")
                if g.dtype is not self._dtype or g.stride() != p.stride() or g.is_neg() or g._is_zerotensor():
                    p.grad = torch.empty_strided(p.size(), p.stride(), dtype=self._dtype, device=p.device).copy_(g)
            changed = self._collect(self._params, self._scalar_type, 0, now.data_ptr())
            if changed == 2:
                now.fill_(-1)
                raise ComprexError("a gradient does not have its parameter's shape, or no memory of its own")
        if changed:
            self._upload("seg_grad")
        return bool(changed)

    def _make_classes(self, steps):
        """Tensors that step with the same settings and step count share a row of settings: (group, steps) of the rows."""
        pair, of = np.unique(np.stack((self._group, steps))[:, self._has], axis=1, return_inverse=True)
        table = np.full(len(steps), -1, dtype=np.int32)
        table[self._has] = of.reshape(-1)
        table = torch.from_numpy(table)
        if not torch.equal(table, self._now["seg_class"]):
            self._now["seg_class"].copy_(table)
            self._upload("seg_class")
        return pair

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for g in self.param_groups:
            self._check_settings(g)
        if self._device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise ComprexError("a step cannot be captured in a CUDA graph: its settings and step count are the launch's own")
        if self._device.type == "cuda" and torch.cuda.current_device() != self._device.index:
            with torch.cuda.device(self._device):
                self._step()
        else:
            self._step()
        return loss

    def _step(self) -> None:
        if self._frozen:
            thawed = _lib.host().graded(self._frozen)
            if thawed:
                self._take_too(thawed)
        self._place()
        if self._grads() or self._classes is None:
            has = (self._now["seg_grad"] != 0).numpy()
            self._same = bool(has.all())
            self._has = has
            self._classes = None
        a = self._args
        steps = self._steps + self._has
        if self._same and self._classes is not None:
            classes = self._classes + _ONE_STEP          # all tensors step: the classes stay what they are, one step further
        else:
            classes = self._make_classes(steps)
        turns = self._turns + bool(self._has.any())
        lib = _lib.load()
        a.noise = lib.cx_adamw_noise((self.seed + turns) & 0xFFFFFFFF)
        rows, stream = classes.T.tolist(), _lib.stream_ptr(self._device)
        for a.first_class in range(0, len(rows), len(a.cls)):        # one launch, where there are more rows than it holds more
            for c, (group, t) in zip(a.cls, rows[a.first_class:]):
                g = self.param_groups[group]
                b1, b2 = g["betas"]
                c.decay = 1.0 - float(g["lr"]) * float(g["weight_decay"])
                c.b1, c.ob1, c.b2, c.ob2 = b1, 1.0 - b1, b2, 1.0 - b2
                c.rate, c.norm, c.eps = float(g["lr"]) / (1.0 - b1 ** t), 1.0 / math.sqrt(1.0 - b2 ** t), g["eps"]
            _lib.check(lib.cx_adamw_step(self._dev, C.byref(a), stream), "cx_adamw_step")
        self._steps, self._classes, self._turns = steps, classes, turns          # a step that was refused does not count
        _lib.host().stepped(self._params, self._now["seg_grad"].data_ptr())

    def flat_state(self) -> dict:
        """The buffers that hold the states of all tensors (not copies): ``master`` for 16-bit tensors, ``exp_avg`` and
        ``exp_avg_sq``, or with 8 bits ``exp_avg`` and ``exp_avg_rms`` with a scale for each 256 elements."""
        return dict(self._flat)

    def spans(self) -> list:
        """(start, elements) of every tensor in the flat buffers, in the order of the parameters."""
        return [(int(a) * _BLOCK, int(n)) for a, n in zip(self._first, self._numel)]

    @torch.no_grad()
    def refresh_master(self) -> None:
        """Take the tensors as they are as the 32-bit weights: after they were overwritten from outside."""
        self._place()
        self._take_master()

    @torch.no_grad()
    def _take_master(self) -> None:
        master = self._flat.get("master")
        if master is not None:
            for p, (a, n) in zip(self._params, self.spans()):
                master[a:a + n].as_strided(p.size(), p.stride()).copy_(p)

    @staticmethod
    def _shape(p) -> list:
        """Size and memory order of a tensor (strides of dimensions of size 1 say nothing)."""
        return [list(p.size()), [s if n != 1 else 0 for n, s in zip(p.size(), p.stride())]]

    # ---- copies: the tables and buffers are made anew, with what is in them --------------------------------------------
    def __getstate__(self):
        return super().__getstate__() | {"comprex_adamw": {
            "bits": self.state_bits, "seed": self.seed, "index": self._index, "shapes": [self._shape(p) for p in self._params],
            "steps": self._steps, "turns": self._turns,
            "flat": {k: t.view(torch.uint8) if t.itemsize == 1 else t for k, t in self._flat.items()}}}     # (pickle knows no e4m3)

    def __setstate__(self, state):
        state = dict(state)
        mine = state.pop("comprex_adamw", None)
        super().__setstate__(state)
        if mine is None:                      # (of load_state_dict: settings alone)
            return
        self.state_bits, self.seed = mine["bits"], mine["seed"]
        every = [p for g in self.param_groups for p in g["params"]]
        self._take([every[i] for i in mine["index"]])
        if mine["shapes"] != [self._shape(p) for p in self._params]:
            raise ComprexError("the copied tensors have other shapes or another memory order")
        with torch.no_grad():
            for k, t in self._flat.items():
                t.view(mine["flat"][k].dtype).copy_(mine["flat"][k])
        self._steps[:] = mine["steps"]
        self._turns = mine["turns"]

    # ---- checkpoint ------------------------------------------------------------------------------------------------
    def state_dict(self):
        sd = super().state_dict()
        sd["comprex_adamw"] = {"version": 1, "bits": self.state_bits, "seed": self.seed, "numel": self._numel.tolist(), "shapes": [self._shape(p) for p in self._params],
                               "index": list(self._index), "steps": self._steps.tolist(), "turns": self._turns, "flat": {k: t.detach().cpu().clone() for k, t in self._flat.items()}}
        return sd

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        state_dict = dict(state_dict)
        mine = state_dict.pop("comprex_adamw", None)
        if mine is None:
            raise ComprexError("not a checkpoint of this optimizer")
        self._place()
        every, index = [p for g in self.param_groups for p in g["params"]], list(mine.get("index", self._index))
        there = [every[i] for i in index if i < len(every)]
        if mine["bits"] != self.state_bits or mine["numel"] != [p.numel() for p in there] or set(mine["flat"]) != set(self._flat):
            raise ComprexError("checkpoint was written for other parameters or another width of states")
        if "shapes" in mine and mine["shapes"] != [self._shape(p) for p in there]:
            raise ComprexError("checkpoint was written for tensors of other shapes or in another memory order")
        super().load_state_dict(state_dict)
        if index != self._index:              # tensors were unfrozen there and not here, or the other way round
            self._take(there)
        for k, t in self._flat.items():
            t.copy_(mine["flat"][k])
        self.seed = int(mine["seed"])
        self._steps = np.array(mine["steps"], dtype=np.int64)
        self._turns = int(mine.get("turns", max(mine["steps"])))
        self._classes = None
        if "master" in self._flat:
            for p, (a, n) in zip(self._params, self.spans()):
                p.copy_(self._flat["master"][a:a + n].as_strided(p.size(), p.stride()))
