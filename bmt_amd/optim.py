"""Fused multi-tensor Adam and gradient clipping on libbmt_hip.so.

Restates what scripts/train_captioning_module.py:46-48 builds (torch.optim.Adam, lr 5e-5, betas (0.9, 0.999),
eps 1e-8, weight_decay 0) and epoch_loops/captioning_epoch_loops.py:138-139 (clip_grad_norm_) as ONE kernel
launch over every parameter.  Subclasses torch.optim.Optimizer so ``state_dict()`` keeps torch's layout
(``exp_avg`` / ``exp_avg_sq`` / ``step`` per parameter) and checkpoints interchange."""
from __future__ import annotations

from typing import Iterable, List, Optional, Sequence

import numpy as np
import torch

from . import _lib
from .ops import _DTYPES, _p, _raw_stream, _run_on, _st, lib


class _PtrTable:
    """Device-side table of tensor pointers + sizes, re-uploaded only when a pointer changes (so a captured
    hipGraph, which needs static gradient buffers anyway, replays without host work)."""

    def __init__(self, device):
        self.device = device
        self.key = None
        self.ptrs = None
        self.sizes = None
        self.max_size = 0
        self.n = 0
        self._retired = []   # tables a captured hipGraph may still read: never freed (a few KB each)

    def update(self, columns: List[List[torch.Tensor]]):
        key = tuple(t.data_ptr() for col in columns for t in col)
        if key == self.key:
            return
        n = len(columns[0])
        host = torch.tensor(key, dtype=torch.int64)
        if self.ptrs is not None:
            self._retired.append((self.ptrs, self.sizes))
            if len(self._retired) > 256:      # gradients re-allocated every step (no static buffers, hence no captured graph): bounded
                del self._retired[:128]
        self.ptrs = host.to(self.device)
        sizes = [t.numel() for t in columns[0]]
        self.sizes = torch.tensor(sizes, dtype=torch.int64).to(self.device)
        self.max_size = max(sizes)
        self.n = n
        self.key = key


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=5e-5, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)
        self._tables = {}
        self._steps = {}
        self.grad_scale = None   # optional device float multiplied into every gradient inside the kernel

    def load_state_dict(self, state_dict):
        """torch.optim.Adam / FusedAdam state (``optimizer_state_dict`` of a reference checkpoint): the pointer tables and the
        device step counters are rebuilt at the next step from the loaded state"""
        super().load_state_dict(state_dict)
        self._tables, self._steps = {}, {}
        for st in self.state.values():      # torch.optim.Adam keeps ``step`` as a tensor (possibly on the device) or a float
            if "step" in st:
                st["step"] = torch.as_tensor(float(st["step"]), dtype=torch.float32)

    def state_dict(self):
        """torch.optim.Adam's layout.  The step count that matters lives on the device (``_steps``: a captured optimizer graph
        advances it without running this Python), so the per-parameter ``step`` entries are refreshed from it first --
        otherwise a checkpoint written after N graph replays would resume Adam's bias correction near step 0 against fully
        warmed moments."""
        for gi, group in enumerate(self.param_groups):
            if gi in self._steps:
                n = float(self._steps[gi].item())
                for p in group["params"]:
                    st = self.state.get(p)
                    if st is not None and "step" in st:
                        st["step"] = torch.as_tensor(n, dtype=torch.float32)
        return super().state_dict()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            ps = [p for p in group["params"] if p.grad is not None]
            if not ps:
                continue
            dev = ps[0].device
            for p in ps:
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = torch.zeros((), dtype=torch.float32)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                if not p.is_contiguous() or not p.grad.is_contiguous() or p.dtype != torch.float32:
                    raise RuntimeError("FusedAdam needs contiguous fp32 parameters and gradients")
            if gi not in self._tables:
                self._tables[gi] = _PtrTable(dev)
                # device-side step counter; resumes from a loaded state_dict (torch layout: one ``step`` per parameter)
                self._steps[gi] = torch.full((1,), int(self.state[ps[0]]["step"]), dtype=torch.int64, device=dev)
            tab = self._tables[gi]
            tab.update([ps, [p.grad for p in ps], [self.state[p]["exp_avg"] for p in ps],
                        [self.state[p]["exp_avg_sq"] for p in ps]])
            b1, b2 = group["betas"]
            _lib.check(lib.bmt_adam_step(_p(tab.ptrs), _p(tab.sizes), tab.n, tab.max_size, _p(self._steps[gi]),
                                         float(group["lr"]), float(b1), float(b2), float(group["eps"]),
                                         float(group["weight_decay"]), _p(self.grad_scale), _st()), "bmt_adam_step")
            from . import ops as _ops
            _ops.WEIGHT_EPOCH[0] += 1      # cached bf16 weight planes are stale now
            for p in ps:   # host-side mirror of the step count (torch's state layout); the kernel uses the device counter
                self.state[p]["step"] += 1
        return loss


_clip_tables = {}      # (device, parameter set) -> (table, sq, coef): one per parameter SET, kept for the life of the process (a captured
                       # optimizer graph has the table's address baked in; _PtrTable.update re-uploads when a gradient pointer moves and
                       # retires the old table, so re-allocated gradients -- zero_grad() sets them to None -- do not add entries)


@torch.no_grad()
def clip_grad_norm_(parameters: Iterable[torch.nn.Parameter], max_norm: float) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ (L2): returns the total norm (device scalar); gradients are scaled in place by
    min(1, max_norm / (norm + 1e-6)) without a host sync."""
    ps = [p for p in parameters if p.grad is not None]
    if not ps:
        return torch.zeros(())
    dev = ps[0].device
    key = (str(dev), tuple(id(p) for p in ps))
    if key not in _clip_tables:
        _clip_tables[key] = (_PtrTable(dev), torch.zeros(1, device=dev), torch.zeros(1, device=dev))
    tab, sq, coef = _clip_tables[key]
    tab.update([[p.grad for p in ps]])
    _lib.check(lib.bmt_grad_sqnorm(_p(tab.ptrs), _p(tab.sizes), tab.n, tab.max_size, _p(sq), float(max_norm), _p(coef), _st()),
               "bmt_grad_sqnorm")
    _lib.check(lib.bmt_scale_tensors(_p(tab.ptrs), _p(tab.sizes), tab.n, tab.max_size, _p(coef), _st()), "bmt_scale_tensors")
    return sq.sqrt().squeeze(0)


_captured_tables = []   # tile tables that a captured hipGraph may still read: never freed (24 bytes per 32 KB of gradients)
CLIP_TILE = 32768       # bytes of gradient per tile of GradClipper's table: 128 per thread of a workgroup


def _dense(t: torch.Tensor) -> bool:
    """whether the elements fill a range of memory, in any order of the dimensions"""
    n = 1
    if t.numel() == 0:
        return True
    for size, stride in sorted(((a, b) for a, b in zip(t.shape, t.stride()) if a != 1), key=lambda x: x[1]):
        if stride != n:
            return False
        n *= size
    return True


class GradClipper:
    """Global norm of many gradient tensors, and clipping -- ``clip_grad_norm_`` for gradients of mixed types, for a captured step and for
    buffers other than the gradients' own:

        clipper = GradClipper([p.grad for p in params], max_norm=1.0)      # static gradient buffers (GradientReducer keeps such)
        total = clipper()                                                  # norm as a device scalar; gradients *= min(1, max_norm / (norm + eps))

    ``grads``: fp32, bf16 or fp16 tensors on one device, dense in any order of their dimensions, none sharing memory with another.  ``out``: one
    tensor per gradient (same shape and order of dimensions, its own type) that takes the clipped values -- what FusedAdam wants of 16-bit
    gradients --; None: in place.  ``norm_type``: 2 or inf.  ``clipper(scale=s)``: s (device float) is a factor the gradients still lack: norm and
    result are those of s * gradient.  ``clipper(apply=False)``: the norm alone.  ``clipper.coef``: the last call's factor min(1, ..) * s, for
    FusedAdam.grad_scale.  A non-finite norm does what it does in torch: inf leaves finite gradients 0, NaN makes them NaN.

    Sums are 64-bit and in one order: the same bits on every run.  The plan holds the tensors, and a call refuses ones whose memory has moved."""

    def __init__(self, grads: Sequence[torch.Tensor], max_norm: float, out: Optional[Sequence[torch.Tensor]] = None, norm_type: float = 2.0, eps: float = 1e-6):
        self.grads = list(grads)
        self.out = self.grads if out is None else list(out)
        self.max_norm, self.eps = max_norm, float(eps)
        if not self.grads:
            raise ValueError("GradClipper: no gradients")
        if norm_type not in (2, float("inf")):
            raise ValueError(f"GradClipper: norm_type {norm_type} (2 or inf)")
        self._inf = int(norm_type != 2)
        if not self.eps >= 0.0:
            raise ValueError(f"GradClipper: eps {eps}")
        if len(self.out) != len(self.grads):
            raise ValueError(f"GradClipper: {len(self.out)} output tensors for {len(self.grads)} gradients")
        for t in self.grads + ([] if out is None else self.out):
            if not t.is_cuda:
                raise RuntimeError("GradClipper: bmt_amd ops need CUDA/HIP tensors: there is no CPU fallback")
            if t.device != self.grads[0].device or t.dtype not in _DTYPES or not _dense(t):
                raise ValueError(f"GradClipper: a tensor of shape {tuple(t.shape)}, strides {t.stride()} and type {t.dtype} on {t.device}: all are dense, "
                                 "float32, bfloat16 or float16, and on one device")
        for g, o in zip(self.grads, self.out):
            if g.shape != o.shape or any(a != 1 and g.numel() > 0 and x != y for a, x, y in zip(g.shape, g.stride(), o.stride())):
                raise ValueError(f"GradClipper: a gradient of shape {tuple(g.shape)} and strides {g.stride()} with an output of {tuple(o.shape)} and {o.stride()}")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("GradClipper: make the plan before the capture (its table is copied from the host); calls of it are captured")
        self.device = self.grads[0].device
        self._ptrs = [t.data_ptr() for t in self.grads], [t.data_ptr() for t in self.out]
        self._in_place = int(all(g.dtype == o.dtype for g, o in zip(self.grads, self.out)) and self._ptrs[0] == self._ptrs[1])
        self._refuse_shared_memory()
        self.coef = None
        self._tiles, self._n = self._table()
        self._stream = _raw_stream(self.device.index)      # whose memory the table is

    @property
    def max_norm(self) -> float:
        """the bound: an argument of every call, so it may be set anew between calls"""
        return self._max_norm

    @max_norm.setter
    def max_norm(self, value: float):
        if not float(value) >= 0.0:
            raise ValueError(f"GradClipper: max_norm {value}")
        self._max_norm = float(value)

    def _refuse_shared_memory(self):
        ranges = []
        for g, o, pg, po in zip(self.grads, self.out, *self._ptrs):
            if g.numel() == 0:
                continue
            ranges.append((pg, pg + g.numel() * g.element_size()))
            if po != pg or o.dtype != g.dtype:
                ranges.append((po, po + o.numel() * o.element_size()))
        ranges.sort()
        if any(a[1] > b[0] for a, b in zip(ranges, ranges[1:])):
            raise ValueError("GradClipper: two of the tensors share memory (a gradient given twice, or an output that overlaps another tensor)")

    def _table(self):
        entry = np.dtype([("g", "<u8"), ("out", "<u8"), ("n", "<i4"), ("kind", "<i4")])
        assert entry.itemsize == lib.bmt_clip_tile_bytes()
        rows = []
        for g, o, pg, po in zip(self.grads, self.out, *self._ptrs):
            tile = CLIP_TILE // g.element_size()
            first = np.arange(0, g.numel(), tile, dtype=np.uint64)
            r = np.empty(len(first), entry)
            r["g"], r["out"] = pg + first * np.uint64(g.element_size()), po + first * np.uint64(o.element_size())
            r["n"] = np.minimum(tile, g.numel() - first.astype(np.int64))
            r["kind"] = _DTYPES[g.dtype] | _DTYPES[o.dtype] << 2
            rows.append(r)
        rows = np.concatenate(rows)
        if len(rows) > 0x7fffffff:
            raise ValueError("GradClipper: too many elements")
        return torch.from_numpy(rows.view(np.uint8)).to(self.device), len(rows)

    @torch.no_grad()
    def __call__(self, scale: Optional[torch.Tensor] = None, apply: bool = True) -> torch.Tensor:
        if ([t.data_ptr() for t in self.grads], [t.data_ptr() for t in self.out]) != self._ptrs:
            raise RuntimeError("GradClipper: a tensor's memory has moved since the plan was made: make a new one")
        if scale is not None and (scale.numel() != 1 or scale.dtype != torch.float32 or scale.device != self.device):
            raise ValueError(f"GradClipper: scale is one float32 value on {self.device}")
        if torch.cuda.is_current_stream_capturing():
            if not any(t is self._tiles for t in _captured_tables):
                _captured_tables.append(self._tiles)
        elif _raw_stream(self.device.index) != self._stream:      # (a plan dropped behind this call: its table outlives what this stream still runs)
            self._tiles.record_stream(torch.cuda.current_stream(self.device))
        result = torch.empty(2, device=self.device, dtype=torch.float32)
        n = lib.bmt_clip_ws_bytes()
        ws = torch.empty(n, device=self.device, dtype=torch.uint8)      # (of this call: two captured graphs, or two streams, share nothing)
        _run_on(self.device.index, "bmt_clip_grads", lib.bmt_clip_grads, self._tiles.data_ptr() if self._n else None, self._n, self._inf, self._max_norm, self.eps,
                None if scale is None else scale.data_ptr(), int(apply), self._in_place, result.data_ptr(), ws.data_ptr(), n)
        if apply:
            torch.autograd.graph.increment_version(self.out)
        self.coef = result[1]
        return result[0]
