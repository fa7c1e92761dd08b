"""Global gradient norm over many tensors, and clipping by it (csrc/clip.cu).

    norm = sqrt(sum g^2)  over all elements of all tensors;    g * min(1, max_norm / norm)

The norm stays on the device: nothing is read back.  A program whose gradients live in the same buffers every step keeps a
``GradSet`` of them, which saves going through the list again::

    grads = GradSet([p.main_grad for p in parameters])
    norm = clip_grad_norm(grads, max_norm=1.0)
"""
from __future__ import annotations

import struct
from operator import attrgetter
from typing import Optional, Sequence, Union

import torch

from ..ops import kernels as K

_ENTRY = struct.Struct("=3q2i")         # ArbGrad of csrc/api.h
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_dtype = attrgetter("dtype")
MAX_TENSORS = 1024                      # per launch
BLOCKS_PER_SM = 5
ITEM = 16384                            # elements of a work item


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one stretch of memory, in any order of the dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= n
    return True


def _order(t: torch.Tensor):
    """Strides of the dimensions that have any use for one."""
    return [s for s, n in zip(t.stride(), t.shape) if n != 1]


def _apart(tensors, what: str) -> None:
    """Refuses tensors that share memory: an element in two of them would count, or be scaled, twice."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors)
    for (_, end), (start, _) in zip(spans, spans[1:]):
        if start < end:
            raise ValueError(f"{what} share memory")


class GradSet:
    """A list of gradients, and optionally as many tensors that take the clipped ones (``out``: same shapes and memory order,
    any of the types).  fp32, bf16 or fp16, dense, on one CUDA device, no two sharing memory."""

    def __init__(self, tensors: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None):
        self._take(tensors, out)
        self._where = self._layout()

    def _take(self, tensors, out) -> None:
        tensors = list(tensors)
        outs = tensors if out is None else list(out)
        if len(outs) != len(tensors):
            raise ValueError(f"{len(outs)} outputs for {len(tensors)} gradients")
        for t in tensors if out is None else tensors + outs:
            if not (torch.is_tensor(t) and t.is_cuda and t.dtype in _TYPES):
                raise TypeError("gradients must be fp32, bf16 or fp16 CUDA tensors")
            if t.device != tensors[0].device:
                raise ValueError("gradients must be on one device")
            if not _dense(t):
                raise ValueError(f"gradients must be dense, got strides {t.stride()} of {tuple(t.shape)}")
        for t, o in zip(tensors, outs):
            if o.shape != t.shape or (o is not t and o.stride() != t.stride() and t.numel() > 1 and _order(o) != _order(t)):
                raise ValueError(f"output {tuple(o.shape)} {o.stride()} does not match its gradient {tuple(t.shape)} {t.stride()}")
        live = [(t, o) for t, o in zip(tensors, outs) if t.numel()]
        _apart([t for t, _ in live], "gradients")
        if out is not None:
            _apart([o for _, o in live], "outputs")
            ins = {t.data_ptr() for t, _ in live}
            for t, o in live:
                if o.data_ptr() == t.data_ptr() and o.dtype == t.dtype:
                    ins.discard(t.data_ptr())                       # in place, this one
            _apart([t for t, _ in live if t.data_ptr() in ins] + [o for _, o in live], "outputs and gradients")
        self.tensors, self.out = tensors, out if out is None else outs
        self.device = tensors[0].device if tensors else None
        rows = [_ENTRY.pack(t.data_ptr(), o.data_ptr(), t.numel(), _TYPES[t.dtype], _TYPES[o.dtype]) for t, o in live]
        # (argument block, tensors in it, blocks of its grid)
        self._parts = []
        if rows:
            most = torch.cuda.get_device_properties(self.device).multi_processor_count * BLOCKS_PER_SM
            for a in range(0, len(rows), MAX_TENSORS):
                items = sum(-(-t.numel() // ITEM) for t, _ in live[a:a + MAX_TENSORS])
                self._parts.append((b"".join(rows[a:a + MAX_TENSORS]), len(rows[a:a + MAX_TENSORS]), min(items, most)))

    def _layout(self):
        """Where the tensors lie, of which size and type: a fifth of a microsecond a tensor, in every call."""
        every = self.tensors if self.out is None else self.tensors + self.out
        return [*map(torch.Tensor.data_ptr, every), *map(torch.Tensor.numel, every), *map(_dtype, every)]

    def _run(self, max_norm: float) -> torch.Tensor:
        if self._layout() != self._where:            # a tensor was given other memory, another size or type since, or the set is a copy
            self.__init__(self.tensors, self.out)
        return self._launch(max_norm)

    def _launch(self, max_norm: float) -> torch.Tensor:
        if not self._parts:
            return torch.zeros((), dtype=torch.float32, device=self.device if self.device is not None else "cuda")
        with K.on_device(self.device):
            total = sum(blocks for _, _, blocks in self._parts)
            work = torch.empty(total, dtype=torch.float64, device=self.device)
            norm = torch.empty((), dtype=torch.float32, device=self.device)
            lib, stream, at = K.lib(), K._stream(), work.data_ptr()
            for args, n, blocks in self._parts:
                K._check(lib.arb_grad_squares(args, n, at, blocks, stream), "grad_squares")
                at += 8 * blocks
            for i, (args, n, blocks) in enumerate(self._parts if max_norm >= 0 else self._parts[:1]):
                K._check(lib.arb_grad_scale(args, n, work.data_ptr(), total, max_norm, norm.data_ptr() if i == 0 else None, blocks, stream),
                         "grad_scale")
        return norm


Grads = Union[GradSet, Sequence[torch.Tensor]]


def _run(grads: Grads, out, max_norm: float) -> torch.Tensor:
    if isinstance(grads, GradSet):
        return grads._run(max_norm)
    once = GradSet.__new__(GradSet)          # for this call alone: nothing to compare it with later
    once._take(grads, out)
    return once._launch(max_norm)


def grad_norm(grads: Grads) -> torch.Tensor:
    """The 2-norm of all gradients together, a 0-dimensional fp32 tensor on their device."""
    return _run(grads, None, -1.0)


def clip_grad_norm(grads: Grads, max_norm: float, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the gradients by min(1, max_norm / norm), in place or into ``out`` (where they are converted to its types), and
    returns their norm before that.  Where a gradient is infinite or NaN they are left as they are (``out`` gets copies), for the
    caller to see in the result; finite gradients are scaled, also those whose norm is infinite as an fp32 number."""
    if not 0.0 < max_norm:
        raise ValueError(f"max_norm must be positive, got {max_norm}")
    if isinstance(grads, GradSet) and out is not None:
        raise ValueError("a GradSet holds its outputs already")
    return _run(grads, out, float(max_norm))
