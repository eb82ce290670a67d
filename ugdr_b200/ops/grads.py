"""The global 2-norm over many gradient tensors, and clipping, in two launches whatever their number.

    clip = GradClip([p.grad for p in params])            # once: the list as the kernels read it
    norm = clip.clip(max_norm=1.0)                       # every step, after the allreduce

Where the gradients of one norm are spread over ranks (each rank's own experts), the ranks add up
their `sum_squares()` and pass the total to `clip`.
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import torch

from .. import _native as N
from ..parallel.peers import check
from .experts import _enqueue, _new_versions

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
PARTIALS = 2048


class _Grad(C.Structure):
    _fields_ = [("grad", C.c_void_p), ("out", C.c_void_p), ("count", C.c_uint64), ("grad_type", C.c_int32),
                ("out_type", C.c_int32)]


_bound: C.CDLL | None = None


def _lib() -> C.CDLL:
    global _bound
    if _bound is None:
        L, vp, i, u64 = N.lib(), C.c_void_p, C.c_int, C.c_uint64
        L.ugdr_x_grad_plan_bytes.restype = C.c_size_t
        L.ugdr_x_grad_plan_bytes.argtypes = [i]
        L.ugdr_x_grad_plan.restype = i
        L.ugdr_x_grad_plan.argtypes = [C.POINTER(_Grad), i, vp, C.POINTER(u64)]
        L.ugdr_x_grad_sum_squares.restype = i
        L.ugdr_x_grad_sum_squares.argtypes = [vp, i, u64, vp, vp, vp]
        L.ugdr_x_grad_clip.restype = i
        L.ugdr_x_grad_clip.argtypes = [vp, i, u64, vp, vp, C.c_float, vp, vp]
        _bound = L
    return _bound


class GradClip:
    """A plan over gradient tensors: contiguous CUDA tensors of one device, bfloat16, float16 or
    float32 in any mix.  `out` (default: the gradients themselves) receives the scaled gradients:
    one tensor each, of the same size, of the gradient's type or float32, the gradient itself or
    memory that overlaps no gradient and no other output.

    The plan holds the tensors and their addresses: gradients that are replaced (not written in
    place) need a new plan.  Its methods are enqueued on `stream` (default: the device's current
    stream), may be captured into a CUDA graph, and can run on several streams at once as far as
    the gradients allow it.  A plan may be dropped with calls still under way, on any stream, but a
    graph that captured a call holds the plan's addresses, not the plan, which has to outlive it."""

    def __init__(self, grads: Sequence[torch.Tensor], out: Sequence[torch.Tensor] | None = None):
        self.grads = tuple(grads)
        self.out = self.grads if out is None else tuple(out)
        if not self.grads:
            raise ValueError("no gradients")
        if len(self.out) != len(self.grads):
            raise ValueError(f"{len(self.out)} outputs for {len(self.grads)} gradients")
        for name, ts in (("gradients", self.grads), ("outputs", self.out)):
            for t in ts:
                if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _TYPES or not t.is_contiguous():
                    raise ValueError(f"{name} must be contiguous CUDA tensors of bfloat16, float16 or float32")
                if t.device != self.grads[0].device:
                    raise ValueError("all tensors must be on one device")
        for g, o in zip(self.grads, self.out):
            if o.shape != g.shape:
                raise ValueError(f"an output of shape {tuple(o.shape)} for a gradient of shape {tuple(g.shape)}")
            if o.dtype not in (g.dtype, torch.float32):
                raise ValueError(f"an output of {o.dtype} for a gradient of {g.dtype}")
            apart = o.data_ptr() >= g.data_ptr() + g.nbytes or g.data_ptr() >= o.data_ptr() + o.nbytes
            if not apart and (o.data_ptr() != g.data_ptr() or o.dtype != g.dtype):
                raise ValueError("an output must be its gradient or not overlap it")
        self._refuse_overlaps()
        self.device = self.grads[0].device
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("build the plan before the capture: it is copied to the device")
        n = len(self.grads)
        table = (_Grad * n)(*[(g.data_ptr(), o.data_ptr(), g.numel(), _TYPES[g.dtype], _TYPES[o.dtype])
                              for g, o in zip(self.grads, self.out)])
        L = _lib()
        plan = torch.empty(L.ugdr_x_grad_plan_bytes(n), dtype=torch.uint8)
        chunks = C.c_uint64()
        check(L.ugdr_x_grad_plan(table, n, plan.data_ptr(), C.byref(chunks)), "ugdr_x_grad_plan")
        self._plan, self._n, self._chunks = plan.to(self.device), n, chunks.value
        # The copy is over: any stream may use the plan.
        torch.cuda.current_stream(self.device).synchronize()
        # The allocator knows of the stream that the table was made on only; _keep tells it of others.
        self._home = torch._C._cuda_getCurrentRawStream(self.device.index)
        self._kept: set[int] = set()
        # Views share their base's version: one of each is enough.
        bases = (o if o._base is None else o._base for o in self.out)
        self._written = tuple({id(b): b for b in bases}.values())

    def _refuse_overlaps(self) -> None:
        """Memory that is written is written for one tensor only, and read for that one only."""
        spans = []
        for g, o in zip(self.grads, self.out):
            size = g.numel()
            if size:
                spans.append((o.data_ptr(), o.data_ptr() + size * o.element_size(), True))
                if o.data_ptr() != g.data_ptr():
                    spans.append((g.data_ptr(), g.data_ptr() + size * g.element_size(), False))
        spans.sort()
        end = written = 0  # the furthest end of the spans so far, and of those that are written
        for a, b, writes in spans:
            if a < written or (writes and a < end):
                raise ValueError("outputs must not overlap other gradients or outputs")
            end = max(end, b)
            written = max(written, b) if writes else written

    def _keep(self, s: int, chosen: bool) -> None:
        """Keep the plan's memory from reuse until the current stream, `s`, is through with it, should
        the plan be dropped before.  (Once per stream: the plan's own references do the rest.)"""
        if s in self._kept or (s == self._home and not chosen):
            return
        stream = torch.cuda.current_stream(self.device)
        for t in (self._plan, *self.grads, *(self.out if self.out is not self.grads else ())):
            t.record_stream(stream)
        self._kept.add(s)

    def sum_squares(self, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """The sum of the squares of all elements, a float64 tensor on the device."""
        def call(s):
            self._keep(s, stream is not None)
            partials = self._plan.new_empty(PARTIALS, dtype=torch.float64)
            total = self._plan.new_empty((), dtype=torch.float64)
            check(_lib().ugdr_x_grad_sum_squares(self._plan.data_ptr(), self._n, self._chunks, partials.data_ptr(),
                                                 total.data_ptr(), s), "ugdr_x_grad_sum_squares")
            return total

        return _enqueue(self.device, stream, (), (), call)

    def clip(self, max_norm: float, sum_squares: torch.Tensor | None = None,
             stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Scale the gradients by min(1, max_norm / (norm + 1e-6)) and return their norm before
        that, a float32 tensor on the device.  `sum_squares` (float64, on the device) takes the
        place of this plan's own sum.  As the formula has it, an infinite norm scales by zero and
        a NaN makes every gradient NaN."""
        max_norm = float(max_norm)
        if not max_norm >= 0.0:
            raise ValueError(f"max_norm must be at least 0, got {max_norm}")
        if sum_squares is not None and (not isinstance(sum_squares, torch.Tensor) or sum_squares.numel() != 1
                                        or sum_squares.dtype != torch.float64 or sum_squares.device != self.device):
            raise ValueError(f"sum_squares must be one float64 on {self.device}")

        def call(s):
            self._keep(s, stream is not None)
            partials = self._plan.new_empty(PARTIALS, dtype=torch.float64)
            norm = self._plan.new_empty((), dtype=torch.float32)
            check(_lib().ugdr_x_grad_clip(self._plan.data_ptr(), self._n, self._chunks, partials.data_ptr(),
                                          None if sum_squares is None else sum_squares.data_ptr(), max_norm,
                                          norm.data_ptr(), s), "ugdr_x_grad_clip")
            return norm

        norm = _enqueue(self.device, stream, () if sum_squares is None else (sum_squares,), (), call)
        _new_versions(self._written)
        return norm
