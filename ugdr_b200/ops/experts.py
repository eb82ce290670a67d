"""The experts' gated feed-forward block on rows grouped by expert, as the MoE dispatch leaves them
in the receive area (`MoEAllToAll.recv_view()` with `MoEAllToAll.expert_rows()`):

    h = act(x Wg^T) * (x Wu^T),   y = h Wo^T

with every row's own expert's weights.  Serving calls `expert_ffn`; a training step calls
`expert_ffn_train`, which keeps what the backward pass needs, and `expert_ffn_backward`.

Tensors are contiguous CUDA tensors on one device, bfloat16 or float16 throughout; sums are fp32, and
h, dg and du are rounded to the type once, as operands of the next product (so with float16 they
must stay within its range, as x and y must):

    x, y, dy, dx   [rows, hidden]             hidden and inner multiples of 8
    counts         [experts] int32            rows of each expert, in order; read on the device
    w_in           [experts, 2, inner, hidden]  the gate's, then the up projection's weights
    w_out          [experts, hidden, inner]

Rows behind the last group (the unused end of a receive area) are left as they were.  Calls are
enqueued on `stream` (default: the device's current stream), whose order the inputs must respect,
and may be captured into a CUDA graph.  They do not take part in autograd: `expert_ffn` refuses tensors
whose gradients it would drop, and the training calls leave the gradients to the caller and
`expert_ffn_backward`.  Counts that are
negative or add up to more than `rows` are recorded on the device: `check_status()` raises for
them, as it does when a bounded wait inside a kernel ran out.
"""
from __future__ import annotations

import ctypes as C
from typing import Iterable, NamedTuple, Sequence

import torch

from .. import _native as N
from ..parallel.peers import check

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_ACTS = {"silu": 0, "gelu": 1}
MAX_EXPERTS = 4096
MAX_ROWS = 1 << 28
MAX_SIZE = 1 << 20  # of hidden and inner


class _Experts(C.Structure):
    _fields_ = [("counts", C.c_void_p), ("w_in", C.c_void_p), ("w_out", C.c_void_p), ("status", C.c_void_p),
                ("rows", C.c_uint64), ("nexp", C.c_int), ("hidden", C.c_int), ("inner", C.c_int),
                ("type", C.c_int), ("act", C.c_int)]


class ExpertFFNSaved(NamedTuple):
    """What a training forward pass keeps for `expert_ffn_backward` (10 * rows * inner bytes)."""

    h: torch.Tensor   # [rows, inner]
    gu: torch.Tensor  # [rows, 2, inner] float32: both projections


_new_versions = torch.autograd.graph.increment_version
_status: dict[int, torch.Tensor] = {}


_bound: C.CDLL | None = None


def _lib() -> C.CDLL:
    global _bound
    if _bound is None:
        L, vp = N.lib(), C.c_void_p
        L.ugdr_x_expert_ffn.restype = C.c_int
        L.ugdr_x_expert_ffn.argtypes = [C.POINTER(_Experts)] + [vp] * 5
        L.ugdr_x_expert_ffn_backward.restype = C.c_int
        L.ugdr_x_expert_ffn_backward.argtypes = [C.POINTER(_Experts)] + [vp] * 9
        _bound = L
    return _bound


def _enqueue(device: torch.device, stream: torch.cuda.Stream | None, read: Iterable[torch.Tensor],
             written: Sequence[torch.Tensor], call):
    """call(raw stream) with the tensors' device current and `stream` (default: the device's current
    one) the stream that outputs and scratch are allocated for.  On a stream of the caller's choice the
    tensors' memory is kept from reuse until the stream is through with it.  Those that are `written`
    get new versions, so that a backward pass which saved one of them raises torch's error."""
    if stream is None:
        if torch.cuda.current_device() == device.index:  # the short way
            result = call(torch._C._cuda_getCurrentRawStream(device.index))
        else:
            with torch.cuda.device(device):
                result = call(torch._C._cuda_getCurrentRawStream(device.index))
    else:
        if stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
        with torch.cuda.device(device), torch.cuda.stream(stream):
            result = call(stream.cuda_stream)
        for t in (*read, *written):
            t.record_stream(stream)
    if written:
        _new_versions(written)
    return result


def _status_word(device: torch.device) -> torch.Tensor:
    word = _status.get(device.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call an expert operator once on this device before capturing it into a graph")
        with torch.inference_mode(False):  # else only inference mode could clear it
            word = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()  # zero before any stream may write it
        word = _status.setdefault(device.index, word)
    return word


def check_status(device: torch.device | int | None = None) -> None:
    """Wait for `device` (default: the current one) and raise RuntimeError if an expert operator on
    it recorded a fault since the last check."""
    index = device if isinstance(device, int) else torch.device(device or "cuda").index
    word = _status.get(torch.cuda.current_device() if index is None else index)
    if word is None:
        return
    torch.cuda.synchronize(word.device)
    st = int(word.item())
    if st:
        word.zero_()
        raise RuntimeError({1: "a bounded wait inside an expert kernel ran out",
                            2: "expert counts are negative or exceed the rows"}.get(st, f"status {st}"))


def _span(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype, device: torch.device) -> tuple[int, int]:
    """The addresses that t begins and ends at, checked to be a dense tensor as described."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor on {device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    at = t.data_ptr()
    if at % 16 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and 16-byte aligned")
    return at, at + t.nbytes


def _checked(x, counts, w_in, w_out, act: str) -> tuple[_Experts, dict[str, tuple[int, int]]]:
    """The call's description, and the addresses that its inputs begin and end at."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _TYPES or x.dim() != 2:
        raise ValueError("x must be a CUDA tensor [rows, hidden] of bfloat16 or float16")
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
    rows, hidden = x.shape
    dtype, device = x.dtype, x.device
    if not isinstance(counts, torch.Tensor) or counts.dtype != torch.int32 or counts.dim() != 1 \
            or counts.device != device or not counts.is_contiguous():
        raise ValueError(f"counts must be a contiguous int32 tensor [experts] on {device}")
    nexp = counts.shape[0]
    if not 1 <= nexp <= MAX_EXPERTS:
        raise ValueError(f"1..{MAX_EXPERTS} experts supported, got {nexp}")
    if not isinstance(w_out, torch.Tensor) or w_out.dim() != 3:
        raise ValueError("w_out must be a tensor [experts, hidden, inner]")
    inner = w_out.shape[2]
    if not 8 <= hidden <= MAX_SIZE or hidden % 8 or not 8 <= inner <= MAX_SIZE or inner % 8:
        raise ValueError(f"hidden and inner must be multiples of 8 up to {MAX_SIZE}, got {hidden} and {inner}")
    if rows > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows, got {rows}")
    at = counts.data_ptr()
    spans = {"x": _span(x, "x", x.shape, dtype, device), "counts": (at, at + 4 * nexp),
             "w_in": _span(w_in, "w_in", (nexp, 2, inner, hidden), dtype, device),
             "w_out": _span(w_out, "w_out", (nexp, hidden, inner), dtype, device)}
    return _Experts(at, spans["w_in"][0], spans["w_out"][0], None, rows, nexp, hidden, inner, _TYPES[dtype],
                    _ACTS[act]), spans


def _apart(name: str, span: tuple[int, int], others: dict[str, tuple[int, int]], same: tuple = ()) -> None:
    """An output overlaps none of the others; those named in `same` it may be as a whole."""
    a, b = span
    for other, (c, d) in others.items():
        if a < d and c < b and not (other in same and a == c):
            raise ValueError(f"{name} must not overlap {other}" + (" unless it is the same tensor" if other in same
                                                                    else ""))


def _forward(x, counts, w_in, w_out, act, out, stream, train):
    m, spans = _checked(x, counts, w_in, w_out, act)
    if out is not None:
        spans_out = _span(out, "out", x.shape, x.dtype, x.device)
        _apart("out", spans_out, spans, () if train else ("x",))

    def call(s):
        m.status = _status_word(x.device).data_ptr()
        y = torch.empty_like(x) if out is None else out
        h = x.new_empty((m.rows, m.inner))
        gu = x.new_empty((m.rows, 2, m.inner), dtype=torch.float32) if train else None
        check(_lib().ugdr_x_expert_ffn(m, spans["x"][0], y.data_ptr(), h.data_ptr(), gu.data_ptr() if train else None,
                                       s), "ugdr_x_expert_ffn")
        return y, ExpertFFNSaved(h, gu) if train else None

    return _enqueue(x.device, stream, (x, counts, w_in, w_out), () if out is None else (out,), call)


def expert_ffn(x: torch.Tensor, counts: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, act: str = "silu",
               out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """y [rows, hidden] of the block, into `out` if given (which may be `x` itself: the experts in
    place in the receive area).  act: "silu" or "gelu" (the exact one).  For serving: where gradients are
    recorded (not under torch.no_grad() or inference_mode()), no tensor may require one."""
    if torch.is_grad_enabled():
        for name, t in (("x", x), ("w_in", w_in), ("w_out", w_out), ("out", out)):
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise ValueError(f"{name} requires a gradient, which expert_ffn does not record: call it under "
                                 "torch.no_grad(), or use expert_ffn_train and expert_ffn_backward")
    return _forward(x, counts, w_in, w_out, act, out, stream, False)[0]


def expert_ffn_train(x: torch.Tensor, counts: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor,
                     act: str = "silu", out: torch.Tensor | None = None,
                     stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, ExpertFFNSaved]:
    """(y, saved): as expert_ffn, keeping what expert_ffn_backward needs beside x, which has to
    stay as it is until then (`out` must not overlap it)."""
    return _forward(x, counts, w_in, w_out, act, out, stream, True)


def expert_ffn_backward(dy: torch.Tensor, x: torch.Tensor, counts: torch.Tensor, w_in: torch.Tensor,
                        w_out: torch.Tensor, saved: ExpertFFNSaved, act: str = "silu",
                        dx: torch.Tensor | None = None, dw_in: torch.Tensor | None = None,
                        dw_out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None
                        ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dw_in, dw_out) from dy = d loss / d y and the forward pass's inputs, into the tensors
    given for them.  dx may be dy or x itself.  Weight gradients of experts without rows are
    zeros."""
    m, spans = _checked(x, counts, w_in, w_out, act)
    dtype, device = x.dtype, x.device
    spans["dy"] = _span(dy, "dy", x.shape, dtype, device)
    spans["saved.h"] = _span(saved.h, "saved.h", (m.rows, m.inner), dtype, device)
    spans["saved.gu"] = _span(saved.gu, "saved.gu", (m.rows, 2, m.inner), torch.float32, device)
    if spans["saved.gu"][0] % 32:
        raise ValueError("saved.gu must be 32-byte aligned")
    given = []
    for name, t, shape in (("dx", dx, x.shape), ("dw_in", dw_in, w_in.shape), ("dw_out", dw_out, w_out.shape)):
        if t is not None:
            span = _span(t, name, shape, dtype, device)
            _apart(name, span, spans, ("dy", "x") if name == "dx" else ())
            spans[name] = span
            given.append(t)

    def call(s):
        m.status = _status_word(device).data_ptr()
        gx = torch.empty_like(x) if dx is None else dx
        gin = torch.empty_like(w_in) if dw_in is None else dw_in
        gout = torch.empty_like(w_out) if dw_out is None else dw_out
        dgu = x.new_empty((m.rows, 2, m.inner))
        check(_lib().ugdr_x_expert_ffn_backward(m, spans["dy"][0], spans["x"][0], spans["saved.h"][0],
                                                spans["saved.gu"][0], dgu.data_ptr(), gx.data_ptr(), gin.data_ptr(),
                                                gout.data_ptr(), s), "ugdr_x_expert_ffn_backward")
        return gx, gin, gout

    return _enqueue(device, stream, (x, counts, w_in, w_out, dy, *saved), given, call)
