"""The model operators' argument checks, which need no GPU: refused calls launch nothing."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

INVALID = 1  # cudaErrorInvalidValue


def _experts(**change):
    from ugdr_b200.ops.experts import _Experts

    a = dict(counts=0x1000, w_in=0x2000, w_out=0x3000, status=0x4000, rows=8, nexp=2, hidden=64, inner=64, type=0,
             act=0) | change
    return _Experts(*[a[n] for n, _ in _Experts._fields_])


@pytest.mark.parametrize("change", [
    dict(counts=None), dict(w_in=None), dict(w_out=None), dict(status=None), dict(w_in=0x2008), dict(w_out=0x3004),
    dict(rows=(1 << 28) + 1), dict(rows=1 << 40), dict(hidden=(1 << 20) + 8), dict(inner=1 << 21), dict(nexp=0), dict(nexp=4097), dict(hidden=0), dict(hidden=12), dict(hidden=-8),
    dict(inner=0), dict(inner=20), dict(type=2), dict(type=-1), dict(act=2), dict(act=-1)])
def test_the_block_refuses_what_it_cannot_do(change):
    from ugdr_b200.ops.experts import _lib

    L = _lib()
    m = _experts(**change)
    assert L.ugdr_x_expert_ffn(C.byref(m), 0x5000, 0x6000, 0x7000, None, None) == INVALID
    assert L.ugdr_x_expert_ffn_backward(C.byref(m), *[0x5000] * 8, None) == INVALID


@pytest.mark.parametrize("pointers", [(None, 0x6000, 0x7000, None), (0x5008, 0x6000, 0x7000, None),
                                      (0x5000, None, 0x7000, None), (0x5000, 0x6000, 0x7002, None),
                                      (0x5000, 0x6000, 0x7000, 0x8001), (0x5000, 0x6000, 0x7000, 0x8010)])
def test_the_forward_refuses_missing_and_misaligned_tensors(pointers):
    from ugdr_b200.ops.experts import _lib

    L = _lib()
    m = _experts()
    assert L.ugdr_x_expert_ffn(C.byref(m), *pointers, None) == INVALID
    assert L.ugdr_x_expert_ffn(None, 0x5000, 0x6000, 0x7000, None, None) == INVALID


@pytest.mark.parametrize("which", range(8))
@pytest.mark.parametrize("value", [None, 0x5008])
def test_the_backward_refuses_missing_and_misaligned_tensors(which, value):
    from ugdr_b200.ops.experts import _lib

    args = [0x5000] * 8
    args[which] = value
    assert _lib().ugdr_x_expert_ffn_backward(C.byref(_experts()), *args, None) == INVALID


def _plan(entries):
    from ugdr_b200.ops.grads import _Grad, _lib

    L = _lib()
    n = len(entries)
    table = (_Grad * n)(*entries)
    size = L.ugdr_x_grad_plan_bytes(n)
    buf, chunks = C.create_string_buffer(size), C.c_uint64()
    rc = L.ugdr_x_grad_plan(table, n, buf, C.byref(chunks))
    first = [int.from_bytes(buf.raw[n * C.sizeof(_Grad) + 4 * i:][:4], "little") for i in range(n + 1)]
    return rc, first, chunks.value


def test_a_plan_counts_every_tensors_chunks():
    """Chunks of 4096 elements that begin at a multiple of 8 elements in memory: a tensor that
    starts behind one begins inside its first chunk."""
    base = 1 << 20
    rc, first, chunks = _plan([(base, base, 4096, 2, 2), (base + 4, base + 4, 4096, 2, 2), (base, base, 0, 0, 0),
                               (base + 2, base + 2, 4095, 0, 0), (base + 2, base + 2, 4096, 0, 0),
                               (base + 14, base, 1, 1, 2)])
    assert rc == 0 and first == [0, 1, 3, 3, 4, 6, 7] and chunks == 7
    rc, first, chunks = _plan([])
    assert rc == 0 and first == [0] and chunks == 0
    rc, first, chunks = _plan([(base, base, 1 << 40, 0, 0)])
    assert rc == 0 and chunks == 1 << 28


@pytest.mark.parametrize("entry", [(None, 64, 1, 0, 0), (64, None, 1, 0, 0), (65, 64, 1, 0, 0), (64, 66, 1, 2, 2),
                                   (64, 66, 1, 0, 2), (64, 64, 1, 3, 3), (64, 64, 1, -1, -1), (64, 64, 1, 0, 1),
                                   (64, 64, 1, 2, 0), (64, 64, 1 << 45, 0, 0), (64, 64, 1 << 44, 0, 0)])
def test_a_plan_refuses_bad_tensors(entry):
    assert _plan([(1 << 20, 1 << 20, 10, 0, 0), entry])[0] == INVALID


def test_clip_refuses_bad_arguments():
    from ugdr_b200.ops.grads import _lib

    L = _lib()
    ok = (0x1000, 1, 1, 0x2000, None, 1.0, 0x3000, None)
    for i, v in ((0, None), (0, 0x1008), (1, -1), (2, 1 << 32), (3, None), (5, -1.0), (5, float("nan")), (6, None)):
        args = list(ok)
        args[i] = v
        assert L.ugdr_x_grad_clip(*args) == INVALID, i
    ok = (0x1000, 1, 1, 0x2000, 0x3000, None)
    for i, v in ((0, None), (1, -1), (2, 1 << 32), (3, None), (4, None)):
        args = list(ok)
        args[i] = v
        assert L.ugdr_x_grad_sum_squares(*args) == INVALID, i
    assert L.ugdr_x_grad_plan_bytes(-1) == 0


def test_python_refuses_host_tensors():
    from ugdr_b200 import ops

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.expert_ffn(x, torch.tensor([4], dtype=torch.int32), torch.zeros(1, 2, 64, 64), torch.zeros(1, 64, 64))
    with pytest.raises(ValueError):
        ops.GradClip([x])
    with pytest.raises(ValueError):
        ops.GradClip([])
