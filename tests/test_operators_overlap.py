"""Gradient tensors whose output overlaps them: only the gradient itself, of the same type, can be
written while it is read.  The argument checks need no GPU."""
from __future__ import annotations

import ctypes as C

import pytest

BF16, FP16, FP32 = 0, 1, 2
AT = 1 << 20


def _plan(entry):
    from ugdr_b200.ops.grads import _Grad, _lib

    L = _lib()
    buf, chunks = C.create_string_buffer(L.ugdr_x_grad_plan_bytes(1)), C.c_uint64()
    return L.ugdr_x_grad_plan((_Grad * 1)(entry), 1, buf, C.byref(chunks))


@pytest.mark.parametrize("grad,out,count,grad_type,out_type", [
    (AT, AT, 1, BF16, FP32), (AT, AT, 1000, FP16, FP32),       # 4 bytes written over every 2 read
    (AT, AT + 4, 8, BF16, FP32), (AT + 12, AT, 8, BF16, FP32),  # begins inside, ends inside
    (AT, AT + 2, 2, BF16, BF16), (AT + 4, AT, 1000, FP32, FP32), (AT, AT + 3996, 1000, FP32, FP32),
    (AT, AT + (1 << 45) - 4, 1 << 44, BF16, FP32)])
def test_a_plan_refuses_an_output_over_its_gradient(grad, out, count, grad_type, out_type):
    assert _plan((grad, out, count, grad_type, out_type)) == 1  # cudaErrorInvalidValue


@pytest.mark.parametrize("grad,out,count,grad_type,out_type", [
    (AT, AT, 1000, BF16, BF16), (AT, AT, 1000, FP32, FP32), (AT, AT, 0, BF16, FP32), (AT, AT + 2000, 1000, BF16, FP32),
    (AT + 4000, AT, 1000, FP16, FP32), (AT, AT + 4000, 1000, FP32, FP32)])
def test_a_plan_takes_an_output_in_place_or_next_to_its_gradient(grad, out, count, grad_type, out_type):
    assert _plan((grad, out, count, grad_type, out_type)) == 0
