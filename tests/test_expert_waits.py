"""Bounded waits inside the experts' kernels: the bound as it is set, and what a call whose waits run out
reports.  No kernel is stopped for that: a single tile whose sum is long enough takes 200 us and more,
and the warps that wait for its end give up after 130 us under a bound of 1 ns (they look at the clock
after every 64 tries of 1 us)."""
from __future__ import annotations

import ctypes as C
import time

import pytest

torch = pytest.importorskip("torch")

DEFAULT = 5 * 10 ** 9


def set_wait_ns(ns):
    from ugdr_b200 import _native as N

    f = N.lib().ugdr_x_set_expert_wait_ns
    f.restype, f.argtypes = C.c_uint64, [C.c_uint64]
    return f(ns)


def test_the_bound_is_set_and_reset():
    try:
        assert set_wait_ns(1000) == DEFAULT
        assert set_wait_ns(0) == 1000
        assert set_wait_ns(0) == DEFAULT
    finally:
        set_wait_ns(0)


@pytest.mark.gpu
@pytest.mark.parametrize("experts,hidden,inner", [(64, 65_536, 8), (1, 524_288, 64)])  # a pair per tile, four pairs
def test_waits_that_run_out_are_reported_and_the_next_call_is_right(experts, hidden, inner):
    from conftest import gpu_count
    from ugdr_b200 import ops

    if gpu_count() < 1:
        pytest.skip("no GPU")
    gen = torch.Generator(device="cuda").manual_seed(1)

    def normal(scale, *shape):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0, scale, generator=gen)

    x, counts = normal(1, experts, hidden), torch.ones(experts, dtype=torch.int32, device="cuda")
    w_in, w_out = normal(hidden ** -0.5, experts, 2, inner, hidden), normal(inner ** -0.5, experts, hidden, inner)
    want = ops.expert_ffn(x, counts, w_in, w_out)
    ops.check_status()
    set_wait_ns(1)
    try:
        t0 = time.monotonic()
        ops.expert_ffn(x, counts, w_in, w_out)
        with pytest.raises(RuntimeError, match="ran out"):
            ops.check_status()
        assert time.monotonic() - t0 < 2.0
    finally:
        set_wait_ns(0)
    for _ in range(2):
        assert torch.equal(ops.expert_ffn(x, counts, w_in, w_out), want)
    ops.check_status()
