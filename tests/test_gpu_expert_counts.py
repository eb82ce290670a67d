"""Counts that do not fit the rows are recorded whatever the number of rows, none among them."""
from __future__ import annotations

import pytest

from conftest import gpu_count

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("counts,bad", [([0, 0, 0], False), ([0, 0, 3], True), ([-1, 0, 0], True), ([2, -2, 0], True),
                                        ([0] * 4095 + [7], True), ([0] * 4096, False)])
def test_counts_that_do_not_fit_are_recorded(rows, counts, bad):
    from ugdr_b200 import ops

    if gpu_count() < 1:
        pytest.skip("no GPU")
    n, hidden, inner = len(counts), 16, 8
    x = torch.ones(rows, hidden, dtype=torch.bfloat16, device="cuda")
    w_in = torch.ones(n, 2, inner, hidden, dtype=torch.bfloat16, device="cuda")
    w_out = torch.ones(n, hidden, inner, dtype=torch.bfloat16, device="cuda")
    c = torch.tensor(counts, dtype=torch.int32, device="cuda")
    good = torch.zeros_like(c)

    def recorded():
        if not bad:
            return ops.check_status()
        with pytest.raises(RuntimeError, match="counts"):
            ops.check_status()

    ops.expert_ffn(x, c, w_in, w_out)
    recorded()
    _, saved = ops.expert_ffn_train(x, good, w_in, w_out)
    ops.check_status()
    _, dw_in, dw_out = ops.expert_ffn_backward(x, x, c, w_in, w_out, saved)
    recorded()
    if not bad:
        assert not bool(dw_in.any()) and not bool(dw_out.any())
