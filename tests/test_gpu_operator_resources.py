"""The model operators' kernels keep everything in registers and shared memory."""
from __future__ import annotations

import pytest

from conftest import gpu_count

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")


def test_no_operator_kernel_uses_local_memory():
    from ugdr_b200 import ops

    if gpu_count() < 1:
        pytest.skip("no GPU")
    kernels = [a for a in ops.kernel_attributes() if a["name"].startswith(("expert_", "grad_", "count_check"))]
    assert {"grad_norm_kernel", "grad_sum_kernel", "grad_scale_kernel", "count_check_kernel"} <= {a["name"] for a in kernels}
    assert [(a["name"], a["local_bytes_per_thread"]) for a in kernels if a["local_bytes_per_thread"]] == []
