"""The serving call of the experts' block does not drop gradients unseen.  It looks at that before anything
else, so this needs no GPU; what the training calls take does."""
from __future__ import annotations

import pytest

from conftest import gpu_count

torch = pytest.importorskip("torch")


def inputs(device):
    t = dict(dtype=torch.bfloat16, device=device)
    return {"x": torch.ones(4, 16, **t), "counts": torch.tensor([4], dtype=torch.int32, device=device),
            "w_in": torch.ones(1, 2, 8, 16, **t), "w_out": torch.ones(1, 16, 8, **t), "out": torch.zeros(4, 16, **t)}


@pytest.mark.parametrize("name", ["x", "w_in", "w_out", "out"])
def test_the_serving_call_refuses_to_drop_a_gradient(name):
    from ugdr_b200 import ops

    a = inputs("cpu")
    a[name].requires_grad_()
    with pytest.raises(ValueError, match=f"{name} requires a gradient"):
        ops.expert_ffn(**a)
    for off in (torch.no_grad(), torch.inference_mode()):  # on to the next check: these are host tensors
        with off, pytest.raises(ValueError, match="CUDA"):
            ops.expert_ffn(**a)


@pytest.mark.gpu
def test_serving_without_gradients_and_training_calls_take_parameters():
    from ugdr_b200 import ops

    if gpu_count() < 1:
        pytest.skip("no GPU")
    a = inputs("cuda")
    want = ops.expert_ffn(a["x"], a["counts"], a["w_in"], a["w_out"])
    for name in ("x", "w_in", "w_out"):
        a[name].requires_grad_()
    with torch.no_grad():
        assert torch.equal(ops.expert_ffn(**a), want)
    y, saved = ops.expert_ffn_train(a["x"], a["counts"], a["w_in"], a["w_out"])
    assert torch.equal(y, want) and not y.requires_grad
    dx, dw_in, dw_out = ops.expert_ffn_backward(torch.ones_like(y), a["x"], a["counts"], a["w_in"], a["w_out"], saved)
    assert not (dx.requires_grad or dw_in.requires_grad or dw_out.requires_grad)
    for p, g in ((a["x"], dx), (a["w_in"], dw_in), (a["w_out"], dw_out)):
        p.grad = g
    ops.check_status()
