"""Tensors that the operators write are seen to have changed: a backward pass that saved one of them, or a
view of the same memory, raises torch's error instead of using what it finds there."""
from __future__ import annotations

import pytest

from conftest import gpu_count

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def one_gpu():
    if gpu_count() < 1:
        pytest.skip("no GPU")


def saved(*shape, dtype):
    """(a tensor that a backward pass has saved, the loss of that pass)"""
    a = torch.ones(*shape, dtype=dtype, device="cuda", requires_grad=True) * 2
    return a, (a * a).float().sum()


def overwritten(loss):
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_clipped_gradients():
    from ugdr_b200.ops import GradClip

    for dtype in (torch.float32, torch.bfloat16):
        whole, loss = saved(1000, dtype=dtype)
        part, part_loss = saved(1000, dtype=dtype)
        out, out_loss = saved(500, dtype=torch.float32)
        plan = GradClip([whole.detach(), part.detach()[:300]])
        apart = GradClip([torch.ones(500, dtype=dtype, device="cuda")], [out.detach()])
        plan.sum_squares()
        versions = whole._version, part._version
        assert versions == (0, 0)  # only read so far
        plan.clip(1.0)
        apart.clip(1.0)
        for t in (loss, part_loss, out_loss):
            overwritten(t)


def test_outputs_of_the_block():
    from ugdr_b200 import ops

    bf16 = torch.bfloat16
    x, counts = torch.ones(4, 16, dtype=bf16, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    w_in, w_out = torch.ones(1, 2, 8, 16, dtype=bf16, device="cuda"), torch.ones(1, 16, 8, dtype=bf16, device="cuda")
    y, y_loss = saved(4, 16, dtype=bf16)
    ops.expert_ffn(x, counts, w_in, w_out, out=y.detach())
    overwritten(y_loss)
    y, y_loss = saved(4, 16, dtype=bf16)
    _, kept = ops.expert_ffn_train(x, counts, w_in, w_out, out=y.detach())
    overwritten(y_loss)
    dx, dw_in, dw_out = (saved(*t.shape, dtype=bf16) for t in (x, w_in, w_out))
    ops.expert_ffn_backward(x, x, counts, w_in, w_out, kept, dx=dx[0].detach(), dw_in=dw_in[0].detach(),
                            dw_out=dw_out[0].detach(), stream=torch.cuda.current_stream())
    for _, loss in (dx, dw_in, dw_out):
        overwritten(loss)
    assert x._version == w_in._version == w_out._version == counts._version == 0


def test_under_inference_mode():
    from ugdr_b200 import ops

    with torch.inference_mode():
        x, counts = torch.ones(4, 16, dtype=torch.bfloat16, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
        w_in, w_out = (torch.ones(*s, dtype=x.dtype, device="cuda") for s in ((1, 2, 8, 16), (1, 16, 8)))
        want = ops.expert_ffn(x, counts, w_in, w_out)
        assert torch.equal(ops.expert_ffn(x, counts, w_in, w_out, out=x), want)
        g = torch.ones(100, device="cuda")
        assert float(ops.GradClip([g[:50], g[50:]]).clip(5.0)) == pytest.approx(10.0, rel=1e-6)
        assert float(g.sum()) == pytest.approx(50.0, rel=1e-5)
    ops.check_status()
