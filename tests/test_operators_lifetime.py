"""Memory that an operator keeps to itself stays until every stream that uses it is through with it.
On the host: the device's streams, the library and the tensors are stand-ins that record."""
from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")


class Block:
    """A tensor, as far as the operators use one."""

    def __init__(self):
        self.streams = []

    def record_stream(self, stream):
        self.streams.append(stream)

    def data_ptr(self):
        return 0x1000

    def new_empty(self, *a, **k):
        return Block()


@pytest.fixture
def plan(monkeypatch):
    """(a plan made on stream 7 over two gradients, one of them scaled elsewhere, a function that makes
    another stream the current one)"""
    from ugdr_b200.ops import grads

    at = [7]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: at[0])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: at[0], raising=False)
    monkeypatch.setattr(grads, "_lib", lambda: types.SimpleNamespace(ugdr_x_grad_clip=lambda *a: 0,
                                                                     ugdr_x_grad_sum_squares=lambda *a: 0))
    p = grads.GradClip.__new__(grads.GradClip)
    p.device, p.grads, p._plan, p._n, p._chunks = torch.device("cuda", 0), (Block(), Block()), Block(), 2, 2
    p.out = (p.grads[0], Block())
    p._home, p._kept, p._written = 7, set(), ()
    return p, lambda s: at.__setitem__(0, s)


def test_a_plan_is_kept_for_every_stream_that_used_it(plan):
    p, switch = plan
    memory = (p._plan, *p.grads, *p.out)
    p.clip(1.0)
    assert all(b.streams == [] for b in memory)  # the allocator knows of the stream it was made on
    switch(9)
    p.clip(1.0)
    assert all(9 in b.streams for b in memory)
    switch(11)
    p.sum_squares()
    assert all(11 in b.streams for b in memory)
    switch(9)
    p.clip(1.0)
    assert p._plan.streams == [9, 11]  # once is enough: the plan holds its tensors


@pytest.mark.gpu
def test_a_plan_used_on_another_stream_is_reported_to_the_allocator(monkeypatch):
    from conftest import gpu_count
    from ugdr_b200.ops import GradClip

    if gpu_count() < 1:
        pytest.skip("no GPU")
    kept = []
    record = torch.Tensor.record_stream
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: (kept.append((t.data_ptr(), s)), record(t, s))[1])
    g, out = torch.ones(5000, device="cuda"), torch.empty(5000, device="cuda")
    plan = GradClip([g], [out])
    plan.clip(1.0)
    assert kept == []
    side, chosen = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        norm = plan.clip(1.0)
    memory = {t.data_ptr() for t in (plan._plan, g, out)}
    assert {a for a, s in kept if s == side} == memory
    plan.sum_squares(stream=chosen)
    assert {a for a, s in kept if s == chosen} == memory
    torch.cuda.synchronize()
    assert float(norm) == pytest.approx(5000 ** 0.5, rel=1e-6)
