"""The word that the expert kernels record faults in, and the check that reads and clears it.  On the host:
the word lies in host memory, and the device's functions are stand-ins."""
from __future__ import annotations

import types

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def experts(monkeypatch):
    from ugdr_b200.ops import experts

    monkeypatch.setattr(experts, "_status", {})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)  # as torch.device("cpu").index
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: types.SimpleNamespace(synchronize=lambda: None))
    return experts


@pytest.mark.parametrize("first", [True, False])  # whether the first call on the device is under inference mode
@pytest.mark.parametrize("check", [True, False])  # and the check
def test_a_fault_is_reported_once_and_cleared(experts, first, check):
    with torch.inference_mode(first):
        word = experts._status_word(torch.device("cpu"))
    for code, text in ((1, "ran out"), (2, "counts")):
        word.numpy()[0] = code  # as a kernel does
        with torch.inference_mode(check), pytest.raises(RuntimeError, match=text):
            experts.check_status()
        with torch.inference_mode(check):
            experts.check_status()
