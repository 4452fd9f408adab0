"""CPU checks of what a call that goes through its stream's workspace asks on the host:
one look where the buffer is long enough, everything else only where it is not (the
library is a stand-in)."""
import pytest
import torch

from tssm import _lib, workspace

KEY = (-1, 7, workspace.SSD)


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(workspace, "_cache", {})
    monkeypatch.setattr(workspace, "_dev_index", lambda device: -1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append((name, *args)))
    return seen


def test_a_buffer_that_is_there_is_looked_up_once(calls, monkeypatch):
    t = torch.zeros(1)
    workspace.call("f", t, 7, 100, 1, 2)
    buf = workspace._cache[KEY]

    def asked(*args):
        raise AssertionError("asked again")

    class Asked:
        __enter__ = __exit__ = asked

    monkeypatch.setattr(workspace, "_dev_index", asked)
    monkeypatch.setattr(workspace, "_raise_if_flagged", asked)
    monkeypatch.setattr(workspace, "_lock", Asked())
    workspace.call("g", t, 7, buf.numel(), 3)
    assert calls == [("f", 1, 2, buf.data_ptr(), buf.numel(), 7),
                     ("g", 3, buf.data_ptr(), buf.numel(), 7)]
    with pytest.raises(AssertionError, match="asked again"):
        workspace.call("h", t, 7, buf.numel() + 1)
    assert len(calls) == 2


def test_a_buffer_that_is_too_short_is_replaced(calls):
    t = torch.zeros(1)
    workspace.call("f", t, 7, 100)
    old = workspace._cache[KEY]
    workspace.call("f", t, 7, old.numel() + 1)
    new = workspace._cache[KEY]
    assert new is not old and new.numel() == old.numel() + 1 and not new.any()
    workspace.call("f", t, 7, 100)
    assert workspace._cache[KEY] is new and calls[2][-3:] == (new.data_ptr(), new.numel(), 7)


def test_other_kinds_are_asked_as_before(calls, monkeypatch):
    """A look-back workspace's flag is read on every request."""
    polled = []
    monkeypatch.setattr(workspace, "_raise_if_flagged", polled.append)
    cpu = torch.device("cpu")
    workspace._cache[(-1, 7, workspace.LOOKBACK)] = torch.zeros(1 << 16, dtype=torch.uint8)
    for _ in range(2):
        workspace.get(cpu, 7, 16)
    assert polled == [(-1, 7, workspace.LOOKBACK)] * 2
