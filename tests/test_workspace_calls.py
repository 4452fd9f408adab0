"""CPU checks of how calls that enqueue several launches use their stream's
workspace: one thread's launches at a time, on a buffer that stays (the library
is a stand-in that records the calls)."""
import threading
import time

import pytest
import torch

from tssm import _lib, delta, fused, groupnorm, launch, workspace


class Library:
    """Answers every size query, the larger the more often it was asked."""

    def __init__(self):
        self.asked = 0

    def __getattr__(self, name):
        def f(*args):
            self.asked += 1
            return 1 << (17 + self.asked) if name.endswith("bytes") else 0
        return f


@pytest.fixture
def stub(monkeypatch):
    """Lets CPU tensors through the checks; returns the list of events."""
    events, library = [], Library()
    for module in (delta, fused, groupnorm, launch):
        monkeypatch.setattr(module, "need_gpu", lambda t, what: t)
        monkeypatch.setattr(module, "stream_handle", lambda t: 7)
    monkeypatch.setattr(workspace, "_dev_index", lambda device: -1)
    monkeypatch.setattr(workspace, "_cache", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(_lib, "lib", lambda: library)
    get = workspace.get

    def recorded(*args):
        buf = get(*args)
        events.append(("workspace", threading.get_ident()))
        return buf

    def call(name, *args):
        events.append(("begin", threading.get_ident()))
        time.sleep(0.005)          # the launches: other threads run meanwhile
        held = workspace._cache[(-1, 7, workspace.SSD)].data_ptr()
        events.append(("end" if held == args[-3] else "buffer replaced", threading.get_ident()))

    monkeypatch.setattr(workspace, "get", recorded)
    monkeypatch.setattr(_lib, "call", call)
    return events


def delta_operands():
    return [torch.zeros(1, 40, 2, 8) for _ in range(3)] + [torch.zeros(1, 40, 2) for _ in range(2)]


def delta_forward():
    delta.gated_delta_forward(*delta_operands())


def delta_backward():
    delta.gated_delta_backward(*delta_operands(), torch.zeros(1, 40, 2, 8))


def norm_forward():
    groupnorm.group_norm_act_forward(torch.zeros(2, 9, 8), 2)


def norm_backward():
    x = torch.zeros(2, 9, 8)
    groupnorm.group_norm_act_backward(x, x, torch.zeros(2, 2, dtype=torch.float64),
                                      torch.zeros(2, 2), 2)


def ssd_forward():
    x, bc = torch.zeros(1, 40, 2, 16), torch.zeros(1, 40, 2, 32)
    fused.ssd_scan_forward(x, torch.zeros(1, 40, 2), torch.zeros(2), bc, bc)


@pytest.mark.parametrize("first,second", [
    (delta_forward, delta_forward), (delta_forward, delta_backward),
    (norm_forward, norm_backward), (norm_forward, delta_backward), (ssd_forward, delta_forward)])
def test_threads_of_one_stream_take_turns(stub, first, second):
    start = threading.Barrier(2)

    def work(f):
        start.wait()
        for _ in range(4):
            f()

    threads = [threading.Thread(target=work, args=(f,)) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(stub) == 2 * 4 * 3
    for i in range(0, len(stub), 3):
        assert [e for e, _ in stub[i:i + 3]] == ["workspace", "begin", "end"], stub
        assert len({t for _, t in stub[i:i + 3]}) == 1, stub


def test_a_failing_call_lets_others_in(stub, monkeypatch):
    def fail(name, *args):
        raise _lib.TssmError("refused")

    with monkeypatch.context() as m:
        m.setattr(_lib, "call", fail)
        with pytest.raises(_lib.TssmError):
            norm_forward()
    done = threading.Thread(target=norm_forward, daemon=True)
    done.start()
    done.join(10)
    assert not done.is_alive() and stub[-1][0] == "end"


@pytest.mark.parametrize("f", [delta_forward, delta_backward, norm_forward, norm_backward,
                               ssd_forward])
def test_captured_calls_have_memory_of_their_own(stub, monkeypatch, f):
    """A graph may outlive the stream's buffer, which larger calls replace."""
    seen = []
    norm_forward()                                   # the stream has a buffer
    before = dict(workspace._cache)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(args[-3:-1]))
    f()
    (address, size), buf = seen[0], before[(-1, 7, workspace.SSD)]
    assert size > 0 and address % 64 == 0
    assert not buf.data_ptr() <= address < buf.data_ptr() + buf.numel()
    assert list(workspace._cache) == list(before) and workspace._cache[(-1, 7, workspace.SSD)] is buf
