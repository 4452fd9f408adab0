"""CPU checks of how linear attention and the norm and rotation use their stream's
workspace: one thread's launches at a time, captured calls on memory of their own
(the library is a stand-in that records the calls)."""
import threading

import pytest
import torch

from test_workspace_calls import delta_forward, stub  # noqa: F401
from tssm import _lib, linear, qknorm, workspace


@pytest.fixture
def calls(stub, monkeypatch):  # noqa: F811
    for module in (linear, qknorm):
        monkeypatch.setattr(module, "need_gpu", lambda t, what: t)
        monkeypatch.setattr(module, "stream_handle", lambda t: 7)
        monkeypatch.setattr(module, "on_device", lambda device, f, *args: f(*args))
    return stub


def operands():
    return [torch.zeros(1, 40, 2, 8) for _ in range(3)] + [torch.zeros(1, 40, 2)]


def forward():
    linear.linear_attention_forward(*operands())


def backward():
    linear.linear_attention_backward(*operands(), torch.zeros(1, 40, 2, 8))


def qk_backward():
    x = torch.zeros(1, 40, 2, 8)
    qknorm.qk_norm_rotary_backward(x, x, x, x, None, None, torch.zeros(8), torch.zeros(8))


@pytest.mark.parametrize("first,second", [
    (forward, forward), (forward, backward), (backward, qk_backward), (qk_backward, delta_forward)])
def test_threads_of_one_stream_take_turns(calls, first, second):
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
    # (a buffer is asked for where the one that is there is too small)
    launches = [e for e in calls if e[0] != "workspace"]
    assert len(launches) == 2 * 4 * 2
    for begin, end in zip(launches[::2], launches[1::2]):
        assert (begin[0], end[0]) == ("begin", "end") and begin[1] == end[1], calls
    for i, (e, thread) in enumerate(calls):
        if e == "workspace":
            assert calls[i + 1] == ("begin", thread), calls


@pytest.mark.parametrize("f", [forward, backward, qk_backward])
def test_captured_calls_have_memory_of_their_own(calls, monkeypatch, f):
    seen = []
    backward()                                       # the stream has a buffer
    before = dict(workspace._cache)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(args[-3:-1]))
    f()
    (address, size), buf = seen[0], before[(-1, 7, workspace.SSD)]
    assert size > 0 and address % 64 == 0
    assert not buf.data_ptr() <= address < buf.data_ptr() + buf.numel()
    assert list(workspace._cache) == list(before)
