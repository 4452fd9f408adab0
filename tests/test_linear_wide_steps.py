"""CPU checks of linear attention's gradients where one step of all heads is so long that
a chunk of them passes 31 bits: what reaches the library can be read by a chunk (nothing
is launched)."""
import pytest
import torch

from test_linear_checks import on
from tssm import linear

MOST = (1 << 31) // (129 * 4)     # floats between two steps


@pytest.fixture
def strides(monkeypatch):
    """The strides (b, l, h) of q, k, v, g and dO that a call hands over."""
    seen = []

    def taken(device, f, *args):
        seen.append([args[-16 + i:-16 + i + 3] for i in range(0, 15, 3)])

    monkeypatch.setattr(linear, "stream_handle", lambda t: 0)
    monkeypatch.setattr(linear, "on_device", taken)
    return seen


@pytest.mark.parametrize("Hk,Hv,K,V,far", [
    (1, 2, 2, 1 << 21, "v"), (1, 64, 2, 1 << 16, "v"),      # heads that are wide, or many
    (1 << 15, 1 << 15, 128, 2, "qk"),
])
def test_backward(strides, Hk, Hv, K, V, far):
    L = 2
    q, k = (on(torch.zeros(1, L, Hk, K)) for _ in range(2))
    v, do = (on(torch.zeros(1, L, Hv, V)) for _ in range(2))
    linear.linear_attention_backward(q, k, v, on(torch.zeros(1, L, Hv)), do)
    sq, sk, sv, sg, sd = strides[0]
    for s, H, N, wide in ((sq, Hk, K, "qk" == far), (sk, Hk, K, "qk" == far),
                          (sv, Hv, V, "v" == far), (sd, Hv, V, "v" == far)):
        # (the batch's stride of one sequence says nothing)
        assert s[1:] == ((N, L * N) if wide else (H * N, N)) and N <= s[1] < MOST


def test_heads_first_stays(strides):
    """Views whose steps are near each other are handed over as they are."""
    L, Hv, V = 2, 64, 1 << 16
    q = on(torch.zeros(1, L, 1, 2))
    v = on(torch.zeros(1, Hv, L, V)).transpose(1, 2)
    linear.linear_attention_backward(q, q, v, on(torch.zeros(1, L, Hv)), v)
    assert strides[0][2][1:] == (V, L * V) and strides[0][4][1:] == (V, L * V)
