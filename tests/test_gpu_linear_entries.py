"""Linear attention's C entry points with what a C caller hands over: a workspace of
exactly the advertised size, whatever it held before, and outputs at any place.  What lies
around either stays."""
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M
from test_gpu_linear import BF16, F16, F32, NAMES, TOL, gradients, inputs, run

pytestmark = pytest.mark.gpu

CODE = {F32: 0, BF16: 1, F16: 2}
AROUND = 4096    # bytes before and behind


class Room:
    """``nbytes`` bytes of NaN on a 256-byte boundary, with a pattern around them."""

    def __init__(self, dev, nbytes):
        self.all = torch.full((nbytes + 2 * AROUND,), 0xA5, dtype=torch.uint8, device=dev)
        self.inside = self.all[AROUND:AROUND + nbytes]
        self.inside.fill_(0xFF)
        assert self.inside.data_ptr() % 256 == 0

    def check(self):
        assert (self.all[:AROUND] == 0xA5).all() and (self.all[-AROUND:] == 0xA5).all()


def strides(*tensors):
    return [s for t in tensors for s in t.stride()[:3]]


def operands(d):
    return [d[n] for n in ("q", "k", "v")]


def call(name, d, *args):
    from tssm import _lib
    _lib.call(name, CODE[d["q"].dtype], *(t.data_ptr() for t in operands(d)), d["g"].data_ptr(),
              d["h0"].data_ptr(), *args, torch.cuda.current_stream().cuda_stream)


def sizes(d):
    return (*d["q"].shape[:3], *d["v"].shape[2:3], d["q"].shape[3], d["v"].shape[3])


CASES = [  # B, L, Hk, Hv, K, V
    (1, 200, 2, 2, 64, 40),       # whole
    (2, 130, 3, 3, 20, 33),
    (1, 3001, 1, 2, 64, 40),      # segments
    (2, 1900, 1, 1, 128, 24),
    (1, 700, 1, 2, 100, 72),      # two segments
    (2, 330, 1, 4, 48, 65),       # gradients: a workgroup for each value head
    (1, 2000, 1, 3, 32, 20),      # that and segments
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,L,Hk,Hv,K,V", CASES)
def test_forward_in_a_workspace_of_its_size(dev, dtype, B, L, Hk, Hv, K, V):
    from tssm import _lib
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L, h0=True, rate=0.1)
    want, last = run(d)
    n = _lib.lib().tssm_linear_attention_workspace_bytes(*sizes(d))
    assert n >= 0
    ws, o, S = Room(dev, n), torch.empty_like(want), torch.empty_like(last)
    call("tssm_linear_attention_forward", d, o.data_ptr(), S.data_ptr(), *sizes(d),
         *strides(*operands(d), d["g"], o), K ** -0.5, ws.inside.data_ptr() if n else None, n)
    ws.check()
    assert torch.equal(o, want) and torch.equal(S, last)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("odd", [None, "dq", "dk", "dv"])
@pytest.mark.parametrize("B,L,Hk,Hv,K,V", CASES)
def test_backward_in_a_workspace_of_its_size(dev, dtype, odd, B, L, Hk, Hv, K, V):
    """``odd``: the output that starts on no 16-byte boundary."""
    from tssm import _lib
    r = torch.Generator().manual_seed(L)
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L, h0=True, rate=0.1)
    do = torch.randn(B, L, Hv, V, generator=r).to(dtype).to(dev)
    dh = torch.randn(B, Hv, K, V, generator=r).to(dev)
    want = gradients(d, do, dh)
    n = _lib.lib().tssm_linear_attention_backward_workspace_bytes(CODE[dtype], *sizes(d))
    ws, rooms, got = Room(dev, n), [], []
    for name, t in zip(NAMES, want):
        rooms.append(Room(dev, (t.numel() + 1) * t.element_size()))
        at = 1 if name == odd else 0
        got.append(rooms[-1].inside.view(t.dtype)[at:at + t.numel()].view(t.shape))
    dq, dk, dv, dg, dh0 = got
    call("tssm_linear_attention_backward", d, do.data_ptr(), dh.data_ptr(),
         *(t.data_ptr() for t in got), *sizes(d), *strides(*operands(d), d["g"], do), K ** -0.5,
         ws.inside.data_ptr(), n)
    ws.check()
    ref = M.linear_backward(*(np64(d[x]) for x in ("q", "k", "v", "g")), np64(do),
                            h0=np64(d["h0"]), dh_last=np64(dh))
    for name, room, x, y, z in zip(NAMES, rooms, got, want, ref):
        room.check()
        spare = room.inside.view(x.dtype)[0 if name == odd else -1]
        assert torch.isnan(spare), name          # the element beside the output
        if odd is None:
            assert torch.equal(x, y), name
        assert_close(x, z, TOL[dtype] if name in ("dq", "dk", "dv") else TOL[F32], name)
