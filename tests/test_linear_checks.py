"""CPU checks of linear attention's arguments: its C entry points' status codes
and its Python entry points' refusals (nothing is launched)."""
import pytest
import torch

from tssm import _lib, linear

P = 1 << 20   # stand-in address, never dereferenced


def _forward(dtype=1, q=P, B=2, L=400, Hk=2, Hv=4, K=64, V=64, ws=P, nbytes=1 << 40):
    return _lib.lib().tssm_linear_attention_forward(
        dtype, q, P, P, P, None, P, None, B, L, Hk, Hv, K, V, *[0] * 15, 0.125, ws, nbytes, None)


def test_forward_status():
    assert _forward(dtype=7) == -4
    assert _forward(q=None) == -1
    assert _forward(Hv=3) == -2 and _forward(Hk=0) == -2 and _forward(L=-1) == -2
    assert _forward(K=0) == -2 and _forward(V=-5) == -2 and _forward(B=-1) == -2
    assert _forward(K=129) == -6 and _forward(V=(1 << 21) + 1) == -6
    assert _forward(B=0) == 0            # nothing to do


def test_step_status():
    f = _lib.lib().tssm_linear_attention_step

    def step(dtype=0, state=P, S=2, Hk=1, Hv=2, K=16, V=16):
        return f(dtype, P, P, P, P, state, P, S, Hk, Hv, K, V, *[0] * 10, 1.0, None)

    assert step(dtype=-1) == -4 and step(state=None) == -1 and step(Hv=0) == -2
    assert step(K=200) == -6 and step(V=1 << 22) == -6 and step(S=0) == 0


def test_workspace():
    f = _lib.lib().tssm_linear_attention_workspace_bytes
    assert f(8, 4096, 16, 16, 64, 64) >= 0 and f(1, 0, 1, 1, 1, 1) == 0
    assert f(1, 4, 2, 3, 8, 8) == -2 and f(1, 4, 1, 1, 129, 8) == -6


def test_backward_status():
    L = _lib.lib()

    def back(dtype=1, q=P, dg=P, B=2, n=400, Hk=2, Hv=4, K=64, V=64, sq=512, sv=256, ws=P,
             nbytes=1 << 40):
        s = [0, sq, 64, 0, sq, 64, 0, sv, 64, 0, 4, 1, 0, sv, 64]
        return L.tssm_linear_attention_backward(dtype, q, P, P, P, None, P, None, P, P, P, dg,
                                                None, B, n, Hk, Hv, K, V, *s, 0.125, ws, nbytes,
                                                None)

    assert back(dtype=5) == -4 and back(q=None) == -1 and back(dg=None) == -1
    assert back(Hv=3) == -2 and back(K=129) == -6 and back(V=1 << 22) == -6
    assert back(sq=8) == -3 and back(sv=0) == -3        # rows that overlap
    assert back(sq=1 << 24) == -3                       # too far apart
    assert back(ws=None) == -5 and back(nbytes=1 << 10) == -5 and back(ws=P + 8) == -5
    assert back(B=0) == 0 and back(n=0) == 0
    f = L.tssm_linear_attention_backward_workspace_bytes
    assert f(1, 2, 400, 2, 4, 64, 64) > L.tssm_linear_attention_workspace_bytes(2, 400, 2, 4, 64,
                                                                               64)
    assert f(0, 2, 384, 2, 4, 128, 64) == f(1, 2, 384, 2, 4, 128, 64)   # chunks of 64 alike
    assert f(3, 1, 4, 1, 1, 8, 8) == -4 and f(1, 1, 4, 2, 3, 8, 8) == -2
    assert f(1, 1, 4, 1, 1, 129, 8) == -6


class On(torch.Tensor):
    """A CPU tensor that is on device ``dev`` by its own account."""
    dev = 0

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return self.dev


class OnOther(On):
    dev = 1


@pytest.fixture(autouse=True)
def no_library(monkeypatch):
    def called(*args):
        raise AssertionError("the library was called")
    monkeypatch.setattr(linear.workspace, "call", called)
    monkeypatch.setattr(linear, "on_device", called)
    monkeypatch.setattr(linear, "stream_handle", lambda t: 0)


def on(t, other=False):
    return t.as_subclass(OnOther if other else On)


def operands(lead=(2, 5), Hk=2, Hv=4, K=8, V=6, dtype=torch.float32, other=None):
    shapes = dict(q=(*lead, Hk, K), k=(*lead, Hk, K), v=(*lead, Hv, V), g=(*lead, Hv))
    return {n: on(torch.zeros(s, dtype=torch.float32 if n == "g" else dtype), n == other)
            for n, s in shapes.items()}


def forward(d, **kw):
    return linear.linear_attention_forward(d["q"], d["k"], d["v"], d["g"], **kw)


def step(d, state, **kw):
    return linear.linear_attention_step(d["q"], d["k"], d["v"], d["g"], state, **kw)


@pytest.mark.parametrize("name", ["k", "v", "g"])
def test_another_device(name):
    with pytest.raises(ValueError, match=f"{name} must be on device 0"):
        forward(operands(other=name))
    with pytest.raises(ValueError, match=f"{name} must be on device 0"):
        step(operands((3,), other=name), on(torch.zeros(3, 4, 8, 6)))


def test_shapes_and_types():
    for change, match in ((dict(k=on(torch.zeros(2, 5, 2, 7))), "k must be"),
                          (dict(v=on(torch.zeros(2, 4, 4, 6))), "v must be"),
                          (dict(v=on(torch.zeros(2, 5, 3, 6))), "multiple of q's"),
                          (dict(g=on(torch.zeros(2, 5, 2))), "g must be"),
                          (dict(q=on(torch.zeros(2, 5, 2))), "expected q, k"),
                          (dict(q=on(torch.zeros(2, 5, 2, 0)), k=on(torch.zeros(2, 5, 2, 0))),
                           "all sizes positive")):
        with pytest.raises(ValueError, match=match):
            forward(dict(operands(), **change))
    with pytest.raises(TypeError, match="v must be torch.bfloat16"):
        forward(dict(operands(dtype=torch.bfloat16), v=on(torch.zeros(2, 5, 4, 6))))
    with pytest.raises(TypeError, match="unsupported dtype"):
        forward(operands(dtype=torch.float64))
    with pytest.raises(TypeError, match="g: expected a float"):
        forward(dict(operands(), g=on(torch.zeros(2, 5, 4, dtype=torch.int32))))
    with pytest.raises(ValueError, match="at most 128"):
        forward(operands(K=129))
    with pytest.raises(TypeError):
        forward(dict(operands(), q=None))
    with pytest.raises(ValueError, match="HIP device"):
        forward(dict(operands(), q=torch.zeros(2, 5, 2, 8)))


def test_backward_refusals():
    d, do = operands(), on(torch.zeros(2, 5, 4, 6))

    def back(do, **kw):
        return linear.linear_attention_backward(d["q"], d["k"], d["v"], d["g"], do, **kw)

    with pytest.raises(ValueError, match="do must be"):
        back(on(torch.zeros(2, 5, 4, 7)))
    with pytest.raises(TypeError, match="do must be"):
        back(do.half())
    with pytest.raises(ValueError, match="do must be on device 0"):
        back(on(torch.zeros(2, 5, 4, 6), True))
    with pytest.raises(ValueError, match="dh_last must be"):
        back(do, dh_last=on(torch.zeros(2, 4, 6, 8)))
    with pytest.raises(ValueError, match="dh_last must be on device 0"):
        back(do, dh_last=on(torch.zeros(2, 4, 8, 6), True))


def test_states_and_outputs():
    d = operands()
    with pytest.raises(ValueError, match="h0 must be"):
        forward(d, h0=on(torch.zeros(2, 4, 6, 8)))
    with pytest.raises(ValueError, match="h0 must be on device"):
        forward(d, h0=on(torch.zeros(2, 4, 8, 6), True))
    with pytest.raises(ValueError, match="out must be"):
        forward(d, out=on(torch.zeros(2, 5, 4, 7)))
    with pytest.raises(TypeError, match="out must be"):
        forward(d, out=on(torch.zeros(2, 5, 4, 6, dtype=torch.float16)))
    with pytest.raises(ValueError, match="share memory"):
        forward(d, out=on(torch.zeros(2, 1, 4, 6)).expand(2, 5, 4, 6))
    d = operands((3,))
    with pytest.raises(TypeError, match="state must be torch.float32"):
        step(d, on(torch.zeros(3, 4, 8, 6, dtype=torch.bfloat16)))
    with pytest.raises(ValueError, match="contiguous"):
        step(d, on(torch.zeros(3, 4, 6, 8)).transpose(2, 3))
    with pytest.raises(ValueError, match="innermost"):
        forward(dict(operands(), q=on(torch.zeros(2, 5, 8, 2)).transpose(2, 3)), out=None)
