"""CPU checks of the mixer's C entry points: argument errors come back as
status codes before anything is launched."""
from tssm import _lib

P = 1 << 20   # stand-in address, never dereferenced
Z = 0


def _forward(dtype=1, q=P, B=2, L=4, Hk=2, Hv=4, K=64, V=64, ws=P, nbytes=1 << 40):
    return _lib.lib().tssm_gated_delta_forward(
        dtype, q, P, P, P, P, None, P, None, B, L, Hk, Hv, K, V, *[Z] * 18, 0.125, ws, nbytes,
        None)


def test_delta_forward_status():
    assert _forward(dtype=7) == -4
    assert _forward(q=None) == -1
    assert _forward(Hv=3) == -2 and _forward(Hk=0) == -2 and _forward(L=-1) == -2
    assert _forward(K=0) == -2 and _forward(V=-5) == -2
    assert _forward(K=129) == -6
    assert _forward(B=0) == 0            # nothing to do


def test_delta_step_status():
    f = _lib.lib().tssm_gated_delta_step

    def step(dtype=0, state=P, S=2, Hk=1, Hv=2, K=16, V=16):
        return f(dtype, P, P, P, P, P, state, P, S, Hk, Hv, K, V, *[Z] * 12, 1.0, None)

    assert step(dtype=-1) == -4 and step(state=None) == -1 and step(Hv=0) == -2
    assert step(K=200) == -6 and step(S=0) == 0


def test_delta_workspace():
    f = _lib.lib().tssm_gated_delta_workspace_bytes
    assert f(8, 4096, 16, 16, 64, 64) > 0 and f(1, 0, 1, 1, 1, 1) >= 0
    assert f(1, 4, 2, 3, 8, 8) == -2 and f(1, 4, 1, 1, 129, 8) == -6


def test_group_norm_status():
    L = _lib.lib()

    def fwd(dtype=0, act=1, x=P, mean=None, rstd=None, N=2, S=3, G=4, Cg=8):
        return L.tssm_group_norm_act_fwd(dtype, act, x, P, P, None, P, mean, rstd, N, S, G, Cg,
                                         *[Z] * 6, 1e-5, P, 1 << 40, None)

    def bwd(dx=P, gate=None, dgate=None, dw=P, ws=P, nbytes=1 << 40, G=4):
        return L.tssm_group_norm_act_bwd(0, 1, P, P, P, P, P, P, gate, dx, dw, P, dgate, 2, 3, G,
                                         8, *[Z] * 10, ws, nbytes, None)

    assert fwd(dtype=3) == -4 and fwd(act=2) == -6 and fwd(x=None) == -1
    assert fwd(mean=P) == -1 and fwd(G=0) == -2 and fwd(N=1 << 31) == -6 and fwd(N=0) == 0
    assert bwd(dx=None) == -1 and bwd(gate=P) == -1 and bwd(dgate=P) == -1 and bwd(dw=None) == -1
    assert bwd(ws=None) == -5 and bwd(nbytes=8) == -5 and bwd(G=-1) == -2
    assert L.tssm_group_norm_workspace_bytes(32768, 1, 16, 64) > 0
    assert L.tssm_group_norm_workspace_bytes(1, 1, 0, 64) < 0


def test_delta_backward_status():
    L = _lib.lib()

    def back(dtype=1, q=P, dg=P, B=2, n=40, Hk=2, Hv=4, K=64, V=64, sq=512, sv=256, ws=P,
             nbytes=1 << 40):
        s = [0, sq, 64, 0, sq, 64, 0, sv, 64, 0, 4, 1, 0, 4, 1, 0, sv, 64]
        return L.tssm_gated_delta_backward(dtype, q, P, P, P, P, None, P, None, P, P, P, dg, P,
                                           None, B, n, Hk, Hv, K, V, *s, 0.125, ws, nbytes, None)

    assert back(dtype=5) == -4 and back(q=None) == -1 and back(dg=None) == -1
    assert back(Hv=3) == -2 and back(K=129) == -6
    assert back(sq=8) == -3 and back(sv=0) == -3        # rows that overlap
    assert back(ws=None) == -5 and back(nbytes=1 << 10) == -5 and back(ws=P + 8) == -5
    assert back(B=0) == 0 and back(n=0) == 0
    f = L.tssm_gated_delta_backward_workspace_bytes
    assert f(2, 40, 2, 4, 64, 64) > L.tssm_gated_delta_workspace_bytes(2, 40, 2, 4, 64, 64)
    assert f(1, 4, 2, 3, 8, 8) == -2 and f(1, 4, 1, 1, 129, 8) == -6
