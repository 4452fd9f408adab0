"""The float64 gradients of the mixer oracle against central differences, and
its properties (CPU)."""
import numpy as np
import pytest

from oracle import mixer_oracle as M


def _delta_case(seed, B=1, L=5, Hk=2, Hv=4, K=3, V=2):
    r = np.random.default_rng(seed)
    k = r.normal(size=(B, L, Hk, K))
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    return dict(q=r.normal(size=(B, L, Hk, K)), k=k, v=r.normal(size=(B, L, Hv, V)),
                g=-r.exponential(0.3, size=(B, L, Hv)), beta=r.uniform(0.1, 1.0, (B, L, Hv)),
                h0=r.normal(size=(B, Hv, K, V))), r


def _differences(f, x, eps=1e-6):
    d = np.empty_like(x)
    for i in np.ndindex(x.shape):
        old = x[i]
        x[i] = old + eps
        hi = f()
        x[i] = old - eps
        lo = f()
        x[i] = old
        d[i] = (hi - lo) / (2 * eps)
    return d


def test_delta_gradients_against_differences():
    c, r = _delta_case(0)
    do, dh = r.normal(size=c["v"].shape), r.normal(size=c["h0"].shape)

    def loss():
        o, S = M.delta_forward(**c)
        return (o * do).sum() + (S * dh).sum()

    got = M.delta_backward(**{n: c[n] for n in ("q", "k", "v", "g", "beta", "h0")}, do=do,
                           dh_last=dh)
    for name, d in zip(("q", "k", "v", "g", "beta", "h0"), got):
        # central differences: truncation and cancellation both ~1e-9 of O(1) values
        np.testing.assert_allclose(d, _differences(loss, c[name]), rtol=1e-6, atol=1e-7,
                                   err_msg=name)


def test_delta_splits_and_padding():
    """A sequence in two calls, and steps with beta = 0 and g = 0 that change nothing."""
    c, r = _delta_case(1, L=7)
    o, S = M.delta_forward(**c)
    one = {n: c[n][:, :3] for n in ("q", "k", "v", "g", "beta")}
    two = {n: c[n][:, 3:] for n in ("q", "k", "v", "g", "beta")}
    o1, S1 = M.delta_forward(**one, h0=c["h0"])
    o2, S2 = M.delta_forward(**two, h0=S1)
    np.testing.assert_allclose(np.concatenate([o1, o2], 1), o, rtol=1e-12)
    np.testing.assert_allclose(S2, S, rtol=1e-12)
    c["beta"][:, 4:], c["g"][:, 4:] = 0.0, 0.0
    _, Sp = M.delta_forward(**c)
    _, S4 = M.delta_forward(**{n: c[n][:, :4] for n in one}, h0=c["h0"])
    np.testing.assert_allclose(Sp, S4, rtol=1e-12)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["silu", "none"])
def test_group_norm_gradients_against_differences(gated, act):
    r = np.random.default_rng(2)
    x, w, b = r.normal(size=(2, 3, 8)), r.normal(size=8), r.normal(size=8)
    gate = r.normal(size=x.shape) if gated else None
    dy = r.normal(size=x.shape)

    def loss():
        return (M.group_norm(x, 2, w, b, gate, act)[0] * dy).sum()

    dx, dw, db, dgate = M.group_norm(x, 2, w, b, gate, act, dy=dy)[3:]
    pairs = [(dx, x), (dw, w), (db, b)] + ([(dgate, gate)] if gated else [])
    for d, t in pairs:
        np.testing.assert_allclose(d, _differences(loss, t), rtol=1e-6, atol=1e-7)
