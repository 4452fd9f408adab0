"""The float64 gradients of the oracle's linear attention and of its norm and
rotation against central differences, and their properties (CPU)."""
import numpy as np
import pytest

from oracle import mixer_oracle as M
from test_oracle_mixer import _differences


def _case(seed, B=1, L=5, Hk=2, Hv=4, K=3, V=2):
    r = np.random.default_rng(seed)
    return dict(q=r.normal(size=(B, L, Hk, K)), k=r.normal(size=(B, L, Hk, K)),
                v=r.normal(size=(B, L, Hv, V)), g=-r.exponential(0.3, size=(B, L, Hv)),
                h0=r.normal(size=(B, Hv, K, V))), r


def test_linear_gradients_against_differences():
    c, r = _case(0)
    do, dh = r.normal(size=c["v"].shape), r.normal(size=c["h0"].shape)

    def loss():
        o, S = M.linear_forward(**c)
        return (o * do).sum() + (S * dh).sum()

    for name, d in zip(("q", "k", "v", "g", "h0"), M.linear_backward(**c, do=do, dh_last=dh)):
        # central differences: truncation and cancellation both ~1e-9 of O(1) values
        np.testing.assert_allclose(d, _differences(loss, c[name]), rtol=1e-6, atol=1e-7,
                                   err_msg=name)


def test_linear_splits_and_closed_form():
    c, _ = _case(1, L=7, Hk=4)
    o, S = M.linear_forward(**c)
    one = {n: c[n][:, :3] for n in ("q", "k", "v", "g")}
    two = {n: c[n][:, 3:] for n in one}
    o1, S1 = M.linear_forward(**one, h0=c["h0"])
    o2, S2 = M.linear_forward(**two, h0=S1)
    np.testing.assert_allclose(np.concatenate([o1, o2], 1), o, rtol=1e-12)
    np.testing.assert_allclose(S2, S, rtol=1e-12)
    # o_t from zero: sum over i <= t of exp(G_t - G_i) (q_t . k_i) v_i
    o, _ = M.linear_forward(**dict(c, h0=None), scale=1.0)
    G = np.cumsum(c["g"], 1)
    for t in range(7):
        want = sum(np.exp(G[:, t] - G[:, i])[..., None] * c["v"][:, i]
                   * (c["q"][:, t] * c["k"][:, i]).sum(-1)[..., None] for i in range(t + 1))
        np.testing.assert_allclose(o[:, t], want, rtol=1e-11)


@pytest.mark.parametrize("norm", ["rms", "l2", "none"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rotary_gradients_against_differences(norm, interleaved):
    r = np.random.default_rng(3)
    x, w, pos = r.normal(size=(2, 3, 2, 7)), r.normal(size=7), r.uniform(0, 9, size=(2, 3))
    kw = dict(pos=pos, freq=np.array([1.0, 0.1]), w=w, norm=norm, interleaved=interleaved,
              amplitude=1.3)
    dy = r.normal(size=x.shape)
    _, dx, dw = M.norm_rotary(x, dy=dy, **kw)
    for d, t in ((dx, x), (dw, w)):
        np.testing.assert_allclose(
            d, _differences(lambda: (M.norm_rotary(x, **kw) * dy).sum(), t), rtol=1e-6, atol=1e-7)


def test_rotation_keeps_lengths_and_distances():
    """Without a norm the rotation keeps each row's length, and q . k depends on the
    difference of positions alone."""
    r = np.random.default_rng(4)
    q, k, freq = r.normal(size=(1, 8)), r.normal(size=(1, 8)), 10.0 ** -np.arange(4.0)
    for interleaved in (False, True):
        def at(x, p):
            return M.norm_rotary(x, np.array(float(p)), freq, norm="none",
                                 interleaved=interleaved)[0]
        np.testing.assert_allclose(np.linalg.norm(at(q, 5)), np.linalg.norm(q), rtol=1e-12)
        np.testing.assert_allclose(at(q, 7) @ at(k, 3), at(q, 104) @ at(k, 100), rtol=1e-12)
