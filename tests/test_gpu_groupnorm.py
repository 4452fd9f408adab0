"""GPU parity of the group norm with an activation against float64.

Tolerances, normwise: fp32 outputs 1e-5 (sums in a fixed tree order, the
variance about the mean), 16-bit outputs twice the rounding of the largest
value (2^-8 bfloat16, 2^-11 float16).  dw and db are fp32 sums of N S terms of
both signs whose normwise error stays near sqrt(N S) 2^-24 of the terms' size:
also 1e-5.
"""
import numpy as np
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 1e-5, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def inputs(dev, N, S, C, dtype, gated, seed=0, offset=0.5):
    r = torch.Generator().manual_seed(seed)

    def n(*shape):
        return torch.randn(*shape, generator=r)

    d = dict(x=(n(N, S, C) + offset * n(C)).to(dtype), w=1.0 + 0.3 * n(C), b=0.3 * n(C),
             gate=n(N, S, C).to(dtype) if gated else None, dy=n(N, S, C).to(dtype))
    return {k: t if t is None else t.to(dev) for k, t in d.items()}


def check(d, groups, act, dtype, x=None, gate=None, dy=None):
    """Forward and backward on the given (possibly strided) tensors against the
    oracle on the dense ones."""
    from tssm import group_norm_act_backward, group_norm_act_forward
    x, gate, dy = (d["x"] if x is None else x, d["gate"] if gate is None else gate,
                   d["dy"] if dy is None else dy)
    ref = M.group_norm(np64(d["x"]), groups, *(None if d[n] is None else np64(d[n])
                                               for n in ("w", "b", "gate")), act, dy=np64(d["dy"]))
    y, mean, rstd = group_norm_act_forward(x, groups, d["w"], d["b"], gate, act=act,
                                           return_stats=True)
    assert torch.equal(y, group_norm_act_forward(x, groups, d["w"], d["b"], gate, act=act))
    got = group_norm_act_backward(dy, x, mean, rstd, groups, d["w"], d["b"], gate, act=act)
    assert_close(y.reshape(d["x"].shape), ref[0], TOL[dtype], "y")
    assert_close(mean, ref[1], TOL[F32], "mean")
    assert_close(rstd, ref[2], TOL[F32], "rstd")
    assert_close(got[0].reshape(d["x"].shape), ref[3], TOL[dtype], "dx")
    for g, r, what, given in ((got[1], ref[4], "dw", d["w"]), (got[2], ref[5], "db", d["b"])):
        if given is None:
            assert g is None
        else:
            assert_close(g, r, TOL[F32], what)
    if d["gate"] is None:
        assert got[3] is None
    else:
        assert_close(got[3].reshape(d["x"].shape), ref[6], TOL[dtype], "dgate")


SIZES = [  # N, S, groups, C
    (1, 1, 1, 1),
    (3, 1, 16, 1024),
    (700, 1, 16, 1024),
    (5, 1, 4, 512),
    (33, 1, 3, 51),
    (2, 1, 1, 2000),
    (129, 1, 31, 62),
    (2, 300, 8, 256),
    (16, 33, 5, 40),
    (1, 4000, 4, 64),
    (3, 1000, 2, 14),
    (1, 2, 7, 1001),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("gated,act", [(False, "silu"), (True, "silu"), (True, "none"),
                                       (False, "none")])
@pytest.mark.parametrize("N,S,G,C", SIZES)
def test_forward_backward(dev, dtype, gated, act, N, S, G, C):
    check(inputs(dev, N, S, C, dtype, gated, seed=C + S), G, act, dtype)


@pytest.mark.parametrize("N,S", [(50, 1), (3, 120)])
def test_strides_and_views(dev, N, S):
    """x and the gate as slices of wider rows, odd offsets, positions before
    batches, and several middle dimensions."""
    C, G = 64, 8
    d = inputs(dev, N, S, C, BF16, True, seed=3)
    wide = torch.zeros(N, S, 2 * C + 3, device=dev, dtype=BF16)
    x, gate = wide[..., :C], wide[..., C + 1:2 * C + 1]
    x.copy_(d["x"])
    gate.copy_(d["gate"])
    check(d, G, "silu", BF16, x=x, gate=gate)
    sb = torch.empty(S, N, C, device=dev, dtype=BF16).transpose(0, 1)
    sb.copy_(d["x"])
    check(d, G, "silu", BF16, x=sb)
    if S > 1:
        four = {n: d[n].reshape(N, 4, S // 4, C) for n in ("x", "gate", "dy")}
        check(d, G, "silu", BF16, **four)


def test_without_weights(dev):
    for w, b in ((True, False), (False, True), (False, False)):
        for N, S in ((40, 1), (3, 100)):
            d = inputs(dev, N, S, 96, F32, False, seed=4)
            d["w"], d["b"] = d["w"] if w else None, d["b"] if b else None
            check(d, 6, "silu", F32)


def test_large_mean(dev):
    """Offsets of a thousand deviations: the variance is formed about the mean,
    so only x's own rounding counts (fp32: 2^-24 of 1000 against 1, 6e-5)."""
    from tssm import group_norm_act_forward
    for N, S in ((64, 1), (2, 500)):
        d = inputs(dev, N, S, 256, F32, False, seed=5)
        d["x"] += 1000.0
        y, mean, rstd = group_norm_act_forward(d["x"], 4, d["w"], d["b"], return_stats=True)
        ref = M.group_norm(np64(d["x"]), 4, np64(d["w"]), np64(d["b"]))
        assert_close(mean, ref[1], 1e-6, "mean")
        assert_close(rstd, ref[2], 1e-5, "rstd")
        assert_close(y, ref[0], 6e-5, "y")


def test_constant_rows_and_empty(dev):
    from tssm import group_norm_act_backward, group_norm_act_forward
    x = torch.full((4, 1, 32), 3.0, device=dev)
    y, mean, rstd = group_norm_act_forward(x, 2, return_stats=True, act="none", eps=1e-4)
    assert not y.any()
    np.testing.assert_allclose(np64(rstd), 100.0, rtol=1e-6)
    for shape in ((0, 1, 32), (4, 0, 32), (0, 32)):
        x = torch.empty(shape, device=dev)
        y, mean, rstd = group_norm_act_forward(x, 2, return_stats=True)
        assert y.shape == x.shape
        w = torch.ones(32, device=dev)
        dx, dw, db, _ = group_norm_act_backward(x, x, mean, rstd, 2, w, w)
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_not_finite_stays_in_its_group(dev):
    for N, S in ((6, 1), (3, 70)):
        d = inputs(dev, N, S, 64, F32, True, seed=6)
        from tssm import group_norm_act_forward
        ref = np64(group_norm_act_forward(d["x"], 4, d["w"], d["b"], d["gate"]))
        d["x"][1, 0, 20] = float("nan")
        y = group_norm_act_forward(d["x"], 4, d["w"], d["b"], d["gate"])
        assert torch.isnan(y[1, :, 16:32]).all()
        y[1, :, 16:32] = torch.from_numpy(ref[1, :, 16:32]).to(y)
        assert_close(y, ref, 1e-7, "other groups")


def test_repeat_gives_the_same_bits(dev):
    from tssm import group_norm_act_backward, group_norm_act_forward
    for N, S in ((3000, 1), (4, 1500)):
        d = inputs(dev, N, S, 128, BF16, True, seed=7)
        runs = []
        for _ in range(2):
            y, mean, rstd = group_norm_act_forward(d["x"], 4, d["w"], d["b"], d["gate"],
                                                   return_stats=True)
            runs.append((y, mean, rstd) + group_norm_act_backward(
                d["dy"], d["x"], mean, rstd, 4, d["w"], d["b"], d["gate"]))
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_refusals(dev):
    from tssm import group_norm_act_backward, group_norm_act_forward
    d = inputs(dev, 3, 4, 16, BF16, True)
    x, gate, w, b, dy = (d[n] for n in ("x", "gate", "w", "b", "dy"))
    for kw, err, match in [
        (dict(groups=3), ValueError, "divide"), (dict(groups=0), ValueError, "divide"),
        (dict(act="relu"), ValueError, "act must be"), (dict(weight=w[:8]), ValueError, "weight"),
        (dict(bias=b[None]), ValueError, "bias"), (dict(gate=gate[:, :2]), ValueError, "gate"),
        (dict(gate=gate.float()), TypeError, "gate"), (dict(x=x.cpu()), ValueError, "HIP device"),
        (dict(x=x.double()), TypeError, "unsupported dtype"),
        (dict(x=x[0, 0]), ValueError, "N, ..., C"),
        (dict(x=x.transpose(1, 2).contiguous().transpose(1, 2)), ValueError, "contiguous"),
        (dict(out=torch.empty_like(x).float()), TypeError, "out"),
    ]:
        a = dict(dict(x=x, groups=4, weight=w, bias=b, gate=gate), **kw)
        with pytest.raises(err, match=match):
            group_norm_act_forward(**a)
    four = torch.zeros(3, 2, 8, 16, device=dev)[:, :, ::2].transpose(1, 2)
    with pytest.raises(ValueError, match="evenly strided"):
        group_norm_act_forward(four.contiguous().transpose(1, 2)[:, :, :3], 4)
    y, mean, rstd = group_norm_act_forward(x, 4, w, b, gate, return_stats=True)
    with pytest.raises(ValueError, match="mean"):
        group_norm_act_backward(dy, x, mean[:2], rstd, 4, w, b, gate)
    with pytest.raises(ValueError, match="dy"):
        group_norm_act_backward(dy[:1], x, mean, rstd, 4, w, b, gate)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,S,G,C", [
    (3, 1, 1, 4099),      # rows past a wave's registers
    (2, 3, 3, 12297),     # series past a workgroup's row
    (2, 40, 1, 8192), (1, 70, 2, 2050), (2, 9, 513, 1026),
])
def test_wide(dev, dtype, N, S, G, C):
    check(inputs(dev, N, S, C, dtype, True, seed=C), G, "silu", dtype)


@pytest.mark.parametrize("N,G,C,dtype", [(140000, 1, 8, F32), (9000, 2, 64, BF16),
                                         (5000, 1, 2048, F16)])
def test_many_rows(dev, N, G, C, dtype):
    """More rows than the gradients' workgroups take at once."""
    check(inputs(dev, N, 1, C, dtype, True, seed=11), G, "silu", dtype)
