"""GPU parity of the norm and rotation of queries and keys against its float64
definition.

Tolerances, normwise (largest difference over largest value).  fp32: a row's sum
of at most 256 squares in a tree of lanes is off by at most 40 roundings of 2^-24,
its root by half of that; the products, the cosine (2 ulp of a value that is
multiplied by at most the largest) and the angle (rounded to fp32 as a fraction of
a turn: 2 pi 2^-25) add 12 more: 32 x 2^-24 = 2e-6, doubled in the gradients, whose
dot product is another such sum; taken as 4e-6.  The weights' gradients add n rows
in fp32, up to some thousands here: sqrt(n) 2^-24 around 4e-6 of the root mean
square of what is added, 1e-5 of the largest sum.  16-bit outputs: one rounding,
2^-8 (bfloat16) or 2^-11 (float16) of the largest value, and a hundredth of it.
"""
import numpy as np
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 4e-6, BF16: 1.01 * 2.0 ** -8, F16: 1.01 * 2.0 ** -11}
TOL_W = 1e-5


def inputs(dev, B, L, Hq, Hk, K, R, dtype, seed=0, weights=True, at="tokens"):
    r = torch.Generator().manual_seed(seed)
    d = dict(q=torch.randn(B, L, Hq, K, generator=r).to(dtype),
             k=(2.0 * torch.randn(B, L, Hk, K, generator=r)).to(dtype),
             dq=torch.randn(B, L, Hq, K, generator=r).to(dtype),
             dk=torch.randn(B, L, Hk, K, generator=r).to(dtype), wq=None, wk=None, pos=None,
             freq=None)
    if weights:
        d["wq"], d["wk"] = (1.0 + 0.3 * torch.randn(2, K, generator=r)).unbind()
    if R:
        d["freq"] = 10000.0 ** (-2.0 * torch.arange(R // 2, dtype=torch.float64) / R)
        n = torch.arange(L) + torch.randint(1000, (B, 1), generator=r)
        d["pos"] = {"tokens": n, "int32": n.int(), "far": n + (1 << 30),
                    "times": torch.rand(B, L, generator=r).cumsum(1),
                    "times64": 1e9 + torch.rand(B, L, generator=r, dtype=torch.float64).cumsum(1),
                    "back": -n}[at]
    return {n: None if t is None else t.to(dev) for n, t in d.items()}


def forward(d, **kw):
    from tssm import qk_norm_rotary_forward
    return qk_norm_rotary_forward(d["q"], d["k"], d["pos"], d["freq"], d["wq"], d["wk"], **kw)


def backward(d, **kw):
    from tssm import qk_norm_rotary_backward
    return qk_norm_rotary_backward(d["dq"], d["dk"], d["q"], d["k"], d["pos"], d["freq"],
                                   d["wq"], d["wk"], **kw)


def oracle(d, n, **kw):
    c = {x: None if t is None else np64(t) for x, t in d.items()}
    return M.norm_rotary(c[n], c["pos"], c["freq"], c["w" + n], dy=c["d" + n], **kw)


def check(d, **kw):
    dtype = d["q"].dtype
    ys, ds = forward(d, **kw), backward(d, **kw)
    for i, n in enumerate("qk"):
        y, dx, dw = oracle(d, n, **kw)
        assert_close(ys[i], y, TOL[dtype], n)
        assert_close(ds[i], dx, TOL[dtype], "d" + n)
        if d["w" + n] is None:
            assert ds[2 + i] is None
        else:
            assert_close(ds[2 + i], dw, TOL_W, "dw" + n)
    return ys, ds


SIZES = [  # B, L, Hq, Hk, K, R
    (1, 1, 1, 1, 1, 0),
    (1, 1, 1, 1, 2, 2),
    (2, 7, 4, 2, 64, 64),
    (1, 33, 3, 1, 128, 64),
    (2, 300, 6, 2, 64, 32),
    (1, 5, 8, 8, 256, 256),
    (3, 11, 5, 3, 40, 20),         # no whole vectors
    (1, 40, 2, 2, 33, 8),          # an odd channel that stays
    (2, 9, 3, 1, 96, 96),          # six lanes of eight
    (1, 64, 2, 1, 200, 100),
    (2, 2500, 2, 1, 16, 16),
    (1, 3, 70, 40, 32, 16),        # more heads than rows side by side
    (1, 70, 2, 2, 48, 0),          # a norm alone
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hk,K,R", SIZES)
def test_sizes(dev, dtype, interleaved, B, L, Hq, Hk, K, R):
    d = inputs(dev, B, L, Hq, Hk, K, R, dtype, seed=K + L)
    if K == 1:
        # d(x / sqrt(x^2 + eps)) is what 1 - x^2 / (x^2 + eps) leaves, eps / x^2: refused
        with pytest.raises(ValueError, match="one channel"):
            forward(d)
        check(d, interleaved=interleaved, norm="none")
    else:
        check(d, interleaved=interleaved)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm", ["rms", "l2", "none"])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("K,R", [(64, 64), (40, 20)])
def test_norms(dev, dtype, norm, weights, K, R):
    check(inputs(dev, 2, 50, 4, 2, K, R, dtype, seed=1, weights=weights), norm=norm,
          eps=1e-3, amplitude=1.25)


@pytest.mark.parametrize("at", ["tokens", "int32", "far", "times", "times64", "back"])
def test_positions(dev, at):
    """Every type of position; angles of 10^9 turns keep their fraction of one."""
    check(inputs(dev, 2, 60, 2, 1, 32, 32, F32, seed=2, at=at))


def test_shared_positions_and_one_token(dev):
    """Positions [L] for all batches, and [S, H, K] rows of single tokens."""
    d = inputs(dev, 3, 20, 2, 2, 32, 16, F32, seed=3)
    d["pos"] = d["pos"][:1].expand(3, 20)
    want = check(d)
    d["pos"] = d["pos"][0]
    for x, y in zip(forward(d) + backward(d), want[0] + want[1]):
        assert torch.equal(x, y)
    one = {n: t if t is None or n in ("wq", "wk", "freq") else t[:, 4] for n, t in d.items()
           if n != "pos"}
    one["pos"] = d["pos"][4:5].expand(3)
    for x, y in zip(forward(one), want[0]):
        assert torch.equal(x, y[:, 4])
    dq, dk, _, _ = backward(one)
    assert torch.equal(dq, want[1][0][:, 4]) and torch.equal(dk, want[1][1][:, 4])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_in_place(dev, dtype):
    """Slices of one projection (at a place that no vector starts on too), heads
    before steps, outputs over the inputs."""
    B, L, Hq, Hk, K = 2, 37, 4, 2, 64
    d = inputs(dev, B, L, Hq, Hk, K, 64, dtype, seed=5)
    want, dwant = check(d)
    for off in (0, 1):
        wide = torch.full((B, L, (Hq + Hk) * K + 16), 7.0, device=dev, dtype=dtype)
        q = wide[..., off:off + Hq * K].view(B, L, Hq, K)
        k = wide[..., off + Hq * K:off + (Hq + Hk) * K].view(B, L, Hk, K)
        q.copy_(d["q"]), k.copy_(d["k"])
        e = dict(d, q=q, k=k, dq=d["dq"].transpose(1, 2).contiguous().transpose(1, 2))
        for x, y in zip(forward(e) + backward(e), want + dwant):
            assert_close(x, np64(y), TOL[dtype] if x.dim() > 1 else TOL_W, "strided")
        yq, yk = forward(e, out_q=q, out_k=k)
        assert yq is q and yk is k
        assert_close(q, np64(want[0]), TOL[dtype], "q in place")
        assert_close(k, np64(want[1]), TOL[dtype], "k in place")
        assert (wide[..., :off] == 7.0).all() and (wide[..., off + (Hq + Hk) * K:] == 7.0).all()


def test_empty(dev):
    from tssm import qk_norm_rotary_backward
    for B, L in ((0, 4), (2, 0)):
        d = inputs(dev, B, L, 2, 1, 32, 32, F32)
        assert [t.shape for t in forward(d)] == [d["q"].shape, d["k"].shape]
        dq, dk, dwq, dwk = backward(d)
        assert dq.shape == d["q"].shape and not dwq.any() and not dwk.any()


def test_rows_apart(dev):
    """A row that is not finite, or zero, changes no other row; a zero row stays zero
    with a finite gradient."""
    d = inputs(dev, 1, 9, 4, 2, 64, 64, F32, seed=6, weights=False)
    d["q"][0, 3, 1] = 0.0
    want, dwant = forward(d), backward(d)
    assert not want[0][0, 3, 1].any() and torch.isfinite(dwant[0]).all()
    d["q"][0, 4, 2, 7] = float("nan")
    d["k"][0, 5, 0, 1] = float("inf")
    got, dgot = forward(d), backward(d)
    for n, at in ((0, (4, 2)), (1, (5, 0))):
        keep = torch.ones(got[n].shape[1:3], dtype=torch.bool)
        keep[at] = False
        assert torch.equal(got[n][0][keep], want[n][0][keep])
        assert torch.equal(dgot[n][0][keep], dwant[n][0][keep])
        assert torch.isnan(got[n][0][at]).any() and torch.isnan(dgot[n][0][at]).any()


def test_repeat_and_stream(dev):
    """The same bits on a repeated call, and on another stream than the tensors' own."""
    d = inputs(dev, 4, 900, 4, 2, 64, 64, BF16, seed=7)
    want = forward(d) + backward(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = forward(d) + backward(d)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_unit_keys_for_the_delta_rule(dev):
    """What comes out is what the delta rule and linear attention read: one rotated
    prompt through both, against the definitions."""
    from tssm import gated_delta_forward, linear_attention_forward
    d = inputs(dev, 2, 70, 2, 2, 64, 64, F32, seed=8, weights=False)
    q, k = forward(d, norm="l2", eps=1e-12)
    r = torch.Generator().manual_seed(9)
    v = torch.randn(2, 70, 4, 48, generator=r).to(dev)
    g = -torch.rand(2, 70, 4, generator=r).to(dev) * 0.1
    beta = torch.rand(2, 70, 4, generator=r).to(dev)
    qr, kr = (oracle(d, n, norm="l2", eps=1e-12)[0] for n in "qk")
    # the inputs' 4e-6 and the operators' own 1e-5
    assert_close(gated_delta_forward(q, k, v, g, beta),
                 M.delta_forward(qr, kr, np64(v), np64(g), np64(beta))[0], 2e-5, "delta")
    assert_close(linear_attention_forward(q, k, v, g),
                 M.linear_forward(qr, kr, np64(v), np64(g))[0], 2e-5, "linear")
