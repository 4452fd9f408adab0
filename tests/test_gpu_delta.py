"""GPU parity of the gated delta rule against its float64 definition.

Tolerances, normwise.  fp32 outputs (states, and everything with fp32 inputs):
1e-5 -- sums of at most 128 products carry about sqrt(128) 2^-24 = 7e-7, a
chunk has five of them in a row, and beta (1 - |k|^2 beta) keeps older errors
from growing.  16-bit outputs: twice the rounding of the largest value, 2^-8
for bfloat16 and 2^-11 for float16.
"""
import numpy as np
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 1e-5, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=0, h0=False, rate=1.0):
    """Unit keys with a shared direction, decays of irregular gaps."""
    r = torch.Generator().manual_seed(seed)

    def unit(t):
        return t / t.norm(dim=-1, keepdim=True)

    d = dict(q=unit(torch.randn(B, L, Hk, K, generator=r)).to(dtype),
             k=unit(torch.randn(B, L, Hk, K, generator=r)
                    + 0.5 * torch.randn(Hk, K, generator=r)).to(dtype),
             v=torch.randn(B, L, Hv, V, generator=r).to(dtype),
             g=-torch.empty(B, L, Hv).exponential_(10.0, generator=r) * rate,
             beta=torch.sigmoid(torch.randn(B, L, Hv, generator=r)))
    d["h0"] = torch.randn(B, Hv, K, V, generator=r) if h0 else None
    return {n: t if t is None else t.to(dev) for n, t in d.items()}


def run(d, **kw):
    from tssm import gated_delta_forward
    return gated_delta_forward(d["q"], d["k"], d["v"], d["g"], d["beta"], h0=d["h0"],
                               return_state=True, **kw)


def oracle(d, **kw):
    c = {n: None if t is None else np64(t) for n, t in d.items()}
    return M.delta_forward(**c, **kw)


SIZES = [  # B, L, Hk, Hv, K, V
    (1, 1, 1, 1, 1, 1),
    (2, 5, 2, 4, 64, 64),
    (1, 31, 1, 1, 16, 16),
    (2, 32, 3, 3, 32, 48),
    (1, 33, 2, 6, 40, 72),
    (3, 64, 1, 2, 128, 128),
    (1, 100, 2, 2, 7, 33),       # no vector access
    (2, 257, 2, 2, 96, 20),
    (1, 1000, 2, 4, 64, 64),
    (1, 130, 1, 1, 100, 300),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,L,Hk,Hv,K,V", SIZES)
def test_forward(dev, dtype, B, L, Hk, Hv, K, V):
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L + K, h0=L % 2 == 1)
    o, S = run(d)
    o_ref, S_ref = oracle(d)
    assert_close(o, o_ref, TOL[dtype], "o")
    assert_close(S, S_ref, TOL[F32], "state")


@pytest.mark.parametrize("B,Hv,K,V", [(1, 4, 64, 40), (64, 8, 16, 16), (1, 2, 128, 8),
                                      (300, 4, 16, 70)])
@pytest.mark.parametrize("L", [2, 12, 13, 24, 25])
def test_few_tokens(dev, B, Hv, K, V, L):
    """Around the lengths where the forward turns from steps to chunks, with few
    and with many heads, narrow and wide waves."""
    d = inputs(dev, B, L, Hv // 2, Hv, K, V, BF16, seed=L + V, h0=True)
    o, S = run(d)
    o_ref, S_ref = oracle(d)
    assert_close(o, o_ref, TOL[BF16], "o")
    assert_close(S, S_ref, TOL[F32], "state")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forward_strides(dev, dtype):
    """q, k and v as slices of one projection, heads before steps, a shared g."""
    B, L, H, K, V = 2, 77, 3, 32, 32
    d = inputs(dev, B, L, H, H, K, V, dtype, seed=5, h0=True)
    packed = torch.zeros(B, L, H * (2 * K + V) + 3, device=dev, dtype=dtype)
    o_ref, S_ref = oracle(d)
    for name, at in (("q", 0), ("k", H * K), ("v", 2 * H * K)):
        view = packed[..., at + 1:at + 1 + H * K].view(B, L, H, K)
        view.copy_(d[name])
        d[name] = view
    d["beta"] = d["beta"].transpose(1, 2).contiguous().transpose(1, 2)
    out = torch.empty(B, H, L, V, device=dev, dtype=dtype).transpose(1, 2)
    o, S = run(d, out=out)
    assert o is out
    assert_close(o, o_ref, TOL[dtype], "o")
    assert_close(S, S_ref, TOL[F32], "state")
    d["g"] = d["g"][:, :1, :1].expand(B, L, H)     # one decay for all steps and heads
    o, S = run(d)
    o_ref, S_ref = oracle(d)
    assert_close(o, o_ref, TOL[dtype], "o")
    assert_close(S, S_ref, TOL[F32], "state")


@pytest.mark.parametrize("dtype,B,L,Hk,Hv,K,V,rate,h0", [
    (BF16, 1, 8200, 1, 2, 64, 64, 0.02, True),    # segments, slow decay across them
    (F32, 1, 5001, 1, 1, 40, 72, 0.05, False),
    (F16, 2, 3000, 1, 1, 128, 30, 0.02, True),
    (BF16, 1, 4096, 2, 2, 16, 16, 0.0, True),     # no decay
])
def test_segments(dev, dtype, B, L, Hk, Hv, K, V, rate, h0):
    """Long sequences over few heads are walked in segments."""
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L, h0=h0, rate=rate)
    o, S = run(d)
    o_ref, S_ref = oracle(d)
    assert_close(o, o_ref, TOL[dtype], "o")
    assert_close(S, S_ref, TOL[F32], "state")


@pytest.mark.parametrize("B,L,H,K,V", [(1, 8200, 2, 64, 64), (2, 100, 2, 64, 48), (2, 9, 3, 32, 32)])
def test_state_in_place(dev, B, L, H, K, V):
    """The C entry point with one buffer for the state before and after, in
    segments, in one walk and step by step: the bits of two buffers."""
    from tssm import _lib
    d = inputs(dev, B, L, H, H, K, V, BF16, seed=9, h0=True, rate=0.05)
    o_ref, S_ref = run(d)
    o, S = torch.empty_like(o_ref), d["h0"].clone()
    n = _lib.lib().tssm_gated_delta_workspace_bytes(B, L, H, H, K, V)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=dev)
    t = [d[x] for x in ("q", "k", "v")]
    _lib.call("tssm_gated_delta_forward", 1, *(x.data_ptr() for x in t), d["g"].data_ptr(),
              d["beta"].data_ptr(), S.data_ptr(), o.data_ptr(), S.data_ptr(), B, L, H, H, K, V,
              *(s for x in t for s in x.stride()[:3]), *d["g"].stride(), *d["beta"].stride(),
              *o.stride()[:3], K ** -0.5, ws.data_ptr() if n else None, n,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(o, o_ref) and torch.equal(S, S_ref)


@pytest.mark.parametrize("L", [0, 1])
def test_empty(dev, L):
    d = inputs(dev, 2, L, 2, 2, 32, 32, F32, h0=True)
    o, S = run(d)
    assert o.shape == (2, L, 2, 32)
    if L == 0:
        assert torch.equal(S, d["h0"])
        d["h0"] = None
        assert not run(d)[1].any()
    none = {n: None if t is None else t[:0] for n, t in d.items()}
    o, S = run(none)
    assert o.shape[0] == 0 and S.shape[0] == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_extreme_decay(dev, dtype):
    """No decay at all, complete resets (g = -inf and the lowest value) among
    slow steps, and steps whose beta is 0 or 1."""
    d = inputs(dev, 2, 150, 2, 2, 64, 64, dtype, seed=8, h0=True, rate=0.05)
    d["g"][:, ::7] = 0.0
    d["g"][0, 40] = -float("inf")
    d["g"][1, 41] = torch.finfo(F32).min
    d["g"][1, 90:100] = -300.0
    d["beta"][:, 10:20] = 0.0
    d["beta"][:, 20:30] = 1.0
    o, S = run(d)
    o_ref, S_ref = oracle(d)
    assert_close(o, o_ref, TOL[dtype], "o")
    assert_close(S, S_ref, TOL[F32], "state")
    # the steps after a reset alone, so that larger earlier outputs hide nothing
    assert_close(o[0, 40:48], o_ref[0, 40:48], TOL[dtype], "o after a reset")


def test_correlated_keys(dev):
    """One key for all steps: products of the chunk's triangular matrix grow
    like binomials, its inverse does not."""
    d = inputs(dev, 1, 200, 1, 1, 64, 32, F32, seed=9)
    d["k"] = d["k"][:, :1].expand_as(d["k"])
    d["beta"] = torch.ones_like(d["beta"])
    d["g"] = torch.zeros_like(d["g"])
    o, S = run(d)
    o_ref, S_ref = oracle(d)
    assert_close(o, o_ref, TOL[F32], "o")
    assert_close(S, S_ref, TOL[F32], "state")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", ["v", "k", "q", "beta"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_not_finite(dev, dtype, name, value):
    """A value that is not finite at one step leaves every earlier output, and
    (in v) every other column, as it was."""
    B, L, H, K, V, t0 = 1, 150, 2, 64, 64, 75
    d = inputs(dev, B, L, H, H, K, V, dtype, seed=11, h0=True)
    o_ref, S_ref = oracle(d)
    if name == "beta":
        d["beta"][0, t0, 1] = value
    else:
        d[name][0, t0, 1, 5] = value
    o, S = run(d)
    assert_close(o[:, :t0], o_ref[:, :t0], TOL[dtype], "earlier steps")
    assert_close(o[:, :, 0], o_ref[:, :, 0], TOL[dtype], "the other head")
    assert not torch.isfinite(o[0, t0, 1]).all()
    if name == "v":
        keep = [c for c in range(V) if c != 5]
        assert_close(o[:, :, 1, keep], o_ref[:, :, 1, keep], TOL[dtype], "other columns")
        assert_close(S[:, 1][..., keep], S_ref[:, 1][..., keep], TOL[F32], "state")
    if name == "q":
        assert_close(o[:, t0 + 1:], o_ref[:, t0 + 1:], TOL[dtype], "later steps")
        assert_close(S, S_ref, TOL[F32], "state")


def test_chained_calls(dev):
    """A sequence in three calls, the state handed on, against one call."""
    d = inputs(dev, 2, 300, 2, 4, 64, 64, BF16, seed=12)
    o, S = run(d)
    parts, h = [], None
    for lo, hi in ((0, 7), (7, 168), (168, 300)):
        p = {n: d[n][:, lo:hi] for n in ("q", "k", "v", "g", "beta")}
        op, h = run(dict(p, h0=h))
        parts.append(op)
    assert_close(torch.cat(parts, 1), np64(o), TOL[BF16], "o")
    assert_close(h, np64(S), TOL[F32], "state")


def test_repeat_and_stream(dev):
    """The same bits on a repeated call, and on another stream than the
    tensors' own."""
    d = inputs(dev, 2, 500, 2, 2, 64, 64, BF16, seed=13)
    o, S = run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, S2 = run(d)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(o, o2) and torch.equal(S, S2)


# ------------------------------------------------------------------ gradients
NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dh0")


def gradients(d, do, dh=None, **kw):
    from tssm import gated_delta_backward
    return gated_delta_backward(d["q"], d["k"], d["v"], d["g"], d["beta"], do, h0=d["h0"],
                                dh_last=dh, **kw)


def check_gradients(dev, d, dtype, seed, dh=True, **kw):
    r = torch.Generator().manual_seed(seed)
    B, L, Hv, V = d["v"].shape
    K = d["q"].shape[-1]
    do = torch.randn(B, L, Hv, V, generator=r).to(dtype).to(dev)
    dh = torch.randn(B, Hv, K, V, generator=r).to(dev) if dh else None
    got = gradients(d, do, dh, **kw)
    ref = M.delta_backward(**{n: None if t is None else np64(t) for n, t in d.items()},
                           do=np64(do), dh_last=None if dh is None else np64(dh), **kw)
    for name, x, y in zip(NAMES, got, ref):
        if name == "dh0" and d["h0"] is None:
            assert x is None
        else:
            assert_close(x, y, TOL[dtype] if name in ("dq", "dk", "dv") else TOL[F32], name)
    return do, dh, got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,L,Hk,Hv,K,V", SIZES)
def test_backward(dev, dtype, B, L, Hk, Hv, K, V):
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L + K, h0=L % 2 == 1)
    check_gradients(dev, d, dtype, seed=V, dh=L % 2 == 1)


@pytest.mark.parametrize("dtype,B,L,Hk,Hv,K,V,rate", [
    (BF16, 1, 6000, 1, 2, 64, 64, 0.05), (F32, 1, 3001, 1, 1, 40, 72, 0.05),
    (F16, 1, 2500, 1, 1, 128, 30, 0.02)])
def test_backward_segments(dev, dtype, B, L, Hk, Hv, K, V, rate):
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L, h0=True, rate=rate)
    check_gradients(dev, d, dtype, seed=1)


def test_backward_scale_and_strides(dev):
    B, L, H, K, V = 2, 77, 3, 32, 32
    d = inputs(dev, B, L, H, H, K, V, BF16, seed=5, h0=True)
    packed = torch.zeros(B, L, H * (2 * K + V) + 3, device=dev, dtype=BF16)
    for name, at in (("q", 0), ("k", H * K), ("v", 2 * H * K)):
        view = packed[..., at + 1:at + 1 + H * K].view(B, L, H, K)
        view.copy_(d[name])
        d[name] = view
    d["g"] = d["g"][:, :1, :1].expand(B, L, H)
    do, dh, got = check_gradients(dev, d, BF16, seed=3, scale=0.7)
    one = do[:, :1].expand_as(do)              # a gradient shared by all steps
    again = gradients(d, one, dh, scale=0.7)
    assert all(torch.equal(x, y) for x, y in zip(again, gradients(d, one.contiguous(), dh,
                                                                  scale=0.7)))


def test_backward_resets(dev):
    d = inputs(dev, 2, 150, 2, 2, 64, 64, F32, seed=8, h0=True, rate=0.05)
    d["g"][:, ::7] = 0.0
    d["g"][1, 90:100] = -300.0
    d["beta"][:, 10:20] = 0.0
    check_gradients(dev, d, F32, seed=2)
    d["g"][0, 40] = -float("inf")
    do = torch.ones_like(d["v"])
    assert all(torch.isfinite(x).all() for x in gradients(d, do))


def test_backward_against_differences(dev):
    """Directional differences of the forward in fp32: the change of
    sum(o do) + sum(S dh) along a random direction.  Step 1e-2 of O(1) inputs:
    third-order truncation 1e-4 of the directional derivative's scale, rounding
    of a sum of 4e3 terms 1e-6 / 1e-2 of it."""
    r = torch.Generator().manual_seed(4)
    d = inputs(dev, 1, 70, 1, 2, 32, 32, F32, seed=4, h0=True)
    do = torch.randn(1, 70, 2, 32, generator=r).to(dev)
    dh = torch.randn(1, 2, 32, 32, generator=r).to(dev)
    got = dict(zip(("q", "k", "v", "g", "beta", "h0"), gradients(d, do, dh)))
    for name in got:
        way = torch.randn(d[name].shape, generator=r).to(dev)
        way = way / way.norm()
        loss = []
        for e in (1e-2, -1e-2):
            o, S = run(dict(d, **{name: d[name] + e * way}))
            loss.append(float((o.double() * do.double()).sum() + (S.double() * dh.double()).sum()))
        want = (loss[0] - loss[1]) / 2e-2
        have = float((got[name].double() * way.double()).sum())
        assert abs(have - want) <= 1e-3 * float(got[name].norm()), (name, have, want)


def test_backward_repeat_and_empty(dev):
    d = inputs(dev, 2, 200, 2, 4, 64, 64, BF16, seed=13, h0=True)
    do, dh, got = check_gradients(dev, d, BF16, seed=6)
    assert all(torch.equal(x, y) for x, y in zip(got, gradients(d, do, dh)))
    none = {n: t[:, :0] if n != "h0" else t for n, t in d.items()}
    got = gradients(none, do[:, :0], dh)
    assert torch.equal(got[5], dh) and got[0].shape == (2, 0, 2, 64)
    assert not gradients(none, do[:, :0])[5].any()


# ------------------------------------------------------------------ decode
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("S,Hk,Hv,K,V", [(1, 1, 1, 1, 1), (1, 8, 16, 128, 128), (7, 2, 2, 64, 64),
                                         (33, 1, 3, 40, 72), (5, 2, 2, 7, 33),
                                         (300, 4, 4, 128, 64), (3, 2, 2, 16, 300)])
def test_step(dev, dtype, S, Hk, Hv, K, V):
    from tssm import gated_delta_step
    d = inputs(dev, 4, S, Hk, Hv, K, V, dtype, seed=S + V)
    state = torch.randn(S, Hv, K, V, generator=torch.Generator().manual_seed(S)).to(dev)
    ref = np64(state)
    for t in range(4):
        x = {n: d[n][t] for n in ("q", "k", "v", "g", "beta")}
        o_ref, ref = M.delta_forward(**{n: np64(a)[:, None] for n, a in x.items()}, h0=ref)
        o = gated_delta_step(**x, state=state)
        assert_close(o, o_ref[:, 0], TOL[dtype], f"o, step {t}")
        assert_close(state, ref, TOL[F32], f"state, step {t}")


def test_step_continues_forward(dev):
    """Prefill, then decode from its state, against one longer prefill."""
    from tssm import gated_delta_step
    d = inputs(dev, 2, 70, 2, 4, 64, 32, BF16, seed=15)
    o, S = run(d)
    _, state = run({n: None if t is None else t[:, :64] for n, t in d.items()})
    for t in range(64, 70):
        x = {n: d[n][:, t] for n in ("q", "k", "v", "g", "beta")}
        assert_close(gated_delta_step(**x, state=state), np64(o[:, t]), TOL[BF16], f"step {t}")
    assert_close(state, np64(S), TOL[F32], "state")


def test_step_graph(dev):
    """A captured step replayed with eager work between the replays."""
    from tssm import gated_delta_step
    d = inputs(dev, 4, 9, 2, 2, 64, 64, BF16, seed=16)
    x = {n: d[n][0].clone() for n in ("q", "k", "v", "g", "beta")}
    state = torch.randn(9, 2, 64, 64, generator=torch.Generator().manual_seed(16)).to(dev)
    eager, out = state.clone(), torch.empty_like(x["v"])
    gated_delta_step(**x, state=state.clone(), out=out)      # loads the kernel
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gated_delta_step(**x, state=state, out=out)
    for t in range(4):
        for n in x:
            x[n].copy_(d[n][t])
        graph.replay()
        torch.cuda.synchronize()
        ref = gated_delta_step(**x, state=eager)
        assert torch.equal(out, ref) and torch.equal(state, eager), f"replay {t}"


# ------------------------------------------------------------------ refusals
def test_refusals(dev):
    from tssm import gated_delta_forward, gated_delta_step
    d = inputs(dev, 2, 6, 2, 4, 16, 8, BF16, h0=True)

    def call(**kw):
        a = dict(d, **kw)
        return gated_delta_forward(a["q"], a["k"], a["v"], a["g"], a["beta"], h0=a["h0"],
                                   out=a.get("out"))

    for bad, match in [
        (dict(k=d["k"][:, :5]), "k must be"),
        (dict(q=d["q"][0]), "expected q"),
        (dict(v=d["v"][:, :, :3]), "multiple"),
        (dict(v=d["v"][:, :5]), "v must be"),
        (dict(g=d["g"][:, :, :2]), "g must be"),
        (dict(beta=d["beta"][0]), "beta must be"),
        (dict(h0=d["h0"][:, :2]), "h0 must be"),
        (dict(out=torch.empty(2, 6, 4, 9, device=dev, dtype=BF16)), "out must be"),
        (dict(q=d["q"].cpu()), "HIP device"),
        (dict(v=d["v"].transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
        (dict(q=torch.zeros(2, 6, 2, 129, device=dev, dtype=BF16)), "at most 128"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(**bad)
    for bad, match in [(dict(k=d["k"].float()), "k must be"), (dict(v=d["v"].half()), "v must be"),
                       (dict(q=d["q"].double()), "unsupported dtype"),
                       (dict(g=d["g"].long()), "float tensor"), (dict(q=None), "torch.Tensor")]:
        with pytest.raises(TypeError, match=match):
            call(**bad)
    for do, err in ((d["v"][:1], ValueError), (d["v"].float(), TypeError),
                    (d["v"].cpu(), ValueError)):
        with pytest.raises(err, match="do"):
            gradients(d, do)
    with pytest.raises(ValueError, match="dh_last must be"):
        gradients(d, d["v"], d["h0"][..., :4])
    x = {n: d[n][:, 0] for n in ("q", "k", "v", "g", "beta")}
    with pytest.raises(ValueError, match="contiguous"):
        gated_delta_step(**x, state=d["h0"].transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(TypeError, match="state must be"):
        gated_delta_step(**x, state=d["h0"].bfloat16())
    with pytest.raises(ValueError, match="state must be"):
        gated_delta_step(**x, state=d["h0"][:1])
