"""GPU parity of linear attention against its float64 definition.

Tolerances, normwise (largest difference over largest value).  fp32 outputs
(states, and everything with fp32 inputs): 1e-5 -- a sum of n products in a fixed
order carries about sqrt(n) 2^-24; here n is K (at most 128), the steps that a
decay leaves (at most some thousands) and the chunks' states, so 100 x 6e-8 = 6e-6.
16-bit outputs: one rounding, 2^-8 (bfloat16) or 2^-11 (float16) of the largest
value, and a fiftieth of it for what precedes it (weights of two planes, 2^-16,
with up to 100 terms that count).
"""
import numpy as np
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TOL = {F32: 1e-5, BF16: 1.02 * 2.0 ** -8, F16: 1.02 * 2.0 ** -11}


def inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=0, h0=False, rate=1.0):
    """Keys and queries with a shared direction, decays of irregular gaps."""
    r = torch.Generator().manual_seed(seed)
    d = dict(q=torch.randn(B, L, Hk, K, generator=r).to(dtype),
             k=((torch.randn(B, L, Hk, K, generator=r)
                 + 0.5 * torch.randn(Hk, K, generator=r)) * K ** -0.5).to(dtype),
             v=torch.randn(B, L, Hv, V, generator=r).to(dtype),
             g=-torch.empty(B, L, Hv).exponential_(10.0, generator=r) * rate)
    d["h0"] = torch.randn(B, Hv, K, V, generator=r) if h0 else None
    return {n: t if t is None else t.to(dev) for n, t in d.items()}


def run(d, **kw):
    from tssm import linear_attention_forward
    return linear_attention_forward(d["q"], d["k"], d["v"], d["g"], h0=d["h0"],
                                    return_state=True, **kw)


def oracle(d, **kw):
    return M.linear_forward(**{n: None if t is None else np64(t) for n, t in d.items()}, **kw)


def check(d, **kw):
    dtype = d["q"].dtype
    o, S = run(d, **kw)
    o_ref, S_ref = oracle(d, **{n: x for n, x in kw.items() if n == "scale"})
    assert_close(o, o_ref, TOL[dtype], "o")
    assert_close(S, S_ref, TOL[F32], "state")
    return o, S, o_ref, S_ref


SIZES = [  # B, L, Hk, Hv, K, V
    (1, 1, 1, 1, 1, 1),
    (2, 5, 2, 4, 64, 64),
    (1, 31, 1, 1, 16, 16),
    (2, 32, 3, 3, 32, 48),
    (1, 33, 2, 6, 40, 72),
    (3, 64, 1, 2, 128, 128),
    (1, 65, 1, 1, 64, 64),
    (1, 100, 2, 2, 7, 33),       # no vector access
    (2, 127, 2, 2, 64, 32),
    (2, 128, 1, 2, 64, 40),
    (1, 129, 2, 2, 64, 8),
    (2, 257, 2, 2, 96, 20),
    (1, 1000, 2, 4, 64, 64),
    (1, 130, 1, 1, 100, 300),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,L,Hk,Hv,K,V", SIZES)
def test_forward(dev, dtype, B, L, Hk, Hv, K, V):
    check(inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L + K, h0=L % 2 == 1))


@pytest.mark.parametrize("B,Hv,K,V", [(1, 4, 64, 40), (64, 8, 16, 16), (1, 2, 128, 8),
                                      (300, 4, 16, 70)])
@pytest.mark.parametrize("L", [2, 8, 16, 17, 24, 33])
def test_few_tokens(dev, B, Hv, K, V, L):
    """Around the lengths where the forward turns from steps to chunks, with few
    and with many heads, narrow and wide waves."""
    check(inputs(dev, B, L, Hv // 2, Hv, K, V, BF16, seed=L + V, h0=True))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forward_strides(dev, dtype):
    """q, k and v as slices of one projection, heads before steps, shared rates."""
    B, L, H, K, V = 2, 77, 3, 32, 32
    d = inputs(dev, B, L, H, H, K, V, dtype, seed=5, h0=True)
    packed = torch.zeros(B, L, H * (2 * K + V) + 3, device=dev, dtype=dtype)
    o_ref, S_ref = oracle(d)
    for name, at in (("q", 0), ("k", H * K), ("v", 2 * H * K)):
        view = packed[..., at + 1:at + 1 + H * K].view(B, L, H, K)
        view.copy_(d[name])
        d[name] = view
    d["g"] = d["g"].transpose(1, 2).contiguous().transpose(1, 2)
    out = torch.empty(B, H, L, V, device=dev, dtype=dtype).transpose(1, 2)
    o, S = run(d, out=out)
    assert o is out
    assert_close(o, o_ref, TOL[dtype], "o")
    assert_close(S, S_ref, TOL[F32], "state")
    for rates in (d["g"][:1, :1, :1], d["g"][:1, :1]):     # for all, for each head
        d["g"] = rates.expand(B, L, H)
        check(d)
    d["q"], d["k"] = (d[n][:, :1].expand(B, L, H, K) for n in "qk")   # rows that overlap
    check(d)


@pytest.mark.parametrize("dtype,B,L,Hk,Hv,K,V,rate,h0", [
    (BF16, 1, 8200, 1, 2, 64, 64, 0.02, True),    # segments, slow decay across them
    (F32, 1, 5001, 1, 1, 40, 72, 0.05, False),
    (F16, 2, 3000, 1, 1, 128, 30, 0.02, True),
    (BF16, 1, 4096, 2, 2, 16, 16, 0.01, True),
])
def test_segments(dev, dtype, B, L, Hk, Hv, K, V, rate, h0):
    """Long sequences over few heads."""
    check(inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L, h0=h0, rate=rate))


def test_no_decay(dev):
    """Everything is kept: 3000 steps add up.  The largest state entry is about
    3 x sqrt(3000) K^-1/2, and the sums' rounding grows like a walk's."""
    check(inputs(dev, 1, 3000, 1, 2, 32, 24, F32, seed=3, h0=True, rate=0.0))


@pytest.mark.parametrize("B,L,H,K,V", [(1, 8200, 2, 64, 64), (2, 100, 2, 64, 48), (2, 9, 3, 32, 32)])
def test_state_in_place(dev, B, L, H, K, V):
    """The C entry point with one buffer for the state before and after, in
    segments, in one walk and step by step: the bits of two buffers."""
    from tssm import _lib
    d = inputs(dev, B, L, H, H, K, V, BF16, seed=9, h0=True, rate=0.05)
    o_ref, S_ref = run(d)
    o, S = torch.empty_like(o_ref), d["h0"].clone()
    n = _lib.lib().tssm_linear_attention_workspace_bytes(B, L, H, H, K, V)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device=dev)
    t = [d[x] for x in ("q", "k", "v")]
    _lib.call("tssm_linear_attention_forward", 1, *(x.data_ptr() for x in t), d["g"].data_ptr(),
              S.data_ptr(), o.data_ptr(), S.data_ptr(), B, L, H, H, K, V,
              *(s for x in t for s in x.stride()[:3]), *d["g"].stride(), *o.stride()[:3],
              K ** -0.5, ws.data_ptr() if n else None, n,
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
    """No decay at all and complete resets (g = -inf and the lowest value) among
    slow steps."""
    d = inputs(dev, 2, 150, 2, 2, 64, 64, dtype, seed=8, h0=True, rate=0.05)
    d["g"][:, ::7] = 0.0
    d["g"][0, 40] = -float("inf")
    d["g"][1, 41] = torch.finfo(F32).min
    d["g"][1, 90:100] = -300.0
    o, S, o_ref, S_ref = check(d)
    # the steps after a reset alone, so that larger earlier outputs hide nothing
    assert_close(o[0, 40:48], o_ref[0, 40:48], TOL[dtype], "o after a reset")


def test_packed_sequences(dev):
    """Three sequences in one row, each started by g = -inf: each one's own result."""
    d = inputs(dev, 1, 300, 1, 2, 64, 48, F32, seed=14, rate=0.1)
    starts = (0, 77, 160, 300)
    for t in starts[:-1]:
        d["g"][:, t] = -float("inf")
    o, S = run(d)
    for lo, hi in zip(starts, starts[1:]):
        one = {n: None if t is None else t[:, lo:hi].clone() for n, t in d.items()}
        one["g"][:, 0] = 0.0
        want, last = oracle(one)
        assert_close(o[:, lo:hi], want, TOL[F32], f"from {lo}")
    assert_close(S, last, TOL[F32], "state")


@pytest.mark.parametrize("dtype,B,L,H,K,V,t0", [
    (F32, 1, 150, 2, 64, 64, 75), (BF16, 1, 150, 2, 64, 64, 75),
    (BF16, 1, 8200, 2, 64, 64, 4000),     # in segments, far from their ends
    (F32, 1, 5001, 1, 40, 72, 3203),
    (F16, 1, 150, 2, 64, 64, 80),
    (F16, 2, 3000, 1, 128, 30, 31),       # in the first chunk of a segmented sequence
    (BF16, 1, 150, 2, 128, 128, 149),     # the last step
    (F32, 1, 150, 2, 128, 64, 64),        # the first step of a chunk
    (BF16, 2, 70, 2, 24, 40, 40),         # K and V that fill no tile
    (BF16, 2, 7, 2, 24, 40, 4),           # step by step
])
@pytest.mark.parametrize("name", ["v", "k", "q", "g"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_not_finite(dev, dtype, B, L, H, K, V, t0, name, value):
    """A value that is not finite at one step of one head changes no earlier output
    and no other head; in v no other column, in q no other step."""
    d = inputs(dev, B, L, H, H, K, V, dtype, seed=L + K, h0=True, rate=0.05)
    o_ref, S_ref = oracle(d)
    if name == "g":
        d[name][B - 1, t0, H - 1] = value
    else:
        d[name][B - 1, t0, H - 1, 5] = value
    o, S = run(d)
    assert_close(o[:, :t0], o_ref[:, :t0], TOL[dtype], "earlier steps")
    rest = [i for i in range(B * H) if i != B * H - 1]
    if rest:
        heads = o.transpose(1, 2).reshape(B * H, L, V)[rest]
        want = o_ref.swapaxes(1, 2).reshape(B * H, L, V)[rest]
        assert_close(heads, want, TOL[dtype], "other heads")
        assert_close(S.reshape(B * H, K, V)[rest], S_ref.reshape(B * H, K, V)[rest], TOL[F32],
                     "other heads' states")
    one, one_ref = o[B - 1, :, H - 1], o_ref[B - 1, :, H - 1]
    last, last_ref = S[B - 1, H - 1], S_ref[B - 1, H - 1]
    if name == "v":
        keep = [c for c in range(V) if c != 5]
        assert not torch.isfinite(one[t0, 5]) and not torch.isfinite(last[:, 5]).any()
        assert_close(one[:, keep], one_ref[:, keep], TOL[dtype], "other columns")
        assert_close(last[:, keep], last_ref[:, keep], TOL[F32], "their state")
    elif name == "q":
        assert not torch.isfinite(one[t0]).any()
        if t0 + 1 < L:
            assert_close(one[t0 + 1:], one_ref[t0 + 1:], TOL[dtype], "later steps")
        assert_close(last, last_ref, TOL[F32], "state")
    else:
        assert not torch.isfinite(one[t0:]).any()
        if name == "k":        # one row of the state
            keep = [c for c in range(K) if c != 5]
            assert not torch.isfinite(last[5]).any()
            assert_close(last[keep], last_ref[keep], TOL[F32], "other rows of the state")
        else:
            assert not torch.isfinite(last).any()


def test_chained_calls(dev):
    """A sequence in three calls and then steps, the state handed on, against one call."""
    from tssm import linear_attention_step
    d = inputs(dev, 2, 310, 2, 4, 64, 64, BF16, seed=12)
    o, S = run(d)
    parts, h = [], None
    for lo, hi in ((0, 7), (7, 168), (168, 300)):
        p = {n: d[n][:, lo:hi] for n in ("q", "k", "v", "g")}
        op, h = run(dict(p, h0=h))
        parts.append(op)
    for t in range(300, 310):
        parts.append(linear_attention_step(*(d[n][:, t] for n in ("q", "k", "v", "g")),
                                           h)[:, None])
    assert_close(torch.cat(parts, 1), np64(o), TOL[BF16], "o")
    assert_close(h, np64(S), TOL[F32], "state")


def test_repeat_and_stream(dev):
    """The same bits on a repeated call, and on another stream than the
    tensors' own."""
    for L, heads in ((500, 2), (9000, 1)):
        d = inputs(dev, 2, L, heads, heads, 64, 64, BF16, seed=13)
        o, S = run(d)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            o2, S2 = run(d)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(o, o2) and torch.equal(S, S2)


def test_rows_past_the_end_stay(dev):
    """Rows behind the last step, columns behind V and other heads of a wider
    output are left as they were."""
    B, L, H, K, V = 2, 150, 2, 64, 40
    for dtype in (F32, BF16):
        d = inputs(dev, B, L, H, H, K, V, dtype, seed=15)
        wide = torch.full((B, L + 9, H + 1, V + 8), 7.0, device=dev, dtype=dtype)
        out = wide[:, :L, :H, :V]
        run(d, out=out)
        assert_close(out, oracle(d)[0], TOL[dtype], "o")
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[:, :L, :H, :V] = False
        assert (wide[keep] == 7.0).all()


# ------------------------------------------------------------------ single steps
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("S,Hk,Hv,K,V", [(1, 1, 1, 1, 1), (3, 2, 4, 64, 64), (5, 1, 3, 40, 72),
                                         (700, 2, 2, 16, 48), (2, 3, 3, 128, 128), (9, 1, 2, 7, 33)])
def test_step(dev, dtype, S, Hk, Hv, K, V):
    from tssm import linear_attention_step
    d = inputs(dev, S, 1, Hk, Hv, K, V, dtype, seed=K + V, h0=True)
    o_ref, S_ref = oracle(d)
    state = d["h0"].clone()
    o = linear_attention_step(d["q"][:, 0], d["k"][:, 0], d["v"][:, 0], d["g"][:, 0], state)
    assert_close(o, o_ref[:, 0], TOL[dtype], "o")
    assert_close(state, S_ref, TOL[F32], "state")


def test_many_streams(dev):
    """More waves than one dimension of a grid holds work-items for: 7e7 streams
    of a 1 x 1 state, whose step is a handful of products."""
    from tssm import linear_attention_step
    S = 70_000_000
    r = torch.Generator(device=dev).manual_seed(26)
    q, k, v, state = (torch.randn(S, generator=r, device=dev) for _ in range(4))
    g = -torch.rand(S, generator=r, device=dev)
    before = state.clone()
    o = linear_attention_step(q.view(S, 1, 1), k.view(S, 1, 1), v.view(S, 1, 1), g.view(S, 1),
                              state.view(S, 1, 1, 1)).view(S)
    for lo in range(0, S, 10_000_000):
        s = slice(lo, lo + 10_000_000)
        x = torch.exp(g[s].double()) * before[s].double() + k[s].double() * v[s].double()
        for got, want in ((state[s], x), (o[s], q[s].double() * x)):
            # a step's few roundings of values that are all below `size`
            size = want.abs().max()
            assert (got.double() - want).abs().max() <= 1e-6 * size, lo


# ------------------------------------------------------------------ gradients
NAMES = ("dq", "dk", "dv", "dg", "dh0")


def gradients(d, do, dh=None, **kw):
    from tssm import linear_attention_backward
    return linear_attention_backward(d["q"], d["k"], d["v"], d["g"], do, h0=d["h0"], dh_last=dh,
                                     **kw)


def compare_gradients(d, do, dh, dtype, **kw):
    got = gradients(d, do, dh, **kw)
    ref = M.linear_backward(**{n: None if t is None else np64(t) for n, t in d.items()},
                            do=np64(do), dh_last=None if dh is None else np64(dh), **kw)
    for name, x, y in zip(NAMES, got, ref):
        if name == "dh0" and d["h0"] is None:
            assert x is None
        else:
            assert_close(x, y, TOL[dtype] if name in ("dq", "dk", "dv") else TOL[F32], name)
    return got


def check_gradients(dev, d, dtype, seed, dh=True, **kw):
    r = torch.Generator().manual_seed(seed)
    B, L, Hv, V = d["v"].shape
    K = d["q"].shape[-1]
    do = torch.randn(B, L, Hv, V, generator=r).to(dtype).to(dev)
    dh = torch.randn(B, Hv, K, V, generator=r).to(dev) if dh else None
    return do, dh, compare_gradients(d, do, dh, dtype, **kw)


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


@pytest.mark.parametrize("dtype,B,L,Hk,Hv,K,V", [
    (BF16, 2, 70, 2, 4, 128, 128), (BF16, 1, 33, 1, 3, 128, 72), (BF16, 1, 3000, 1, 2, 128, 64),
    (F16, 2, 100, 1, 2, 128, 128), (BF16, 1, 5000, 1, 1, 24, 20), (F32, 1, 70, 1, 2, 128, 200),
    (F32, 1, 100, 1, 3, 64, 130)])
def test_backward_wide(dev, dtype, B, L, Hk, Hv, K, V):
    """Keys of 128, shared key heads, V in several slices, segments."""
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L + V, h0=True, rate=0.1)
    check_gradients(dev, d, dtype, seed=27)


@pytest.mark.parametrize("rate", [30.0, 1.0, 0.01])
def test_gradient_of_the_decays(dev, rate):
    """dg alone at strong and slow decays: each chunk sums its own terms, so that what
    strong decays leave is not the difference of large sums."""
    d = inputs(dev, 1, 700, 1, 2, 32, 32, F32, seed=31, h0=True, rate=rate)
    check_gradients(dev, d, F32, seed=32)


def test_backward_resets(dev):
    """g = -inf and the lowest value: nothing flows past, and dg is 0 there."""
    d = inputs(dev, 2, 150, 1, 2, 64, 48, F32, seed=33, h0=True, rate=0.1)
    d["g"][0, 40], d["g"][0, 64] = -float("inf"), -float("inf")
    d["g"][1, 41] = torch.finfo(F32).min
    dg = check_gradients(dev, d, F32, seed=34)[2][3]
    assert not dg[0, 40].any() and not dg[0, 64].any() and not dg[1, 41].any()


def test_backward_against_differences(dev):
    """Central differences of the forward itself, in fp32: a step of 2^-6 of inputs of
    size 1 leaves a truncation of 2^-12 / 6 of third derivatives (none in q, k, v and
    h0, of which the loss is linear one at a time) and a rounding of 64 x 2^-24 of the
    loss over the step: 1e-3 of the largest gradient holds both."""
    B, L, H, K, V = 1, 9, 1, 5, 4
    d = inputs(dev, B, L, H, H, K, V, F32, seed=35, h0=True)
    r = torch.Generator().manual_seed(36)
    do = torch.randn(B, L, H, V, generator=r).to(dev)
    dh = torch.randn(B, H, K, V, generator=r).to(dev)

    def loss():
        o, S = run(d)
        return float((o.double() * do.double()).sum() + (S.double() * dh.double()).sum())

    for name, got in zip(("q", "k", "v", "g", "h0"), gradients(d, do, dh)):
        flat, want, eps = d[name].view(-1), [], 2.0 ** -6
        for i in range(flat.numel()):
            old = flat[i].item()
            flat[i] = old + eps
            hi = loss()
            flat[i] = old - eps
            lo = loss()
            flat[i] = old
            want.append((hi - lo) / (2 * eps))
        assert_close(got.reshape(-1), np.array(want), 1e-3, name)


def one_step(t, layout):
    """t [B, 1, H, N] as a view whose step stride is no row's length."""
    B, _, H, N = t.shape
    if layout == "innermost":       # [B, H, N, L] with L = 1
        return t.new_empty(B, H, N, 1).permute(0, 3, 1, 2).copy_(t)
    if layout == "shared":          # one head for all
        return t[:, 0, 0][:, None].expand(B, H, N).unsqueeze(1)
    # 31 rows of this stride pass 32 bits
    return t.contiguous().as_strided(t.shape, (H * N, 1 << 30, N, 1))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["innermost", "shared", "far"])
def test_backward_of_one_step(dev, dtype, layout):
    """The stride of a dimension of one element says nothing."""
    r = torch.Generator().manual_seed(22)
    d = inputs(dev, 2, 1, 3, 3, 32, 32, dtype, seed=21, h0=True)
    do = torch.randn(2, 1, 3, 32, generator=r).to(dtype).to(dev)
    dh = torch.randn(2, 3, 32, 32, generator=r).to(dev)
    for n in ("q", "k", "v"):
        d[n] = one_step(d[n], layout)
    compare_gradients(d, one_step(do, layout), dh, dtype)


def test_backward_strides(dev):
    """Slices of one projection, rows that overlap, steps further apart than a chunk's
    31 bits reach, shared rates, an expanded gradient."""
    B, L, H, K, V = 2, 77, 2, 32, 32
    d = inputs(dev, B, L, H, H, K, V, F32, seed=5, h0=True)
    packed = torch.zeros(B, L, H * (2 * K + V) + 3, device=dev)
    for name, at in (("q", 0), ("k", H * K), ("v", 2 * H * K)):
        view = packed[..., at + 1:at + 1 + H * K].view(B, L, H, K)
        view.copy_(d[name])
        d[name] = view
    d["g"] = d["g"][:1, :1].expand(B, L, H)
    check_gradients(dev, d, F32, seed=6)
    d["k"] = d["k"][:, :1].expand(B, L, H, K)
    compare_gradients(d, torch.ones(B, 1, H, V, device=dev).expand(B, L, H, V), None, F32)
    far = 17_000_000
    base = torch.empty(3 * H * K + 2 * far, device=dev)
    e = {n: t if t is None or n == "h0" else t[:1, :3] for n, t in d.items()}
    e["h0"] = d["h0"][:1]
    for i, n in enumerate(("q", "k", "v")):
        view = base.as_strided((1, 3, H, K), (1, far, K, 1), i * H * K)
        view.copy_(e[n])
        e[n] = view
    check_gradients(dev, e, F32, seed=7)


def test_backward_empty_and_repeat(dev):
    d = inputs(dev, 2, 0, 2, 2, 32, 32, F32, h0=True)
    dh = torch.ones_like(d["h0"])
    assert torch.equal(gradients(d, d["v"], dh)[4], dh)
    assert not gradients(d, d["v"])[4].any()
    for L in (300, 9000):
        d = inputs(dev, 1, L, 1, 2, 64, 64, BF16, seed=41)
        do = d["v"].flip(1).contiguous()
        want = gradients(d, do)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = gradients(d, do)
        torch.cuda.current_stream().wait_stream(side)
        assert all(x is y is None or torch.equal(x, y) for x, y in zip(got, want))
