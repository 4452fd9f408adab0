"""GPU parity of the gated delta rule at its edges: step strides that are no
row's length, tensors past launch limits, values that are not finite in every
form of the kernels.  Tolerances as in test_gpu_delta."""
import pytest
import torch

from helpers import assert_close, np64
from oracle import mixer_oracle as M
from test_gpu_delta import BF16, F16, F32, NAMES, TOL, gradients, inputs, oracle, run

pytestmark = pytest.mark.gpu


def compare_gradients(d, do, dh, dtype):
    ref = M.delta_backward(**{n: None if t is None else np64(t) for n, t in d.items()},
                           do=np64(do), dh_last=None if dh is None else np64(dh))
    for name, x, y in zip(NAMES, gradients(d, do, dh), ref):
        assert_close(x, y, TOL[dtype] if name in ("dq", "dk", "dv") else TOL[F32], name)


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
@pytest.mark.parametrize("layout,step", [("innermost", 1), ("shared", 0), ("far", 1 << 30)])
def test_backward_of_one_step(dev, dtype, layout, step):
    """The stride of a dimension of one element says nothing."""
    r = torch.Generator().manual_seed(22)
    d = inputs(dev, 2, 1, 3, 3, 32, 32, dtype, seed=21, h0=True)
    do = torch.randn(2, 1, 3, 32, generator=r).to(dtype).to(dev)
    dh = torch.randn(2, 3, 32, 32, generator=r).to(dev)
    for n in ("q", "k", "v"):
        d[n] = one_step(d[n], layout)
        assert d[n].stride(1) == step
    compare_gradients(d, one_step(do, layout), dh, dtype)


def test_many_streams(dev):
    """More waves than one dimension of a grid holds work-items for: 7e7 streams
    of a 1 x 1 state, whose step is a handful of products."""
    from tssm import gated_delta_step
    S = 70_000_000
    r = torch.Generator(device=dev).manual_seed(26)
    q, k, v, state = (torch.randn(S, generator=r, device=dev) for _ in range(4))
    beta = torch.rand(S, generator=r, device=dev)
    g = -torch.rand(S, generator=r, device=dev)
    before = state.clone()
    o = gated_delta_step(q.view(S, 1, 1), k.view(S, 1, 1), v.view(S, 1, 1), g.view(S, 1),
                         beta.view(S, 1), state.view(S, 1, 1, 1)).view(S)
    for lo in range(0, S, 10_000_000):
        s = slice(lo, lo + 10_000_000)
        x = torch.exp(g[s].double()) * before[s].double()
        k64 = k[s].double()
        x = x + k64 * beta[s].double() * (v[s].double() - k64 * x)
        for got, want in ((state[s], x), (o[s], q[s].double() * x)):
            # a step's few roundings of values that are all below `size`
            size = want.abs().max()
            assert (got.double() - want).abs().max() <= 1e-5 * size, lo


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("odd", ["dq", "dk", "dv"])
def test_packed_gradients(dev, dtype, odd):
    """The C entry point with gradients in one allocation, one of which starts on
    no 16-byte boundary."""
    from tssm import _lib
    B, L, H, K, V = 2, 70, 2, 64, 48
    r = torch.Generator().manual_seed(29)
    d = inputs(dev, B, L, H, H, K, V, dtype, seed=30, h0=True)
    do = torch.randn(B, L, H, V, generator=r).to(dtype).to(dev)
    want = gradients(d, do)
    sizes = dict(dq=d["q"], dk=d["k"], dv=d["v"])
    pack = torch.full((sum(t.numel() for t in sizes.values()) + 64,), 7.0, device=dev, dtype=dtype)
    got, used, at = {}, torch.zeros_like(pack, dtype=torch.bool), 8
    for name, t in sizes.items():
        at += 1 if name == odd else 0
        got[name] = pack[at:at + t.numel()].view(t.shape)
        used[at:at + t.numel()] = True
        at = (at + t.numel() + 7) // 8 * 8
    dg, dbeta, dh0 = (torch.empty_like(d[n]) for n in ("g", "beta", "h0"))
    n = _lib.lib().tssm_gated_delta_backward_workspace_bytes(B, L, H, H, K, V)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    t = [d[x] for x in ("q", "k", "v")]
    _lib.call("tssm_gated_delta_backward", {F32: 0, BF16: 1}[dtype], *(x.data_ptr() for x in t),
              d["g"].data_ptr(), d["beta"].data_ptr(), d["h0"].data_ptr(), do.data_ptr(), None,
              *(g.data_ptr() for g in got.values()), dg.data_ptr(), dbeta.data_ptr(),
              dh0.data_ptr(), B, L, H, H, K, V, *(s for x in t for s in x.stride()[:3]),
              *d["g"].stride(), *d["beta"].stride(), *do.stride()[:3], K ** -0.5, ws.data_ptr(), n,
              torch.cuda.current_stream().cuda_stream)
    for name, x, y in zip(NAMES, (*got.values(), dg, dbeta, dh0), want):
        assert_close(x, np64(y), 2.0 ** -8 if dtype == BF16 and name in got else 1e-6, name)
    assert (pack[~used] == 7.0).all()


def test_backward_of_far_steps(dev):
    """Steps that lie further apart than a chunk's 31 bits reach."""
    L, H, N, far = 3, 2, 16, 17_000_000
    r = torch.Generator().manual_seed(24)
    d = inputs(dev, 1, L, H, H, N, N, F32, seed=25, h0=True)
    do = torch.randn(1, L, H, N, generator=r).to(dev)
    base = torch.empty(4 * H * N + (L - 1) * far, device=dev)
    views = [base.as_strided((1, L, H, N), (1, far, N, 1), i * H * N) for i in range(4)]
    for view, t in zip(views, (d["q"], d["k"], d["v"], do)):
        view.copy_(t)
    d["q"], d["k"], d["v"], do = views
    compare_gradients(d, do, torch.randn(1, H, N, N, generator=r).to(dev), F32)


@pytest.mark.parametrize("dtype,B,L,H,K,V,t0", [
    (BF16, 1, 8200, 2, 64, 64, 4000),     # in segments, far from their ends
    (F32, 1, 5001, 1, 40, 72, 3203),
    (F16, 1, 150, 2, 64, 64, 75),
    (F16, 2, 3000, 1, 128, 30, 31),       # in the first chunk of a segmented sequence
    (BF16, 1, 150, 2, 128, 128, 149),     # the last step
    (F32, 1, 150, 2, 128, 64, 64),        # the first step of a chunk
    (BF16, 2, 70, 2, 24, 40, 40),         # K and V that fill no tile
])
@pytest.mark.parametrize("name", ["v", "k", "q", "beta", "g"])
def test_not_finite_in_every_form(dev, dtype, B, L, H, K, V, t0, name):
    """A NaN at one step of one head changes no earlier output and no other head;
    in v no other column, in q no other step."""
    d = inputs(dev, B, L, H, H, K, V, dtype, seed=L + K, h0=True, rate=0.05)
    o_ref, S_ref = oracle(d)
    if name in ("beta", "g"):
        d[name][B - 1, t0, H - 1] = float("nan")
    else:
        d[name][B - 1, t0, H - 1, 5] = float("nan")
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
        assert torch.isnan(one[t0, 5]) and torch.isnan(last[:, 5]).all()
        assert_close(one[:, keep], one_ref[:, keep], TOL[dtype], "other columns")
        assert_close(last[:, keep], last_ref[:, keep], TOL[F32], "their state")
    elif name == "q":
        assert torch.isnan(one[t0]).all()
        if t0 + 1 < L:
            assert_close(one[t0 + 1:], one_ref[t0 + 1:], TOL[dtype], "later steps")
        assert_close(last, last_ref, TOL[F32], "state")
    else:
        assert torch.isnan(one[t0:]).all() and torch.isnan(last).all()


@pytest.mark.parametrize("dtype,B,L,Hk,Hv,K,V", [
    (BF16, 2, 70, 2, 4, 128, 128), (BF16, 1, 33, 1, 3, 128, 72), (BF16, 1, 3000, 1, 2, 128, 64),
    (F16, 2, 100, 1, 2, 128, 128), (BF16, 1, 5000, 1, 1, 24, 20), (F32, 1, 70, 1, 2, 128, 200)])
def test_backward_wide(dev, dtype, B, L, Hk, Hv, K, V):
    """Keys of 128, shared key heads, V in several slices, segments."""
    r = torch.Generator().manual_seed(27)
    d = inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L + V, h0=True, rate=0.1)
    do = torch.randn(B, L, Hv, V, generator=r).to(dtype).to(dev)
    compare_gradients(d, do, torch.randn(B, Hv, K, V, generator=r).to(dev), dtype)


def test_long_sequence_of_shared_rows(dev):
    """The C entry point with one key and one query for all steps (stride 0): rows
    that overlap go step by step at any length, without a workspace."""
    from tssm import _lib
    B, L, H, K, V = 2, 100, 2, 64, 48
    d = inputs(dev, B, L, H, H, K, V, BF16, seed=28, h0=True)
    d["q"], d["k"] = d["q"][:, :1].expand(B, L, H, K), d["k"][:, :1].expand(B, L, H, K)
    o, S = torch.empty_like(d["v"]), torch.empty_like(d["h0"])
    t = [d[x] for x in ("q", "k", "v")]
    assert d["q"].stride(1) == 0
    _lib.call("tssm_gated_delta_forward", 1, *(x.data_ptr() for x in t), d["g"].data_ptr(),
              d["beta"].data_ptr(), d["h0"].data_ptr(), o.data_ptr(), S.data_ptr(), B, L, H, H, K,
              V, *(s for x in t for s in x.stride()[:3]), *d["g"].stride(), *d["beta"].stride(),
              *o.stride()[:3], K ** -0.5, None, 0, torch.cuda.current_stream().cuda_stream)
    o_ref, S_ref = oracle(d)
    assert_close(o, o_ref, TOL[BF16], "o")
    assert_close(S, S_ref, TOL[F32], "state")
