"""Calls of linear attention and of the norm and rotation that their own tests leave
out: captured and replayed ones, two threads on a stream, the lengths where the form of a
call changes, gradients of unaligned and transposed operands, and the operators
together as a layer uses them, in training and in serving."""
import threading

import pytest
import torch

from helpers import assert_close
import test_gpu_linear as lin
import test_gpu_qknorm as qk

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


# ------------------------------------------------------------------ graphs and threads
def forward(d):
    return lin.run(d)


def backward(d):
    from tssm import linear_attention_backward
    do = d["v"].flip(1)
    return linear_attention_backward(d["q"], d["k"], d["v"], d["g"], do, h0=d["h0"],
                                     dh_last=d["h0"])


def step(d):
    from tssm import linear_attention_step
    state = d["h0"].clone()
    o = linear_attention_step(*(d[n][:, 0] for n in ("q", "k", "v", "g")), state)
    return o, state


def qk_both(d):
    return (*qk.forward(d), *qk.backward(d))


def tokens(L, dtype=BF16, K=64, V=64, H=2):
    return lambda dev, seed: lin.inputs(dev, 1, L, H, 2 * H, K, V, dtype, seed=seed, h0=True,
                                        rate=0.1)


def rows(L, dtype=BF16):
    return lambda dev, seed: qk.inputs(dev, 2, L, 3, 2, 64, 32, dtype, seed=seed)


FORMS = [
    (forward, tokens(5), tokens(3000)),              # step by step
    (forward, tokens(100), tokens(30000)),
    (forward, tokens(3000), tokens(30000)),          # segments
    (forward, tokens(1200, F32, K=100, V=40), tokens(9000, F32)),
    (backward, tokens(100), tokens(5000)),
    (backward, tokens(4000, F16), tokens(9000, F32)),  # segments
    (step, tokens(1), tokens(2)),
    (qk_both, rows(70), rows(2000)),
    (qk_both, rows(500, F32), rows(9000, F32)),
]


@pytest.mark.parametrize("run,make,larger", FORMS)
def test_replays(dev, run, make, larger):
    """Two graphs of one call with other inputs, replayed in turn, with the stream's
    workspace replaced and eager work between: the eager call's bits every time."""
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        inputs = [make(dev, seed) for seed in (1, 2)]
        run(inputs[0])                             # loads the kernels, fills a workspace
        stream.synchronize()
        graphs, outs = [], []
        for d in inputs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(run(d))
            graphs.append(graph)
        run(larger(dev, 3))
        for seed in (4, 5, 6):
            for i, d in enumerate(inputs):
                for t, new in zip(d.values(), make(dev, seed + 10 * i).values()):
                    if t is not None:
                        t.copy_(new)
            rest = [torch.full((1 << 16,), seed, device=dev) for _ in range(8)]
            for graph in graphs:
                graph.replay()
            stream.synchronize()
            for d, out in zip(inputs, outs):
                assert all(x is None or torch.equal(x, y) for x, y in zip(out, run(d))), seed
            assert all((t == seed).all() for t in rest)


def test_two_threads_on_a_stream(dev):
    """Segments and gradients, whose launches hand data on through one workspace."""
    cases = [(forward, tokens(3000)(dev, 1)), (backward, tokens(2000)(dev, 2)),
             (qk_both, rows(300)(dev, 3))]
    want = [run(d) for run, d in cases]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(cases))

    def work(i):
        start.wait()
        for n in range(20):
            got = cases[i][0](cases[i][1])
            if not all(x is None or torch.equal(x, y) for x, y in zip(got, want[i])):
                wrong.append((i, n))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------ where forms change
@pytest.mark.parametrize("dtype,B,L,Hv,K,V", [
    (BF16, 1, 12, 2, 16, 16), (BF16, 1, 13, 2, 16, 16),          # one by one or a chunk
    (F32, 64, 51, 16, 8, 8), (F32, 64, 52, 16, 8, 8),            # the same for 1024 heads
    (F16, 130, 64, 16, 8, 16), (F16, 130, 65, 16, 8, 16),        # and for 2080
    (BF16, 1, 767, 1, 32, 32), (BF16, 1, 768, 1, 32, 32),        # whole or in segments
    (F16, 4, 600, 8, 72, 72),                                    # two segments
    (F32, 5, 800, 14, 16, 20),                                   # three
    (BF16, 5, 6200, 14, 16, 16),                                 # long ones are halved
    (BF16, 3, 900, 86, 16, 16),                                  # a full chip: whole
])
def test_forms(dev, dtype, B, L, Hv, K, V):
    lin.check(lin.inputs(dev, B, L, Hv, Hv, K, V, dtype, seed=L + Hv, h0=True, rate=0.1))


@pytest.mark.parametrize("dtype,B,L,Hv,K,V", [
    (BF16, 1, 1535, 1, 32, 32), (BF16, 1, 1536, 1, 32, 32),      # whole or in segments
    (F32, 1, 1700, 2, 100, 24), (F16, 2, 1800, 3, 48, 40),
])
def test_forms_of_the_gradients(dev, dtype, B, L, Hv, K, V):
    d = lin.inputs(dev, B, L, Hv, Hv, K, V, dtype, seed=L, h0=True, rate=0.1)
    lin.check_gradients(dev, d, dtype, seed=L)


@pytest.mark.parametrize("dtype,B,L,Hk,Hv,K,V", [
    (BF16, 6, 2017, 1, 2, 16, 16), (F16, 3, 2100, 2, 6, 24, 40), (F32, 3, 1024, 4, 8, 32, 8),
    (F32, 6, 1040, 1, 3, 100, 36),
    (BF16, 2, 6080, 1, 2, 32, 32), (F32, 1, 6110, 2, 4, 16, 20),   # one chunk too few for it
])
def test_gradients_of_shared_heads(dev, dtype, B, L, Hk, Hv, K, V):
    """Value heads one after the other in a workgroup, or in workgroups of their own."""
    d = lin.inputs(dev, B, L, Hk, Hv, K, V, dtype, seed=L, h0=True, rate=0.1)
    lin.check_gradients(dev, d, dtype, seed=L)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 40), (24, 72)])
def test_gradients_of_views(dev, dtype, K, V):
    """q, k and v packed at an odd offset, dO with the heads first, g a transposed
    view: the same bits as of contiguous tensors."""
    B, L, H = 2, 150, 2
    d = lin.inputs(dev, B, L, H, H, K, V, dtype, seed=K, h0=True)
    do, dh, want = lin.check_gradients(dev, d, dtype, seed=2)
    packed = torch.zeros(B, L, H * (2 * K + V) + 3, device=dev, dtype=dtype)
    at, views = 1, {}
    for n, N in (("q", K), ("k", K), ("v", V)):
        views[n] = packed[..., at:at + H * N].view(B, L, H, N)
        views[n].copy_(d[n])
        at += H * N
    views["g"] = d["g"].transpose(1, 2).contiguous().transpose(1, 2)
    views["h0"] = d["h0"]
    do = do.transpose(1, 2).contiguous().transpose(1, 2)
    got = lin.gradients(views, do, dh)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_the_same_tensor_twice(dev):
    """q, k and v are one tensor, dO is its output's own."""
    B, L, H, K = 1, 200, 2, 32
    d = lin.inputs(dev, B, L, H, H, K, K, BF16, seed=3)
    d["k"] = d["v"] = d["q"]
    o = lin.check(d)[0]
    lin.compare_gradients(d, o, None, BF16)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("K,V", [(100, 117), (40, 30), (64, 65), (128, 5), (17, 4), (8, 3),
                                 (33, 47), (64, 64), (16, 18)])
@pytest.mark.parametrize("at", [0, 3])
def test_states_of_odd_places(dev, dtype, K, V, at):
    """States whose rows are no whole pieces, at any 4-byte address: what lies before and
    behind stays, in a step, in few tokens and where a chunk reads it."""
    from tssm import linear_attention_forward, linear_attention_step
    S, H = 3, 2
    d = lin.inputs(dev, S, 70, H, H, K, V, dtype, seed=K + V, h0=True)
    n = S * H * K * V
    for L in (1, 6, 70):
        room = torch.full((n + 8,), 5.0, device=dev)
        h = room[at:at + n].view(S, H, K, V)
        h.copy_(d["h0"])
        c = {x: t if x == "h0" else t[:, :L] for x, t in d.items()}
        o_ref, S_ref = lin.oracle(c)
        o, last = linear_attention_forward(*(c[x] for x in ("q", "k", "v", "g")), h0=h,
                                           return_state=True)
        assert_close(o, o_ref, lin.TOL[dtype], "o")
        assert_close(last, S_ref, lin.TOL[F32], "state")
        if L == 1:
            o = linear_attention_step(*(c[x][:, 0] for x in ("q", "k", "v", "g")), h)
            assert_close(o[:, None], o_ref, lin.TOL[dtype], "o")
            assert_close(h, S_ref, lin.TOL[F32], "state")
        else:
            assert torch.equal(h, d["h0"])
        assert (room[:at] == 5.0).all() and (room[at + n:] == 5.0).all()


# ------------------------------------------------------------------ together
# The longest sums have 140 terms (a weight's gradient over the tokens): 12 x 6e-8, 1e-6
# of their size, behind four stages of which each adds 1e-5 of its largest value at
# most; a row that the group norm stretches has a third of the largest row's size at
# least (its state starts from normal values): 5e-5 of the largest value.
TOL = 5e-5


def layer(q, k, v, z, g, t, freq, wq, wk, wn, h0):
    """The operators' formulas in the precision of the inputs, one token at a time."""
    B, L, Hk, K = q.shape
    Hv, V = v.shape[2:]

    def turned(x, w):
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        angle = (t[..., None] * freq)[:, :, None]
        R = 2 * freq.shape[0]
        a, b, rest = x[..., :R // 2], x[..., R // 2:R], x[..., R:]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(),
                          rest], -1).repeat_interleave(Hv // Hk, dim=2)

    q, k, S, o = turned(q, wq), turned(k, wk), h0, []
    for i in range(L):
        S = S * g[:, i, :, None, None].exp() + k[:, i, :, :, None] * v[:, i, :, None]
        o.append((S * q[:, i, :, :, None]).sum(2) * K ** -0.5)
    o = torch.stack(o, 1)
    o = o - o.mean(-1, keepdim=True)
    o = o * (o.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    return o.reshape(B, L, Hv * V) * wn * torch.nn.functional.silu(z), S


def values(B, L, Hk, Hv, K, V, R):
    r = torch.Generator().manual_seed(B + L)
    x = dict(q=torch.randn(B, L, Hk, K, generator=r), k=torch.randn(B, L, Hk, K, generator=r),
             v=torch.randn(B, L, Hv, V, generator=r), z=torch.randn(B, L, Hv * V, generator=r),
             g=-0.2 * torch.rand(B, L, Hv, generator=r),
             t=torch.rand(B, L, generator=r).cumsum(1),
             freq=1000.0 ** (-2.0 * torch.arange(R // 2) / R),
             wq=1 + 0.2 * torch.randn(K, generator=r), wk=1 + 0.2 * torch.randn(K, generator=r),
             wn=1 + 0.2 * torch.randn(Hv * V, generator=r),
             h0=torch.randn(B, Hv, K, V, generator=r))
    return {n: y.double() for n, y in x.items()}


def on_gpu(x, dev):
    y = {n: t.to(dev, F32) for n, t in x.items()}
    y["t"], y["freq"] = x["t"].to(dev), x["freq"].to(dev)
    return y


@pytest.mark.parametrize("B,L,Hk,Hv,K,V,R", [(2, 70, 1, 2, 32, 32, 32), (1, 21, 2, 4, 24, 40, 12),
                                             (1, 140, 2, 2, 64, 48, 64)])
def test_layer_and_its_gradients(dev, B, L, Hk, Hv, K, V, R):
    from tssm import (group_norm_act_backward, group_norm_act_forward, linear_attention_backward,
                      linear_attention_forward, qk_norm_rotary_backward, qk_norm_rotary_forward)
    x = values(B, L, Hk, Hv, K, V, R)
    leaves = ("q", "k", "v", "z", "g", "wq", "wk", "wn", "h0")
    for n in leaves:
        x[n].requires_grad_()
    want, last = layer(**x)
    dy = torch.randn(B, L, Hv * V, generator=torch.Generator().manual_seed(1)).double()
    dh = torch.randn(B, Hv, K, V, generator=torch.Generator().manual_seed(2)).double()
    ((want * dy).sum() + (last * dh).sum()).backward()

    c = on_gpu({n: t.detach() for n, t in x.items()}, dev)
    q, k = qk_norm_rotary_forward(c["q"], c["k"], c["t"], c["freq"], c["wq"], c["wk"])
    o, S = linear_attention_forward(q, k, c["v"], c["g"], h0=c["h0"], return_state=True)
    flat, gate = o.view(B * L, 1, Hv * V), c["z"].view(B * L, 1, Hv * V)
    y, mean, rstd = group_norm_act_forward(flat, Hv, c["wn"], None, gate, return_stats=True)
    do, dwn, _, dz = group_norm_act_backward(dy.to(dev, F32).view_as(flat), flat, mean, rstd, Hv,
                                             c["wn"], None, gate)
    dq, dk, dv, dg, dh0 = linear_attention_backward(
        q, k, c["v"], c["g"], do.view_as(o), h0=c["h0"], dh_last=dh.to(dev, F32))
    dq, dk, dwq, dwk = qk_norm_rotary_backward(dq, dk, c["q"], c["k"], c["t"], c["freq"],
                                               c["wq"], c["wk"])
    got = dict(q=dq, k=dk, v=dv, z=dz.view(B, L, -1), g=dg, wq=dwq, wk=dwk, wn=dwn, h0=dh0)
    assert_close(y.view(B, L, -1), want.detach().numpy(), TOL, "y")
    assert_close(S, last.detach().numpy(), TOL, "state")
    for n in leaves:
        assert_close(got[n], x[n].grad.numpy(), TOL, "d" + n)


def test_prompt_turns_and_steps(dev):
    """A prompt, a second turn and single tokens, each from the state that the one before
    left, against the whole."""
    from tssm import (group_norm_act_forward, linear_attention_forward, linear_attention_step,
                      qk_norm_rotary_forward)
    B, L, Hk, Hv, K, V, R = 3, 60, 2, 4, 32, 24, 16
    x = values(B, L, Hk, Hv, K, V, R)
    want, last = layer(**x)
    c = on_gpu(x, dev)

    def norm(o, z):
        n = o.numel() // (Hv * V)
        return group_norm_act_forward(o.reshape(n, 1, -1), Hv, c["wn"], None,
                                      z.reshape(n, 1, -1)).view(*z.shape)

    S, parts = c["h0"], []
    for s in (slice(0, 37), slice(37, 44)):
        q, k = qk_norm_rotary_forward(c["q"][:, s], c["k"][:, s], c["t"][:, s], c["freq"], c["wq"],
                                      c["wk"])
        o, S = linear_attention_forward(q, k, c["v"][:, s], c["g"][:, s], h0=S, return_state=True)
        parts.append(norm(o, c["z"][:, s]))
    for i in range(44, L):
        q, k = qk_norm_rotary_forward(c["q"][:, i], c["k"][:, i], c["t"][:, i], c["freq"],
                                      c["wq"], c["wk"])
        o = linear_attention_step(q, k, c["v"][:, i], c["g"][:, i], S)
        parts.append(norm(o, c["z"][:, i])[:, None])
    assert_close(torch.cat(parts, 1), want.numpy(), TOL, "y")
    assert_close(S, last.numpy(), TOL, "state")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("K,R,pad", [(40, 40, 0), (40, 20, 0), (72, 72, 4), (24, 8, 2), (56, 28, 0),
                                     (128, 64, 4), (128, 64, 2), (36, 36, 0), (68, 4, 0)])
def test_norm_of_narrow_pieces(dev, dtype, interleaved, K, R, pad):
    """Rows that are made of 8- or 4-byte pieces, by their sizes or by where they begin."""
    d = qk.inputs(dev, 2, 37, 3, 2, K, R, dtype, seed=K + R)
    for n in ("q", "k", "dq", "dk"):
        t = d[n]
        wide = torch.zeros(*t.shape[:3], K + pad, device=dev, dtype=dtype)
        d[n] = wide[..., pad:]
        d[n].copy_(t)
    qk.check(d, interleaved=interleaved)
