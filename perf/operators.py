"""The delta-rule mixer's operators: what their speed is judged by.

One case is one pass through the gated delta rule (whole sequences, with or
without its gradients, or one decoding step of many streams) or through the
group norm with an activation, channels last, that follows it (with or without
its gradients).

Gated delta rule, per batch and value head, with a state S [K, V], keys k_t and
queries q_t of the head's key group, alpha_t = exp(g_t):

    u_t = beta_t (v_t - alpha_t S_{t-1}^T k_t)
    S_t = alpha_t S_{t-1} + k_t u_t^T
    o_t = K^-1/2 S_t^T q_t

Group norm of x [N, S, C] in G groups of channels, xhat normalised over (S, C/G):

    y = act(xhat w + b)            without a gate
    y = (xhat w + b) act(gate)     with one

Where ``own`` is false, ``run`` computes both with elementary torch operations
in 32 bits (the delta rule in its chunked form); where it is true it calls the
framework's operators.  ``exact`` is the step-by-step definition in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CHUNK = 64  # steps of a chunk of the plain form


def listed():
    return [
        # prefill of one mixer layer at the multihead benchmark's shapes
        dict(name="prefill_bf16", kind="scan", B=8, L=4096, Hk=16, Hv=16, K=64, V=64,
             dtype="bf16", h0=False),
        # one very long sequence over few heads
        dict(name="prefill_long_bf16", kind="scan", B=1, L=65536, Hk=8, Hv=8, K=64, V=64,
             dtype="bf16", h0=False),
        # a wide state, two value heads to a key head: a prompt continued from a cached state
        # whose length ends inside a chunk
        dict(name="prefill_wide_bf16", kind="scan", B=2, L=2000, Hk=8, Hv=16, K=128, V=128,
             dtype="bf16", h0=True),
        # fp32 with sizes that fill no tile, resumed from a state
        dict(name="prefill_f32", kind="scan", B=3, L=1111, Hk=4, Hv=12, K=40, V=72,
             dtype="f32", h0=True),
        # the smallest: a few tokens of one stream, where latency counts
        dict(name="prefill_few", kind="scan", B=1, L=5, Hk=4, Hv=8, K=64, V=64, dtype="bf16",
             h0=True),
        # training: the forward pass and every gradient
        dict(name="train_bf16", kind="train", B=4, L=4096, Hk=16, Hv=16, K=64, V=64,
             dtype="bf16", h0=False),
        # the same in fp32 with shared key heads, truncated back-propagation (state in and out)
        dict(name="train_f32", kind="train", B=2, L=777, Hk=4, Hv=8, K=64, V=96, dtype="f32",
             h0=True),
        # decode: one step of the streaming benchmark's streams, 4 GiB of state in place
        dict(name="step_many", kind="step", S=4096, Hk=32, Hv=32, K=128, V=64, dtype="bf16"),
        # decode of one stream
        dict(name="step_one", kind="step", S=1, Hk=8, Hv=16, K=128, V=128, dtype="bf16"),
        # the mixer's output norm: per token and head, gated by SiLU
        dict(name="norm_token_bf16", kind="norm", N=32768, S=1, G=16, Cg=64, dtype="bf16",
             gate=True, act="silu", grad=False),
        # the same with its gradients, in training
        dict(name="norm_token_train", kind="norm", N=8192, S=1, G=16, Cg=64, dtype="bf16",
             gate=True, act="silu", grad=True),
        # statistics over whole sequences (a classifier over sampled series), with gradients
        dict(name="norm_series_f32", kind="norm", N=16, S=2048, G=8, Cg=32, dtype="f32",
             gate=False, act="silu", grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "train", "train", "step", "step", "norm", "norm",
                       "norm"])
    if kind == "norm":
        C = _log(rng, 16, 2048)
        G = max(g for g in range(1, 33) if C % g == 0) if rng.random() < 0.5 else \
            rng.choice([g for g in range(1, 33) if C % g == 0])
        token = rng.random() < 0.5
        grad = rng.random() < 0.5
        most = (32768 * 1024 if not grad else 8192 * 1024) // C
        N = _log(rng, 1, min(32768, most)) if token else _log(rng, 1, min(32, most))
        S = 1 if token else _log(rng, 2, max(2, min(8192, most // N)))
        return dict(kind=kind, N=N, S=S, G=G, Cg=C // G, dtype=rng.choice(["bf16", "f32", "f16"]),
                    gate=rng.random() < 0.5, act=rng.choice(["silu", "silu", "none"]), grad=grad)
    Hk, per = rng.randint(1, 16), rng.choice([1, 1, 2, 3])
    K = rng.choice([16, 32, 64, 64, 128, 128, 8 * rng.randint(1, 16)])
    V = rng.choice([16, 32, 64, 64, 128, 128, 8 * rng.randint(1, 16), rng.randint(1, 128)])
    size = Hk * per * K * V
    if kind == "step":
        return dict(kind=kind, S=_log(rng, 1, min(4096, 4096 * 32 * 128 * 64 // size)), Hk=Hk,
                    Hv=Hk * per, K=K, V=V, dtype=rng.choice(["bf16", "f32", "f16"]))
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    B = _log(rng, 1, 4)
    # at most half of the work of the largest listed sequence
    most = (8 * 4096 * 16 * 64 * 64 if kind == "scan" else 4 * 4096 * 16 * 64 * 64) // 2 // (
        B * size)
    L = _log(rng, 1, max(1, min(65536 if kind == "scan" else 4096, most)))
    return dict(kind=kind, B=B, L=L, Hk=Hk, Hv=Hk * per, K=K, V=V, dtype=dtype,
                h0=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=gen, device="cuda") * (hi - lo) + lo

    def unit(t):
        return (t / t.norm(dim=-1, keepdim=True)).to(dtype)

    if c["kind"] == "norm":
        N, S, G, C = c["N"], c["S"], c["G"], c["G"] * c["Cg"]
        # activations whose channels have offsets of their own
        s = dict(x=(normal(N, S, C) + 0.5 * normal(C)).to(dtype), G=G, act=c["act"],
                 w=1.0 + 0.2 * normal(C), b=0.2 * normal(C), gate=None, dy=None)
        if c["gate"]:
            s["gate"] = normal(N, S, C).to(dtype)
        if c["grad"]:
            s["dy"] = normal(N, S, C).to(dtype)
        return s
    rows = (c["S"],) if c["kind"] == "step" else (c["B"], c["L"])
    Hk, Hv, K, V = c["Hk"], c["Hv"], c["K"], c["V"]
    # unit keys and queries that share a direction within a head, irregular time gaps with a
    # rate for each head, step sizes in (0, 1)
    s = dict(q=unit(normal(*rows, Hk, K)), k=unit(normal(*rows, Hk, K) + 0.5 * normal(Hk, K)),
             v=normal(*rows, Hv, V).to(dtype), beta=torch.sigmoid(normal(*rows, Hv)))
    gap = torch.empty(*rows, 1, device="cuda").exponential_(20.0, generator=gen).clamp_(1e-3, 1.0)
    s["g"] = -gap * torch.exp(uniform(Hv, lo=math.log(0.5), hi=math.log(5.0)))
    if c["kind"] == "step":
        s["state"] = 0.3 * normal(c["S"], Hv, K, V)
        return s
    s["h0"] = 0.3 * normal(c["B"], Hv, K, V) if c["h0"] else None
    if c["kind"] == "train":
        s["do"] = normal(*rows, Hv, V).to(dtype)
        s["dh"] = normal(c["B"], Hv, K, V) if c["h0"] else None
    return s


def prepare(case, seed):
    return dict(_inputs(case, seed), case=case)


# ------------------------------------------------------------------ plain forms
def _delta_plain(q, k, v, g, beta, h0):
    """The chunked form in 32 bits.  Within a chunk, with G the sums of g and
    D[t, i] = exp(G_t - G_i): (I + A) U = beta (V - e^G K S), A the strict lower part of
    beta D K K^T; O = e^G Q S + (Q K^T D) U; S' = e^G_end S + K^T (e^(G_end - G) U)."""
    B, L, Hv, V = v.shape
    K, pad = q.shape[-1], (-L) % CHUNK

    def cut(t):  # [B, L, H, ...] -> [B, Hv, chunk, CHUNK, ...]
        t = torch.nn.functional.pad(t.float(), (0, 0) * (t.dim() - 2) + (0, pad))
        t = t.reshape(B, -1, CHUNK, *t.shape[2:]).movedim(3, 1)
        return t.repeat_interleave(Hv // t.shape[1], 1) if t.shape[1] != Hv else t.contiguous()

    q, k, v, g, beta = cut(q) * K ** -0.5, cut(k), cut(v), cut(g), cut(beta)
    G = torch.cumsum(g, -1)
    keep = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    D = (G[..., :, None] - G[..., None, :]).masked_fill(~keep, -math.inf).exp()
    kt = k.transpose(-1, -2).contiguous()
    P = torch.matmul(q, kt) * D
    A = (torch.matmul(k, kt) * D * beta[..., None]).masked_fill(
        torch.eye(CHUNK, dtype=torch.bool, device=q.device), 0.0)
    T = torch.eye(CHUNK, device=q.device).expand_as(A)
    n = 1
    while n < CHUNK:  # inverse of the diagonal blocks of 2n from those of n
        at = torch.arange(CHUNK, device=q.device) // n
        low = (at[:, None] == at[None, :] + 1) & (at[:, None] % 2 == 1)
        T = T - torch.matmul(T, torch.matmul(A * low, T))
        n *= 2
    eG, end = torch.exp(G), torch.exp(G[..., -1:] - G)
    TV = torch.matmul(T, beta[..., None] * v)
    TK = torch.matmul(T, (beta * eG)[..., None] * k)
    qe, ke, last = eG[..., None] * q, kt * end[..., None, :], eG[..., -1, None, None]
    S = torch.zeros(B, Hv, K, V, device=q.device) if h0 is None else h0.float()
    o = []
    for i in range(q.shape[2]):
        U = TV[:, :, i] - torch.matmul(TK[:, :, i], S)
        o.append(torch.matmul(qe[:, :, i], S) + torch.matmul(P[:, :, i], U))
        S = last[:, :, i] * S + torch.matmul(ke[:, :, i], U)
    return torch.stack(o, 2).movedim(1, 3).reshape(B, -1, Hv, V)[:, :L], S


def _delta_train_plain(s):
    names = ["q", "k", "v", "g", "beta"] + (["h0"] if s["h0"] is not None else [])
    leaves = {n: s[n].float().detach().requires_grad_() for n in names}
    o, S = _delta_plain(*(leaves[n] for n in names[:5]), leaves.get("h0"))
    outs, grads = [o], [s["do"].float()]
    if s["dh"] is not None:
        outs, grads = outs + [S], grads + [s["dh"]]
    d = torch.autograd.grad(outs, [leaves[n] for n in names], grads)
    dtype = s["q"].dtype
    return (o.detach().to(dtype), S.detach()) + tuple(t.to(dtype) for t in d[:3]) + tuple(d[3:])


def _step_plain(s):
    q, k, v, state = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    per = state.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(per, 1) * q.shape[-1] ** -0.5, k.repeat_interleave(per, 1)
    state.mul_(torch.exp(s["g"])[..., None, None])
    u = s["beta"][..., None] * (v - torch.matmul(k[..., None, :], state)[..., 0, :])
    state.addcmul_(k[..., None], u[..., None, :])
    return torch.matmul(q[..., None, :], state)[..., 0, :].to(s["v"].dtype), state


def _act(t, act):
    return t * torch.sigmoid(t) if act == "silu" else t


def _norm_plain(x, w, b, gate, G, act):
    N, S, C = x.shape
    xg = x.reshape(N, S, G, C // G)
    mean = xg.mean((1, 3), keepdim=True)
    var = (xg - mean).square().mean((1, 3), keepdim=True)
    z = ((xg - mean) * torch.rsqrt(var + 1e-5)).reshape(N, S, C) * w + b
    return _act(z, act) if gate is None else z * _act(gate, act)


def _norm_pass_plain(s):
    gate = None if s["gate"] is None else s["gate"].float()
    if s["dy"] is None:
        return _norm_plain(s["x"].float(), s["w"], s["b"], gate, s["G"], s["act"]).to(s["x"].dtype)
    leaves = [t.detach().requires_grad_() for t in (s["x"].float(), s["w"], s["b"], gate)
              if t is not None]
    y = _norm_plain(*leaves[:3], leaves[3] if gate is not None else None, s["G"], s["act"])
    dx, dw, db, *dgate = torch.autograd.grad(y, leaves, s["dy"].float())
    dtype = s["x"].dtype
    return (y.detach().to(dtype), dx.to(dtype), dw, db) + tuple(t.to(dtype) for t in dgate)


# ------------------------------------------------------------------ the framework's operators
def _framework():
    path = os.path.abspath("triton-ssm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tssm
    return tssm


def _run_own(s):
    tssm, kind = _framework(), s["case"]["kind"]
    if kind == "scan":
        return tssm.gated_delta_forward(s["q"], s["k"], s["v"], s["g"], s["beta"], h0=s["h0"],
                                        return_state=True)
    if kind == "train":
        o, S = tssm.gated_delta_forward(s["q"], s["k"], s["v"], s["g"], s["beta"], h0=s["h0"],
                                        return_state=True)
        d = tssm.gated_delta_backward(s["q"], s["k"], s["v"], s["g"], s["beta"], s["do"],
                                      h0=s["h0"], dh_last=s["dh"])
        return (o, S) + tuple(t for t in d if t is not None)
    if kind == "step":
        return tssm.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"],
                                     s["state"]), s["state"]
    if s["dy"] is None:
        return tssm.group_norm_act_forward(s["x"], s["G"], s["w"], s["b"], s["gate"],
                                           act=s["act"])
    y, mean, rstd = tssm.group_norm_act_forward(s["x"], s["G"], s["w"], s["b"], s["gate"],
                                                act=s["act"], return_stats=True)
    d = tssm.group_norm_act_backward(s["dy"], s["x"], mean, rstd, s["G"], s["w"], s["b"],
                                     s["gate"], act=s["act"])
    return (y,) + tuple(t for t in d if t is not None)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "scan":
        o, S = _delta_plain(state["q"], state["k"], state["v"], state["g"], state["beta"],
                            state["h0"])
        return o.to(state["v"].dtype), S
    if kind == "train":
        return _delta_train_plain(state)
    if kind == "step":
        return _step_plain(state)
    return _norm_pass_plain(state)


# ------------------------------------------------------------------ cost
def work(c):
    e = BYTES[c["dtype"]]
    if c["kind"] == "norm":
        n, C = c["N"] * c["S"] * c["G"] * c["Cg"], c["G"] * c["Cg"]
        passes = 3 if c["gate"] else 2          # x (and the gate) in, y out
        if c["grad"]:
            passes += 3 if c["gate"] else 2     # dy in, dx (and the gate's gradient) out
        return dict(bytes=passes * n * e + (16 if c["grad"] else 8) * C,
                    flops=(40 if c["grad"] else 12) * n)
    Hk, Hv, K, V = c["Hk"], c["Hv"], c["K"], c["V"]
    rows = c["S"] if c["kind"] == "step" else c["B"] * c["L"]
    each = rows * (2 * Hk * K + 2 * Hv * V) * e + rows * Hv * 8     # q, k, v, o, g, beta
    state = (c["S"] if c["kind"] == "step" else c["B"]) * Hv * K * V * 4
    flops = 7 * rows * Hv * K * V
    if c["kind"] == "step":
        return dict(bytes=each + 2 * state, flops=flops)
    if c["kind"] == "scan":
        return dict(bytes=each + state * (2 if c["h0"] else 1), flops=flops)
    # forward as above; its gradients: do in, those of q, k, v, g and beta out (the inputs are
    # the forward's, read once), of the states where they are given
    grads = rows * (2 * Hk * K + 2 * Hv * V) * e + rows * Hv * 8
    return dict(bytes=each + grads + state * (4 if c["h0"] else 1), flops=3 * flops)


# ------------------------------------------------------------------ 64-bit definitions
def _norm_exact(s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    N, S, C = x.shape
    G = s["G"]
    n = S * (C // G)
    wide = lambda t: t[:, None, :, None].expand(N, S, G, C // G).reshape(N, S, C)  # noqa: E731
    over = lambda t: t.reshape(N, S, G, C // G).sum((1, 3))                        # noqa: E731
    m = over(x) / n
    r = 1.0 / torch.sqrt(over((x - wide(m)) ** 2) / n + 1e-5)
    xhat = (x - wide(m)) * wide(r)
    z = xhat * w + b
    at = z if s["gate"] is None else s["gate"].double()   # what the activation is applied to
    if s["act"] == "silu":
        sg = 1.0 / (1.0 + torch.exp(-at))
        f, df = at * sg, sg * (1.0 + at * (1.0 - sg))
    else:
        f, df = at, torch.ones_like(at)
    y = f if s["gate"] is None else z * f
    if s["dy"] is None:
        return y
    dy = s["dy"].double()
    dz = dy * df if s["gate"] is None else dy * f
    dxhat = dz * w
    dx = wide(r) * (dxhat - wide(over(dxhat) / n) - xhat * wide(over(dxhat * xhat) / n))
    out = (y, dx, (dz * xhat).sum((0, 1)), dz.sum((0, 1)))
    return out if s["gate"] is None else out + (dy * z * df,)


def _delta_exact(s, c):
    per = c["Hv"] // c["Hk"]
    q = s["q"].double().repeat_interleave(per, 2) * c["K"] ** -0.5
    k = s["k"].double().repeat_interleave(per, 2)
    v, alpha, beta = s["v"].double(), torch.exp(s["g"].double()), s["beta"].double()
    B, L, Hv, V = v.shape
    S = torch.zeros(B, Hv, c["K"], V, dtype=torch.float64, device=v.device) \
        if s["h0"] is None else s["h0"].double()
    o, train = torch.empty_like(v), c["kind"] == "train"
    u, before = torch.empty_like(v), []
    for t in range(L):
        if train:
            before.append(S)
        S = S * alpha[:, t, :, None, None]
        u[:, t] = beta[:, t, :, None] * (v[:, t] - (k[:, t, :, :, None] * S).sum(2))
        S.addcmul_(k[:, t, :, :, None], u[:, t, :, None, :])
        o[:, t] = torch.matmul(q[:, t, :, None, :], S)[:, :, 0]
    if not train:
        return o, S
    do = s["do"].double()
    dS = torch.zeros_like(S) if s["dh"] is None else s["dh"].double()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg, dbeta = torch.empty_like(alpha), torch.empty_like(beta)
    for t in range(L - 1, -1, -1):
        prev = before.pop()
        a, kt, bt = alpha[:, t, :, None, None], k[:, t, :, :, None], beta[:, t, :, None]
        now = a * prev + kt * u[:, t, :, None, :]
        dq[:, t] = torch.matmul(now, do[:, t, :, :, None])[..., 0]
        dS = dS + q[:, t, :, :, None] * do[:, t, :, None, :]
        du = (kt * dS).sum(2)
        seen = (kt * prev).sum(2)                     # S_{t-1}^T k_t
        dv[:, t] = bt * du
        dbeta[:, t] = (du * (v[:, t] - a[..., 0] * seen)).sum(-1)
        dseen = -(a[..., 0] * bt) * du
        dk[:, t] = torch.matmul(dS, u[:, t, :, :, None])[..., 0] + \
            torch.matmul(prev, dseen[..., None])[..., 0]
        dg[:, t] = a[..., 0, 0] * (dS * prev).sum((2, 3)) + (dseen * seen).sum(-1)
        dS = a * dS + kt * dseen[..., None, :]
    share = lambda t: t.reshape(B, L, c["Hk"], per, c["K"]).sum(3)  # noqa: E731
    out = (o, S, share(dq) * c["K"] ** -0.5, share(dk), dv, dg, dbeta)
    return out if s["h0"] is None else out + (dS,)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "norm":
        return _norm_exact(s)
    if case["kind"] != "step":
        return _delta_exact(s, case)
    per = case["Hv"] // case["Hk"]
    k = s["k"].double().repeat_interleave(per, 1)
    q = s["q"].double().repeat_interleave(per, 1) * case["K"] ** -0.5
    S = s.pop("state").double().mul_(torch.exp(s["g"].double())[..., None, None])
    u = s["beta"].double()[..., None] * (s["v"].double() - torch.matmul(k[..., None, :], S)[..., 0, :])
    S.addcmul_(k[..., None], u[..., None, :])
    return torch.matmul(q[..., None, :], S)[..., 0, :], S
