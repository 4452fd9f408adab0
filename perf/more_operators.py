"""Linear attention with a decay for each head, and what prepares its queries and
keys: what their speed is judged by.

One case is one pass through linear attention (whole sequences, with or without
their gradients, or one decoding step of many streams) or through the norm of
queries and keys for each head with the rotation by their positions (with or
without its gradients).

Linear attention, per batch and value head, with a state S [K, V], keys k_t and
queries q_t of the head's key group:

    S_t = exp(g_t) S_{t-1} + k_t v_t^T
    o_t = K^-1/2 S_t^T q_t

Norm and rotation of a row x of a head, r = (mean x^2 + eps)^-1/2 ("rms"),
(sum x^2 + eps)^-1/2 ("l2") or 1 ("none"), w a weight for each channel:

    n = r x w;  (n_a, n_b) -> (n_a cos - n_b sin, n_a sin + n_b cos)

for the R/2 pairs of the first R channels, (j, j + R/2) or (2 j, 2 j + 1), by the
angle position * frequency_j; the other channels stay n.

Where ``own`` is false, ``run`` computes both with elementary torch operations
in 32 bits (linear attention in its chunked form, angles in 64 bits); where it
is true it calls the framework's operators.  ``exact`` is the definition in 64
bits, step by step.
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
EPS = 1e-6


def listed():
    return [
        # prefill of one mixer layer at the multihead benchmark's shapes, irregular time gaps
        dict(name="prefill_bf16", kind="scan", B=8, L=4096, Hk=16, Hv=16, K=64, V=64,
             dtype="bf16", h0=False, gaps=True),
        # one very long sequence over few heads
        dict(name="prefill_long_bf16", kind="scan", B=1, L=65536, Hk=8, Hv=8, K=64, V=64,
             dtype="bf16", h0=False, gaps=True),
        # a wide state, two value heads to a key head, one rate for each head and even steps: a
        # prompt continued from a cached state whose length ends inside a chunk
        dict(name="prefill_wide_f16", kind="scan", B=2, L=2000, Hk=8, Hv=16, K=128, V=128,
             dtype="f16", h0=True, gaps=False),
        # fp32 with sizes that fill no tile, resumed from a state
        dict(name="prefill_f32", kind="scan", B=3, L=1111, Hk=4, Hv=12, K=40, V=72,
             dtype="f32", h0=True, gaps=True),
        # training: the forward pass and every gradient
        dict(name="train_bf16", kind="train", B=4, L=4096, Hk=16, Hv=16, K=64, V=64,
             dtype="bf16", h0=False, gaps=True),
        # the same in fp32 with shared key heads, truncated back-propagation (state in and out)
        dict(name="train_f32", kind="train", B=2, L=777, Hk=4, Hv=8, K=64, V=96, dtype="f32",
             h0=True, gaps=True),
        # decode: one step of the streaming benchmark's streams, 4 GiB of state in place
        dict(name="step_many", kind="step", S=4096, Hk=32, Hv=32, K=128, V=64, dtype="bf16",
             gaps=True),
        # decode of one stream, where latency counts
        dict(name="step_one", kind="step", S=1, Hk=8, Hv=16, K=128, V=128, dtype="bf16",
             gaps=False),
        # queries and keys of the prefill above, slices of one projection, positions of tokens
        dict(name="qk_prefill_bf16", kind="qk", B=8, L=4096, Hq=16, Hk=16, K=64, R=64,
             dtype="bf16", norm="rms", weights=True, interleaved=False, at="tokens", packed=True,
             grad=False),
        # training with shared key heads: half of a wide head is rotated, in neighbouring pairs
        dict(name="qk_train_bf16", kind="qk", B=4, L=4096, Hq=16, Hk=8, K=128, R=64,
             dtype="bf16", norm="rms", weights=True, interleaved=True, at="tokens", packed=True,
             grad=True),
        # fp32 unit keys at irregular sampling times, odd sizes, with gradients
        dict(name="qk_times_f32", kind="qk", B=3, L=1111, Hq=12, Hk=4, K=40, R=20, dtype="f32",
             norm="l2", weights=False, interleaved=False, at="times", packed=False, grad=True),
        # decode: one token of each of 64 streams, far into long contexts
        dict(name="qk_step", kind="qk", B=64, L=1, Hq=16, Hk=8, K=128, R=128, dtype="bf16",
             norm="rms", weights=True, interleaved=False, at="far", packed=True, grad=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "scan", "train", "train", "step", "step", "qk", "qk", "qk",
                       "qk"])
    if kind == "qk":
        K = rng.choice([32, 64, 64, 128, 128, 8 * rng.randint(1, 16), rng.randint(2, 128)])
        R = rng.choice([0, 2 * rng.randint(1, K // 2)] + 4 * [K // 2 * 2] + 2 * [K // 4 * 2])
        Hk, per, B, grad = rng.randint(1, 16), rng.choice([1, 1, 2, 4]), _log(rng, 1, 64), \
            rng.random() < 0.5
        # at most the elements of the largest listed case of the kind
        most = (8 * 4096 * 32 * 64 if not grad else 4 * 4096 * 24 * 128) // (
            B * Hk * (1 + per) * K)
        return dict(kind=kind, B=B, L=_log(rng, 1, max(1, min(8192, most))), Hq=Hk * per, Hk=Hk,
                    K=K, R=R, dtype=rng.choice(["bf16", "bf16", "f32", "f16"]),
                    norm=rng.choice(["rms", "rms", "l2", "none"]), weights=rng.random() < 0.6,
                    interleaved=rng.random() < 0.5, at=rng.choice(["tokens", "times", "far"]),
                    packed=rng.random() < 0.5, grad=grad)
    Hk, per = rng.randint(1, 16), rng.choice([1, 1, 2, 3])
    K = rng.choice([16, 32, 64, 64, 128, 128, 8 * rng.randint(1, 16)])
    V = rng.choice([16, 32, 64, 64, 128, 128, 8 * rng.randint(1, 16), rng.randint(1, 128)])
    size, gaps = Hk * per * K * V, rng.random() < 0.7
    if kind == "step":
        return dict(kind=kind, S=_log(rng, 1, min(4096, 4096 * 32 * 128 * 64 // size)), Hk=Hk,
                    Hv=Hk * per, K=K, V=V, dtype=rng.choice(["bf16", "f32", "f16"]), gaps=gaps)
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    B = _log(rng, 1, 4)
    # at most half of the work of the largest listed sequence
    most = (8 * 4096 * 16 * 64 * 64 if kind == "scan" else 4 * 4096 * 16 * 64 * 64) // 2 // (
        B * size)
    L = _log(rng, 1, max(1, min(65536 if kind == "scan" else 4096, most)))
    return dict(kind=kind, B=B, L=L, Hk=Hk, Hv=Hk * per, K=K, V=V, dtype=dtype,
                h0=rng.random() < 0.5, gaps=gaps)


# ------------------------------------------------------------------ inputs
def _inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, generator=gen, device="cuda") * (hi - lo) + lo

    def gap(*shape):
        return torch.empty(*shape, device="cuda").exponential_(20.0, generator=gen).clamp_(1e-3,
                                                                                           1.0)

    if c["kind"] == "qk":
        B, L, Hq, Hk, K, R = (c[n] for n in ("B", "L", "Hq", "Hk", "K", "R"))
        s = dict(wq=None, wk=None, dq=None, dk=None)

        def rows():
            # activations whose channels differ in size; queries and keys lie beside the values
            # and gates of one projection, or in tensors of their own
            heads = (Hq + Hk) * K
            t = (normal(B, L, heads) * torch.exp(0.3 * normal(heads))).to(dtype)
            if c["packed"]:
                wide = torch.empty(B, L, 2 * heads, device="cuda", dtype=dtype)
                wide[..., :heads] = t
                t = wide[..., :heads]
            q, k = t[..., :Hq * K].unflatten(-1, (Hq, K)), t[..., Hq * K:].unflatten(-1, (Hk, K))
            return (q, k) if c["packed"] else (q.contiguous(), k.contiguous())

        s["q"], s["k"] = rows()
        if c["weights"]:
            s["wq"], s["wk"] = 1.0 + 0.2 * normal(K), 1.0 + 0.2 * normal(K)
        s["freq"] = s["pos"] = None
        if R:
            j = torch.arange(R // 2, device="cuda", dtype=torch.float64)
            if c["at"] == "times":   # angular rates for gaps that differ, in the data's time unit
                s["freq"] = 10.0 ** (1.0 - 4.0 * j / (R // 2))
                s["pos"] = torch.cumsum(gap(B, L), 1)
            else:
                s["freq"] = 10000.0 ** (-2.0 * j / R)
                lo, hi = (1 << 17, 1 << 20) if c["at"] == "far" else (0, 4096)
                first = torch.randint(lo, hi, (B, 1), generator=gen, device="cuda")
                s["pos"] = first + torch.arange(L, device="cuda")
        if c["grad"]:
            s["dq"], s["dk"] = normal(B, L, Hq, K).to(dtype), normal(B, L, Hk, K).to(dtype)
        return s
    rows = (c["S"],) if c["kind"] == "step" else (c["B"], c["L"])
    Hk, Hv, K, V = c["Hk"], c["Hv"], c["K"], c["V"]
    # queries and keys that share a direction within a head
    s = dict(q=normal(*rows, Hk, K).to(dtype),
             k=((normal(*rows, Hk, K) + 0.5 * normal(Hk, K)) * K ** -0.5).to(dtype),
             v=normal(*rows, Hv, V).to(dtype))
    if c["gaps"]:  # irregular time gaps with a rate for each head
        s["g"] = -gap(*rows, 1) * torch.exp(uniform(Hv, lo=math.log(0.5), hi=math.log(5.0)))
    else:          # one decay for each head, memories of 8 to 1000 steps
        s["g"] = (-torch.exp(uniform(Hv, lo=math.log(1e-3), hi=math.log(0.125)))).expand(*rows, Hv)
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
def _linear_plain(q, k, v, g, h0):
    """The chunked form in 32 bits, sums of g in 64.  Within a chunk, with G the sums of g and
    D[t, i] = exp(G_t - G_i): O = e^G Q S + (Q K^T D) V, and the chunk adds K^T (e^(G_end - G) V)
    to the state; the state before chunk n is the sum of what earlier chunks added, decayed by
    what lies between."""
    B, L, Hv, V = v.shape
    K, pad = q.shape[-1], (-L) % CHUNK

    def cut(t):  # [B, L, H, ...] -> [B, Hv, chunk, CHUNK, ...]
        t = torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, pad))
        t = t.reshape(B, -1, CHUNK, *t.shape[2:]).movedim(3, 1)
        return t.repeat_interleave(Hv // t.shape[1], 1) if t.shape[1] != Hv else t.contiguous()

    q, k, v, g = cut(q.float()) * K ** -0.5, cut(k.float()), cut(v.float()), cut(g.double())
    G = torch.cumsum(g, -1)
    keep = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    D = (G[..., :, None] - G[..., None, :]).masked_fill(~keep, -math.inf).float().exp()
    kt = k.transpose(-1, -2).contiguous()
    o = torch.matmul(torch.matmul(q, kt) * D, v)
    eG, end = torch.exp(G.float()), torch.exp((G[..., -1:] - G).float())
    added = torch.matmul(kt * end[..., None, :], v).flatten(-2)      # [B, Hv, chunk, K V]
    E = torch.cumsum(G[..., -1], -1)                                 # sums over whole chunks
    n = E.shape[-1]
    # state after chunk c: of chunk m <= c, exp(E_c - E_m) of what it added
    low = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
    between = (E[..., :, None] - E[..., None, :]).masked_fill(~low, -math.inf).float().exp()
    after = torch.matmul(between, added)
    if h0 is not None:
        after = after + E.float().exp()[..., None] * h0.float().flatten(-2)[:, :, None]
    first = torch.zeros_like(after[:, :, :1]) if h0 is None else h0.float().flatten(-2)[:, :, None]
    S = torch.cat([first, after[:, :, :-1]], 2).unflatten(-1, (K, V))
    o = o + torch.matmul(eG[..., None] * q, S)
    return o.movedim(1, 3).reshape(B, -1, Hv, V)[:, :L], after[:, :, -1].unflatten(-1, (K, V))


def _linear_train_plain(s):
    names = ["q", "k", "v", "g"] + (["h0"] if s["h0"] is not None else [])
    leaves = {n: s[n].float().detach().clone().requires_grad_() for n in names}
    o, S = _linear_plain(*(leaves[n] for n in names[:4]), leaves.get("h0"))
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
    state.addcmul_(k[..., None], v[..., None, :])
    return torch.matmul(q[..., None, :], state)[..., 0, :].to(s["v"].dtype), state


def _pairs(t, R, interleaved):
    """The two members of every rotated pair, and the channels that stay."""
    if interleaved:
        return t[..., 0:R:2], t[..., 1:R:2], t[..., R:]
    return t[..., :R // 2], t[..., R // 2:R], t[..., R:]


def _join(a, b, rest, interleaved):
    both = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([both, rest], -1)


def _qk_plain(x, w, cos, sin, c):
    n = x
    if c["norm"] != "none":
        square = x.square()
        n = x * torch.rsqrt((square.mean(-1, keepdim=True) if c["norm"] == "rms"
                             else square.sum(-1, keepdim=True)) + EPS)
    if w is not None:
        n = n * w
    if not c["R"]:
        return n
    a, b, rest = _pairs(n, c["R"], c["interleaved"])
    return _join(a * cos - b * sin, a * sin + b * cos, rest, c["interleaved"])


def _qk_pass_plain(s):
    c, dtype, cos, sin = s["case"], s["q"].dtype, None, None
    if c["R"]:
        angle = (s["pos"].double()[..., None] * s["freq"])[:, :, None]
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if not c["grad"]:
        return tuple(_qk_plain(s[n].float(), s["w" + n], cos, sin, c).to(dtype) for n in "qk")
    outs, grads, weights = [], [], []
    for n in "qk":
        leaves = [t.detach().requires_grad_() for t in (s[n].float(), s["w" + n]) if t is not None]
        y = _qk_plain(leaves[0], leaves[1] if len(leaves) > 1 else None, cos, sin, c)
        d = torch.autograd.grad(y, leaves, s["d" + n].float())
        outs.append(y.detach().to(dtype))
        grads.append(d[0].to(dtype))
        weights += d[1:]
    return tuple(outs + grads + weights)


# ------------------------------------------------------------------ the framework's operators
def _framework():
    path = os.path.abspath("triton-ssm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tssm
    return tssm


def _run_own(s):
    tssm, c = _framework(), s["case"]
    if c["kind"] == "scan":
        return tssm.linear_attention_forward(s["q"], s["k"], s["v"], s["g"], h0=s["h0"],
                                             return_state=True)
    if c["kind"] == "train":
        o, S = tssm.linear_attention_forward(s["q"], s["k"], s["v"], s["g"], h0=s["h0"],
                                             return_state=True)
        d = tssm.linear_attention_backward(s["q"], s["k"], s["v"], s["g"], s["do"], h0=s["h0"],
                                           dh_last=s["dh"])
        return (o, S) + tuple(t for t in d if t is not None)
    if c["kind"] == "step":
        return tssm.linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"]), s["state"]
    how = dict(norm=c["norm"], eps=EPS, interleaved=c["interleaved"])
    outs = tssm.qk_norm_rotary_forward(s["q"], s["k"], s["pos"], s["freq"], s["wq"], s["wk"],
                                       **how)
    if not c["grad"]:
        return outs
    d = tssm.qk_norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], s["pos"], s["freq"],
                                     s["wq"], s["wk"], **how)
    return tuple(outs) + tuple(t for t in d if t is not None)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "scan":
        o, S = _linear_plain(state["q"], state["k"], state["v"], state["g"], state["h0"])
        return o.to(state["v"].dtype), S
    if kind == "train":
        return _linear_train_plain(state)
    if kind == "step":
        return _step_plain(state)
    return _qk_pass_plain(state)


# ------------------------------------------------------------------ cost
def work(c):
    e = BYTES[c["dtype"]]
    if c["kind"] == "qk":
        n, rows = c["B"] * c["L"] * (c["Hq"] + c["Hk"]) * c["K"], c["B"] * c["L"]
        side = rows * (4 if c["at"] == "times" else 8) + 4 * c["R"] if c["R"] else 0
        side += 8 * c["K"] * (2 if c["grad"] else 1) if c["weights"] else 0
        # x in, y out; with gradients dy in, dx out too (x is the forward's, read once)
        return dict(bytes=(4 if c["grad"] else 2) * n * e + side, flops=(24 if c["grad"] else 8) * n)
    Hk, Hv, K, V = c["Hk"], c["Hv"], c["K"], c["V"]
    rows = c["S"] if c["kind"] == "step" else c["B"] * c["L"]
    decays = rows * Hv * 4 if c["gaps"] else Hv * 4
    each = rows * (2 * Hk * K + 2 * Hv * V) * e + decays             # q, k, v, o, g
    state = (c["S"] if c["kind"] == "step" else c["B"]) * Hv * K * V * 4
    flops = 5 * rows * Hv * K * V
    if c["kind"] == "step":
        return dict(bytes=each + 2 * state, flops=flops)
    if c["kind"] == "scan":
        return dict(bytes=each + state * (2 if c["h0"] else 1), flops=flops)
    # forward as above; its gradients: do in, those of q, k, v and g out (the inputs are the
    # forward's, read once), of the states where they are given
    grads = rows * (2 * Hk * K + 2 * Hv * V) * e + rows * Hv * 4
    return dict(bytes=each + grads + state * (4 if c["h0"] else 1), flops=3 * flops)


# ------------------------------------------------------------------ 64-bit definitions
def _qk_exact(s, c):
    K, R = c["K"], c["R"]
    if c["interleaved"]:
        one, two = list(range(0, R, 2)), list(range(1, R, 2))
    else:
        one, two = list(range(R // 2)), list(range(R // 2, R))
    if R:
        angle = s["pos"].double()[:, :, None, None] * s["freq"].double()
        cos, sin = angle.cos(), angle.sin()
    outs, grads, weights = [], [], []
    for n in "qk":
        x, w = s[n].double(), s["w" + n]
        w = torch.ones(K, dtype=torch.float64, device=x.device) if w is None else w.double()
        mean = 1.0 / K if c["norm"] == "rms" else 1.0
        r = torch.ones_like(x[..., :1]) if c["norm"] == "none" else \
            1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) * mean + EPS)
        y = r * x * w
        if R:
            a, b = y[..., one], y[..., two]
            y[..., one], y[..., two] = a * cos - b * sin, b * cos + a * sin
        outs.append(y)
        if s["d" + n] is None:
            continue
        d = s["d" + n].double()
        if R:
            a, b = d[..., one], d[..., two]
            d[..., one], d[..., two] = a * cos + b * sin, b * cos - a * sin
        weights.append((d * r * x).sum((0, 1, 2)))
        d = d * w
        if c["norm"] != "none":
            d = d - r * r * mean * x * (d * x).sum(-1, keepdim=True)
        grads.append(r * d)
    return tuple(outs + grads + (weights if s["wq"] is not None else []))


def _linear_exact(s, c):
    per = c["Hv"] // c["Hk"]
    q = s["q"].double().repeat_interleave(per, 2) * c["K"] ** -0.5
    k = s["k"].double().repeat_interleave(per, 2)
    v, alpha = s["v"].double(), torch.exp(s["g"].double())
    B, L, Hv, V = v.shape
    S = torch.zeros(B, Hv, c["K"], V, dtype=torch.float64, device=v.device) \
        if s["h0"] is None else s["h0"].double()
    o, train, decayed = torch.empty_like(v), c["kind"] == "train", []
    for t in range(L):
        S = S * alpha[:, t, :, None, None]
        if train:
            decayed.append(S.clone())
        S.addcmul_(k[:, t, :, :, None], v[:, t, :, None, :])
        o[:, t] = torch.matmul(q[:, t, :, None, :], S)[:, :, 0]
    if not train:
        return o, S
    do = s["do"].double()
    dS = torch.zeros_like(S) if s["dh"] is None else s["dh"].double()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    dg = torch.empty_like(alpha)
    for t in range(L - 1, -1, -1):
        before, kt, vt = decayed.pop(), k[:, t, :, :, None], v[:, t, :, None, :]
        dq[:, t] = torch.matmul(before + kt * vt, do[:, t, :, :, None])[..., 0]
        dS = dS + q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = (dS * vt).sum(3)
        dv[:, t] = (dS * kt).sum(2)
        dg[:, t] = (dS * before).sum((2, 3))
        dS = alpha[:, t, :, None, None] * dS
    share = lambda t: t.reshape(B, L, c["Hk"], per, c["K"]).sum(3)  # noqa: E731
    out = (o, S, share(dq) * c["K"] ** -0.5, share(dk), dv, dg)
    return out if s["h0"] is None else out + (dS,)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "qk":
        return _qk_exact(s, case)
    if case["kind"] != "step":
        return _linear_exact(s, case)
    per = case["Hv"] // case["Hk"]
    k = s["k"].double().repeat_interleave(per, 1)
    q = s["q"].double().repeat_interleave(per, 1) * case["K"] ** -0.5
    S = s.pop("state").double().mul_(torch.exp(s["g"].double())[..., None, None])
    S.addcmul_(k[..., None], s["v"].double()[..., None, :])
    return torch.matmul(q[..., None, :], S)[..., 0, :], S
