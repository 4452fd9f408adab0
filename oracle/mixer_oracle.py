"""float64 restatement of the gated delta rule and of the group norm with an
activation, with their gradients, step by step from the definitions (numpy;
test infrastructure only)."""
from __future__ import annotations

import numpy as np


def _heads(t, Hv):
    return np.repeat(t, Hv // t.shape[-2], axis=-2)


def delta_forward(q, k, v, g, beta, scale=None, h0=None):
    """q, k [B,L,Hk,K], v [B,L,Hv,V], g, beta [B,L,Hv], h0 [B,Hv,K,V] or None;
    returns o [B,L,Hv,V] and the final state."""
    B, L, Hv, V = v.shape
    K = q.shape[-1]
    scale = K ** -0.5 if scale is None else scale
    qe, ke = _heads(q, Hv) * scale, _heads(k, Hv)
    S = np.zeros((B, Hv, K, V)) if h0 is None else h0.copy()
    o = np.empty_like(v)
    for t in range(L):
        S = S * np.exp(g[:, t])[..., None, None]
        u = beta[:, t][..., None] * (v[:, t] - np.einsum("bhk,bhkv->bhv", ke[:, t], S))
        S = S + ke[:, t][..., :, None] * u[..., None, :]
        o[:, t] = np.einsum("bhk,bhkv->bhv", qe[:, t], S)
    return o, S


def delta_backward(q, k, v, g, beta, do, scale=None, h0=None, dh_last=None):
    """Gradients (dq, dk, dv, dg, dbeta, dh0) of sum(o do) + sum(S_L dh_last)."""
    B, L, Hv, V = v.shape
    Hk, K = q.shape[-2:]
    scale = K ** -0.5 if scale is None else scale
    qe, ke = _heads(q, Hv) * scale, _heads(k, Hv)
    S = np.zeros((B, Hv, K, V)) if h0 is None else h0.copy()
    decayed, after = [], []           # e^g S_{t-1} and S_t
    us = np.empty_like(v)
    for t in range(L):
        S = S * np.exp(g[:, t])[..., None, None]
        decayed.append(S)
        us[:, t] = beta[:, t][..., None] * (v[:, t] - np.einsum("bhk,bhkv->bhv", ke[:, t], S))
        S = S + ke[:, t][..., :, None] * us[:, t][..., None, :]
        after.append(S)
    dS = np.zeros((B, Hv, K, V)) if dh_last is None else dh_last.copy()
    dq, dk, dv = np.empty_like(qe), np.empty_like(ke), np.empty_like(v)
    dg, dbeta = np.empty_like(g), np.empty_like(beta)
    for t in range(L - 1, -1, -1):
        kt, bt, R = ke[:, t], beta[:, t][..., None], decayed[t]
        dq[:, t] = np.einsum("bhkv,bhv->bhk", after[t], do[:, t])
        dS = dS + qe[:, t][..., :, None] * do[:, t][..., None, :]
        du = np.einsum("bhk,bhkv->bhv", kt, dS)
        gap = v[:, t] - np.einsum("bhk,bhkv->bhv", kt, R)
        dv[:, t] = bt * du
        dbeta[:, t] = (du * gap).sum(-1)
        dk[:, t] = np.einsum("bhkv,bhv->bhk", dS, us[:, t]) \
            - np.einsum("bhkv,bhv->bhk", R, bt * du)
        dR = dS - kt[..., :, None] * (bt * du)[..., None, :]
        dg[:, t] = (dR * R).sum((-2, -1))
        dS = dR * np.exp(g[:, t])[..., None, None]

    def shared(t):
        return t.reshape(B, L, Hk, Hv // Hk, K).sum(3)

    return shared(dq) * scale, shared(dk), dv, dg, dbeta, dS


def _act(t, act):
    """act(t) and its derivative."""
    if act == "none":
        return t, np.ones_like(t)
    s = 1.0 / (1.0 + np.exp(-t))
    return t * s, s + t * s * (1.0 - s)


def group_norm(x, groups, w=None, b=None, gate=None, act="silu", eps=1e-5, dy=None):
    """x [N,S,C]; returns y, mean, rstd and, with dy, also dx, dw, db, dgate."""
    N, S, C = x.shape
    xg = x.reshape(N, S, groups, C // groups)
    mean = xg.mean((1, 3))
    rstd = 1.0 / np.sqrt(((xg - mean[:, None, :, None]) ** 2).mean((1, 3)) + eps)
    xhat = ((xg - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(N, S, C)
    w = np.ones(C) if w is None else w
    z = xhat * w + (0.0 if b is None else b)
    f, df = _act(z if gate is None else gate, act)
    y = f if gate is None else z * f
    if dy is None:
        return y, mean, rstd
    dz = dy * df if gate is None else dy * f
    e = (dz * w).reshape(xg.shape)
    xh = xhat.reshape(xg.shape)
    m1 = e.mean((1, 3), keepdims=True)
    m2 = (e * xh).mean((1, 3), keepdims=True)
    dx = (rstd[:, None, :, None] * (e - m1 - xh * m2)).reshape(N, S, C)
    dgate = None if gate is None else dy * z * df
    return y, mean, rstd, dx, (dz * xhat).sum((0, 1)), dz.sum((0, 1)), dgate
