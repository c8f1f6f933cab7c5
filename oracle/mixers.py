"""Float64 restatements of the operators beside the linear-attention scans: gated delta rule, rotary positions, group norm,
with their gradients.  Token by token and group by group as the definitions have them; numpy only.
"""

from __future__ import annotations

import numpy as np

__all__ = ["delta_rule", "delta_rule_bwd", "rotary", "group_norm", "group_norm_bwd"]


def _per_value_head(t, H):
    return np.repeat(t, H // t.shape[1], axis=1)


def _gates(v, g, beta):
    return (np.zeros(v.shape[:3]) if g is None else g), (np.ones(v.shape[:3]) if beta is None else beta)


def delta_rule(q, k, v, g=None, beta=None, scale=None, state=None):
    """(o, final state) of S_t = e^g S + beta k (v - e^g S^T k)^T, o = scale S^T q; q, k (B, HK, L, dk), v (B, H, L, dv)."""
    B, H, L, dv = v.shape
    dk = q.shape[-1]
    scale = dk ** -0.5 if scale is None else scale
    q, k = _per_value_head(q, H), _per_value_head(k, H)
    g, beta = _gates(v, g, beta)
    S = np.zeros((B, H, dk, dv)) if state is None else state.copy()
    o = np.zeros(v.shape)
    for t in range(L):
        S = S * np.exp(g[:, :, t])[..., None, None]
        kt = k[:, :, t]
        u = beta[:, :, t, None] * (v[:, :, t] - (S * kt[..., None]).sum(-2))
        S = S + kt[..., None] * u[..., None, :]
        o[:, :, t] = scale * (S * q[:, :, t, :, None]).sum(-2)
    return o, S


def delta_rule_bwd(do, q, k, v, g=None, beta=None, scale=None, state=None, d_final=None):
    """(dq, dk, dv, dg, dbeta, d_state) of ``delta_rule``, by its steps taken backwards."""
    B, H, L, dv_ = v.shape
    HK, dk_ = q.shape[1], q.shape[-1]
    scale = dk_ ** -0.5 if scale is None else scale
    qh, kh = _per_value_head(q, H), _per_value_head(k, H)
    g, beta = _gates(v, g, beta)
    S = np.zeros((B, H, dk_, dv_)) if state is None else state.copy()
    before, after, us = [], [], []               # the decayed state, the state, v - S^T k of each token
    for t in range(L):
        S = S * np.exp(g[:, :, t])[..., None, None]
        before.append(S)
        u = v[:, :, t] - (S * kh[:, :, t, :, None]).sum(-2)
        S = S + kh[:, :, t, :, None] * (beta[:, :, t, None] * u)[..., None, :]
        after.append(S)
        us.append(u)
    dS = np.zeros_like(S) if d_final is None else d_final.copy()
    dq, dk, dv = np.zeros(qh.shape), np.zeros(kh.shape), np.zeros(v.shape)
    dg, db = np.zeros(g.shape), np.zeros(g.shape)
    for t in range(L - 1, -1, -1):
        dot, kt, bt = do[:, :, t], kh[:, :, t], beta[:, :, t]
        dq[:, :, t] = scale * (after[t] * dot[..., None, :]).sum(-1)
        dS = dS + scale * qh[:, :, t, :, None] * dot[..., None, :]
        dSu = (dS * us[t][..., None, :]).sum(-1)
        db[:, :, t] = (kt * dSu).sum(-1)
        du = bt[..., None] * (dS * kt[..., None]).sum(-2)
        dv[:, :, t] = du
        dk[:, :, t] = bt[..., None] * dSu - (before[t] * du[..., None, :]).sum(-1)
        dS = dS - kt[..., None] * du[..., None, :]
        dg[:, :, t] = (dS * before[t]).sum((-2, -1))
        dS = dS * np.exp(g[:, :, t])[..., None, None]
    shape = (B, HK, H // HK, L, dk_)
    return dq.reshape(shape).sum(2), dk.reshape(shape).sum(2), dv, dg, db, dS


def rotary(x, inv_freq, positions, interleaved=False, scale=1.0, inverse=False):
    """x (B, H, L, D), positions (L,) or (B, L): pairs of the first 2 n channels turned by positions * inv_freq."""
    n = len(inv_freq)
    pos = np.broadcast_to(positions, (x.shape[0], x.shape[2])).astype(np.float64)
    a = pos[:, None, :, None] * np.asarray(inv_freq, np.float64) * (-1 if inverse else 1)
    first = slice(0, 2 * n, 2) if interleaved else slice(0, n)
    second = slice(1, 2 * n, 2) if interleaved else slice(n, 2 * n)
    y = x.copy()
    y[..., first] = scale * (x[..., first] * np.cos(a) - x[..., second] * np.sin(a))
    y[..., second] = scale * (x[..., first] * np.sin(a) + x[..., second] * np.cos(a))
    return y


def _groups(x, G):
    return x.reshape(x.shape[0], -1, G, x.shape[-1] // G)


def group_norm(x, G, w=None, b=None, eps=1e-5, silu=False):
    """(y, stats) of x (N, ..., C): stats (N, G, 2) = mean, 1 / sqrt(var + eps) over a group's channels and all positions."""
    xg = _groups(x, G)
    mu = xg.mean((1, 3))
    r = 1 / np.sqrt(((xg - mu[:, None, :, None]) ** 2).mean((1, 3)) + eps)
    z = ((xg - mu[:, None, :, None]) * r[:, None, :, None]).reshape(x.shape)
    if w is not None:
        z = z * w
    if b is not None:
        z = z + b
    return z / (1 + np.exp(-z)) if silu else z, np.stack([mu, r], -1)


def group_norm_bwd(dy, x, stats, G, w=None, b=None, silu=False):
    """(dx, dw, db) of ``group_norm``."""
    mu, r = stats[:, None, :, :1], stats[:, None, :, 1:]
    c = ((_groups(x, G) - mu) * r)
    cx = c.reshape(x.shape)
    dz = dy
    if silu:
        z = cx if w is None else cx * w
        z = z if b is None else z + b
        s = 1 / (1 + np.exp(-z))
        dz = dy * s * (1 + z * (1 - s))
    gg = _groups(dz if w is None else dz * w, G)
    dx = r * (gg - gg.mean((1, 3), keepdims=True) - c * (gg * c).mean((1, 3), keepdims=True))
    axes = tuple(range(x.ndim - 1))
    return dx.reshape(x.shape), (dz * cx).sum(axes), dz.sum(axes)
