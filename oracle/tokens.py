"""Float64 restatements of the operators at the ends of a language model: token table, layer norm, 8-bit activations and
log probabilities, with their gradients.  Loops and sums as the definitions have them; numpy only.
"""

from __future__ import annotations

import numpy as np

__all__ = ["embedding", "embedding_bwd", "layer_norm", "layer_norm_bwd", "pack", "unpack", "token_logprobs",
           "token_logprobs_bwd"]


def embedding(ids, W, scale=1.0):
    out = np.zeros((*ids.shape, W.shape[1]))
    for t in np.ndindex(*ids.shape):
        if 0 <= ids[t] < W.shape[0]:
            out[t] = scale * W[ids[t]]
    return out


def embedding_bwd(dy, ids, V, scale=1.0, padding_idx=None):
    dW = np.zeros((V, dy.shape[-1]))
    for t in np.ndindex(*ids.shape):
        if 0 <= ids[t] < V and ids[t] != padding_idx:
            dW[ids[t]] += scale * dy[t]
    return dW


def layer_norm(h, w=None, b=None, eps=1e-5):
    """(y, stats) of rows h (R, D), stats (R, 2) = mean, 1 / sqrt(var + eps)."""
    mu = h.mean(-1)
    r = 1 / np.sqrt(((h - mu[:, None]) ** 2).mean(-1) + eps)
    y = (h - mu[:, None]) * r[:, None]
    if w is not None:
        y = y * w
    if b is not None:
        y = y + b
    return y, np.stack([mu, r], -1)


def layer_norm_bwd(dy, h, stats, w=None, d_h=None):
    """(dx, dw, db); h may differ from the rows that stats are of (their 8-bit form)."""
    mu, r = stats[:, :1], stats[:, 1:]
    c = (h - mu) * r
    g = dy if w is None else dy * w
    dx = r * (g - g.mean(-1, keepdims=True) - c * (g * c).mean(-1, keepdims=True))
    if d_h is not None:
        dx = dx + d_h
    return dx, (dy * c).sum(0), dy.sum(0)


def pack(x):
    """Rows x (R, D) -> codes (R, dp) int8 and exponent bytes (R, dp / 64) uint8, dp = D up to a multiple of 64."""
    R, D = x.shape
    dp = (D + 63) // 64 * 64
    codes, exps = np.zeros((R, dp), np.int8), np.zeros((R, dp // 64), np.uint8)
    for r in range(R):
        for g in range(dp // 64):
            v = x[r, 64 * g:min(D, 64 * g + 64)]
            if not np.isfinite(v).all():
                exps[r, g] = 255
                continue
            e = -132
            while np.abs(v).max() > 127 * 2.0 ** e:
                e += 1
            exps[r, g] = e + 132
            codes[r, 64 * g:64 * g + v.size] = np.rint(v / 2.0 ** e)           # rint: to nearest even
    return codes, exps


def unpack(codes, exps, D):
    e = np.repeat(exps.astype(np.int64), 64, -1)
    return np.where(e == 255, np.nan, codes * 2.0 ** (e - 132))[:, :D]


def token_logprobs(logits, targets, temperature=1.0, top=0, ignore_index=-100):
    """(logprobs, entropy, top_ids, top_logprobs, lnp): lnp (R, V) the log probabilities of every token."""
    R, V = logits.shape
    lnp = np.full((R, V), -np.inf)
    lp, ent = np.zeros(R), np.zeros(R)
    ids, alt = np.zeros((R, top), np.int64), np.zeros((R, top))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        for r in range(R):
            z = logits[r] / temperature
            if not (z == -np.inf).all():
                m = z.max()
                lnp[r] = z - m - np.log(np.exp(z - m).sum())
                p = np.exp(lnp[r])
                ent[r] = -np.where(p == 0, 0.0, p * lnp[r]).sum()
            if 0 <= targets[r] < V and targets[r] != ignore_index:
                lp[r] = lnp[r, targets[r]]
            if top:
                v = np.where(np.isnan(logits[r]), np.inf, logits[r])
                nan = np.isnan(logits[r])
                ids[r] = np.lexsort((np.arange(V), -v, ~nan))[:top]
                alt[r] = lnp[r, ids[r]]
    return lp, ent, ids, alt, lnp


def token_logprobs_bwd(lnp, ent, targets, d_lp=None, d_ent=None, temperature=1.0, ignore_index=-100):
    R, V = lnp.shape
    d = np.zeros((R, V))
    for r in range(R):
        keep = 0 <= targets[r] < V and targets[r] != ignore_index
        g = d_lp[r] if d_lp is not None and keep else 0.0
        h = d_ent[r] if d_ent is not None else 0.0
        if (g == 0 and h == 0) or (lnp[r] == -np.inf).all():
            continue
        p = np.exp(lnp[r])
        d[r] = -g * p - h * np.where(p == 0, 0.0, p * (lnp[r] + ent[r]))
        if keep:
            d[r, targets[r]] += g
        d[r] /= temperature
    return d
