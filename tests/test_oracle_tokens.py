"""The float64 oracle of the token operators on the CPU: its gradients against central differences, the 8-bit form's
bounds and edges, and the rows that a mask leaves empty."""

import numpy as np
import pytest

from oracle import tokens as tk

EPS = 1e-5            # step of the central differences: truncation O(1e-10), rounding 1e-16 / 1e-5 = 1e-11
TOL = 1e-8


def diff(f, x, dy):
    """Gradient of sum(dy * f(x)) by central differences."""
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        a, b = x.copy(), x.copy()
        a[i] += EPS
        b[i] -= EPS
        g[i] = ((f(a) - f(b)) * dy).sum() / (2 * EPS)
    return g


def test_embedding_gradient(rng):
    ids = np.array([[3, 0, 3], [-1, 7, 2]])
    W, dy = rng.standard_normal((5, 4)), rng.standard_normal((2, 3, 4))
    want = diff(lambda w: tk.embedding(ids, w, 1.7), W, dy)
    np.testing.assert_allclose(tk.embedding_bwd(dy, ids, 5, 1.7), want, atol=TOL)
    pad = tk.embedding_bwd(dy, ids, 5, 1.7, padding_idx=3)
    assert (pad[3] == 0).all() and np.allclose(np.delete(pad, 3, 0), np.delete(want, 3, 0), atol=TOL)


def test_layer_norm_gradient(rng):
    h, dy, d_h = rng.standard_normal((3, 3, 11))
    w, b = rng.standard_normal((2, 11))
    _, stats = tk.layer_norm(h, w, b)
    dx, dw, db = tk.layer_norm_bwd(dy, h, stats, w, d_h)
    np.testing.assert_allclose(dx, diff(lambda v: tk.layer_norm(v, w, b)[0], h, dy) + d_h, atol=TOL)
    np.testing.assert_allclose(dw, diff(lambda v: tk.layer_norm(h, v, b)[0], w, dy), atol=TOL)
    np.testing.assert_allclose(db, diff(lambda v: tk.layer_norm(h, w, v)[0], b, dy), atol=TOL)


@pytest.mark.parametrize("masked", [False, True])
def test_logprob_gradient(rng, masked):
    z = 2 * rng.standard_normal((4, 9))
    if masked:
        z[:, 5] = -np.inf
    t = np.array([2, -100, 8, 11])
    d_lp, d_ent = rng.standard_normal((2, 4))

    def f(v):
        lp, ent, *_ = tk.token_logprobs(v, t, 0.7)
        return np.stack([lp, ent])

    _, ent, _, _, lnp = tk.token_logprobs(z, t, 0.7)
    got = tk.token_logprobs_bwd(lnp, ent, t, d_lp, d_ent, 0.7)
    want = diff(f, z, np.stack([d_lp, d_ent]))
    np.testing.assert_allclose(got, np.where(np.isfinite(z), want, 0.0), atol=TOL)


def test_logprob_ranks_and_empty_rows():
    z = np.array([[1.0, 3.0, 3.0, np.nan], [-np.inf] * 4, [2.0, -np.inf, 5.0, 5.0]])
    lp, ent, ids, alt, _ = tk.token_logprobs(z, np.array([0, 1, 0]), top=3)
    assert ids.tolist() == [[3, 1, 2], [0, 1, 2], [2, 3, 0]]
    assert np.isnan(lp[0]) and lp[1] == -np.inf and ent[1] == 0 and (alt[1] == -np.inf).all()


def test_pack_edges():
    x = np.zeros((7, 70))
    x[1] = 127.0
    x[2] = 127.5                                   # above 127: the next exponent, where it is a tie (63.75 -> 64)
    x[3] = 2.0 ** -140                             # below the least exponent
    x[4, 3] = np.inf
    x[5, 66] = np.nan
    x[6] = np.linspace(-1e30, 3e30, 70)
    codes, exps = tk.pack(x)
    back = tk.unpack(codes, exps, 70)
    assert (back[0] == 0).all() and (exps[0] == 0).all() and (back[1] == 127).all() and (back[2] == 128).all()
    assert (back[3] == 0).all()
    assert np.isnan(back[4, :64]).all() and (back[4, 64:] == 0).all()
    assert (back[5, :64] == 0).all() and np.isnan(back[5, 64:]).all()
    for g in (slice(0, 64), slice(64, 70)):
        assert np.abs(back[6, g] - x[6, g]).max() <= np.abs(x[6, g]).max() / 127
