"""The float64 oracle of the gated delta rule, rotary positions and group norm on the CPU: gradients against central
differences, and properties that the definitions imply."""

import math

import numpy as np
import pytest
import torch

import mamformer_amd as mh
from oracle import mixers as mx
from tests.test_oracle_tokens import diff

TOL = 1e-8                                       # as for the token operators: central differences of step 1e-5


def delta_inputs(rng, B=1, H=2, HK=1, L=5, dk=3, dv=4):
    q, k = rng.standard_normal((2, B, HK, L, dk))
    k /= np.linalg.norm(k, axis=-1, keepdims=True)
    return [q, k, rng.standard_normal((B, H, L, dv)), -rng.random((B, H, L)), rng.random((B, H, L)),
            rng.standard_normal((B, H, dk, dv))]


def test_delta_gradient(rng):
    x = delta_inputs(rng)
    do, d_final = rng.standard_normal(x[2].shape), rng.standard_normal(x[5].shape)
    grads = mx.delta_rule_bwd(do, *x[:5], 0.7, x[5], d_final)

    for i, grad in enumerate(grads):
        def f(v, j):
            y = [v if m == i else x[m] for m in range(6)]
            return mx.delta_rule(*y[:5], 0.7, y[5])[j]
        want = diff(lambda v: f(v, 0), x[i], do) + diff(lambda v: f(v, 1), x[i], d_final)
        np.testing.assert_allclose(grad, want, atol=TOL)


def test_delta_pieces_and_padding(rng):
    q, k, v, g, beta, s = delta_inputs(rng, L=9)
    o, final = mx.delta_rule(q, k, v, g, beta, None, s)
    o1, mid = mx.delta_rule(q[:, :, :4], k[:, :, :4], v[:, :, :4], g[:, :, :4], beta[:, :, :4], None, s)
    o2, end = mx.delta_rule(q[:, :, 4:], k[:, :, 4:], v[:, :, 4:], g[:, :, 4:], beta[:, :, 4:], None, mid)
    np.testing.assert_allclose(np.concatenate([o1, o2], 2), o, atol=1e-12)
    np.testing.assert_allclose(end, final, atol=1e-12)
    g[:, :, 4:], beta[:, :, 4:] = 0, 0           # tokens that change nothing
    np.testing.assert_allclose(mx.delta_rule(q, k, v, g, beta, None, s)[1], mid, atol=1e-12)
    # beta = 1 and keys of norm 1: the state answers a key with the last value written to it
    _, last = mx.delta_rule(q, k, v, None, None, None, s)
    np.testing.assert_allclose((last[0, 0] * k[0, 0, -1][:, None]).sum(0), v[0, 0, -1], atol=1e-12)


def test_delta_is_the_gradient_step(rng):
    """Without a decay a token takes a step of size beta down the gradient of |S^T k - v|^2 / 2."""
    q, k, v, _, beta, s = delta_inputs(rng, L=1, H=1)
    _, S = mx.delta_rule(q, k, v, None, beta, None, s)
    kt, vt = k[0, 0, 0], v[0, 0, 0]
    np.testing.assert_allclose(S[0, 0], s[0, 0] - beta[0, 0, 0] * np.outer(kt, s[0, 0].T @ kt - vt), atol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(rng, interleaved):
    x, dy = rng.standard_normal((2, 2, 3, 4, 7))
    f, pos = np.array([1.0, 0.3]), np.array([[0, 1, -5, 100], [3, 3, 2, 10 ** 6]])
    y = mx.rotary(x, f, pos, interleaved, 1.5)
    back = mx.rotary(y, f, pos, interleaved, 1 / 1.5, inverse=True)
    np.testing.assert_allclose(back, np.where(np.arange(7) < 4, x, x), atol=1e-9)
    assert (y[..., 4:] == x[..., 4:]).all()
    np.testing.assert_allclose(mx.rotary(dy, f, pos, interleaved, 1.5, True),
                               diff(lambda v: mx.rotary(v, f, pos, interleaved, 1.5), x, dy), atol=TOL)
    # the products of turned queries and keys depend on the distance alone
    a, b = rng.standard_normal((2, 1, 1, 1, 4))
    p = [(mx.rotary(a, f, np.array([i]), interleaved) * mx.rotary(b, f, np.array([i + 3]), interleaved)).sum() for i in (0, 9)]
    assert abs(p[0] - p[1]) < 1e-12


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("affine", [False, True])
def test_group_norm_gradient(rng, silu, affine):
    x, dy = rng.standard_normal((2, 2, 3, 2, 6))
    w, b = rng.standard_normal((2, 6)) if affine else (None, None)
    y, stats = mx.group_norm(x, 3, w, b, 1e-3, silu)
    assert y.shape == x.shape and stats.shape == (2, 3, 2)
    dx, dw, db = mx.group_norm_bwd(dy, x, stats, 3, w, b, silu)
    np.testing.assert_allclose(dx, diff(lambda v: mx.group_norm(v, 3, w, b, 1e-3, silu)[0], x, dy), atol=TOL)
    if affine:
        np.testing.assert_allclose(dw, diff(lambda v: mx.group_norm(x, 3, v, b, 1e-3, silu)[0], w, dy), atol=TOL)
        np.testing.assert_allclose(db, diff(lambda v: mx.group_norm(x, 3, w, v, 1e-3, silu)[0], b, dy), atol=TOL)


def test_group_norm_is_torchs(rng):
    x = rng.standard_normal((2, 5, 6))
    w, b = rng.standard_normal((2, 6))
    t = [torch.as_tensor(v) for v in (x.transpose(0, 2, 1).copy(), w, b)]
    want = torch.nn.functional.group_norm(t[0], 2, t[1], t[2], 1e-5).numpy().transpose(0, 2, 1)
    np.testing.assert_allclose(mx.group_norm(x, 2, w, b)[0], want, atol=1e-12)


def test_rotary_frequencies():
    f, s = mh.rotary_frequencies(64, 1e4, device="cpu")
    assert f.dtype is torch.float64 and s == 1.0
    np.testing.assert_allclose(f, 1e4 ** (-np.arange(0, 64, 2) / 64), rtol=1e-14)
    np.testing.assert_allclose(mh.rotary_frequencies(64, 1e4, scaling="linear", factor=4, device="cpu")[0], f / 4, rtol=1e-14)
    n, _ = mh.rotary_frequencies(64, 1e4, scaling="ntk", factor=4, device="cpu")
    assert n[0] == 1 and abs(n[-1] / (f[-1] / 4) - 1) < 1e-12        # the slowest wave is 4 times as long
    y, s = mh.rotary_frequencies(64, 1e4, scaling="yarn", factor=4, original_length=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert abs(s - (0.1 * math.log(4) + 1)) < 1e-12
    np.testing.assert_allclose(y[turns > 40], f[turns > 40], rtol=1e-12)
    np.testing.assert_allclose(y[turns < 0.7], f[turns < 0.7] / 4, rtol=1e-12)
    assert ((y <= f) & (y >= f / 4)).all() and (y[1:] <= y[:-1]).all()
    for kw in (dict(dim=63), dict(dim=0), dict(dim=64, scaling="cubic"), dict(dim=64, factor=0.5), dict(dim=64, base=0.0),
               dict(dim=64, scaling="yarn", factor=2.0), dict(dim=64, scaling="yarn", original_length=64, beta_fast=1.0)):
        with pytest.raises(ValueError):
            mh.rotary_frequencies(kw.pop("dim"), kw.pop("base", 1e4), device="cpu", **kw)
