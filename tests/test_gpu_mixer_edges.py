"""Gated delta rule, rotary positions and group norm on the GPU where results cancel, variants meet and sizes end, against the
float64 oracle; tolerances are counted as in test_gpu_mixer_ops."""

import numpy as np
import pytest
import torch

import mamformer_amd as mh
from oracle import mixers as mx
from tests.gpu_helpers import host, say
from tests.test_gpu_mixer_ops import compare, delta_inputs

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def both(a, dtype):
    """a rounded to dtype: (float64 array, GPU tensor)."""
    t = torch.as_tensor(np.asarray(a)).to(dtype)
    return t.double().numpy(), t.cuda()


def rows_within(name, out, ref, enter, k):
    """Rows' errors in norm against half a step of the result and k 2^-20 of the norm that enters, a number."""
    half = torch.finfo(out.dtype).eps / 2
    o = host(out)
    assert o.shape == ref.shape and np.isfinite(o).all(), name
    tol = half * np.linalg.norm(ref, axis=-1) + k * 2.0 ** -20 * enter
    worst = (np.linalg.norm(o - ref, axis=-1) / tol).max()
    say(f"{name}: error at most {worst:.3f} of the tolerance")
    assert worst <= 1, f"{name}: {worst:.3f} times the tolerance"


# ------------------------------------------------------------------------------------------------ results that cancel
# o, dq and dk are sums whose terms may cancel far below what enters them.  Their error before the one rounding is 2^-20 of
# the norms that enter for each product (12 on the way to o, 24 to a gradient), whatever is left of the sum.

def cancelling(rng, *shape):
    """(r, -r (1 + about 2^-8)) along a new first axis of 2, in fp32."""
    r = rng.standard_normal(shape).astype(np.float32)
    return np.stack([r, -r * (1 + 2.0 ** -8 * rng.uniform(0.5, 1, shape))]).astype(np.float32)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("H,L,dk,dv", [(4, 5, 2, 64), (3, 130, 70, 16), (40, 70, 2, 130), (2, 1500, 2, 64)])
def test_delta_of_a_state_that_cancels(dtype, H, L, dk, dv):
    """o = scale q^T S with two rows of S that nearly cancel (beta = 0: no token writes)."""
    rng = np.random.default_rng(L)
    s = np.zeros((1, H, dk, dv), np.float32)
    s[:, :, 0], s[:, :, -1] = cancelling(rng, 1, H, dv)
    q = np.zeros((1, H, L, dk))
    q[..., 0] = q[..., -1] = rng.uniform(1, 2, (1, H, L))
    (qh, qg), (kh, kg), (vh, vg) = both(q, dtype), both(rng.standard_normal(q.shape) / dk ** 0.5, dtype), both(rng.standard_normal((1, H, L, dv)), dtype)
    (sh, sg), (bh, bg) = both(s, F32), both(np.zeros((1, H, L)), F32)
    say(f"state that cancels H={H} L={L} {dk} {dv} {dtype}")
    o = mh.gated_delta_rule(qg, kg, vg, None, bg, initial_state=sg)
    ref, _ = mx.delta_rule(qh, kh, vh, None, bh, None, sh)
    enter = dk ** -0.5 * np.linalg.norm(qh, axis=-1).max() * np.linalg.norm(sh, axis=(-2, -1)).max()
    rows_within("o", o, ref, enter, 12 * np.sqrt((L + 63) // 64))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("H,dv,given", [(8, 64, "beta"), (8, 64, "state"), (40, 130, "beta"), (40, 130, "state")])
def test_delta_of_corrections_that_cancel(dtype, H, dv, given):
    """o of a second token whose two terms nearly cancel: equal values with nearly equal beta, or what two rows of the state
    are corrected by.  Keys are the unit vectors, so that each token's correction is v less its row of the state."""
    rng = np.random.default_rng(dv)
    k, q = np.broadcast_to(np.eye(2), (1, H, 2, 2)), np.ones((1, H, 2, 2))
    v, beta, s = np.zeros((1, H, 2, dv)), np.ones((1, H, 2)), np.zeros((1, H, 2, dv))
    if given == "beta":
        v[:, :, 0] = rng.standard_normal((1, H, dv))
        v[:, :, 1] = -v[:, :, 0]
        beta[..., 0] = rng.uniform(0.5, 1, (1, H))
        beta[..., 1] = beta[..., 0] * (1 + 2.0 ** -8 * rng.uniform(0.5, 1, (1, H)))
    else:
        s[:, :, 0], s[:, :, 1] = cancelling(rng, 1, H, dv)
        q[:, :, 0] = 0.5
    (qh, qg), (kh, kg), (vh, vg), (bh, bg), (sh, sg) = (both(a, t) for a, t in ((q, dtype), (k, dtype), (v, dtype), (beta, F32), (s, F32)))
    say(f"corrections that cancel, {given}, H={H} {dv} {dtype}")
    o = mh.gated_delta_rule(qg, kg, vg, None, bg, scale=1.0, initial_state=sg)
    ref, _ = mx.delta_rule(qh, kh, vh, None, bh, 1.0, sh)
    enter = np.sqrt(2) * (np.linalg.norm(sh, axis=(-2, -1)).max() + np.linalg.norm(vh, axis=(-2, -1)).max())
    rows_within("o", o, ref, enter, 12)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("H,dv", [(16, 64), (40, 130)])
def test_delta_gradients_that_cancel(dtype, H, dv):
    """dq and dk whose pair terms nearly cancel.  Three tokens of one key: values v0 and -v0 written with nearly the same small
    beta, and a third that reads and corrects nearly nothing, whose dq and dk are the sum of both; and a key that two opposite
    queries read under nearly the same decay, whose dk is the sum of theirs."""
    rng = np.random.default_rng(dv)
    v0, one = rng.standard_normal((1, H, dv)), np.ones((1, H))
    v, do, g, beta = np.zeros((1, H, 3, dv)), np.zeros((1, H, 3, dv)), np.zeros((1, H, 3)), np.zeros((1, H, 3))
    v[:, :, 0], v[:, :, 1], do[:, :, 2] = v0, -v0, v0
    beta[..., 0] = 2.0 ** -8 * rng.uniform(0.5, 1, (1, H))
    beta[..., 1] = beta[..., 0] * (1 + 2.0 ** -8 * rng.uniform(0.5, 1, (1, H)))
    beta[..., 2] = 1
    key = np.stack([0.6 * one, 0.8 * one], -1)
    k = np.stack([key] * 3, 2)
    q = np.zeros_like(k)
    q[:, :, 2] = key
    args = [both(a, t) for a, t in ((do, dtype), (q, dtype), (k, dtype), (v, dtype), (g, F32), (beta, F32))]
    say(f"dq and dk of values that cancel H={H} {dv} {dtype}")
    got = mh.gated_delta_rule_bwd(*(a for _, a in args), scale=1.0)
    ref = mx.delta_rule_bwd(*(a for a, _ in args), 1.0)
    # each of the two terms: do . v0 times beta, by a key of norm 1
    enter = 2 * (args[0][0] ** 2).sum(-1).max() * args[5][0][..., :2].max()
    rows_within("dq", got[0][:, :, 2:], ref[0][:, :, 2:], enter, 24)
    rows_within("dk", got[1][:, :, 2:], ref[1][:, :, 2:], enter, 24)

    v, do, beta = v * 0, do * 0, beta * 0
    v[:, :, 0] = do[:, :, 1] = do[:, :, 2] = v0
    beta[..., 0] = rng.uniform(0.5, 1, (1, H))
    g[..., 1:] = -2.0 ** -8 * rng.uniform(0.5, 1, (1, H, 2))
    k, q = np.zeros_like(k), np.zeros_like(q)
    k[..., 0] = 1
    q[:, :, 1, 1], q[:, :, 2, 1] = 1, -1
    args = [both(a, t) for a, t in ((do, dtype), (q, dtype), (k, dtype), (v, dtype), (g, F32), (beta, F32))]
    say("dk of queries that cancel")
    got = mh.gated_delta_rule_bwd(*(a for _, a in args), scale=1.0)
    ref = mx.delta_rule_bwd(*(a for a, _ in args), 1.0)
    enter = 2 * (args[0][0] ** 2).sum(-1).max() * args[5][0].max()
    rows_within("dk", got[1][:, :, :1], ref[1][:, :, :1], enter, 24)


# ------------------------------------------------------------------------------------------------ two pairs a workgroup
# bf16 scans take two pairs of waves a workgroup, 32 columns of v, where batch * heads * segments * ceil(dv / 16) passes 256.

@pytest.mark.parametrize("B,H,HK,L,dk,dv,opts", [
    (4, 24, 12, 70, 40, 37, {}),                 # 288 blocks, three a head: a workgroup's second pair without columns
    (2, 15, 5, 131, 100, 130, {}),               # 270, nine a head, the last of two columns
    (3, 30, 30, 64, 128, 48, dict(state=False)), (11, 12, 6, 1, 64, 31, {}), (5, 20, 4, 65, 17, 33, dict(gates=False)),
    (1, 260, 26, 200, 24, 8, dict(decay=3.0)),
    (1, 8, 4, 2100, 16, 130, {}),                # in segments as well
])
def test_delta_of_many_columns(B, H, HK, L, dk, dv, opts):
    say(f"delta {B} {H} {HK} {L} {dk} {dv} {opts}")
    compare(*delta_inputs(B, H, HK, L, dk, dv, BF, **opts))


@pytest.mark.parametrize("B,H,HK,L,dk,dv", [(4, 24, 12, 70, 40, 37), (3, 20, 10, 190, 100, 130), (5, 20, 20, 129, 64, 48)])
def test_delta_of_many_columns_is_that_of_few(B, H, HK, L, dk, dv):
    """The last sequence of a batch alone, which takes one pair a workgroup: the same bits, recomputed or kept."""
    _, t = delta_inputs(B, H, HK, L, dk, dv, BF)
    last = [a[-1:] for a in t]
    do, df = torch.randn_like(t[2]), torch.randn_like(t[5])
    say(f"last of {B} {H} {HK} {L} {dk} {dv}")

    def run(t, do, df, recompute):
        leaves = [a.detach().requires_grad_(True) for a in t]
        out = mh.gated_delta_rule(*leaves[:5], initial_state=leaves[5], return_final_state=True, recompute=recompute)
        return [a.detach() for a in (*out, *torch.autograd.grad(out, leaves, (do, df)))]

    for recompute in (False, True):
        for a, b in zip(run(t, do, df, recompute), run(last, do[-1:], df[-1:], recompute)):
            assert torch.equal(a[-1:], b)


# ------------------------------------------------------------------------------------------------ far from one

def scaled(t, x, i, size):
    t[i] = t[i] * size
    x[i] = t[i].double().cpu().numpy()


def sized(name, out, ref, k):
    """rows_within in units of the largest of ref (squares of its values may leave fp32's range); k products, and the result's
    rounding in its type."""
    size = np.abs(ref).max()
    half = 2.0 ** 20 * torch.finfo(out.dtype).eps / 2
    rows_within(name, out.double() / size, ref / size, np.linalg.norm(ref / size, axis=-1).max(), k + half)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("values", [1e-34, 1e-30, 1e-18, 1e12, 1e30])
@pytest.mark.parametrize("L", [130, 1100])
def test_delta_far_from_one(dtype, values, L):
    """Values and states far outside fp16's range and near the ends of fp32's: no power of two on the way leaves it before."""
    x, t = delta_inputs(1, 4, 2, L, 32, 24, dtype)
    for i in (2, 5):
        scaled(t, x, i, values)
    say(f"values of {values}, L={L} {dtype}")
    o, s = mh.gated_delta_rule(*t[:5], initial_state=t[5], return_final_state=True)
    ro, rs = mx.delta_rule(*x[:5], None, x[5])
    sized("o", o, ro, 12 * np.sqrt((L + 63) // 64))
    sized("state", s, rs, 12 * np.sqrt((L + 63) // 64))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("values,grads", [(1e-18, 1e12), (1e12, 1e-18), (1e12, 1e12), (1e-9, 1e-18), (1e-18, 1e-18),
                                          (1e-30, 1.0), (1.0, 1e-30), (1.0, 1e-33), (1e-20, 1e-14), (1e18, 1e17)])
def test_delta_gradients_far_from_one(dtype, values, grads):
    """The same of gradients, whose products with the values stay within fp32's normal range."""
    x, t = delta_inputs(1, 4, 2, 130, 32, 24, dtype)
    for i in (2, 5):
        scaled(t, x, i, values)
    do, df = torch.randn_like(t[2]) * grads, torch.randn_like(t[5]) * grads
    say(f"values of {values}, gradients of {grads}, {dtype}")
    got = mh.gated_delta_rule_bwd(do, *t[:5], initial_state=t[5], d_final_state=df)
    ref = mx.delta_rule_bwd(host(do), *x[:5], None, x[5], host(df))
    for name, a, r in zip(("dq", "dk", "dv", "dg", "dbeta", "d_state"), got, ref):
        sized(name, *((a, r) if a.dim() == 4 else (a[:, :, None], r[:, :, None])), 24 * np.sqrt(3))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("L", [20, 130, 1500])
def test_delta_gradients_of_zeros(dtype, L):
    """Nothing written and no state, or nothing that comes back: what does not depend on it has its gradient, all else is 0."""
    x, t = delta_inputs(1, 4, 2, L, 32, 24, dtype)
    do, zero = torch.randn_like(t[2]), torch.zeros_like(t[2])
    say(f"zeros L={L} {dtype}")
    for state in (None, torch.zeros_like(t[5])):
        xs = None if state is None else host(state)
        got = mh.gated_delta_rule_bwd(do, *t[:2], zero, *t[3:5], initial_state=state)
        ref = mx.delta_rule_bwd(host(do), *x[:2], host(zero), *x[3:5], None, xs)
        for name, a, r in zip(("dq", "dk", "dv", "dg", "dbeta", "d_state"), got, ref):
            if name in ("dv", "d_state"):
                if a is not None:
                    rows_within(name, a, r, np.linalg.norm(r, axis=-1).max(), 24 * np.sqrt((L + 63) // 64))
            else:
                assert (a == 0).all(), name
        for a in mh.gated_delta_rule_bwd(zero, *t[:5], initial_state=t[5], d_final_state=state):
            assert (a == 0).all()
    o, s = mh.gated_delta_rule(*t[:2], zero, *t[3:5], return_final_state=True)
    assert (o == 0).all() and (s == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_delta_gradients_nonfinite_stay_in_their_head(dtype, bad):
    """What comes back of a value or a gradient that is not finite: other heads keep their bits, the head's own tell."""
    _, t = delta_inputs(1, 3, 3, 200, 32, 32, dtype)
    do = torch.randn_like(t[2])
    want = mh.gated_delta_rule_bwd(do, *t[:5], initial_state=t[5])
    for i in (1, 2, 6):
        u = [a.clone() for a in (*t, do)]
        u[i][0, 1, 70, 5] = bad
        got = mh.gated_delta_rule_bwd(u[6], *u[:5], initial_state=u[5])
        for a, b in zip(got, want):
            assert torch.equal(a[:, [0, 2]], b[:, [0, 2]])
        assert not torch.isfinite(got[2][0, 1]).all() or i == 2
        assert not torch.isfinite(got[1][0, 1]).all()


# ------------------------------------------------------------------------------------------------ rotary positions

def test_rotary_without_queries():
    """q of no heads: keys are turned all the same, and their gradient."""
    f, _ = mh.rotary_frequencies(16)
    k = torch.randn(2, 3, 9, 24, device="cuda", requires_grad=True)
    for H in (0, 1):
        q = torch.randn(2, H, 9, 24, device="cuda", requires_grad=True)
        a, b = mh.rotary(q, k, f)
        assert a.shape == q.shape and torch.equal(b, mh.rotary(k, None, f))
        dk, = torch.autograd.grad(b, k, torch.ones_like(b), retain_graph=True)
        assert torch.equal(dk, mh.rotary(torch.ones_like(b), None, f, inverse=True))
        dq, dk2 = torch.autograd.grad((a, b), (q, k), (torch.ones_like(a), torch.ones_like(b)))
        assert dq.shape == q.shape and torch.equal(dk, dk2)
    assert mh.rotary(q[:, :0], None, f).shape == (2, 0, 9, 24)
    assert [t.shape[1] for t in mh.rotary(q[:, :0], k[:, :0], f)] == [0, 0]


# ------------------------------------------------------------------------------------------------ strides

@pytest.mark.parametrize("dtype", [F32, BF])
def test_sliding_windows(dtype):
    """Tokens that are windows of one signal, an element apart, as unfold gives them: inputs may overlap themselves, the
    results do not, and they have the bits of a copy."""
    L, D = 9, 16                                 # fewer tokens than channels: torch would lay a like tensor out by tokens
    x = torch.randn(2, 3, L + D - 1, device="cuda").to(dtype)
    w = x.unfold(-1, D, 1)
    assert w.shape == (2, 3, L, D) and w.stride()[-2:] == (1, 1)
    c = w.contiguous()
    f, _ = mh.rotary_frequencies(D)
    for a, b in zip(mh.rotary(w, w, f), mh.rotary(c, c, f)):
        assert torch.equal(a, b)
    assert torch.equal(mh.gated_delta_rule(w, w, w), mh.gated_delta_rule(c, c, c))
    for a, b in zip(mh.gated_delta_rule_bwd(w, w, w, w)[:3], mh.gated_delta_rule_bwd(c, c, c, c)[:3]):
        assert torch.equal(a, b)
    state = torch.randn(2, L, D, D, device="cuda")
    w3, s2 = w[:, 0], state.clone()
    assert torch.equal(mh.gated_delta_step(state, w3, w3, w3), mh.gated_delta_step(s2, *(w3.contiguous(),) * 3))
    assert torch.equal(state, s2)
    assert torch.equal(mh.group_norm(w[:, 0], 4), mh.group_norm(w[:, 0].contiguous(), 4))


# ------------------------------------------------------------------------------------------------ grids of 2^32 threads

def test_step_of_many_heads():
    B, H, dv = 1 << 20, 8, 33                    # 2^24 workgroups of 256 threads
    state = torch.randn(B, H, 1, dv, device="cuda")
    q, k, v = (torch.randn(B, H, d, device="cuda", dtype=BF) for d in (1, 1, dv))
    say("step of 2^23 heads")
    first, last = state[:2].clone(), state[-2:].clone()
    o = mh.gated_delta_step(state, q, k, v)
    for part, s in ((slice(None, 2), first), (slice(-2, None), last)):
        assert torch.equal(o[part], mh.gated_delta_step(s, q[part], k[part], v[part])) and torch.equal(state[part], s)


def test_rotary_of_many_tokens():
    x = torch.randn(4, 1, 1 << 30, 2, device="cuda", dtype=BF)
    f = torch.full((1,), 1e-3, device="cuda", dtype=torch.float64)
    say("rotary of 2^32 tokens")
    y = mh.rotary(x, None, f)
    for b in (0, 3):
        for at in (0, (1 << 30) - 300):
            assert torch.equal(y[b:b + 1, :, at:at + 300], mh.rotary(x[b:b + 1, :, at:at + 300], None, f, offset=at))


def test_state_through_no_tokens():
    """2^32 elements of a state that passes a sequence of none."""
    B, dk, dv = 1 << 17, 128, 256
    s = torch.empty(B, 1, dk, dv, device="cuda")
    s.view(-1)[:] = 1.5
    s[-1] = torch.randn(1, dk, dv, device="cuda")
    q, v = torch.zeros(B, 1, 0, dk, device="cuda"), torch.zeros(B, 1, 0, dv, device="cuda")
    say("no tokens, 16 GiB of state")
    _, out = mh.gated_delta_rule(q, q, v, initial_state=s, return_final_state=True)
    assert torch.equal(out[-1], s[-1]) and bool((out[:-1] == 1.5).all())
    back = mh.gated_delta_rule_bwd(v, q, q, v, initial_state=s, d_final_state=out)[5]
    assert torch.equal(back[-1], s[-1]) and bool((back[0] == 1.5).all())


# ------------------------------------------------------------------------------------------------ group norm

@pytest.mark.parametrize("shape,G", [((48, 256), 4), ((3, 500, 64), 4), ((2, 4001, 20), 4), ((1, 70, 4800), 2)])
@pytest.mark.parametrize("mean", [4096.0, -1e6, 3e7])
def test_group_norm_of_a_far_mean(shape, G, mean):
    """Values far from zero, in either way of taking the sums: centred values keep their digits, whatever fp32 leaves of the
    mean.  fp32 near 3e7 has steps of 2, so that the values are what they were rounded to."""
    x = (torch.randn(*shape, generator=torch.Generator().manual_seed(1)) * max(1.0, abs(mean) * 2.0 ** -21) + mean).cuda()
    b = torch.randn(shape[-1], device="cuda")
    say(f"group norm of {shape} around {mean}")
    y, stats = mh.group_norm(x, G, None, b, 1e-5, return_stats=True)
    ry, rs = mx.group_norm(host(x), G, None, host(b), 1e-5)
    z = ry - host(b)
    # x - mean is exact (both within a factor 2 of each other); then what the mean's rounding left, 1 / deviation (the variance
    # as fp32, eps, the root, the quotient), the product and the sum with b: 8 roundings of what enters them; in the one-position
    # way the deviations of a first mean off by 4 roundings of it, mended by their own mean, whose sum has another 8 of those
    first = 4 * 2.0 ** -24 * abs(mean) * rs[..., 1].max()
    tol = 2.0 ** -24 * (8 * (np.abs(z) + np.abs(host(b))) + 8 * (1 + np.abs(z)) + 8 * first)
    worst = (np.abs(host(y) - ry) / tol).max()
    say(f"error at most {worst:.3f} of the tolerance")
    assert worst <= 1
    assert np.abs(host(stats[..., 1]) / rs[..., 1] - 1).max() <= 2.0 ** -20
    assert np.abs(host(stats[..., 0]) - rs[..., 0]).max() <= 2.0 ** -23 * abs(mean)


def test_group_norm_of_an_outlier_first():
    """The value that all others are taken from may lie far from them."""
    for first in (1e8, -3e12):
        x = torch.randn(2, 300, 64, device="cuda")
        x[:, 0, ::16] = first
        y, stats = mh.group_norm(x, 4, return_stats=True)
        ry, rs = mx.group_norm(host(x), 4)
        # all but the first end at -mean / deviation, apart by their own differences over it
        assert np.abs(host(y) - ry).max() <= 2.0 ** -20 * np.abs(ry).max()
        assert np.abs(host(stats[..., 1]) / rs[..., 1] - 1).max() <= 2.0 ** -20


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape,G", [((6, 64), 4), ((2, 300, 64), 4)])
def test_group_norm_beyond_fp32s_squares(dtype, shape, G):
    """A group whose variance leaves fp32 says so, and not its bias; the others keep their bits.  Near the end it is right."""
    x = torch.randn(*shape, device="cuda").to(dtype)
    w, b = torch.randn(2, 64, device="cuda")
    want, ws = mh.group_norm(x, G, w, b, return_stats=True)
    for size in (1e25, 3e38):
        y = x.clone()
        y[1, ..., 16:32] = torch.sign(y[1, ..., 16:32]) * size
        got, st = mh.group_norm(y, G, w, b, return_stats=True)
        assert got[1, ..., 16:32].isnan().all() and st[1, 1, 1].isnan()
        got[1, ..., 16:32], st[1, 1] = want[1, ..., 16:32], ws[1, 1]
        assert torch.equal(got, want) and torch.equal(st, ws)
    y = x * 1e17
    got, st = mh.group_norm(y, G, w, b, return_stats=True)
    ry, rs = mx.group_norm(host(y), G, host(w), host(b))
    half = torch.finfo(dtype).eps / 2
    # 16 roundings of what enters, as everywhere (a deviation is taken of at most 4 of them)
    assert (np.abs(host(got) - ry) <= half * np.abs(ry) + 2.0 ** -19 * (np.abs(ry) + 2 * np.abs(host(b)) + 4 * np.abs(host(w)))).all()
    assert np.abs(host(st[..., 1]) / rs[..., 1] - 1).max() <= 2.0 ** -19


def test_group_norm_statistics_of_no_positions():
    torch.full((3, 4, 2), 5.0, device="cuda")    # what the next allocation of this size holds
    y, stats = mh.group_norm(torch.zeros(3, 0, 64, device="cuda"), 4, return_stats=True)
    assert y.shape == (3, 0, 64) and stats.shape == (3, 4, 2) and stats.isnan().all()
    y, stats = mh.group_norm(torch.zeros(0, 7, 64, device="cuda"), 4, return_stats=True)
    assert stats.shape == (0, 4, 2)
    x, st = torch.zeros(3, 0, 64, device="cuda"), torch.full((3, 4, 2), float("nan"), device="cuda")
    dx, dw, db = mh.group_norm_bwd(x, x, st, 4, torch.ones(64, device="cuda"))
    assert dx.shape == (3, 0, 64) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("offset", [1 << 63, -(1 << 63) - 1, 1 << 64])
def test_rotary_offset_out_of_range(offset):
    q, f = torch.randn(1, 1, 2, 8, device="cuda"), torch.ones(4, device="cuda")
    with pytest.raises(ValueError, match="offset"):
        mh.rotary(q, None, f, offset=offset)
    mh.rotary(q, None, f, offset=(1 << 63) - 2)


def test_gradients_of_many_positions():
    """2^31 elements of one sequence: dx and db against sums in fp64 over all of it, a piece at a time."""
    n, C, G = (1 << 24) + 5, 128, 4
    x = torch.randn(1, n, C, device="cuda", dtype=BF)
    say("group norm's gradients over 2^24 positions")
    _, st = mh.group_norm(x, G, return_stats=True)
    db = mh.group_norm_bwd(torch.ones_like(x), x, st, G, dtype=F32)[2]
    # sums of ones are exact up to 2^24; a few roundings of half a step of 2 above
    assert (db.double() - n).abs().max() <= 4
    rows = torch.arange(n, device="cuda")
    dy = ((rows * 7919 % 13 - 6)[:, None] * (1 + torch.arange(C, device="cuda") % 3)).to(BF)[None]
    dx, _, db = mh.group_norm_bwd(dy, x, st, G, dtype=F32)
    m, r = (st[0, :, i].double().repeat_interleave(C // G) for i in (0, 1))
    s1, s2, mag = (torch.zeros(C, device="cuda", dtype=torch.float64) for _ in range(3))
    for a in range(0, n, 1 << 20):
        d = dy[0, a:a + (1 << 20)].double()
        xh = (x[0, a:a + (1 << 20)].double() - m) * r
        s1, s2, mag = s1 + d.sum(0), s2 + (d * xh).sum(0), mag + (d * xh).abs().sum(0)
    mean1, mean2, meanmag = ((t.view(G, -1).sum(-1) / (n * C // G)).repeat_interleave(C // G) for t in (s1, s2, mag))
    # a thread's sum of up to 1100 terms in fp32, then 16 and a fourth of 1100 of those: 2^11 roundings of their magnitude
    for part in (slice(0, 9), slice(n // 2, n // 2 + 9), slice(n - 9, n)):
        d, xh = dy[0, part].double(), (x[0, part].double() - m) * r
        want = r * (d - mean1 - xh * mean2)
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -20 * r * (d.abs() + 18) + 2.0 ** -13 * r * xh.abs() * meanmag
        assert ((dx[0, part].double() - want).abs() <= tol).all()
    assert ((db.double() - s1).abs() <= 2.0 ** -13 * (dy.abs().float().mean((0, 1)).double() * n)).all()
