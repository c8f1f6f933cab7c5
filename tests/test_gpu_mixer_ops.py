"""Gated delta rule, rotary positions and group norm on the GPU against the float64 oracle.

Tolerances.  A result of type T is rounded once: half a step, ``finfo(T).eps / 2`` of the value.  Before that:

Gated delta rule.  Operands of its products are fp16 in two parts of their column's or matrix's largest value (22 bits and
a sign: 2^-23 of it), the product of the two small parts is left out (2^-22) and the sum of 64 or 128 terms is fp32 (under
2^-21 of the terms' magnitude): below 2^-20 of the norms that enter for each product.  From inputs to a result a piece takes
at most 12 of them (K K^T, the system's inverse in 6 levels, K S, T R, Q S, P delta, K^T U), the gradients twice as many.
Errors of different pieces are independent: their sum grows with the square root of their number.  So a row's error, in
norm, is within ``half * |row| + 12 * 2^-20 * sqrt(pieces) * max |rows of its head|``, for the gradients with 24.  Where o
and the gradients are bf16, their last products take one part each of two operands (2 * 2^-12) and bf16 inputs are exact.

Rotary, group norm.  Elementwise ``near`` as for the token operators: k fp32 roundings of 2^-24 of what enters.
"""

import numpy as np
import pytest
import torch

import mamformer_amd as mh
from oracle import mixers as mx
from tests.gpu_helpers import host, say
from tests.test_gpu_token_ops import draw, near

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def rows_near(name, out, ref, k, pieces=1):
    """out, ref (B, heads, rows, ...): each row's error in norm."""
    half = torch.finfo(out.dtype).eps / 2
    o = host(out)
    assert o.shape == ref.shape, f"{name}: shape {o.shape}, expected {ref.shape}"
    assert np.isfinite(o).all(), f"{name}: not finite"
    if o.size == 0:
        return
    o, r = (x.reshape(*ref.shape[:3], -1) for x in (o, ref))
    rows = np.linalg.norm(r, axis=-1)
    part = 2.0 ** -11 if out.dtype is BF else 0.0
    tol = half * rows + (k * 2.0 ** -20 * np.sqrt(pieces) + part) * rows.max(-1, keepdims=True) + 1e-30
    worst = (np.linalg.norm(o - r, axis=-1) / tol).max()
    say(f"{name}: error at most {worst:.3f} of the tolerance")
    assert worst <= 1, f"{name}: {worst:.3f} times the tolerance"


# ------------------------------------------------------------------------------------------------ gated delta rule

def delta_inputs(B, H, HK, L, dk, dv, dtype=F32, *, gates=True, state=True, decay=0.2, seed=0):
    """(float64 arrays, GPU tensors) of q, k, v, g, beta, state: keys of norm 1 (rounded to dtype)."""
    q, qg = draw(seed, B, HK, L, dk, dtype=dtype)
    k = torch.nn.functional.normalize(torch.as_tensor(draw(seed + 1, B, HK, L, dk)[0]), dim=-1).to(dtype)
    v, vg = draw(seed + 2, B, H, L, dv, dtype=dtype)
    gen = torch.Generator().manual_seed(seed + 3)
    g = (-decay * torch.rand(B, H, L, generator=gen)) if gates else None
    b = torch.rand(B, H, L, generator=gen) if gates else None
    s = torch.randn(B, H, dk, dv, generator=gen) if state else None
    np_, gpu = (lambda t: None if t is None else t.double().numpy()), (lambda t: None if t is None else t.cuda())
    return [q, np_(k), v, np_(g), np_(b), np_(s)], [qg, k.cuda(), vg, gpu(g), gpu(b), gpu(s)]


def compare(x, t, scale=None, d_final=True, seed=9, names=("dq", "dk", "dv", "dg", "dbeta", "d_state")):
    """Forward, explicit backward and autograd's of one case against the oracle; the results."""
    B, H, L, dv = x[2].shape
    pieces = max((L + 63) // 64, 1)
    o, final = mh.gated_delta_rule(*t[:5], scale=scale, initial_state=t[5], return_final_state=True)
    ro, rf = mx.delta_rule(*x[:5], scale, x[5])
    assert o.dtype is t[2].dtype and final.dtype is F32
    rows_near("o", o, ro, 12, pieces)
    rows_near("final", final, rf, 12, pieces)
    do, dog = draw(seed, *x[2].shape, dtype=t[2].dtype)
    df, dfg = draw(seed + 1, *final.shape) if d_final else (None, None)
    grads = mh.gated_delta_rule_bwd(dog, *t[:5], scale=scale, initial_state=t[5], d_final_state=dfg)
    refs = mx.delta_rule_bwd(do, *x[:5], scale, x[5], df)
    leaves = [None if a is None else a.detach().requires_grad_(True) for a in t]
    for recompute in (False, True):
        out, fin = mh.gated_delta_rule(*leaves[:5], scale=scale, initial_state=leaves[5], return_final_state=True,
                                       recompute=recompute)
        assert torch.equal(out, o) and torch.equal(fin, final)
        loss = [(out, dog)] + ([(fin, dfg)] if d_final else [])
        auto = torch.autograd.grad([a for a, _ in loss], [a for a in leaves if a is not None], [b for _, b in loss])
        auto = iter(auto)
        for name, leaf, got in zip(names, leaves, grads):
            assert leaf is None or torch.equal(next(auto), got.to(leaf.dtype)), (name, recompute)
    for name, leaf, got, want in zip(names, leaves, grads, refs):
        if leaf is None:
            assert got is None, name
        elif got.dim() == 3:                     # dg, dbeta: a number a token; the head's is the scale
            rows_near(name, got[:, :, None], want[:, :, None], 24, pieces)
            worst = np.abs(host(got) - want) / (np.abs(want).max(-1, keepdims=True) + 1e-30) if L else np.zeros(1)
            assert worst.max() <= 24 * 2.0 ** -20 * np.sqrt(64 * pieces), name
        else:
            rows_near(name, got, want, 24, pieces)
    return o, final, grads


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,H,HK,L,dk,dv,opts", [
    (1, 1, 1, 1, 1, 1, {}), (2, 3, 1, 2, 8, 8, {}), (1, 2, 2, 31, 16, 33, {}), (1, 2, 1, 63, 64, 16, dict(gates=False)),
    (2, 4, 2, 64, 64, 64, {}), (1, 2, 1, 65, 65, 31, {}), (1, 6, 2, 127, 128, 17, dict(state=False)),
    (2, 2, 1, 128, 37, 128, {}), (1, 2, 1, 129, 128, 256, {}), (1, 4, 4, 200, 96, 80, dict(gates=False, state=False)),
    (3, 2, 1, 191, 3, 130, dict(decay=3.0)), (1, 9, 3, 257, 33, 65, dict(decay=0.0)),
])
def test_delta(dtype, B, H, HK, L, dk, dv, opts):
    say(f"delta {B} {H} {HK} {L} {dk} {dv} {dtype} {opts}")
    compare(*delta_inputs(B, H, HK, L, dk, dv, dtype, **opts))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,H,HK,L,dk,dv", [(1, 2, 1, 1500, 24, 40), (1, 1, 1, 2100, 128, 100), (1, 3, 1, 3001, 64, 16)])
def test_delta_in_segments(dtype, B, H, HK, L, dk, dv):
    """Few heads and many pieces: segments, the last ones ragged; the last head's decay leaves nothing of a segment."""
    x, t = delta_inputs(B, H, HK, L, dk, dv, dtype)
    t[3][:, -1] *= 100
    x[3] = t[3].double().cpu().numpy()
    say(f"delta in segments {B} {H} {HK} {L} {dk} {dv} {dtype}")
    compare(x, t)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("only", ["g", "beta"])
def test_delta_with_one_gate(dtype, only):
    x, t = delta_inputs(1, 2, 1, 100, 32, 32, dtype)
    i = 4 if only == "g" else 3
    x[i] = t[i] = None
    say(f"delta with {only} alone, {dtype}")
    compare(x, t, scale=-0.75, d_final=False)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_delta_gates_at_their_ends(dtype):
    """g = -inf and far below exp's range clears the state (its own gradient 0), beta = 0 writes nothing, beta = 2 reflects."""
    x, t = delta_inputs(1, 4, 1, 150, 32, 24, dtype)
    g, b = t[3], t[4]
    g[:, 0, [0, 40, 64, 65, 149]] = -float("inf")
    g[:, 1, ::7] = -1000.0
    g[:, 2] = 0
    b[:, 2, 64:128] = 0
    b[:, 3], g[:, 3] = 2.0, 0
    x[3], x[4] = g.double().cpu().numpy(), b.double().cpu().numpy()
    say(f"gates at their ends, {dtype}")
    _, _, grads = compare(x, t)
    assert (grads[3][:, 0, [0, 40, 64, 65, 149]] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_delta_padding(dtype):
    """Tokens with beta = 0 and g = 0 behind a sequence leave its results and its state."""
    x, t = delta_inputs(2, 2, 1, 200, 64, 48, dtype)
    short = [a[:, :, :70] if i < 5 else a for i, a in enumerate(t)]
    t[3][:, :, 70:], t[4][:, :, 70:] = 0, 0
    o, s = mh.gated_delta_rule(*t[:5], initial_state=t[5], return_final_state=True)
    xs = [a[:, :, :70] if i < 5 else a for i, a in enumerate(x)]
    ro, rs = mx.delta_rule(*xs[:5], None, xs[5])
    rows_near("o", o[:, :, :70], ro, 12, 2)
    rows_near("state", s, rs, 12, 2)
    o2, s2 = mh.gated_delta_rule(*short[:5], initial_state=t[5], return_final_state=True)
    rows_near("short o", o2, ro, 12, 2)
    rows_near("short state", s2, rs, 12, 2)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_delta_strides(dtype):
    """One packed projection (B, L, (q | k | v) heads) read as it lies, from an odd element on; o and the gradients of views;
    inputs that are broadcast over the batch and the heads."""
    B, H, HK, L, dk, dv = 2, 4, 2, 130, 24, 40
    x, t = delta_inputs(B, H, HK, L, dk, dv, dtype)
    W = 2 * HK * dk + H * dv + 5
    room = torch.zeros(B * L * W + 3, device="cuda", dtype=dtype)[3:].view(B, L, W)
    parts = room[..., 1:1 + HK * dk], room[..., 1 + HK * dk:1 + 2 * HK * dk], room[..., 1 + 2 * HK * dk:W - 4]
    views = []
    for part, src in zip(parts, t[:3]):
        v = part.unflatten(-1, (src.shape[1], -1)).transpose(1, 2)
        v.copy_(src)
        views.append(v)
    gates = [a.transpose(1, 2).contiguous().transpose(1, 2) for a in t[3:5]]
    say(f"delta of views, {dtype}")
    got = compare(x, [*views, *gates, t[5]])
    for a, b in zip((*got[:2], *got[2]), (lambda r: (*r[:2], *r[2]))(compare(x, t))):
        assert torch.equal(a, b)
    x2, t2 = [a.copy() for a in x], list(t)
    x2[0][1:], x2[2][:, 1:], x2[3][:] = x2[0][:1], x2[2][:, :1], x2[3][:, :1, :1]
    t2[0], t2[2] = t[0][:1].expand(B, -1, -1, -1), t[2][:, :1].expand(-1, H, -1, -1)
    t2[3] = t[3][:, :1, :1].expand(-1, H, L)
    say("broadcast inputs")
    compare(x2, t2)


def test_delta_of_a_channel_stride():
    x, t = delta_inputs(1, 2, 1, 70, 16, 16)
    wide = [torch.stack([a, a], -1).flatten(-2)[..., ::2] for a in t[:3]]
    say("channels two apart")
    compare(x, [*wide, *t[3:]])


def test_delta_far_apart_rows():
    """Rows and batch entries whose distance in bytes passes 32 bits (fp32 and bf16 take other paths)."""
    for dtype in (F32, BF):
        n = (1 << 32) // torch.empty((), dtype=dtype).element_size()
        x, t = delta_inputs(1, 1, 1, 35, 16, 16, dtype)
        room = torch.empty(n // 2 * 3, device="cuda", dtype=dtype)
        stride = n // 24
        v = room.as_strided(t[2].shape, (0, 0, stride, 1))
        v.copy_(t[2])
        say(f"rows {stride} apart, {dtype}")
        got = mh.gated_delta_rule(t[0], t[1], v, *t[3:5], initial_state=t[5])
        rows_near("o", got, mx.delta_rule(*x[:5], None, x[5])[0], 12)
        del room, v


@pytest.mark.parametrize("dtype", [F32, BF])
def test_delta_without_tokens(dtype):
    x, t = delta_inputs(2, 2, 1, 0, 16, 24, dtype)
    compare(x, t)
    x, t = delta_inputs(2, 2, 1, 0, 16, 24, dtype, state=False)
    o, s = mh.gated_delta_rule(*t[:5], return_final_state=True)
    assert o.shape == (2, 2, 0, 24) and (s == 0).all()
    x, t = delta_inputs(0, 2, 1, 5, 16, 24, dtype)
    o, s = mh.gated_delta_rule(*t[:5], initial_state=t[5], return_final_state=True)
    assert o.shape == (0, 2, 5, 24) and s.shape == (0, 2, 16, 24)
    assert [g.shape for g in mh.gated_delta_rule_bwd(o, *t[:5], initial_state=t[5])] == [a.shape for a in t]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("L", [200, 2000])
def test_delta_nonfinite_stays_in_its_head(dtype, bad, L):
    """Other heads and the pieces before keep their bits; the head's later results tell."""
    _, t = delta_inputs(1, 3, 3, L, 32, 32, dtype)
    want, ws = mh.gated_delta_rule(*t[:5], initial_state=t[5], return_final_state=True)
    for i in range(3):
        u = [a.clone() for a in t]
        u[i][0, 1, 70, 5] = bad
        o, s = mh.gated_delta_rule(*u[:5], initial_state=u[5], return_final_state=True)
        keep = [0, 2]
        assert torch.equal(o[:, keep], want[:, keep]) and torch.equal(s[:, keep], ws[:, keep])
        assert torch.equal(o[:, 1, :64], want[:, 1, :64])
        assert not torch.isfinite(o[:, 1, 70:128]).all()


def test_delta_beyond_fp16():
    """Values, states and gradients far outside fp16's range: the parts are scaled."""
    for size in (1e-18, 1e12):
        x, t = delta_inputs(1, 2, 1, 130, 32, 32)
        x[2], x[5] = x[2] * size, x[5] * size
        t[2], t[5] = (torch.as_tensor(a).float().cuda() for a in (x[2], x[5]))
        x[2], x[5] = t[2].double().cpu().numpy(), t[5].double().cpu().numpy()
        say(f"values of {size}")
        o, s = mh.gated_delta_rule(*t[:5], initial_state=t[5], return_final_state=True)
        ro, rs = mx.delta_rule(*x[:5], None, x[5])
        rows_near("o", o, ro, 12, 3)
        rows_near("state", s, rs, 12, 3)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_delta_step_is_the_sequence(dtype):
    """Pieces, then single tokens: the results of one sequence; in place and into another state, on another stream."""
    x, t = delta_inputs(3, 4, 2, 90, 40, 72, dtype)
    ro, rs = mx.delta_rule(*x[:5], 0.3, x[5])
    o, state = mh.gated_delta_rule(*(a[:, :, :75] for a in t[:5]), scale=0.3, initial_state=t[5], return_final_state=True)
    rows_near("first", o, ro[:, :, :75], 12, 2)
    stream = torch.cuda.Stream()
    for i in range(75, 90):
        args = [a[:, :, i] for a in t[:5]]
        if i % 2:
            before, other = state.clone(), torch.full_like(state, float("nan"))
            o = mh.gated_delta_step(state, *args, scale=0.3, state_out=other)
            assert torch.equal(before, state)
            state = other
        else:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                o = mh.gated_delta_step(state, *args, scale=0.3)
            torch.cuda.current_stream().wait_stream(stream)
        rows_near(f"token {i}", o[:, :, None], ro[:, :, i:i + 1], 12, 2)
    rows_near("state", state, rs, 12, 2)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,H,HK,dk,dv", [(1, 1, 1, 1, 1), (2, 3, 1, 17, 9), (5, 4, 2, 128, 256), (1, 16, 4, 96, 80), (33, 2, 2, 64, 65)])
def test_delta_step(dtype, B, H, HK, dk, dv):
    x, t = delta_inputs(B, H, HK, 1, dk, dv, dtype)
    for gates in (True, False):
        xs, ts = (a[:3] + (a[3:5] if gates else [None, None]) for a in (x, t))
        if gates:
            ts[3] = ts[3].clone()
            ts[3][0, 0] = -float("inf")
            xs[3] = ts[3].double().cpu().numpy()
        state = t[5].clone()
        o = mh.gated_delta_step(state, *(None if a is None else a[:, :, 0] for a in ts))
        ro, rs = mx.delta_rule(*xs, None, x[5])
        say(f"step {B} {H} {HK} {dk} {dv} {dtype} gates={gates}")
        rows_near("o", o[:, :, None], ro, 2)
        rows_near("state", state, rs, 2)


def test_delta_step_refusals():
    x, t = delta_inputs(1, 2, 1, 1, 16, 16)
    args, state = [a[:, :, 0] for a in t[:5]], t[5]
    with pytest.raises(RuntimeError, match="no backward"):
        mh.gated_delta_step(state, args[0].clone().requires_grad_(True), *args[1:])
    with pytest.raises(ValueError, match="contiguous"):
        mh.gated_delta_step(state.transpose(2, 3), *args)
    with pytest.raises(ValueError, match="contiguous"):
        mh.gated_delta_step(state, *args, state_out=torch.empty_like(state).transpose(2, 3))
    for bad in (state[:, :1], state.bfloat16(), state.cpu()):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            mh.gated_delta_step(bad, *args)
    v = state._version
    mh.gated_delta_step(state, *args)
    assert state._version > v
    with torch.inference_mode():
        mh.gated_delta_step(state.clone(), *args)


def test_delta_refusals():
    x, t = delta_inputs(1, 4, 2, 10, 16, 16)
    q, k, v, g, b, s = t
    for call in (lambda: mh.gated_delta_rule(q, k[:, :1], v), lambda: mh.gated_delta_rule(q[:, :, :9], k[:, :, :9], v),
                 lambda: mh.gated_delta_rule(q[0], k[0], v[0]), lambda: mh.gated_delta_rule(q, k, v, g[..., :9]),
                 lambda: mh.gated_delta_rule(q, k.bfloat16(), v), lambda: mh.gated_delta_rule(q.half(), k.half(), v.half()),
                 lambda: mh.gated_delta_rule(q, k, v, g.double()), lambda: mh.gated_delta_rule(q, k, v, initial_state=s[..., :8]),
                 lambda: mh.gated_delta_rule(q, k, v, initial_state=s.bfloat16()),
                 lambda: mh.gated_delta_rule(q, k, v[:, :3]), lambda: mh.gated_delta_rule(q, k, torch.zeros(1, 4, 10, 257, device="cuda")),
                 lambda: mh.gated_delta_rule(*(torch.zeros(1, 2, 10, 129, device="cuda"),) * 2, v),
                 lambda: mh.gated_delta_rule_bwd(v[..., :8], q, k, v), lambda: mh.gated_delta_rule_bwd(v, q, k, v, d_final_state=s[:, :1]),
                 lambda: mh.gated_delta_rule(q.cpu(), k, v)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()


def test_delta_autograd_of_parts():
    """Gates in bf16, some inputs without a gradient, either result alone, a graph used twice, a second backward refused."""
    x, t = delta_inputs(1, 4, 2, 100, 32, 32)
    g, b = t[3].bfloat16().requires_grad_(True), t[4].bfloat16().requires_grad_(True)
    o, s = mh.gated_delta_rule(*t[:3], g, b, initial_state=t[5], return_final_state=True)
    full = mh.gated_delta_rule_bwd(torch.ones_like(o), *t[:3], g.detach(), b.detach(), initial_state=t[5])
    dg, db = torch.autograd.grad(o.sum(), (g, b), retain_graph=True)
    assert dg.dtype is BF and torch.equal(dg, full[3].to(BF)) and torch.equal(db, full[4].to(BF))
    again = torch.autograd.grad(o.sum(), (g, b), retain_graph=True)
    assert torch.equal(again[0], dg) and torch.equal(again[1], db)
    df = mh.gated_delta_rule_bwd(torch.zeros_like(o), *t[:3], g.detach(), b.detach(), initial_state=t[5], d_final_state=torch.ones_like(s))
    assert torch.equal(torch.autograd.grad(s.sum(), g)[0], df[3].to(BF))
    k = t[1].clone().requires_grad_(True)
    dk, = torch.autograd.grad(mh.gated_delta_rule(t[0], k, *t[2:5], initial_state=t[5]).sum(), k)
    assert torch.equal(dk, mh.gated_delta_rule_bwd(torch.ones_like(o), t[0], k.detach(), *t[2:5], initial_state=t[5])[1])
    out = mh.gated_delta_rule(t[0], k, *t[2:5])
    d, = torch.autograd.grad(out.sum(), k, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    out = mh.gated_delta_rule(t[0], k * 1.0, *t[2:5])
    _ = out.detach().zero_()                     # a result is not read again
    out = mh.gated_delta_rule(t[0], kk := k * 1.0, *t[2:5])
    kk.detach().mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad
    x, t = delta_inputs(1, 1, 1, 4, 8, 8)
    f = torch.ones(4, device="cuda", dtype=torch.float64)
    for call in (lambda v: mh.gated_delta_rule(v, *t[1:5]), lambda v: mh.rotary(v, None, f), lambda v: mh.group_norm(v, 2)):
        with forward_ad.dual_level(), pytest.raises(RuntimeError):
            call(forward_ad.make_dual(t[0], torch.ones_like(t[0])))


def on_stream_and_captured(fn, inputs):
    """fn(*inputs) twice, on another stream, and replayed from a graph with eager work between: one result's bits."""
    want = [a.clone() for a in fn(*inputs)]
    assert all(torch.equal(a, b) for a, b in zip(fn(*inputs), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fn(*inputs)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn(*inputs)
    for i in range(4):
        for a in out:
            a.fill_(float(i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {i}"
        eager = fn(*inputs)
        assert all(torch.equal(a, b) for a, b in zip(eager, want))
    new = [a.clone() for a in inputs]
    for a in inputs:                             # a replay reads what its inputs hold then
        a.mul_(0.5) if a.is_floating_point() else a.add_(1)
    want2 = [a.clone() for a in fn(*inputs)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want2))
    for a, b in zip(inputs, new):
        a.copy_(b)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("L", [150, 2000])
def test_delta_streams_and_graphs(dtype, L):
    _, t = delta_inputs(1, 2, 1, L, 64, 48, dtype)
    do = torch.randn_like(t[2])
    say(f"streams and graphs L={L} {dtype}")

    def forward(*a):
        return mh.gated_delta_rule(*a[:5], initial_state=a[5], return_final_state=True)

    def backward(*a):
        return mh.gated_delta_rule_bwd(a[6], *a[:5], initial_state=a[5])

    def train(*a):
        leaves = [x.detach().requires_grad_(True) for x in a[:6]]
        out = mh.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
        return torch.autograd.grad(out, leaves, a[6])

    on_stream_and_captured(forward, t)
    on_stream_and_captured(backward, [*t, do])
    on_stream_and_captured(train, [*t, do])
    on_stream_and_captured(lambda s, *a: (mh.gated_delta_step(s, *a, state_out=torch.empty_like(s)),),
                           [t[5], *(a[:, :, 0].contiguous() for a in t[:5])])


def test_two_graphs_of_one_forward():
    """Two captured backward passes of one eager forward, replayed on two streams at once: they only read what it kept."""
    _, t = delta_inputs(1, 2, 1, 700, 64, 64, BF)
    leaves = [a.detach().requires_grad_(True) for a in t]
    out = mh.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
    dos = [torch.randn_like(out) for _ in range(2)]
    want = [[a.clone() for a in torch.autograd.grad(out, leaves, d, retain_graph=True)] for d in dos]
    node = out.grad_fn
    q, k, v, g, b, s, kept = node.saved_tensors
    from mamformer_amd import mixer_ops
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for d in dos:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(mixer_ops._delta_bwd(d, *(a.detach() for a in (q, k, v, g, b, s)), None, node.scale, kept))
    for _ in range(3):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))


# ------------------------------------------------------------------------------------------------ rotary positions

@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,H,HK,L,D,n,pos", [
    (1, 1, 0, 1, 2, 1, None), (2, 3, 1, 7, 64, 32, "row"), (1, 2, 2, 33, 37, 5, "batch"), (2, 4, 2, 5, 128, 64, "far"),
    (3, 2, 1, 17, 100, 50, "int32"), (1, 5, 5, 64, 80, 20, None), (2, 1, 0, 130, 256, 128, "batch"),
])
def test_rotary(dtype, interleaved, B, H, HK, L, D, n, pos):
    q, qg = draw(1, B, H, L, D, dtype=dtype)
    k, kg = draw(2, B, HK, L, D, dtype=dtype) if HK else (None, None)
    f, scale = mh.rotary_frequencies(2 * n, 1e4, scaling="yarn", factor=2.0, original_length=512)
    rng = np.random.default_rng(n)
    offset = {"far": 10 ** 9, "int32": -40}.get(pos, 3)
    p = None if pos is None else rng.integers(-50, 5000, (L,) if pos == "row" else (B, L))
    if pos == "far":
        p = p * 100000
    pg = None if p is None else torch.as_tensor(p).to(torch.int32 if pos == "int32" else torch.int64).cuda()
    ph = (np.arange(L) if p is None else p) + offset
    fh = f.cpu().numpy()
    say(f"rotary {B} {H} {HK} {L} {D} {n} {pos} interleaved={interleaved} {dtype}")
    for inverse in (False, True):
        out = mh.rotary(qg, kg, f, pg, offset=offset, interleaved=interleaved, scale=scale, inverse=inverse)
        for name, x, got in (("q", q, out[0] if HK else out), ("k", k, out[1] if HK else None))[:2 if HK else 1]:
            # sine and cosine, two products, their sum, the scale: 6 roundings of the pair's magnitude; the angle is rounded
            # in fp64, where one of 1e9 turns is off by 2^-23 radians
            pair = np.zeros_like(x)
            a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
            pair[..., a] = pair[..., b] = scale * (np.abs(x[..., a]) + np.abs(x[..., b]))
            far = 1 + np.abs(ph).max() * fh.max() * 2.0 ** -53 / U
            near(name, got, mx.rotary(x, fh, ph, interleaved, scale, inverse), pair * far, 6)
            assert torch.equal(got[..., 2 * n:], (qg if name == "q" else kg)[..., 2 * n:])
    # fp32 frequencies are taken as they are
    f32 = f.float()
    got = mh.rotary(qg, None, f32, pg, interleaved=interleaved)
    near("fp32 frequencies", got, mx.rotary(q, f32.double().cpu().numpy(), ph - offset, interleaved), np.abs(q).max() * 2, 16)


def test_rotary_gradient_and_strides():
    B, H, HK, L, D = 2, 4, 2, 19, 24
    f, _ = mh.rotary_frequencies(16, 1e4)
    room = torch.randn(B, L, (H + HK) * D + 3, device="cuda")
    q = room[..., 1:1 + H * D].unflatten(-1, (H, D)).transpose(1, 2)
    k = room[..., 1 + H * D:-2].unflatten(-1, (HK, D)).transpose(1, 2)
    pos = torch.arange(L, device="cuda").expand(B, L)
    a, b = mh.rotary(q, k, f, pos)
    near("q", a, mx.rotary(host(q), f.cpu().numpy(), np.arange(L)), np.abs(host(q)).max() * 2, 8)
    near("k", b, mx.rotary(host(k), f.cpu().numpy(), np.arange(L)), np.abs(host(k)).max() * 2, 8)
    assert torch.equal(mh.rotary(q[:1].expand(B, -1, -1, -1), None, f, pos)[1], mh.rotary(q[:1], None, f, pos[:1])[0])
    ql, kl = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    da, db = torch.randn_like(a), torch.randn_like(b)
    o = mh.rotary(ql, kl, f, pos, scale=1.3)
    dq, dk = torch.autograd.grad(o, (ql, kl), (da, db), retain_graph=True)
    want = mh.rotary(da, db, f, pos, scale=1.3, inverse=True)
    assert torch.equal(dq, want[0]) and torch.equal(dk, want[1])
    assert torch.equal(torch.autograd.grad(o[1], kl, db)[0], dk)
    assert torch.equal(torch.autograd.grad(mh.rotary(ql, None, f, pos, scale=1.3), ql, da)[0], dq)
    for e in (torch.zeros(0, 2, 5, 24, device="cuda"), torch.zeros(2, 2, 0, 24, device="cuda")):
        assert mh.rotary(e, e, f)[0].shape == e.shape


def test_rotary_streams_and_graphs():
    q, k = torch.randn(2, 4, 33, 64, device="cuda", dtype=BF), torch.randn(2, 2, 33, 64, device="cuda", dtype=BF)
    f, _ = mh.rotary_frequencies(64)
    on_stream_and_captured(lambda q, k, p: mh.rotary(q, k, f, p), [q, k, torch.arange(33, device="cuda")])


def test_rotary_refusals():
    q = torch.zeros(1, 2, 3, 8, device="cuda")
    f = torch.ones(4, device="cuda")
    for call in (lambda: mh.rotary(q[0], None, f), lambda: mh.rotary(q, q[:, :, :2], f), lambda: mh.rotary(q, q.bfloat16(), f),
                 lambda: mh.rotary(q, None, torch.ones(5, device="cuda")), lambda: mh.rotary(q, None, f[:0]),
                 lambda: mh.rotary(q, None, f.half()), lambda: mh.rotary(q, None, f, torch.zeros(3, device="cuda")),
                 lambda: mh.rotary(q, None, f, torch.zeros(4, device="cuda", dtype=torch.int64)),
                 lambda: mh.rotary(q.half(), None, f), lambda: mh.rotary(q, None, f.cpu()),
                 lambda: mh.rotary(q, None, f.clone().requires_grad_(True))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()


# ------------------------------------------------------------------------------------------------ group norm

def norm_inputs(shape, dtype, wdtype, mean=0.0, seed=0):
    x = (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) + mean).to(dtype)
    C = shape[-1]
    w, wg = draw(seed + 1, C, dtype=wdtype) if wdtype else (None, None)
    b, bg = draw(seed + 2, C, dtype=wdtype) if wdtype else (None, None)
    return (x.double().numpy(), w, b), (x.cuda(), wg, bg)


def norm_scales(x, w, b, G, stats, eps):
    """|x - mean| as fp32 sees it, turned to z's scale: the value, the group's own deviation and a rounding of the mean."""
    mu, r = np.abs(stats[:, None, :, :1]), stats[:, None, :, 1:]
    xg = x.reshape(x.shape[0], -1, G, x.shape[-1] // G)
    c = (np.abs(xg - stats[:, None, :, :1]) + mu + np.abs(xg)) * r
    c = np.broadcast_to(c, xg.shape).reshape(x.shape)
    c = c if w is None else c * np.abs(w)
    return c if b is None else c + np.abs(b)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("shape,G,wdtype,mean", [
    ((1, 1), 1, F32, 0), ((5, 8), 2, None, 0), ((300, 96), 4, F32, 0), ((7, 1, 2048), 16, BF, 2), ((33, 1000), 1, F32, 0),
    ((9, 1, 520), 1, F32, -1), ((2, 37, 30), 5, F32, 0), ((3, 5, 7, 48), 3, BF, 1), ((2, 1000, 512), 32, F32, 3),
    ((1, 4097, 24), 24, None, 0), ((2, 3, 5000), 2, F32, 0), ((4, 64, 64), 64, F32, 0),
])
def test_group_norm(dtype, silu, shape, G, wdtype, mean):
    (x, w, b), (xg, wg, bg) = norm_inputs(shape, dtype, wdtype, mean)
    act = "silu" if silu else None
    say(f"group norm {shape} G={G} {dtype} {wdtype} {act}")
    y, stats = mh.group_norm(xg, G, wg, bg, 1e-3, activation=act, return_stats=True)
    ry, rs = mx.group_norm(x, G, w, b, 1e-3, silu)
    mag = norm_scales(x, w, b, G, rs, 1e-3)
    # mean and deviation, centring, two products, the bias, and for the activation an exponential, a sum, a quotient
    # whose slope is at most 1.1: 16 roundings
    near("y", y, ry, mag, 16)
    near("mean", stats[..., 0], rs[..., 0], np.abs(rs[..., 0]) + 1 / rs[..., 1], 4)
    near("rstd", stats[..., 1], rs[..., 1], rs[..., 1] * (1 + np.abs(rs[..., 0]) * rs[..., 1]), 16)
    assert y.shape == xg.shape and y.dtype is dtype
    dy, dyg = draw(5, *shape, dtype=dtype)
    sh = stats.double().cpu().numpy()
    rdx, rdw, rdb = mx.group_norm_bwd(dy, x, sh, G, w, b, silu)
    dx, dw, db = mh.group_norm_bwd(dyg, xg, stats, G, wg, bg, activation=act)
    # what enters dx: the terms' magnitudes through the same formula.  c is off by 8 roundings of mag, g by as many
    amag = norm_scales(x, None, None, G, rs, 1e-3)
    slope = 1.1 + 0.25 * mag if silu else 1.0    # the activation's slope, and how far z's error moves it
    gmag = np.abs(dy) * slope * (1 if w is None else np.abs(w)) * (1 + mag * (0.5 if silu else 0))
    gg, cg = (a.reshape(shape[0], -1, G, shape[-1] // G) for a in (gmag, amag))
    r = rs[:, None, :, 1:]
    scale = r * (gg + gg.mean((1, 3), keepdims=True) + cg * (gg * cg).mean((1, 3), keepdims=True))
    near("dx", dx, rdx, scale.reshape(shape), 32)
    if wdtype:
        axes = tuple(range(len(shape) - 1))
        dmag = np.abs(dy) * slope * (1 + mag * (0.5 if silu else 0))
        near("dw", dw, rdw, (dmag * amag).sum(axes), 32)
        near("db", db, rdb, dmag.sum(axes), 32)
    else:
        assert dw is None and db.dtype is dtype
    leaves = [None if a is None else a.detach().requires_grad_(True) for a in (xg, wg, bg)]
    out = mh.group_norm(*(leaves[0], G, *leaves[1:]), 1e-3, activation=act)
    assert torch.equal(out, y)
    auto = torch.autograd.grad(out, [a for a in leaves if a is not None], dyg)
    for got, want in zip(auto, (dx, dw, db) if wdtype else (dx,)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape,G", [((64, 256), 4), ((2, 500, 64), 4)])
def test_group_norm_of_constant_and_far_values(dtype, shape, G):
    """Groups without a deviation give the bias; a mean far above the deviation keeps the deviation's digits."""
    x = torch.full(shape, 3.25, dtype=dtype, device="cuda")
    b = torch.randn(shape[-1], device="cuda")
    y, stats = mh.group_norm(x, G, None, b, 1e-5, return_stats=True)
    assert torch.equal(y, b.to(dtype).expand(shape)) and (stats[..., 0] == 3.25).all()
    if dtype is F32:
        x = torch.randn(*shape, device="cuda") + 4096.0
        y, stats = mh.group_norm(x, G, return_stats=True)
        ry, rs = mx.group_norm(host(x), G)
        # the fp32 mean is off by half a step of 4096 (2^-12): relative to the deviation as much
        assert np.abs(host(y) - ry).max() <= 2.0 ** -12 * 1.5
        assert np.abs(host(stats[..., 1]) / rs[..., 1] - 1).max() <= 2.0 ** -16


def test_group_norm_nonfinite_stays_in_its_group():
    for shape, G in (((6, 64), 4), ((2, 300, 64), 4)):
        x = torch.randn(*shape, device="cuda")
        want = mh.group_norm(x, G)
        x[1, ..., 20] = float("nan")             # group 1 of entry 1
        got = mh.group_norm(x, G)
        keep = torch.ones(shape, dtype=torch.bool)
        keep[1, ..., 16:32] = False
        assert torch.equal(got.cpu()[keep], want.cpu()[keep]) and got.cpu()[~keep].isnan().all()


def test_group_norm_strides_and_empty():
    x = torch.randn(3, 50, 200, device="cuda")
    w = torch.randn(64, device="cuda")
    for view in (x[..., 7:71], x[:, ::3, :64], x[:, :64].transpose(1, 2)[..., :48], x[:1, :, :64].expand(3, -1, -1), x[:, 0, 3:67]):
        G, wv = 4, w[:view.shape[-1]]
        assert torch.equal(mh.group_norm(view, G, wv), mh.group_norm(view.contiguous(), G, wv))
        _, st = mh.group_norm(view, G, wv, return_stats=True)
        for a, b in zip(mh.group_norm_bwd(view, view, st, G, wv), mh.group_norm_bwd(*(view.contiguous(),) * 2, st, G, wv)):
            assert torch.equal(a, b)
    for shape in ((0, 5, 64), (3, 0, 64)):
        e = torch.zeros(shape, device="cuda", requires_grad=True)
        wl = w.clone().requires_grad_(True)
        y = mh.group_norm(e, 4, wl)
        assert y.shape == shape
        de, dw = torch.autograd.grad(y.sum(), (e, wl))
        assert de.shape == shape and (dw == 0).all()


def test_group_norm_autograd_of_parts():
    x, w, b = torch.randn(10, 3, 64, device="cuda"), *torch.randn(2, 64, device="cuda")
    dy = torch.randn_like(x)
    _, st = mh.group_norm(x, 4, w, b, return_stats=True)
    want = mh.group_norm_bwd(dy, x, st, 4, w, b, activation="silu")
    for i in range(3):
        t = [a.detach().requires_grad_(j == i) for j, a in enumerate((x, w, b))]
        got, = torch.autograd.grad(mh.group_norm(t[0], 4, t[1], t[2], activation="silu"), t[i], dy)
        assert torch.equal(got, want[i])
    assert mh.group_norm_bwd(dy, x, st, 4, w, b, need_bias=False)[2] is None
    y, stats = mh.group_norm(x.requires_grad_(True), 4, w, b, return_stats=True)
    assert y.requires_grad and not stats.requires_grad
    assert mh.group_norm_bwd(dy.bfloat16(), x.detach().bfloat16(), st, 4, dtype=F32)[2].dtype is F32


def test_group_norm_refusals():
    x = torch.zeros(2, 3, 12, device="cuda")
    st = torch.zeros(2, 4, 2, device="cuda")
    for call in (lambda: mh.group_norm(x, 5), lambda: mh.group_norm(x, 0), lambda: mh.group_norm(x[0, 0], 1),
                 lambda: mh.group_norm(x, 4, torch.zeros(11, device="cuda")), lambda: mh.group_norm(x.half(), 4),
                 lambda: mh.group_norm(x, 4, torch.zeros(12, device="cuda"), torch.zeros(12, device="cuda", dtype=BF)),
                 lambda: mh.group_norm(x, 4, activation="gelu"), lambda: mh.group_norm(x, 4, eps=-1.0),
                 lambda: mh.group_norm_bwd(x[:1], x, st, 4), lambda: mh.group_norm_bwd(x, x, st[:1], 4),
                 lambda: mh.group_norm_bwd(x, x, st, 4, dtype=torch.float16), lambda: mh.group_norm(x.cpu(), 4),
                 lambda: mh.group_norm(torch.zeros(1, 65537, device="cuda"), 1)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()


def test_group_norm_streams_and_graphs():
    for shape, G in (((40, 256), 4), ((2, 300, 96), 8)):
        x, w = torch.randn(*shape, device="cuda"), torch.randn(shape[-1], device="cuda")

        def step(x, w):
            xl, wl = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
            y = mh.group_norm(xl, G, wl, activation="silu")
            return (y.detach(), *torch.autograd.grad(y, (xl, wl), x))
        on_stream_and_captured(step, [x, w])


# ------------------------------------------------------------------------------------------------ past 32 bits

def test_large_delta():
    """Workspaces of more than 4 GiB and results of 2^29 elements: the last sequence's bits are those of it alone, which
    takes other workgroups."""
    B, H, HK, L, dk, dv = 16, 32, 16, 8192, 128, 128
    gen = torch.Generator("cuda").manual_seed(1)
    q, k = (torch.nn.functional.normalize(torch.randn(B, HK, L, dk, device="cuda", generator=gen), dim=-1).to(BF) for _ in range(2))
    v, do = (torch.randn(B, H, L, dv, device="cuda", generator=gen, dtype=BF) for _ in range(2))
    g, beta = -torch.rand(B, H, L, device="cuda", generator=gen), torch.rand(B, H, L, device="cuda", generator=gen)
    say("delta with more than 4 GiB of workspace")
    o, s = mh.gated_delta_rule(q, k, v, g, beta, return_final_state=True)
    last = [a[-1:] for a in (q, k, v, g, beta)]
    o1, s1 = mh.gated_delta_rule(*last, return_final_state=True)
    assert torch.equal(o[-1:], o1) and torch.equal(s[-1:], s1)
    grads = mh.gated_delta_rule_bwd(do, q, k, v, g, beta)
    for a, b in zip(grads[:5], mh.gated_delta_rule_bwd(do[-1:], *last)[:5]):
        assert torch.equal(a[-1:], b)


def test_large_step():
    B, H = 4097, 32
    state = torch.randn(B, H, 128, 128, device="cuda")
    q, k, v = (torch.randn(B, H, 128, device="cuda", dtype=BF) for _ in range(3))
    say("step of 2^31 state elements")
    tail, out = state[-2:].clone(), mh.gated_delta_step(state, q, k, v)
    assert torch.equal(out[-2:], mh.gated_delta_step(tail, q[-2:], k[-2:], v[-2:])) and torch.equal(state[-2:], tail)


def test_large_rotary_and_norm():
    n = (1 << 24) + 5
    x = torch.randn(1, 1, n, 128, device="cuda", dtype=BF)
    f, _ = mh.rotary_frequencies(128)
    say("rotary of 2^31 elements")
    y = mh.rotary(x, None, f)
    assert torch.equal(y[:, :, -9:], mh.rotary(x[:, :, -9:], None, f, offset=n - 9))
    for x in (x.view(n, 128), x.view(1, n, 128)):
        say(f"group norm of {tuple(x.shape)}")
        y, st = mh.group_norm(x, 4, return_stats=True)
        dx, _, db = mh.group_norm_bwd(x, x, st, 4, dtype=F32)
        if x.dim() == 2:
            y1, st1 = mh.group_norm(x[-9:], 4, return_stats=True)
            assert torch.equal(y[-9:], y1) and torch.equal(dx[-9:], mh.group_norm_bwd(x[-9:], x[-9:], st1, 4)[0])
        else:
            m, r = st[0, :, 0].repeat_interleave(32), st[0, :, 1].repeat_interleave(32)
            want = (x[0, -9:].float() - m) * r
            assert (y[0, -9:].float() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
        assert torch.isfinite(db).all()


# ------------------------------------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", [F32, BF])
def test_a_mixer_of_all_three(dtype):
    """Rotary positions, the delta rule and a norm of its heads as a layer runs them: a prompt in two parts, then single
    tokens, and the gradients of the whole, each against the operators of the oracle in a row."""
    B, H, HK, L, dk, dv = 2, 4, 2, 150, 32, 48
    x, t = delta_inputs(B, H, HK, L, dk, dv, dtype)
    w, wg = draw(20, H * dv)
    f, _ = mh.rotary_frequencies(16, 1e4)
    fh = f.cpu().numpy()

    def norm(o):                                 # (B, H, l, dv) -> a group a head of each token
        return mh.group_norm(o.transpose(1, 2).reshape(-1, H * dv), H, wg, activation="silu").view(B, -1, H, dv)

    def layer(q, k, v, g, b, state, at):
        q, k = mh.rotary(q, k, f, offset=at)
        return mh.gated_delta_rule(q, k, v, g, b, initial_state=state, return_final_state=True)

    xq, xk = mx.rotary(x[0], fh, np.arange(L)), mx.rotary(x[1], fh, np.arange(L))
    ro, rs = mx.delta_rule(xq, xk, *x[2:5], None, x[5])
    ry, rst = mx.group_norm(ro.transpose(0, 2, 1, 3).reshape(-1, H * dv), H, w, None, 1e-5, True)
    ry = ry.reshape(B, L, H, dv)
    # q, k and o are rounded to the type: each half a step of its norm, and the norm divides by o's own size
    half = torch.finfo(dtype).eps / 2
    got, state = [], t[5]
    for a, b in ((0, 70), (70, 146)):
        o, state = layer(*(c[:, :, a:b] for c in t[:5]), state, a)
        got.append(norm(o))
    for i in range(146, L):
        q, k = mh.rotary(t[0][:, :, i:i + 1], t[1][:, :, i:i + 1], f, offset=i)
        o = mh.gated_delta_step(state, q[:, :, 0], k[:, :, 0], *(c[:, :, i] for c in t[2:5]))
        got.append(norm(o[:, :, None]))
    y = torch.cat(got, 1)
    norm_of = lambda a: np.linalg.norm(a.reshape(-1))
    err, size = norm_of(host(y) - ry), norm_of(ry)
    say(f"layer {dtype}: {err / size:.2e}")
    # five roundings (q, k, o, y; k enters twice) and the fp32 arithmetic, on a norm whose slope is at most 3 here
    assert err <= 3 * (5 * half + 24 * 2.0 ** -20 * 2) * size
    whole, s = layer(*t[:5], t[5], 0)
    assert norm_of(host(s) - host(state)) <= (5 * half + 24 * 2.0 ** -20) * norm_of(rs)

    leaves = [a.detach().requires_grad_(True) for a in t]
    o, s = layer(*leaves[:5], leaves[5], 0)
    dy, dyg = draw(30, B, L, H, dv, dtype=dtype)
    grads = torch.autograd.grad(norm(o), leaves, dyg)
    rows = ro.transpose(0, 2, 1, 3).reshape(-1, H * dv)
    dro = mx.group_norm_bwd(dy.reshape(-1, H * dv), rows, rst, H, w, None, True)[0]
    dro = dro.reshape(B, L, H, dv).transpose(0, 2, 1, 3)
    refs = list(mx.delta_rule_bwd(dro, xq, xk, *x[2:5], None, x[5]))
    refs[0], refs[1] = (mx.rotary(a, fh, np.arange(L), inverse=True) for a in refs[:2])
    for name, got, want in zip(("dq", "dk", "dv", "dg", "dbeta", "dstate"), grads, refs):
        e = norm_of(host(got) - want) / norm_of(want)
        say(f"{name}: {e:.2e}")
        # the way back doubles it: o's rounding moves the norm's slope, do and the gradients are rounded too
        assert e <= 3 * (10 * half + 48 * 2.0 ** -20 * 2), name
