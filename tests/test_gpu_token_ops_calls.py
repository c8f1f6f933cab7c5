"""Token operators as torch sees their calls: in-place writes and autograd's checks, results that are overwritten, forward-mode
levels, gradients written beside or in place of the logits, outputs at the C entry points that are their inputs."""

import ctypes as ct

import pytest
import torch
from torch.autograd import forward_ad

import mamformer_amd as mh
from mamformer_amd import _lib
from tests.gpu_helpers import say

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------ in-place gradient

def loss_inputs(R=6, V=500):
    z = torch.randn(R, V, device="cuda")
    return z, torch.arange(R, device="cuda") % V


@pytest.mark.parametrize("reader", ["token_logprobs", "logsumexp"])
def test_gradient_in_place_of_saved_logits(reader):
    """Logits that a backward pass still has to read are written over: that pass must say so, not go on from the gradient."""
    z, t = loss_inputs()
    leaf = z.clone().requires_grad_(True)
    logits = leaf * 1.0
    y = mh.token_logprobs(logits, t).logprobs if reader == "token_logprobs" else torch.logsumexp(logits, -1)
    out = mh.token_logprobs(z, t)
    buf, was = logits.detach(), logits._version
    mh.token_logprobs_bwd(buf, t, out.stats, torch.ones(6, device="cuda"), out=buf)
    assert logits._version > was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradient_in_place_where_nothing_reads_the_logits_again():
    """The use that the argument is for: logits of a product, whose backward does not need them."""
    h, W = torch.randn(6, 32, device="cuda"), torch.randn(500, 32, device="cuda", requires_grad=True)
    t = torch.arange(6, device="cuda")
    logits = h @ W.t()
    want, = torch.autograd.grad(mh.token_logprobs(logits, t).logprobs.sum(), W, retain_graph=True)
    buf = logits.detach()
    out = mh.token_logprobs(buf, t)
    mh.token_logprobs_bwd(buf, t, out.stats, torch.ones(6, device="cuda"), out=buf)
    got, = torch.autograd.grad(logits, W, buf)
    assert torch.equal(got, want)
    with torch.inference_mode():                 # tensors without a version
        z = torch.randn(6, 500, device="cuda")
        out = mh.token_logprobs(z, t)
        want = mh.token_logprobs_bwd(z, t, out.stats, out.entropy)
        assert torch.equal(mh.token_logprobs_bwd(z, t, out.stats, out.entropy, out=z), want)


def test_gradient_into_a_leaf_is_refused():
    z, t = loss_inputs()
    out = mh.token_logprobs(z, t)
    g = torch.ones(6, device="cuda")
    leaf = z.clone().requires_grad_(True)
    for target in (leaf, leaf[:, :]):            # the leaf, and a view of it
        with pytest.raises(RuntimeError, match="leaf"):
            mh.token_logprobs_bwd(z, t, out.stats, g, out=target)
    assert torch.equal(leaf.detach(), z)
    with torch.no_grad():                        # as torch's own in-place operations
        mh.token_logprobs_bwd(z, t, out.stats, g, out=leaf)
    assert torch.equal(leaf.detach(), mh.token_logprobs_bwd(z, t, out.stats, g))


# ------------------------------------------------------------------------------------------------ results that are changed

def test_results_changed_in_place():
    """Log probabilities masked in place, entropies overwritten before the backward: the gradient is that of the masked sum."""
    z, t = loss_inputs()
    z.requires_grad_(True)
    drop = torch.arange(6, device="cuda") % 2 == 0
    out = mh.token_logprobs(z, t)
    want, = torch.autograd.grad((out.logprobs.masked_fill(drop, 0.0) * 3).sum() + out.entropy.clamp(min=0).sum(), z)
    out = mh.token_logprobs(z, t)
    out.logprobs.masked_fill_(drop, 0.0)
    out.logprobs.mul_(3)
    out.entropy.clamp_(min=0)
    got, = torch.autograd.grad(out.logprobs.sum() + out.entropy.sum(), z)
    assert torch.equal(got, want)
    out = mh.token_logprobs(z, t)
    want, = torch.autograd.grad((out.logprobs ** 2).sum(), z)
    out = mh.token_logprobs(z, t)
    loss = (out.logprobs ** 2).sum()             # keeps the log probabilities for its backward
    with torch.no_grad():
        out.entropy.zero_()
    got, = torch.autograd.grad(loss, z)
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------ forward mode

def test_forward_mode_is_refused():
    """The operators have no forward-mode rule: a call that a tangent reaches raises rather than drop it."""
    W, x = torch.randn(20, 8, device="cuda"), torch.randn(3, 8, device="cuda")
    w, b = torch.randn(2, 8, device="cuda")
    ids = torch.tensor([0, 4, 7], device="cuda")
    calls = {
        "embedding": (lambda p: mh.embedding(ids, p), W),
        "layer_norm x": (lambda p: mh.layer_norm(p, w, b), x),
        "layer_norm residual": (lambda p: mh.layer_norm(x, w, b, residual=p), x),
        "layer_norm weight": (lambda p: mh.layer_norm(x, p, b), w),
        "layer_norm bias": (lambda p: mh.layer_norm(x, w, p), b),
        "layer_norm packed": (lambda p: mh.layer_norm(p, w, b, packed=True, return_stats=True), x),
        "token_logprobs": (lambda p: mh.token_logprobs(p, ids), x),
    }
    first = lambda r: r if torch.is_tensor(r) else r[0]
    for what, (f, p) in calls.items():
        want = first(f(p))
        with forward_ad.dual_level():
            d = forward_ad.make_dual(p, torch.ones_like(p))
            for grad in (True, False):
                say(f"{what}, grad mode {grad}")
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    f(d)
            assert torch.equal(first(f(p)), want)        # a level alone, without a tangent, changes nothing


# ------------------------------------------------------------------------------------------------ temperature

@pytest.mark.parametrize("temp", [4.5e-39, 3e38])
def test_temperatures_at_the_ends_of_the_range(temp):
    """Towards 0 the largest logit has all the weight, towards infinity all have the same."""
    z = torch.tensor([[1.0, 3.0, 2.0, -5.0], [7.0, 7.0, -float("inf"), 0.0]], device="cuda")
    out = mh.token_logprobs(z, torch.tensor([1, 0], device="cuda"), temperature=temp, top=2)
    counts = torch.tensor([1.0, 2.0] if temp < 1 else [4.0, 3.0], device="cuda")
    # exponents, the sum, its base-2 logarithm and the way back: up to 16 roundings of numbers below 4
    assert (out.logprobs + counts.log()).abs().max() <= 16 * 4 * 2 ** -24
    assert (out.entropy - counts.log()).abs().max() <= 16 * 4 * 2 ** -24
    assert out.top_ids.tolist() == [[1, 2], [0, 1]]


@pytest.mark.parametrize("temp", [3.5e-39, 4.2e-39])
def test_temperature_whose_scale_leaves_the_range(temp):
    z, t = loss_inputs()
    st = mh.token_logprobs(z, t).stats
    with pytest.raises(_lib.MHError, match="temperature"):
        mh.token_logprobs(z, t, temperature=temp)
    with pytest.raises(_lib.MHError, match="temperature"):
        mh.token_logprobs_bwd(z, t, st, st[:, 2], temperature=temp)


# ------------------------------------------------------------------------------------------------ where outputs may lie

@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient_in_other_columns_of_the_logits_buffer(dtype):
    R, V = 7, 501
    t = torch.arange(R, device="cuda")
    for gap in (0, 3):
        wide = torch.randn(R, 2 * V + gap, device="cuda").to(dtype)
        left, right = wide[:, :V], wide[:, V + gap:]
        for z, d in ((left, right), (right, left)):
            keep = z.clone()
            out = mh.token_logprobs(z, t)
            want = mh.token_logprobs_bwd(keep, t, out.stats, out.entropy)
            assert torch.equal(mh.token_logprobs_bwd(z, t, out.stats, out.entropy, out=d), want)
            assert torch.equal(z, keep)
        with pytest.raises(_lib.MHError, match="overlap"):
            mh.token_logprobs_bwd(left, t, out.stats, out.entropy, out=wide[:, V - 1:2 * V - 1])


def test_gradient_of_one_row_of_any_stride():
    """A single row that is the transpose of a column has a row stride of 1."""
    z, t = torch.randn(500, 1, device="cuda").t(), torch.tensor([7], device="cuda")
    assert z.stride(0) == 1
    leaf = torch.randn(500, 1, device="cuda", requires_grad=True)
    got, = torch.autograd.grad(mh.token_logprobs(leaf.t(), t).logprobs.sum(), leaf)
    row = leaf.detach().reshape(1, 500).requires_grad_(True)
    want, = torch.autograd.grad(mh.token_logprobs(row, t).logprobs.sum(), row)
    assert torch.equal(got, want.t())
    out = mh.token_logprobs(z, t)
    want = mh.token_logprobs_bwd(z, t, out.stats, out.entropy)
    assert torch.equal(mh.token_logprobs_bwd(z, t, out.stats, out.entropy, out=torch.empty(500, 1, device="cuda").t()), want)
    assert torch.equal(mh.token_logprobs_bwd(z, t, out.stats, out.entropy, out=z), want)


@pytest.mark.parametrize("R,D", [(9, 64), (40, 1000), (1100, 1000), (5, 3000), (3, 9000)])
def test_layer_norm_in_place_at_the_c_entry(R, D):
    """y, h and dx may be the row tensors that they are computed from."""
    st = torch.cuda.current_stream().cuda_stream
    x, res, dy, d_h = torch.randn(4, R, D, device="cuda").to(BF)
    w, b = torch.randn(2, D, device="cuda")
    y, h, stats = mh.layer_norm(x, w, b, residual=res, return_stats=True)
    want = mh.layer_norm_bwd(dy, h, stats, w, d_h=d_h)

    def fwd(x, res, y, h):
        s = torch.empty(R, 2, device="cuda")
        a = _lib.LayerNormArgs(R, D, _lib.MH_BF16, _lib.MH_F32, 1e-5, x.data_ptr(), D, res.data_ptr(), D, w.data_ptr(),
                               b.data_ptr(), y.data_ptr(), D, h.data_ptr(), D, s.data_ptr(), None, None)
        _lib.call("mh_layer_norm_fwd", ct.byref(a), st)

    def bwd(dy, h, d_h, dx):
        dw, db = torch.empty(2, D, device="cuda")
        n = ct.c_size_t()
        a = _lib.LayerNormBwdArgs(R, D, _lib.MH_BF16, _lib.MH_F32, dy.data_ptr(), D, h.data_ptr(), D, None, None,
                                  stats.data_ptr(), w.data_ptr(), d_h.data_ptr(), D, dx.data_ptr(), D, dw.data_ptr(),
                                  db.data_ptr())
        _lib.call("mh_layer_norm_bwd_workspace_bytes", ct.byref(a), ct.byref(n))
        ws = torch.empty(max(n.value, 16), device="cuda", dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
        _lib.call("mh_layer_norm_bwd", ct.byref(a), st)
        torch.cuda.synchronize()
        return dw, db

    for y_in, h_in in ((0, 1), (1, 0)):                  # y over x and h over residual, and the other way round
        both = [x.clone(), res.clone()]
        fwd(*both, both[y_in], both[h_in])
        assert torch.equal(both[y_in], y) and torch.equal(both[h_in], h)
    for over in range(3):
        bufs = [dy.clone(), h.clone(), d_h.clone()]
        dw, db = bwd(*bufs, bufs[over])
        assert torch.equal(bufs[over], want[0]) and torch.equal(dw, want[1]) and torch.equal(db, want[2])


# ------------------------------------------------------------------------------------------------ rows out of range

@pytest.mark.parametrize("D", [40, 600, 2048, 5000, 12000])
def test_layer_norm_of_rows_out_of_range(D):
    """Squares or sums beyond fp32: NaN in that row, its statistics' scale and its gradient, and nowhere else."""
    x = torch.randn(5, D, device="cuda")
    want, ws = mh.layer_norm(x, return_stats=True)
    good = [0, 2, 4]
    x[1] *= 1e25
    x[3] = 3e38
    y, st = mh.layer_norm(x, return_stats=True)
    assert torch.equal(y[good], want[good]) and torch.equal(st[good], ws[good])
    assert y[[1, 3]].isnan().all() and st[[1, 3], 1].isnan().all()
    dx, _, _ = mh.layer_norm_bwd(torch.ones_like(x), x, st, bias=False)
    assert dx[good].isfinite().all() and dx[[1, 3]].isnan().all()
