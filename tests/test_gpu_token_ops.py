"""Token table, layer norm, 8-bit activations and log probabilities on the GPU against the float64 oracle.

Tolerances.  A result of type T is rounded once: half a step, ``finfo(T).eps / 2`` of the value.  Before that come fp32
operations of 2^-24 each relative to the magnitudes that enter: ``near`` takes that scale (elementwise) and the number k of
roundings on the longest chain, counted in each test.  Where nothing is rounded the comparison is equality.
"""

import numpy as np
import pytest
import torch

import mamformer_amd as mh
from mamformer_amd._lib import MHError
from oracle import tokens as tk
from tests.gpu_helpers import dev, host, say

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def draw(seed, *shape, std=1.0, dtype=F32):
    """Normal values that `dtype` holds, as float64 on the host and on the GPU."""
    t = (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)
    return t.double().numpy(), t.cuda()


def near(name, out, ref, scale, k):
    half = torch.finfo(out.dtype).eps / 2
    o = host(out)
    assert o.shape == ref.shape, f"{name}: shape {o.shape}, expected {ref.shape}"
    fin = np.isfinite(ref)
    assert (np.isnan(o) == np.isnan(ref)).all(), f"{name}: NaN in other places"
    assert (o[~fin & ~np.isnan(ref)] == ref[~fin & ~np.isnan(ref)]).all(), f"{name}: infinities in other places"
    if not fin.any():
        return
    tol = half * np.abs(ref) + k * U * np.broadcast_to(scale, ref.shape) * (1 + half) + 1e-42
    worst = (np.abs(o - ref)[fin] / tol[fin]).max()
    say(f"{name}: error at most {worst:.2f} of the tolerance")
    assert worst <= 1, f"{name}: {worst:.2f} times the tolerance"


# ------------------------------------------------------------------------------------------------ token table

@pytest.mark.parametrize("shape,V,D,dtype,idx", [
    ((1,), 1, 1, BF, torch.int64), ((0,), 5, 8, F32, torch.int64), ((7,), 10, 3, BF, torch.int32),
    ((4, 16), 513, 64, BF, torch.int64), ((300,), 511, 65, F32, torch.int32), ((2, 513), 130, 2056, BF, torch.int64),
    ((1025,), 2000, 130, F32, torch.int64), ((3, 1000), 7, 16, BF, torch.int32),
    ((700,), 300001, 9, BF, torch.int64),                # three passes of the sort
])
def test_embedding(shape, V, D, dtype, idx):
    rng = np.random.default_rng(V + D)
    ids = rng.integers(0, V, shape)
    if ids.size > 6:                                     # out of range on both sides
        ids.reshape(-1)[[1, 5]] = [-3, V]
    W, Wg = draw(1, V, D, dtype=dtype)
    dy, dyg = draw(2, *shape, D, dtype=dtype)
    idg = torch.as_tensor(ids).to(idx).cuda()
    say(f"embedding {shape} V={V} D={D} {dtype}")
    out = mh.embedding(idg, Wg, scale=1.5)
    near("out", out, tk.embedding(ids, W, 1.5), 0.0, 0)  # 1.5 x is exact in fp32
    pad = V - 1
    for kw in (dict(), dict(padding_idx=pad), dict(padding_idx=-1, dtype=F32)):
        p = pad if "padding_idx" in kw else None
        dw = mh.embedding_bwd(dyg, idg, V, scale=1.5, **kw)
        assert dw.dtype is kw.get("dtype", dtype)
        ref = tk.embedding_bwd(dy, ids, V, 1.5, p)
        n = np.bincount(ids[(ids >= 0) & (ids < V)].reshape(-1), minlength=V).max() if ids.size else 0
        near(f"dweight {kw}", dw, ref, tk.embedding_bwd(np.abs(dy), ids, V, 1.5, p), n + 2)
        assert torch.equal(dw, mh.embedding_bwd(dyg, idg, V, scale=1.5, **kw))


@pytest.mark.parametrize("T,V,D", [(5000, 50, 40), (140000, 1000, 8), (20000, 30000, 24)])
def test_embedding_gradient_of_frequent_tokens(T, V, D):
    """Runs of one token over many pieces, tiles beyond the smallest, and a row that every other token asks for."""
    rng = np.random.default_rng(T)
    ids = np.minimum((V ** rng.random(T)).astype(np.int64) - 1, V - 1)
    ids[::2] = V // 2
    ids[T // 3:T // 2] = -1
    dy, dyg = draw(3, T, D, dtype=BF)
    say(f"embedding gradient T={T} V={V} D={D}")
    dw = mh.embedding_bwd(dyg, torch.as_tensor(ids).cuda(), V, dtype=F32)
    ref, mag = np.zeros((V, D)), np.zeros((V, D))
    np.add.at(ref, ids[ids >= 0], dy[ids >= 0])
    np.add.at(mag, ids[ids >= 0], np.abs(dy[ids >= 0]))
    near("dweight", dw, ref, mag, np.bincount(ids[ids >= 0]).max())
    assert torch.equal(dw, mh.embedding_bwd(dyg, torch.as_tensor(ids).cuda(), V, dtype=F32))


def test_embedding_of_one_token_only():
    dy, dyg = draw(4, 3000, 33)
    ids = torch.full((3000,), 2, dtype=torch.int32, device="cuda")
    dw = mh.embedding_bwd(dyg, ids, 4)
    ref = np.zeros((4, 33))
    ref[2] = dy.sum(0)
    mag = np.zeros((4, 33))
    mag[2] = np.abs(dy).sum(0)
    near("dweight", dw, ref, mag, 3000)
    assert not mh.embedding_bwd(dyg, ids, 4, padding_idx=2).any()
    assert not mh.embedding_bwd(dyg, ids + 2, 4).any()


def test_embedding_of_very_many_tokens():
    """More workgroups than a grid takes along one axis (64 tokens of one column each)."""
    W = torch.randn(5, 1, device="cuda")
    ids = torch.arange((1 << 26) + 3, device="cuda", dtype=torch.int32) % 5
    assert torch.equal(mh.embedding(ids, W), W[ids.long()])


@pytest.mark.parametrize("T", [1023, 1024, 1025, 16384, 16385])
def test_embedding_gradient_at_the_borders_of_the_sort(T):
    """Whole tiles, one token more and less, and both ways of counting; whole numbers, so every sum is exact."""
    V, D = 1500, 5
    g = torch.Generator(device="cuda").manual_seed(T)
    ids = torch.randint(-1, V, (T,), generator=g, device="cuda")
    dy = torch.randint(-8, 9, (T, D), generator=g, device="cuda").float()
    live = ids >= 0
    want = torch.zeros(V, D, device="cuda", dtype=torch.float64).index_add_(0, ids[live], dy[live].double())
    assert torch.equal(mh.embedding_bwd(dy, ids, V), want.float())


@pytest.mark.parametrize("T,D", [(2047, 40), (2048, 7), (2049, 40), (30000, 3), (70000, 130), (200000, 8)])
@pytest.mark.parametrize("V", [1, 40, 600, 300000])
def test_embedding_gradient_runs(T, D, V):
    """Runs shorter and longer than the pieces, over many of them, in every way of sorting (one workgroup, several that count
    by themselves, several that are counted for), with one to three passes; whole numbers, so every sum is exact."""
    if V == 300000 and D > 40:
        D = 40
    g = torch.Generator(device="cuda").manual_seed(T + V)
    ids = (torch.rand(T, generator=g, device="cuda") ** 4 * V).long().clamp_(0, V - 1)
    ids[torch.rand(T, generator=g, device="cuda") < 0.1] = V           # out of range
    dy = torch.randint(-4, 5, (T, D), generator=g, device="cuda").to(BF)
    say(f"embedding gradient runs T={T} V={V} D={D}")
    live = ids < V
    want = torch.zeros(V, D, device="cuda", dtype=torch.float64).index_add_(0, ids[live], dy[live].double())
    assert torch.equal(mh.embedding_bwd(dy, ids, V, dtype=F32), want.float())


@pytest.mark.parametrize("V", [1, 2, 33, 4096, 262144, 262145])
@pytest.mark.parametrize("T,D", [(1, 5), (16, 600), (17, 512), (31, 8), (33, 520), (1000, 513), (2048, 64)])
def test_embedding_gradient_of_few_tokens(T, D, V):
    """Rows with one token, with as many as a wave takes and with more, all rows alike, several columns' worth of workgroups."""
    g = torch.Generator(device="cuda").manual_seed(T + V)
    ids = torch.where(torch.rand(T, generator=g, device="cuda") < 0.5, min(V, 3) - 1,
                      torch.randint(-1, V + 1, (T,), generator=g, device="cuda"))
    dy = torch.randint(-4, 5, (T, D), generator=g, device="cuda").float()
    say(f"embedding gradient of few tokens T={T} V={V} D={D}")
    for pad in (None, V - 1):
        live = (ids >= 0) & (ids < V) if pad is None else (ids >= 0) & (ids < V) & (ids != pad)
        want = torch.zeros(V, D, device="cuda", dtype=torch.float64).index_add_(0, ids[live], dy[live].double())
        for dtype in (F32, BF):                  # sums up to 4096: bf16 rounds them once
            assert torch.equal(mh.embedding_bwd(dy, ids, V, padding_idx=pad, dtype=dtype), want.float().to(dtype))


def test_offsets_beyond_32_bits():
    """Rows 2^31 elements apart: every operator reads and writes them where they are."""
    D, far = 200, (1 << 31) + 64
    big = torch.empty(2 * far + D, device="cuda", dtype=BF)
    rows = big.as_strided((3, D), (far, 1))
    x = torch.randn(3, D, device="cuda").to(BF)
    rows.copy_(x)
    ids, w = torch.tensor([2, 0, 1, 2], device="cuda"), torch.randn(D, device="cuda").to(BF)
    assert torch.equal(mh.embedding(ids, rows), x[ids])
    assert torch.equal(mh.embedding_bwd(rows, ids[:3], 5), mh.embedding_bwd(x, ids[:3], 5))
    for p, q in zip(mh.layer_norm(rows, w, residual=rows, return_stats=True), mh.layer_norm(x, w, residual=x, return_stats=True)):
        assert torch.equal(p, q)
    _, st = mh.layer_norm(x, w, return_stats=True)
    for p, q in zip(mh.layer_norm_bwd(rows, rows, st, w, d_h=rows), mh.layer_norm_bwd(x, x, st, w, d_h=x)):
        assert torch.equal(p, q)
    assert torch.equal(mh.pack_activations(rows).codes, mh.pack_activations(x).codes)
    out, want = mh.token_logprobs(rows, ids[:3], top=3), mh.token_logprobs(x, ids[:3], top=3)
    assert all(torch.equal(p, q) for p, q in zip(out, want))
    d = mh.token_logprobs_bwd(x, ids[:3], want.stats, want.entropy)
    mh.token_logprobs_bwd(rows, ids[:3], want.stats, want.entropy, out=rows)
    assert torch.equal(rows, d)


def test_embedding_strides_and_autograd():
    W, Wg = draw(5, 20, 24, dtype=BF)
    wide = torch.zeros(20, 50, device="cuda", dtype=BF)
    wide[:, 3:27] = Wg
    ids = torch.arange(40, device="cuda").reshape(5, 8).t() % 21        # strided ids, one out of range
    want = tk.embedding(host(ids).astype(np.int64), W)
    assert np.array_equal(host(mh.embedding(ids, wide[:, 3:27])), want)
    assert np.array_equal(host(mh.embedding(ids, Wg.t().contiguous().t())), want)
    leaf = Wg.clone().requires_grad_(True)
    g = torch.randn(24, device="cuda").to(BF).expand(8, 5, 24)          # a gradient that is broadcast
    mh.embedding(ids, leaf, scale=2.0, padding_idx=4).backward(g)
    ref = tk.embedding_bwd(host(g), host(ids).astype(np.int64), 20, 2.0, 4)
    near("grad", leaf.grad, ref, np.abs(ref), 4)
    assert torch.equal(leaf.grad, mh.embedding_bwd(g, ids, 20, scale=2.0, padding_idx=4))


# ------------------------------------------------------------------------------------------------ layer norm

def norm_scales(h, w, b, eps):
    """Magnitudes that enter y: the products, the mean's share and the bias."""
    _, st = tk.layer_norm(h, None, None, eps)
    c = np.abs((h - st[:, :1]) * st[:, 1:])
    wa = np.abs(w) if w is not None else 1.0
    return (c.max(-1, keepdims=True) + (st[:, 1:] * np.abs(h).mean(-1, keepdims=True))) * wa \
        + (np.abs(b) if b is not None else 0.0)


# A row's sums: at most 32 values a thread one after another, 6 levels of a wave, 16 waves: 54 roundings, in the mean and
# again (halved by the root) in r, and 10 more on the way to y.
K_Y = 54 + 27 + 10


@pytest.mark.parametrize("dtype,wdtype", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("D", [1, 7, 64, 65, 100, 128, 200, 256, 500, 512, 999, 1024, 2048, 2050, 4095, 4096, 8192, 12000,
                               16384])
def test_layer_norm(D, dtype, wdtype):
    R = 19 if D <= 128 else 5
    x, xg = draw(D, R, D, std=3.0, dtype=dtype)
    x2, xg2 = draw(D + 1, R, D, dtype=dtype)
    w, wg = draw(D + 2, D, dtype=wdtype)
    b, bg = draw(D + 3, D, dtype=wdtype)
    say(f"layer norm R={R} D={D} {dtype} {wdtype}")
    y, st = mh.layer_norm(xg, wg, bg, return_stats=True)
    ref, rst = tk.layer_norm(x, w, b)
    near("y", y, ref, norm_scales(x, w, b, 1e-5), K_Y)
    y, h, packed, st = mh.layer_norm(xg, wg, None, 0.1, residual=xg2, packed=True, return_stats=True)
    hs = (x + x2).astype(np.float32)                     # both types: fp32 holds the sum of two bf16 well enough
    hs = torch.as_tensor(hs).to(dtype).double().numpy()
    assert np.array_equal(host(h), hs)
    ref, rst = tk.layer_norm(hs, w, None, 0.1)
    near("y of the sum", y, ref, norm_scales(hs, w, None, 0.1), K_Y)
    near("stats", st, rst, np.stack([np.abs(hs).mean(-1), rst[:, 1]], -1), K_Y)
    codes, exps = tk.pack(hs)
    assert np.array_equal(packed.codes.cpu().numpy(), codes) and np.array_equal(packed.exponents.cpu().numpy(), exps)
    # the backward, from the rows and from their 8-bit form
    dy, dyg = draw(D + 4, R, D, dtype=dtype)
    dh, dhg = draw(D + 5, R, D, dtype=dtype)
    st64 = host(st)
    for kept, src in ((h, hs), (packed, tk.unpack(codes, exps, D))):
        dx, dw, db = mh.layer_norm_bwd(dyg, kept, st, wg, d_h=dhg)
        check_bwd(dx, dw, db, dy, src, st64, w, dh)
        again = mh.layer_norm_bwd(dyg, kept, st, wg, d_h=dhg)
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def check_bwd(dx, dw, db, dy, h, st, w, dh, extra=0):
    rx, rw, rb = tk.layer_norm_bwd(dy, h, st, w, dh)
    c = np.abs((h - st[:, :1]) * st[:, 1:])
    # c carries 3 roundings relative to r (|h| + |mu|)
    cm = (np.abs(h) + np.abs(st[:, :1])) * st[:, 1:]
    g = np.abs(dy if w is None else dy * w)
    scale = st[:, 1:] * (g + g.mean(-1, keepdims=True) + cm * (g * cm).mean(-1, keepdims=True))
    near("dx", dx, rx, scale + (0 if dh is None else np.abs(dh)), 54 + 12)
    n = h.shape[0] + 32                                  # the rows one after another, and the joins
    if dw is not None:
        near("dweight", dw, rw, (np.abs(dy) * cm).sum(0), n + 4)
    if db is not None:
        near("dbias", db, rb, np.abs(dy).sum(0), n)


@pytest.mark.parametrize("R,D,dtype", [(5000, 64, BF), (9001, 128, BF), (2500, 100, F32), (3000, 512, BF), (2300, 1024, F32),
                                       (2100, 2048, BF), (700, 4096, BF), (600, 8000, F32), (300, 16384, BF)])
def test_layer_norm_backward_of_many_rows(R, D, dtype):
    """More rows than the workgroups take at once: every workgroup walks several."""
    x, xg = draw(R, R, D, dtype=dtype)
    dy, dyg = draw(R + 1, R, D, dtype=dtype)
    w, wg = draw(R + 2, D)
    _, st = mh.layer_norm(xg, wg, return_stats=True)
    say(f"layer norm backward R={R} D={D} {dtype}")
    check_bwd(*mh.layer_norm_bwd(dyg, xg, st, wg), dy, x, host(st), w, None)
    dx, dw, db = mh.layer_norm_bwd(dyg, xg, st, bias=False)
    assert dw is None and db is None
    check_bwd(dx, None, None, dy, x, host(st), None, None)


def test_layer_norm_edges():
    D = 96
    x = torch.randn(6, D, device="cuda")
    x[1] = 5.0                                           # no variance
    x[2, 7] = float("nan")
    x[3, 8] = float("inf")
    x[4] *= 1e18                                         # squares near the top of fp32
    y, st = mh.layer_norm(x, return_stats=True)
    good = mh.layer_norm(x[:1])
    assert torch.equal(y[0], good[0]) and not y[1].any()
    assert y[2].isnan().all() and y[3].isnan().any()
    ref, _ = tk.layer_norm(host(x[4:5]))
    near("large values", y[4:5], ref, norm_scales(host(x[4:5]), None, None, 1e-5), K_Y)
    dy = torch.randn(6, D, device="cuda")
    dx, _, db = mh.layer_norm_bwd(dy, x, st)
    assert dx[0].isfinite().all() and dx[1].isfinite().all() and dx[5].isfinite().all() and db.isfinite().all()
    # nothing at all
    y, st = mh.layer_norm(x[:0], return_stats=True)
    w = torch.ones(D, device="cuda")
    dx, dw, db = mh.layer_norm_bwd(dy[:0], x[:0], st, w)
    assert y.shape == (0, D) and dx.shape == (0, D) and not dw.any() and not db.any()


def test_layer_norm_strides():
    wide = torch.randn(3, 10, 100, device="cuda").to(BF)
    x = wide[:, :, 1:92]                                 # rows of 91 channels at odd addresses
    w = torch.randn(200, device="cuda")[::2][:91]
    want = mh.layer_norm(x.contiguous(), w.contiguous())
    assert torch.equal(mh.layer_norm(x, w), want)
    t = x.transpose(0, 1)
    assert torch.equal(mh.layer_norm(t, w), want.transpose(0, 1))
    assert torch.equal(mh.layer_norm(x.transpose(1, 2).contiguous().transpose(1, 2), w), want)
    one = torch.randn(91, device="cuda").to(BF).expand(4, 91)           # one row read four times
    assert torch.equal(mh.layer_norm(one, w), mh.layer_norm(one.contiguous(), w))
    _, st = mh.layer_norm(x, w, return_stats=True)
    dy = wide[:, :, 5:96]
    for p, q in zip(mh.layer_norm_bwd(dy, x, st, w, d_h=t.transpose(0, 1)),
                    mh.layer_norm_bwd(dy.contiguous(), x.contiguous(), st, w.contiguous(), d_h=x.contiguous())):
        assert torch.equal(p, q)


@pytest.mark.parametrize("packed", [False, True])
def test_layer_norm_autograd(packed):
    D = 72
    x, res = (torch.randn(2, 5, D, device="cuda", requires_grad=True) for _ in range(2))
    w, b = (torch.randn(D, device="cuda", requires_grad=True) for _ in range(2))
    out = mh.layer_norm(x, w, b, residual=res, packed=packed, return_stats=True)
    y, h = out[:2]
    dy, dh = torch.randn(2, 2, 5, D, device="cuda")
    gx, gr, gw, gb = torch.autograd.grad([y, h], [x, res, w, b], [dy, dh], retain_graph=True)
    dx, dw, db = mh.layer_norm_bwd(dy, out[2] if packed else h.detach(), out[-1], w, d_h=dh)
    assert torch.equal(gx, dx) and torch.equal(gr, dx) and torch.equal(gw, dw) and torch.equal(gb, db)
    assert torch.equal(torch.autograd.grad(h, x, dh, retain_graph=True)[0], dh)
    only, = torch.autograd.grad(y, [b], [dy])
    assert torch.equal(only, db)


def test_layer_norm_bias_alone():
    """A bias of 32 bits without a weight: its gradient is not rounded to the rows' 16."""
    x, dy = torch.randn(2, 700, 40, device="cuda").to(BF)
    b = torch.randn(40, device="cuda", requires_grad=True)
    y = mh.layer_norm(x, None, b)
    gb, = torch.autograd.grad(y, b, dy)
    ref, mag = host(dy).sum(0), np.abs(host(dy)).sum(0)
    assert gb.dtype is F32
    near("dbias", gb, ref, mag, 700 + 32)
    _, st = mh.layer_norm(x, return_stats=True)
    _, dw, db = mh.layer_norm_bwd(dy, x, st, dtype=F32)
    assert dw is None and torch.equal(db, gb) and mh.layer_norm_bwd(dy, x, st)[2].dtype is BF
    with pytest.raises(TypeError):
        mh.layer_norm_bwd(dy, x, st, dtype=torch.half)


def test_layer_norm_against_differences():
    """The directional derivative of the kernels' own forward: steps of 2^-6 leave a truncation of about 2^-12 (third
    order) and a rounding of 2^-24 * 2^6 of y's size, both against a derivative of the order of sqrt(R D)."""
    R, D, e = 4, 300, 2.0 ** -6
    x, w, b, dy, vx, vw, vb = (torch.randn(*s, device="cuda") for s in ((R, D), (D,), (D,), (R, D), (R, D), (D,), (D,)))
    y, st = mh.layer_norm(x, w, b, return_stats=True)
    dx, dw, db = mh.layer_norm_bwd(dy, x, st, w)
    f = lambda s: (mh.layer_norm(x + s * vx, w + s * vw, b + s * vb).double() * dy.double()).sum()
    num = float((f(e) - f(-e)) / (2 * e))
    got = float((dx.double() * vx).sum() + (dw.double() * vw).sum() + (db.double() * vb).sum())
    size = float((dx.norm() ** 2 + dw.norm() ** 2 + db.norm() ** 2) ** 0.5)
    say(f"derivative {got:.6f}, by differences {num:.6f}")
    assert abs(got - num) <= 2e-3 * size


# ------------------------------------------------------------------------------------------------ 8-bit activations

@pytest.mark.parametrize("D", [1, 9, 63, 64, 65, 128, 1000])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_pack(D, dtype):
    x, _ = draw(D, 40, D, dtype=F32)
    x[1] = 0
    x[2] *= 1e-38                                        # subnormal in both types
    x[3] *= 1e38 / np.abs(x[3]).max() * 3.3
    x[4] = 127
    x[5] = 127.5
    x[6] = -128
    x[7, D // 2] = np.inf
    x[8, 0] = np.nan
    x[9] = np.round(x[9] * 64) + 0.5                     # ties
    x[9, 0] = 127
    x[10] *= 2.0 ** np.arange(-60, D - 60).clip(-60, 60)
    xg = torch.as_tensor(x).to(dtype).cuda()
    x = host(xg)
    say(f"pack D={D} {dtype}")
    p = mh.pack_activations(xg)
    codes, exps = tk.pack(x)
    assert np.array_equal(p.exponents.cpu().numpy(), exps) and np.array_equal(p.codes.cpu().numpy(), codes)
    want = tk.unpack(codes, exps, D)
    for t in (BF, F32):
        assert np.array_equal(host(mh.unpack_activations(p, t)), want, equal_nan=True)
    assert mh.unpack_activations(p).dtype is dtype
    wide = torch.zeros(40, D + 3, device="cuda", dtype=dtype)
    wide[:, 1:D + 1] = xg
    q = mh.pack_activations(wide[:, 1:D + 1])
    assert torch.equal(q.codes, p.codes) and torch.equal(q.exponents, p.exponents)
    e = mh.pack_activations(xg[:0])
    assert mh.unpack_activations(e).shape == (0, D)


def test_packed_of_a_diverged_row():
    x = torch.randn(3, 128, device="cuda")
    x[1, 70] = float("nan")
    y, p, st = mh.layer_norm(x, packed=True, return_stats=True)
    dx, _, _ = mh.layer_norm_bwd(torch.ones_like(x), p, st, bias=False)
    assert dx[0].isfinite().all() and dx[1].isnan().all() and dx[2].isfinite().all()


# ------------------------------------------------------------------------------------------------ log probabilities

def logit_rows(seed, R, V, dtype):
    z, zg = draw(seed, R, V, std=3.0, dtype=dtype)
    rng = np.random.default_rng(seed)
    t = rng.integers(0, V, R)
    if R > 4:
        t[1], t[3] = -100, V + 7
    return z, zg, t, torch.as_tensor(t).cuda()


def check_logprobs(out, z, t, temp, top):
    lp, ent, ids, alt, lnp = tk.token_logprobs(z, t, temp, top)
    V = z.shape[1]
    fin = np.where(np.isfinite(z), np.abs(z), 0).max(-1) / temp
    # S: at most V / 256 + 8 sums of a thread, 6 + 4 joins of 4 roundings; the exponents' 2 roundings of |l|, entering by
    # their weights, at most ln V + 1 each; the same again through U
    k = 2 * (V / 256 + 48) + 4 * np.log(V + 1) + 16
    near("logprobs", out.logprobs, lp, 1 + fin, k)
    near("entropy", out.entropy, ent, 1 + np.log(V + 1) + fin, k)
    if top:
        assert np.array_equal(out.top_ids.cpu().numpy(), ids)
        near("top_logprobs", out.top_logprobs, alt, (1 + fin)[:, None], k)
    return lnp, ent, k


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,top,temp", [(1, 1, 1.0), (2, 0, 1.0), (7, 7, 0.5), (8, 3, 1.0), (255, 64, 1.3), (2048, 1, 1.0),
                                        (2049, 20, 0.7), (5003, 0, 1.0), (32000, 5, 1.0), (70001, 64, 1.0)])
def test_token_logprobs(V, top, temp, dtype):
    R = 9
    z, zg, t, tg = logit_rows(V, R, V, dtype)
    say(f"token logprobs V={V} top={top} temp={temp} {dtype}")
    out = mh.token_logprobs(zg, tg, temperature=temp, top=top)
    lnp, ent, k = check_logprobs(out, z, t, temp, top)
    g, gg = draw(V + 1, R)
    e, eg = draw(V + 2, R)
    for d_lp, d_ent in ((g, e), (g, None), (None, e)):
        d = mh.token_logprobs_bwd(zg, tg, out.stats, None if d_lp is None else gg, None if d_ent is None else eg,
                                  temperature=temp)
        ref = tk.token_logprobs_bwd(lnp, ent, t, d_lp, d_ent, temp)
        p, hit = np.exp(lnp), np.zeros((R, V))
        for r in range(R):
            if 0 <= t[r] < V:
                hit[r, t[r]] = 1
        ga = np.zeros(R) if d_lp is None else np.abs(d_lp) * hit.sum(-1)
        ea = np.zeros(R) if d_ent is None else np.abs(d_ent)
        scale = (ga[:, None] * (p + hit) + ea[:, None] * p * (1 - lnp + ent[:, None])) / temp
        near("dlogits", d, ref, scale, k + 4 * np.abs(lnp).max() + 8)


def test_token_logprobs_masks():
    V = 3001
    for dtype in (BF, F32):
        low = torch.finfo(dtype).min
        z = torch.randn(8, V, device="cuda").to(dtype)
        z[0, 5:] = -float("inf")
        z[1] = -float("inf")
        z[2] = low                                       # the type's lowest value everywhere: an even distribution
        z[3, 100:] = low
        z[4, 77] = float("nan")
        z[5, 78] = float("inf")
        z[6] = 0
        z[6, ::2] = -0.0
        z[7, 1:] = -float("inf")
        t = torch.tensor([7, 3, 11, 5, 0, 0, 9, 0], device="cuda")
        say(f"masked rows {dtype}")
        out = mh.token_logprobs(z, t, top=6)
        with np.errstate(invalid="ignore"):
            lnp, ent, k = check_logprobs_masked(out, host(z), host(t).astype(int))
        assert out.logprobs[7] == 0 and out.entropy[7] == 0
        g = torch.ones(8, device="cuda")
        d = mh.token_logprobs_bwd(z, t, out.stats, g, g)
        assert not d[1].any() and d[4].isnan().all() and d[5].isnan().any()
        ok = [0, 2, 3, 6, 7]
        assert d[ok].isfinite().all() and not d[0, 8:].any() and not d[7].any()
        assert not mh.token_logprobs_bwd(z, t, out.stats, 0 * g, None).any()


def check_logprobs_masked(out, z, t):
    lp, ent, ids, alt, lnp = tk.token_logprobs(z, t, 1.0, 6)
    bad = [5]                                            # +inf: NaN by the formula, whatever the order of operations
    assert np.isnan(host(out.logprobs)[bad]).all() and np.isnan(host(out.entropy)[bad]).all()
    keep = [0, 1, 2, 3, 4, 6, 7]
    assert np.array_equal(out.top_ids.cpu().numpy(), ids)
    near("logprobs", out.logprobs[keep], lp[keep], 16.0, 200)
    near("entropy", out.entropy[keep], ent[keep], 16.0, 200)
    near("top_logprobs", out.top_logprobs[keep], alt[keep], 16.0, 200)
    return lnp, ent, 200


@pytest.mark.parametrize("dtype", [BF, F32])
def test_alternatives_in_hard_orders(dtype):
    """Equal logits, rising and falling rows, and large values in few threads' shares, more than are ranked at once."""
    V = 65536
    z = torch.zeros(5, V, device="cuda")
    z[1] = torch.arange(V, device="cuda") / 64.0
    z[2] = -torch.arange(V, device="cuda") / 64.0
    at = (torch.arange(V // 2048, device="cuda")[:, None] * 2048 + torch.arange(0, 160, device="cuda")).reshape(-1)
    z[3, at] = 10 + torch.rand(at.numel(), device="cuda")
    z[4, at] = 7.0
    z = z.to(dtype)
    t = torch.zeros(5, dtype=torch.int64, device="cuda")
    for top in (1, 20, 64):
        say(f"alternatives {dtype} top={top}")
        out = mh.token_logprobs(z, t, top=top)
        order = np.lexsort((np.broadcast_to(np.arange(V), (5, V)), -host(z)))[:, :top]
        assert np.array_equal(out.top_ids.cpu().numpy(), order)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("temp", [0.4, 1.0, 3.0])
def test_long_rows_with_masks(temp, dtype):
    """Few long rows, which are cut into spans: spans that hold nothing, the type's lowest value in whole spans and in whole
    rows (over a temperature below 1 it leaves the type's range), a NaN, equal values over the borders."""
    V, top = 20011, 64
    low = torch.finfo(dtype).min
    z = torch.randn(7, V, device="cuda").to(dtype)
    z[0, 9000:] = -float("inf")
    z[0, :30] = -float("inf")
    z[1] = -float("inf")
    z[1, V - 3:] = torch.tensor([1.0, 3.0, 2.0], dtype=dtype, device="cuda")
    z[2] = low
    z[3, 5000:] = low
    z[4, 12345] = float("nan")
    z[5] = 0.25
    z[6] = low
    z[6, ::7] = -float("inf")
    t = torch.tensor([100, V - 2, 5, 3, 0, V - 1, 8], device="cuda")
    say(f"long masked rows {dtype} T={temp}")
    out = mh.token_logprobs(z, t, temperature=temp, top=top)
    with np.errstate(invalid="ignore"):
        lp, ent, ids, alt, lnp = tk.token_logprobs(host(z), host(t).astype(int), temp, top)
    assert np.array_equal(out.top_ids.cpu().numpy(), ids)
    with np.errstate(invalid="ignore"):                  # infinite and NaN entries are compared by their places
        # sums of V / 256 + 8 values a thread at most, 6 + 4 + 6 joins of 4 roundings, and |l| <= ln V + 6 / temp
        k = 2 * (V / 256 + 64) + 4 * np.log(V) + 16
        scale = 1 + np.log(V) + 6 / temp
        near("logprobs", out.logprobs, lp, scale, k)
        near("entropy", out.entropy, ent, scale, k)
        near("top_logprobs", out.top_logprobs, alt, scale, k)
        g = torch.linspace(0.5, 1.5, 7, device="cuda")
        d = mh.token_logprobs_bwd(z, t, out.stats, g, -g, temperature=temp)
        ok = [0, 1, 2, 3, 5, 6]
        ref = tk.token_logprobs_bwd(lnp, ent, host(t).astype(int), host(g), -host(g), temp)
        mag = np.exp(lnp) * (2 + ent[:, None] + np.where(np.isfinite(lnp), np.abs(lnp), 0))
        mag[np.arange(7), host(t).astype(int)] += 1
        near("dlogits", d[ok], ref[ok], mag[ok] * host(g)[ok, None] / temp, k + 4 * np.abs(lnp[ok][np.isfinite(lnp[ok])]).max() + 8)
    assert d[4].isnan().all()


def test_token_logprobs_of_very_many_rows():
    """More rows than a grid takes along one axis: each row is the same as in a call of its own."""
    R = (1 << 20) + 5
    z = torch.randn(R, 3, device="cuda").to(BF)
    t = torch.arange(R, device="cuda") % 3
    out = mh.token_logprobs(z, t, top=2)
    d = mh.token_logprobs_bwd(z, t, out.stats, out.entropy)
    for s in (slice(0, 9), slice(R - 9, R)):
        want = mh.token_logprobs(z[s], t[s], top=2)
        assert all(torch.equal(p[s], q) for p, q in zip(out, want))
        assert torch.equal(d[s], mh.token_logprobs_bwd(z[s], t[s], want.stats, want.entropy))


@pytest.mark.parametrize("V", [9, 65, 500, 520, 1024, 1537, 2047, 2048, 2056])
def test_alternatives_of_short_rows(V):
    """Rows with fewer chunks than threads, some with a wave that has none; small whole numbers make many ties."""
    g = torch.Generator(device="cuda").manual_seed(V)
    z = torch.randint(-3, 4, (6, V), generator=g, device="cuda").float()
    z[1, V // 3:] = -float("inf")
    z[2] = torch.randn(V, generator=g, device="cuda")
    z[3, V - 2] = float("nan")
    t = torch.zeros(6, dtype=torch.int64, device="cuda")
    for top in (1, 5, min(V, 64)):
        out = mh.token_logprobs(z, t, top=top)
        v = host(z)
        order = np.lexsort((np.broadcast_to(np.arange(V), v.shape), -np.where(np.isnan(v), np.inf, v), ~np.isnan(v)))[:, :top]
        assert np.array_equal(out.top_ids.cpu().numpy(), order)


def test_token_logprobs_strides_and_in_place():
    wide = torch.randn(2, 6, 515, device="cuda").to(BF)
    z = wide[:, :, 1:502]
    t = torch.randint(501, (6, 2), device="cuda", dtype=torch.int32).t()
    out = mh.token_logprobs(z, t, top=3, temperature=0.8)
    want = mh.token_logprobs(z.contiguous(), t.contiguous().long(), top=3, temperature=0.8)
    assert all(torch.equal(p, q) for p, q in zip(out, want)) and out.top_ids.shape == (2, 6, 3)
    g = torch.randn(1, device="cuda").expand(2, 6)
    d = mh.token_logprobs_bwd(z, t, out.stats, g, temperature=0.8)
    buf = z.contiguous()
    d2 = mh.token_logprobs_bwd(buf, t, out.stats, g, temperature=0.8, out=buf)
    assert d2 is buf and torch.equal(d, buf)
    with pytest.raises(RuntimeError):
        mh.token_logprobs_bwd(buf, t, out.stats, g, out=buf.transpose(0, 1).contiguous().transpose(0, 1))
    none = mh.token_logprobs(z[:, :0], t[:, :0], top=2)
    assert none.logprobs.shape == (2, 0) and none.top_ids.shape == (2, 0, 2)


def test_token_logprobs_autograd():
    z = torch.randn(5, 300, device="cuda", requires_grad=True)
    t = torch.tensor([0, 3, -100, 299, 7], device="cuda")
    out = mh.token_logprobs(z, t, top=2)
    g, e = torch.randn(2, 5, device="cuda")
    gz, = torch.autograd.grad([out.logprobs, out.entropy], [z], [g, e], retain_graph=True)
    assert torch.equal(gz, mh.token_logprobs_bwd(z.detach(), t, out.stats, g, e))
    gz, = torch.autograd.grad(out.logprobs.sum(), [z])
    assert torch.equal(gz, mh.token_logprobs_bwd(z.detach(), t, out.stats, torch.ones_like(g)))
    assert not out.top_logprobs.requires_grad and not gz[2].any()


def test_token_logprobs_against_differences():
    """As for the layer norm: steps of 2^-6, a truncation of about 2^-12 and a rounding of 2^-18 of the results' size."""
    z, v = torch.randn(2, 6, 500, device="cuda")
    z = 2 * z
    t = torch.arange(6, device="cuda")
    g, h = torch.randn(2, 6, device="cuda")
    out = mh.token_logprobs(z, t, temperature=0.9)
    d = mh.token_logprobs_bwd(z, t, out.stats, g, h, temperature=0.9)

    def f(s):
        o = mh.token_logprobs(z + s * v, t, temperature=0.9)
        return float((o.logprobs.double() * g + o.entropy.double() * h).sum())

    e = 2.0 ** -6
    num, got = (f(e) - f(-e)) / (2 * e), float((d.double() * v).sum())
    say(f"derivative {got:.6f}, by differences {num:.6f}")
    assert abs(got - num) <= 4e-3 * float(g.norm() + h.norm())


# ------------------------------------------------------------------------------------------------ streams, graphs, refusals

def test_another_stream_and_graphs():
    """Every operator on a stream of its own and in a graph that is replayed on changed inputs."""
    V, D, T = 700, 192, 1500
    W, x, res = torch.randn(V, D, device="cuda"), torch.randn(T, D, device="cuda"), torch.randn(T, D, device="cuda")
    w, b, z = torch.randn(D, device="cuda"), torch.randn(D, device="cuda"), torch.randn(T, V, device="cuda")
    ids = torch.randint(V, (T,), device="cuda")

    def all_of():
        y, h, p, st = mh.layer_norm(x, w, b, residual=res, packed=True, return_stats=True)
        o = mh.token_logprobs(z, ids, top=4)
        return [mh.embedding(ids, W), mh.embedding_bwd(x, ids, V), y, h, mh.unpack_activations(p),
                *mh.layer_norm_bwd(x, p, st, w), *mh.layer_norm_bwd(x, h, st, w), *o,
                mh.token_logprobs_bwd(z, ids, o.stats, st[:, 0].contiguous(), st[:, 1].contiguous()),
                mh.unpack_activations(mh.pack_activations(x))]

    want = all_of()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = all_of()
    for turn in range(3):
        for t in (x, res, z, W):
            t.copy_(torch.randn_like(t))
        ids.copy_(torch.randint(V, (T,), device="cuda"))
        want = all_of()
        graph.replay()
        torch.cuda.synchronize()
        say(f"replay {turn}")
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_python_refusals():
    x = torch.zeros(3, 8, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    st = torch.zeros(3, 2, device="cuda")
    p = mh.pack_activations(x)
    bad = [
        (TypeError, lambda: mh.embedding(ids.float(), x)), (TypeError, lambda: mh.embedding(ids, x.half())),
        (ValueError, lambda: mh.embedding(ids, x[0])), (ValueError, lambda: mh.embedding(ids, x, padding_idx=3)),
        (ValueError, lambda: mh.embedding_bwd(x, ids[:2], 4)), (TypeError, lambda: mh.embedding_bwd(x, ids, 4, dtype=torch.half)),
        (ValueError, lambda: mh.embedding_bwd(x, ids, 0)),
        (TypeError, lambda: mh.layer_norm(x.half())), (ValueError, lambda: mh.layer_norm(x, x[0, :4])),
        (ValueError, lambda: mh.layer_norm(x, residual=x[:2])), (TypeError, lambda: mh.layer_norm(x, x[0], x[0].to(BF))),
        (MHError, lambda: mh.layer_norm(torch.zeros(1, 16385, device="cuda"))),
        (ValueError, lambda: mh.layer_norm_bwd(x, x, st[:2])), (ValueError, lambda: mh.layer_norm_bwd(x, x[:2], st)),
        (ValueError, lambda: mh.layer_norm_bwd(x[:, :4], p, st)), (ValueError, lambda: mh.layer_norm_bwd(x, p._replace(dim=65), st)),
        (ValueError, lambda: mh.unpack_activations(p._replace(codes=p.codes[:, :32]))),
        (TypeError, lambda: mh.pack_activations(ids)),
        (ValueError, lambda: mh.token_logprobs(x, ids[:2])), (TypeError, lambda: mh.token_logprobs(x, ids.short())),
        (MHError, lambda: mh.token_logprobs(x, ids, top=9)), (MHError, lambda: mh.token_logprobs(x, ids, temperature=0)),
        (ValueError, lambda: mh.token_logprobs_bwd(x, ids, st)),
    ]
    for i, (err, call) in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {i} was taken")
