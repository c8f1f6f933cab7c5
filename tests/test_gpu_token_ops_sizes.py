"""Token operators at sizes of training batches: the kernels that only many rows, long pieces or tensors beyond the 256 MB cache
reach, against the float64 oracle (of large calls on rows that include the first, the last and those at the cache's border).

Tolerances as for the small sizes: half a step of the result's type and a counted number of fp32 roundings.
"""

import numpy as np
import pytest
import torch

import mamformer_amd as mh
from oracle import tokens as tk
from tests.gpu_helpers import host, say
from tests.test_gpu_token_ops import K_Y, check_bwd, check_logprobs, near, norm_scales

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
CACHE = 256 << 20


def normal(seed, *shape, std=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def rows_of(R, *extra):
    """The first and last rows, some between, and rows around each of `extra`."""
    around = [e + d for e in extra for d in (-2, -1, 0, 1)]
    some = np.random.default_rng(R).integers(0, R, 40).tolist()
    return torch.tensor(sorted({r for r in [0, 1, 2, R - 3, R - 2, R - 1, *around, *some] if 0 <= r < R}), device="cuda")


# ------------------------------------------------------------------------------------------------ token table

# pieces of 16, 32 and 8 tokens in two and three slabs of columns; pieces of 128 and of 256 in one
@pytest.mark.parametrize("T,V,D", [(20001, 3000, 2050), (40003, 700, 4100), (9000, 5000, 4096), (300007, 1500, 520),
                                   (600011, 90, 520)])
def test_embedding_gradient_of_training_batches(T, V, D):
    """Runs that cross pieces of every length in several slabs of columns; whole numbers, so every sum is exact."""
    g = torch.Generator(device="cuda").manual_seed(T)
    ids = (torch.rand(T, generator=g, device="cuda") ** 4 * V).long().clamp_(0, V - 1)
    ids[torch.rand(T, generator=g, device="cuda") < 0.05] = V - 1
    ids[torch.rand(T, generator=g, device="cuda") < 0.02] = -7         # out of range
    dy = torch.randint(-4, 5, (T, D), generator=g, device="cuda", dtype=torch.int8).to(BF)
    say(f"embedding gradient T={T} V={V} D={D}")
    live = ids >= 0
    for pad in (None, V - 1):
        keep = live if pad is None else live & (ids != pad)
        want = torch.zeros(V, D, device="cuda", dtype=torch.float64)
        for lo in range(0, T, 65536):
            s = slice(lo, lo + 65536)
            want.index_add_(0, ids[s][keep[s]], dy[s][keep[s]].double())
        for dtype in (F32, BF):
            got = mh.embedding_bwd(dy, ids, V, padding_idx=pad, dtype=dtype)
            assert torch.equal(got, want.float().to(dtype)), (pad, dtype)


# ------------------------------------------------------------------------------------------------ layer norm

# more than 1024 rows of 513 to 2048 channels (a wave a row), 8 million elements of up to 512 channels (two rows a group, and one left)
@pytest.mark.parametrize("R,D,dtype", [(1100, 1000, BF), (1500, 1024, F32), (1200, 2048, BF), (1031, 1537, F32), (131075, 64, BF),
                                       (70001, 128, BF), (35003, 250, F32), (17001, 500, BF)])
def test_layer_norm_forward_of_many_rows(R, D, dtype):
    x, res = normal(R, R, D, std=3.0, dtype=dtype), normal(R + 1, R, D, dtype=dtype)
    w, b = normal(R + 2, D), normal(R + 3, D)
    say(f"layer norm R={R} D={D} {dtype}")
    y, st = mh.layer_norm(x, w, b, return_stats=True)
    hs = host(x)
    ref, rst = tk.layer_norm(hs, host(w), host(b))
    near("y", y, ref, norm_scales(hs, host(w), host(b), 1e-5), K_Y)
    near("stats", st, rst, np.stack([np.abs(hs).mean(-1), rst[:, 1]], -1), K_Y)
    y, h, packed, st = mh.layer_norm(x, w, b, residual=res, packed=True, return_stats=True)
    assert torch.equal(h, (x.float() + res.float()).to(dtype))
    hs = host(h)
    ref, rst = tk.layer_norm(hs, host(w), host(b))
    near("y of the sum", y, ref, norm_scales(hs, host(w), host(b), 1e-5), K_Y)
    near("stats of the sum", st, rst, np.stack([np.abs(hs).mean(-1), rst[:, 1]], -1), K_Y)
    at = rows_of(R)
    codes, exps = tk.pack(hs[at.cpu().numpy()])
    assert np.array_equal(packed.codes[at].cpu().numpy(), codes) and np.array_equal(packed.exponents[at].cpu().numpy(), exps)
    alone = mh.pack_activations(h)                       # checked against the oracle at small sizes
    assert torch.equal(packed.codes, alone.codes) and torch.equal(packed.exponents, alone.exponents)


# each width's group of threads once; the four tensors of the forward, and of the backward, are above the cache's size
@pytest.mark.parametrize("R,D,dtype", [(600011, 60, BF), (350003, 100, BF), (90001, 200, F32), (70003, 512, BF), (35001, 1000, BF),
                                       (11003, 2047, F32), (17001, 2050, BF), (4501, 5000, F32), (3001, 12000, F32),
                                       (3001, 16384, BF)])
def test_layer_norm_beyond_the_cache(R, D, dtype):
    x, res = normal(R, R, D, dtype=dtype), normal(R + 1, R, D, dtype=dtype)
    assert 4 * x.nbytes > CACHE
    w, b = normal(R + 2, D), normal(R + 3, D)
    at = rows_of(R)
    say(f"layer norm beyond the cache R={R} D={D} {dtype}")
    y, h, packed, st = mh.layer_norm(x, w, b, residual=res, packed=True, return_stats=True)
    assert torch.equal(h, (x.float() + res.float()).to(dtype))
    hs = host(h[at])
    ref, rst = tk.layer_norm(hs, host(w), host(b))
    near("y", y[at], ref, norm_scales(hs, host(w), host(b), 1e-5), K_Y)
    near("stats", st[at], rst, np.stack([np.abs(hs).mean(-1), rst[:, 1]], -1), K_Y)
    alone = mh.pack_activations(h)
    assert torch.equal(packed.codes, alone.codes) and torch.equal(packed.exponents, alone.exponents)
    del x, res, y
    dy, d_h = normal(R + 4, R, D, dtype=dtype), normal(R + 5, R, D, dtype=dtype)
    for kept in (h, packed):
        dx, _, _ = mh.layer_norm_bwd(dy, kept, st, w, d_h=d_h)
        src = mh.unpack_activations(packed, F32) if kept is packed else h
        check_bwd(dx[at], None, None, host(dy[at]), host(src[at]), host(st[at]), host(w), host(d_h[at]))
        del dx, src


@pytest.mark.parametrize("R,D", [(600011, 60), (350003, 100), (131077, 200), (70003, 512), (35001, 1000), (20011, 2047),
                                 (17001, 2050), (9001, 5000), (5003, 12000)])
def test_layer_norm_parameter_sums_of_many_rows(R, D):
    """Every row enters dweight and dbias once: whole numbers and statistics (0, 1), so both sums are exact (below 2^24)."""
    g = torch.Generator(device="cuda").manual_seed(R)
    dy, h, d_h = (torch.randint(-4, 5, (R, D), generator=g, device="cuda", dtype=torch.int8).to(BF) for _ in range(3))
    st = torch.tensor([0.0, 1.0], device="cuda").expand(R, 2).contiguous()
    want = torch.zeros(2, D, device="cuda", dtype=torch.float64)
    for s in range(0, R, 8192):
        p = dy[s:s + 8192].double()
        want += torch.stack([(p * h[s:s + 8192]).sum(0), p.sum(0)])
    w = torch.ones(D, device="cuda")
    packed = mh.pack_activations(h)                      # holds whole numbers up to 127 exactly
    say(f"layer norm parameter sums R={R} D={D}")
    for kept in (h, packed):
        for dh in (None, d_h):                           # with it four tensors, above the cache's size
            _, dw, db = mh.layer_norm_bwd(dy, kept, st, w, d_h=dh)
            assert torch.equal(dw, want[0].float()) and torch.equal(db, want[1].float())


# ------------------------------------------------------------------------------------------------ log probabilities

@pytest.mark.parametrize("R,V,dtype", [(5003, 30011, BF), (1031, 70001, F32)])
def test_token_logprobs_beyond_the_cache(R, V, dtype):
    """Rows that go past the cache and rows that stay in it, forward and backward, into a tensor of its own and in place."""
    z = normal(R, R, V, std=3.0, dtype=dtype)
    border = R - CACHE // (V * z.element_size())         # the first row that stays
    assert 8 < border < R - 8
    at = rows_of(R, border)
    t = torch.randint(V, (R,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(V))
    t[at[1]], t[at[3]] = -100, V
    say(f"token logprobs beyond the cache R={R} V={V} {dtype} border={border}")
    out = mh.token_logprobs(z, t, temperature=0.9)
    zs, ts = host(z[at]), host(t[at]).astype(int)
    lnp, ent, k = check_logprobs(out._replace(logprobs=out.logprobs[at], entropy=out.entropy[at]), zs, ts, 0.9, 0)
    g, e = normal(1, R), normal(2, R)
    d = mh.token_logprobs_bwd(z, t, out.stats, g, e, temperature=0.9)
    ref = tk.token_logprobs_bwd(lnp, ent, ts, host(g[at]), host(e[at]), 0.9)
    p, hit = np.exp(lnp), np.zeros(zs.shape)
    live = (ts >= 0) & (ts < V)
    hit[np.nonzero(live)[0], ts[live]] = 1
    ga, ea = np.abs(host(g[at])) * live, np.abs(host(e[at]))
    scale = (ga[:, None] * (p + hit) + ea[:, None] * p * (1 - lnp + ent[:, None])) / 0.9
    near("dlogits", d[at], ref, scale, k + 4 * np.abs(lnp).max() + 8)
    mh.token_logprobs_bwd(z, t, out.stats, g, e, temperature=0.9, out=z)
    assert torch.equal(z, d)
