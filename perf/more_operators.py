"""The operators around a linear-attention scan that corrects its state, as cases that can be timed and compared.

================  ===================================================================================
``delta``         gated delta rule over whole sequences, from a state and to one (prompts)
``delta_grad``    the same with the gradients of everything that enters (a training step)
``delta_step``    one token of every sequence, from a state into the next
``rotary``        rotary positions of queries and keys
``rotary_grad``   the same and its gradient
``gnorm``         group norm, channels last, with an activation
``gnorm_grad``    the same with the gradients of the rows, the weight and the bias
================  ===================================================================================

``run`` computes an operator from elementary torch operations in 32 bits, or, where ``own`` is true, by this package's
kernels; ``exact`` restates the definitions in float64, token by token.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_DEV = "cuda"
_C = 64                      # tokens that the plain form of the delta rule takes at once


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one sequence's next token through one layer of 16 heads: the smallest call, latency alone
        dict(name="step_one", kind="delta_step", dtype="bf16", B=1, H=16, HK=16, DK=128, DV=128),
        # the next token of a serving batch of 64, key heads shared by two value heads each
        dict(name="step_batch", kind="delta_step", dtype="bf16", B=64, H=32, HK=16, DK=128, DV=128),
        # a short prompt of odd length in 32 bits with odd head sizes, as a small verification run has it
        dict(name="prompt_odd", kind="delta", dtype="fp32", B=1, H=16, HK=8, L=333, DK=96, DV=80, init=False),
        # a serving batch's prompts, each going on from a cached state
        dict(name="prefill", kind="delta", dtype="bf16", B=4, H=16, HK=16, L=2048, DK=128, DV=128, init=True),
        # one long document in few heads: the scan's sequential case
        dict(name="document", kind="delta", dtype="bf16", B=1, H=8, HK=8, L=32768, DK=128, DV=128, init=False),
        # a training step's two sequences of 4096 tokens: the largest call
        dict(name="train", kind="delta_grad", dtype="bf16", B=2, H=16, HK=8, L=4096, DK=128, DV=128, init=False),
        # one token of 64 sequences at far positions
        dict(name="rotary_decode", kind="rotary", dtype="bf16", B=64, H=16, HK=8, L=1, D=128, RD=128, far=True,
             inter=False),
        # the queries and keys of a training step, both directions
        dict(name="rotary_train", kind="rotary_grad", dtype="bf16", B=2, H=16, HK=8, L=4096, D=128, RD=128, far=False,
             inter=False),
        # part of odd heads in 32 bits, neighbouring channels as pairs
        dict(name="rotary_part", kind="rotary_grad", dtype="fp32", B=3, H=10, HK=10, L=777, D=80, RD=48, far=True,
             inter=True),
        # the norm of each of 16 heads behind the scan, per token, with its backward pass
        dict(name="gnorm_heads", kind="gnorm_grad", dtype="bf16", wdtype="bf16", N=8192, S=1, C=2048, G=16, act="silu"),
        # sequences normalised over all their positions, forward only
        dict(name="gnorm_seq", kind="gnorm", dtype="bf16", wdtype="fp32", N=8, S=4096, C=512, G=32, act="silu"),
        # odd positions and channels in 32 bits without an activation, with the backward pass
        dict(name="gnorm_odd", kind="gnorm_grad", dtype="fp32", wdtype="fp32", N=3, S=1999, C=300, G=6, act=None),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))


def draw(rng):
    """A case of the ranges around the listed ones: sizes log-uniform, most of them odd."""
    kind = rng.choice(["delta", "delta", "delta", "delta_grad", "delta_grad", "delta_grad", "delta_step", "delta_step",
                       "rotary", "rotary_grad", "gnorm", "gnorm_grad", "gnorm_grad"])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if kind.startswith("delta"):
        HK = rng.choice([1, 2, 4, 8, 16, rng.randint(1, 12)])
        c.update(H=HK * rng.choice([1, 1, 2, 3]), HK=HK, DK=rng.choice([64, 128, 128, rng.randint(8, 128)]),
                 DV=rng.choice([64, 128, 128, rng.randint(8, 256)]))
        if kind == "delta_step":
            c["B"] = _log_int(rng, 1, 2048 // c["H"])
            return c
        top = (262144 if kind == "delta" else 131072) // c["H"] // (2 if c["dtype"] == "fp32" else 1) // (1 + c["DV"] // 129)
        c["L"] = _log_int(rng, 1, min(16384 if kind == "delta" else 4096, top))
        c.update(B=_log_int(rng, 1, min(64, max(1, top // c["L"]))), init=rng.random() < 0.5)
    elif kind.startswith("rotary"):
        D = rng.choice([64, 128, 256, 2 * rng.randint(8, 100)])
        HK = rng.choice([1, 4, 8, rng.randint(1, 16)])
        H = HK * rng.choice([1, 2, 4])
        L = _log_int(rng, 1, 8192)
        top = max(1, 16_000_000 // (D * (H + HK) * L))
        c.update(B=_log_int(rng, 1, min(256, top)), H=H, HK=HK, L=L, D=D,
                 RD=rng.choice([D, D, D // 4 * 2, 2 * rng.randint(1, D // 2)]), far=rng.random() < 0.5,
                 inter=rng.random() < 0.5)
    else:
        G = rng.choice([1, 4, 8, 16, 32, rng.randint(1, 40)])
        C = G * rng.choice([16, 32, 64, 128, rng.randint(2, 150)])
        per_token = rng.random() < 0.5
        most = 16_000_000 // (2 if c["dtype"] == "fp32" else 1)
        S = 1 if per_token else _log_int(rng, 2, min(8192, most // C))
        c.update(wdtype=rng.choice([c["dtype"], "fp32"]), C=C, G=G, S=S,
                 N=_log_int(rng, 1, max(1, min(32768 if per_token else 64, most // (C * S)))),
                 act=rng.choice(["silu", "silu", None]))
    return c


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dt = _DT[case["dtype"]]
    s = dict(case)
    kind = case["kind"]

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=_DEV).mul_(std).to(dtype)

    if kind.startswith("delta"):
        B, H, HK, DK, DV = (case[k] for k in ("B", "H", "HK", "DK", "DV"))
        L = case.get("L", 1)

        def unit(h):                                     # queries and keys as a layer normalises them
            x = torch.randn(B, L, h, DK, generator=g, device=_DEV)
            return (x * (x.square().sum(-1, keepdim=True) + 1e-6).rsqrt()).to(dt)

        # projections leave (B, L, heads, channels); the operators take the heads before the tokens
        s["q"], s["k"] = unit(HK).transpose(1, 2), unit(HK).transpose(1, 2)
        s["v"] = normal(B, L, H, DV).transpose(1, 2)
        rate = 16 * torch.rand(H, generator=g, device=_DEV)
        step = torch.exp(math.log(1e-3) + math.log(1e2) * torch.rand(B, L, H, generator=g, device=_DEV))
        s["g"] = (-rate * step).transpose(1, 2)
        s["beta"] = torch.sigmoid(1.5 * torch.randn(B, L, H, generator=g, device=_DEV)).transpose(1, 2)
        s["state"] = None
        if kind == "delta_step" or case["init"]:
            s["state"] = normal(B, H, DK, DV, std=0.3, dtype=torch.float32)
        if kind == "delta_step":
            for name in ("q", "k", "v", "g", "beta"):
                s[name] = s[name][:, :, 0].contiguous()
            s["next"] = torch.empty_like(s["state"])
        if kind == "delta_grad":
            s["do"] = normal(B, L, H, DV).transpose(1, 2)
            s["d_final"] = normal(B, H, DK, DV, std=0.1, dtype=torch.float32)
            s["leaves"] = tuple(s[n].requires_grad_() for n in ("q", "k", "v", "g", "beta", "state") if s[n] is not None)
    elif kind.startswith("rotary"):
        B, H, HK, L, D, RD = (case[k] for k in ("B", "H", "HK", "L", "D", "RD"))
        s["q"], s["k"] = normal(B, L, H, D).transpose(1, 2), normal(B, L, HK, D).transpose(1, 2)
        s["inv_freq"] = 10000.0 ** (-torch.arange(0, RD, 2, device=_DEV, dtype=torch.float64) / RD)
        start = torch.randint(900_000 if case["far"] else 1, (B, 1), generator=g, device=_DEV)
        s["positions"] = start + torch.arange(L, device=_DEV)
        s["scale"] = 1.0 if RD == D else 1.1
        if kind == "rotary_grad":
            s["dq"], s["dk"] = normal(B, L, H, D).transpose(1, 2), normal(B, L, HK, D).transpose(1, 2)
    else:
        N, S, C = case["N"], case["S"], case["C"]
        wd = _DT[case["wdtype"]]
        chan = torch.exp(0.5 * torch.randn(C, generator=g, device=_DEV))
        s["x"] = (torch.randn(N, S, C, generator=g, device=_DEV) * chan + 0.3).to(dt)
        s["weight"] = (1 + 0.1 * torch.randn(C, generator=g, device=_DEV)).to(wd)
        s["bias"] = (0.1 * torch.randn(C, generator=g, device=_DEV)).to(wd)
        s["eps"] = 1e-5
        if kind == "gnorm_grad":
            s["dy"] = normal(N, S, C)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


def _run_own(s):
    import mamformer_amd as mh

    kind = s["kind"]
    if kind == "delta_step":
        return mh.gated_delta_step(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"], state_out=s["next"]), s["next"]
    if kind.startswith("delta"):
        out = mh.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["state"],
                                  return_final_state=True)
        if kind == "delta":
            return out
        return *(t.detach() for t in out), *torch.autograd.grad(out, s["leaves"], (s["do"], s["d_final"]))
    if kind.startswith("rotary"):
        how = dict(interleaved=s["inter"], scale=s["scale"])
        out = mh.rotary(s["q"], s["k"], s["inv_freq"], s["positions"], **how)
        if kind == "rotary":
            return out
        return *out, *mh.rotary(s["dq"], s["dk"], s["inv_freq"], s["positions"], inverse=True, **how)
    y, stats = mh.group_norm(s["x"], s["G"], s["weight"], s["bias"], s["eps"], activation=s["act"], return_stats=True)
    if kind == "gnorm":
        return y
    return y, *mh.group_norm_bwd(s["dy"], s["x"], stats, s["G"], s["weight"], s["bias"], activation=s["act"])


def _run_plain(s):
    kind = s["kind"]
    if kind == "delta_step":
        return _plain_step(s)
    if kind.startswith("delta"):
        return _plain_delta(s, kind == "delta_grad")
    if kind.startswith("rotary"):
        angle = s["positions"].double()[:, None, :, None] * s["inv_freq"]
        c, sn = angle.cos().float() * s["scale"], angle.sin().float() * s["scale"]
        out = tuple(_plain_turn(x, c, sn, s["inter"]) for x in (s["q"], s["k"]))
        if kind == "rotary":
            return out
        return *out, *(_plain_turn(x, c, -sn, s["inter"]) for x in (s["dq"], s["dk"]))
    return _plain_gnorm(s, kind == "gnorm_grad")


def _plain_step(s):
    r = s["H"] // s["HK"]
    q, k = (s[n].float().repeat_interleave(r, 1) for n in ("q", "k"))
    S = s["state"] * s["g"].exp()[..., None, None]
    delta = s["beta"][..., None] * (s["v"].float() - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * delta[..., None, :]
    return ((S * q[..., None]).sum(-2) * s["DK"] ** -0.5).to(s["v"].dtype), S


def _plain_delta(s, grad):
    """Pieces of 64 tokens: what the tokens of a piece do to one another as a triangular system, the state between them."""
    B, H, L, DV = s["v"].shape
    DK, r, dt = s["DK"], H // s["HK"], s["v"].dtype
    scale = DK ** -0.5
    n = -(-L // _C)

    def pieces(x, rep=1):
        x = x.float().repeat_interleave(rep, 1) if rep > 1 else x.float()
        x = torch.cat([x, x.new_zeros(B, H, n * _C - L, *x.shape[3:])], 2)
        return x.view(B, H, n, _C, *x.shape[3:])

    q, k, v, beta = pieces(s["q"], r), pieces(s["k"], r), pieces(s["v"]), pieces(s["beta"])
    G = pieces(s["g"]).double().cumsum(-1)
    low = torch.ones(_C, _C, device=q.device, dtype=torch.bool).tril()
    D = torch.where(low, G[..., :, None] - G[..., None, :], -math.inf).exp().float() * beta[..., None, :]
    eG, eEnd = G.exp().float()[..., None], (G[..., -1:] - G).exp().float()[..., None] * beta[..., None]
    last = G[..., -1].exp().float()[..., None, None]
    kT = k.transpose(-1, -2).contiguous()
    A = (k @ kT).mul_(D).tril_(-1)
    P = (q @ kT).mul_(D).mul_(scale)
    T = torch.eye(_C, device=q.device).expand(B, H, n, _C, _C).contiguous()
    for i in range(1, _C):                               # rows of the inverse, each from those above it
        T[..., i, :i] = -(A[..., i, :i, None] * T[..., :i, :i]).sum(-2)
    S = s["state"].detach().clone() if s["state"] is not None else q.new_zeros(B, H, DK, DV)
    first, deltas = [], []
    keT = (k * eEnd).transpose(-1, -2).contiguous()
    for c in range(n):
        first.append(S)
        d = T[:, :, c] @ (v[:, :, c] - (k[:, :, c] * eG[:, :, c]) @ S)
        deltas.append(d)
        S = last[:, :, c] * S + keT[:, :, c] @ d
    S0, d = torch.stack(first, 2), torch.stack(deltas, 2)
    o = scale * (q * eG) @ S0 + P @ d

    def whole(x, dtype):
        return x.reshape(B, H, n * _C, *x.shape[4:])[:, :, :L].to(dtype)

    if not grad:
        return whole(o, dt), S
    do = pieces(s["do"])
    Tt, Pt, St = (x.transpose(-1, -2).contiguous() for x in (T, P, S0))
    qeT, kgT = ((x * eG).transpose(-1, -2).contiguous() for x in (q, k))
    dS, after, ys = s["d_final"], [], []
    for c in range(n - 1, -1, -1):
        after.append(dS)
        y = Tt[:, :, c] @ (Pt[:, :, c] @ do[:, :, c] + (k[:, :, c] * eEnd[:, :, c]) @ dS)
        ys.append(y)
        dS = last[:, :, c] * dS + scale * qeT[:, :, c] @ do[:, :, c] - kgT[:, :, c] @ y
    y, dN = torch.stack(ys[::-1], 2), torch.stack(after[::-1], 2)
    dT = d.transpose(-1, -2).contiguous()
    rawA, rawP = (y @ dT).neg_().tril_(-1), (do @ dT).mul_(scale).tril_()
    X, Xp = rawA * D, rawP * D
    back = d @ dN.transpose(-1, -2).contiguous()
    dq1, dk1, dk2 = scale * eG * (do @ St), -eG * (y @ St), eEnd * back
    dq = dq1 + Xp @ k
    dkl = dk1 + X @ k
    dkr = dk2 + X.transpose(-1, -2).contiguous() @ k + Xp.transpose(-1, -2).contiguous() @ q
    # D without beta, and what beta scales of each token
    Db = torch.where(low, G[..., :, None] - G[..., None, :], -math.inf).exp().float()
    kk, qk = k @ kT, q @ kT
    dbeta = ((rawA * kk + rawP * qk) * Db).sum(-2) + ((G[..., -1:] - G).exp().float()[..., None] * back * k).sum(-1)
    dG = (q * dq).sum(-1) + (k * dkl).sum(-1) - (k * dkr).sum(-1)
    dG[..., -1] += (last * S0 * dN).sum((-1, -2)) + (k * dk2).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1)

    def shared(x):
        return x.view(B, s["HK"], r, n, _C, DK).sum(2).reshape(B, s["HK"], n * _C, DK)[:, :, :L].to(dt)

    out = (whole(o, dt), S, shared(dq), shared(dkl + dkr), whole(y, dt), whole(dg, torch.float32),
           whole(dbeta, torch.float32))
    return out if s["state"] is None else (*out, dS)


def _plain_turn(x, c, sn, inter):
    x32, n = x.float(), c.shape[-1]
    if inter:
        a, b = x32[..., 0:2 * n:2], x32[..., 1:2 * n:2]
        t = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    else:
        a, b = x32[..., :n], x32[..., n:2 * n]
        t = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.cat([t, x32[..., 2 * n:]], -1).to(x.dtype)


def _plain_gnorm(s, grad):
    N, S, C = s["x"].shape
    G, dt = s["G"], s["x"].dtype
    x = s["x"].float().view(N, S, G, C // G)
    w, b = s["weight"].float().view(G, -1), s["bias"].float().view(G, -1)
    cen = x - x.mean((1, 3), keepdim=True)
    r = (cen.square().mean((1, 3), keepdim=True) + s["eps"]).rsqrt()
    xh = cen * r
    z = xh * w + b
    sig = 1 / (1 + (-z).exp()) if s["act"] else None
    y = (z * sig if s["act"] else z).view(N, S, C).to(dt)
    if not grad:
        return y
    dz = s["dy"].float().view(N, S, G, C // G)
    if s["act"]:
        dz = dz * sig * (1 + z * (1 - sig))
    gw = dz * w
    dx = r * (gw - gw.mean((1, 3), keepdim=True) - xh * (gw * xh).mean((1, 3), keepdim=True))
    wd = s["weight"].dtype
    return y, dx.view(N, S, C).to(dt), (dz * xh).sum((0, 1)).view(C).to(wd), dz.sum((0, 1)).view(C).to(wd)


# ------------------------------------------------------------------------------------------------ work and definition

def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    kind = case["kind"]
    if kind.startswith("delta"):
        B, H, HK, DK, DV = (case[k] for k in ("B", "H", "HK", "DK", "DV"))
        L = case.get("L", 1)
        tokens, state = B * L, 4 * B * H * DK * DV
        rows = tokens * es * (2 * HK * DK + 2 * H * DV) + 8 * tokens * H      # q, k, v, o, g, beta
        mults = tokens * H * DK * DV
        if kind == "delta_step":
            return {"bytes": rows + 2 * state, "flops": 7 * mults}
        if kind == "delta":
            return {"bytes": rows + state * (1 + case["init"]), "flops": 7 * mults}
        # the output's and the final state's gradients in, those of all inputs out
        more = tokens * es * (2 * HK * DK + 2 * H * DV) + 8 * tokens * H + state * (1 + case["init"])
        return {"bytes": rows + state * (1 + case["init"]) + more, "flops": 21 * mults}
    if kind.startswith("rotary"):
        rows = case["B"] * case["L"] * (case["H"] + case["HK"])
        passes = 2 if kind == "rotary_grad" else 1
        return {"bytes": passes * (2 * rows * case["D"] * es + 8 * case["B"] * case["L"]),
                "flops": passes * 3 * rows * case["RD"]}
    n = case["N"] * case["S"] * case["C"]
    if kind == "gnorm":
        return {"bytes": 2 * n * es, "flops": 12 * n}
    return {"bytes": 4 * n * es, "flops": 30 * n}        # x, dy, y, dx


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        kind = case["kind"]
        if kind.startswith("delta"):
            return _exact_delta(s, kind)
        if kind.startswith("rotary"):
            pairs = [(s["q"], 1), (s["k"], 1)] + ([(s["dq"], -1), (s["dk"], -1)] if kind == "rotary_grad" else [])
            turn = torch.polar(torch.full_like(s["inv_freq"], s["scale"]).expand(*s["positions"].shape, -1).contiguous(),
                               s["positions"][..., None] * s["inv_freq"])[:, None]
            return tuple(_exact_turn(x, turn if sign > 0 else turn.conj(), s["inter"]) for x, sign in pairs)
        return _exact_gnorm(s, kind == "gnorm_grad")


def _exact_delta(s, kind):
    """Token by token, the gradients by walking back over the kept states."""
    step = kind == "delta_step"
    q, k, v, g, beta = (s[n].double() for n in ("q", "k", "v", "g", "beta"))
    if step:
        q, k, v, g, beta = (t.unsqueeze(2) for t in (q, k, v, g, beta))
    B, H, L, DV = v.shape
    HK, DK = q.shape[1], q.shape[3]
    head = torch.arange(H, device=v.device) // (H // HK)                     # the key head of each value head
    q, k = q.index_select(1, head), k.index_select(1, head)
    scale = 1 / math.sqrt(DK)
    S = torch.zeros(B, H, DK, DV, device=v.device, dtype=torch.float64)
    if s["state"] is not None:
        S += s["state"]
    kept = torch.empty(L, B, H, DK, DV, device=v.device, dtype=torch.float64) if kind == "delta_grad" else None
    o, err = torch.empty_like(v), torch.empty_like(v)
    decay = torch.exp(g)
    for t in range(L):
        if kept is not None:
            kept[t] = S
        S = S * decay[:, :, t, None, None]
        kt = k[:, :, t, :, None]
        err[:, :, t] = v[:, :, t] - (kt.mT @ S).squeeze(-2)
        S = torch.addcmul(S, kt, (beta[:, :, t, None] * err[:, :, t]).unsqueeze(-2))
        o[:, :, t] = (q[:, :, t, None, :] @ S).squeeze(-2)
    o *= scale
    if step:
        return o[:, :, 0], S
    if kind == "delta":
        return o, S
    end, dS = S, s["d_final"].double()
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    dv, dg, db = torch.empty_like(v), torch.empty_like(g), torch.empty_like(g)
    do = s["do"].double() * scale
    for t in range(L - 1, -1, -1):
        kt, e, bt = k[:, :, t], err[:, :, t], beta[:, :, t, None]
        before = kept[t] * decay[:, :, t, None, None]                        # the decayed state that the token meets
        now = before + kt[..., :, None] * (bt * e)[..., None, :]
        dq[:, :, t] = (now @ do[:, :, t, :, None]).squeeze(-1)
        dS = dS + q[:, :, t, :, None] * do[:, :, t, None, :]
        du = (kt[..., None, :] @ dS).squeeze(-2)                             # of beta (v - S^T k)
        db[:, :, t] = (du * e).sum(-1)
        de = bt * du
        dv[:, :, t] = de
        dk[:, :, t] = (dS @ (bt * e)[..., :, None]).squeeze(-1) - (before @ de[..., :, None]).squeeze(-1)
        dS = dS - kt[..., :, None] * de[..., None, :]
        dg[:, :, t] = (dS * before).sum((-1, -2))
        dS = dS * decay[:, :, t, None, None]
    dq, dk = (torch.zeros(B, HK, L, DK, device=v.device, dtype=torch.float64).index_add_(1, head, t) for t in (dq, dk))
    out = (o, end, dq, dk, dv, dg, db)
    return out if s["state"] is None else (*out, dS)


def _exact_turn(x, turn, inter):
    n = turn.shape[-1]
    out = x.double().contiguous()
    if inter:
        z = torch.complex(out[..., 0:2 * n:2].contiguous(), out[..., 1:2 * n:2].contiguous()) * turn
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = z.real, z.imag
    else:
        z = torch.complex(out[..., :n].contiguous(), out[..., n:2 * n].contiguous()) * turn
        out[..., :n], out[..., n:2 * n] = z.real, z.imag
    return out


def _exact_gnorm(s, grad):
    N, S, C = s["x"].shape
    G = s["G"]
    x = s["x"].double().view(N, S, G, C // G).permute(0, 2, 1, 3).reshape(N, G, -1)
    n = x.shape[-1]
    w, b = (s[p].double().view(1, G, 1, -1).expand(N, G, S, -1).reshape(N, G, n) for p in ("weight", "bias"))
    mu = x.sum(-1, keepdim=True) / n
    r = 1 / torch.sqrt(((x - mu) ** 2).sum(-1, keepdim=True) / n + s["eps"])
    xh = (x - mu) * r
    z = torch.addcmul(b, xh, w)
    p = torch.sigmoid(z)
    y = z * p if s["act"] else z

    def rows(t):
        return t.view(N, G, S, C // G).permute(0, 2, 1, 3).reshape(N, S, C)

    if not grad:
        return rows(y)
    dz = s["dy"].double().view(N, S, G, C // G).permute(0, 2, 1, 3).reshape(N, G, n)
    if s["act"]:
        dz = dz * (p + y * (1 - p))
    t = dz * w
    dx = (t - t.sum(-1, keepdim=True) / n - xh * ((t * xh).sum(-1, keepdim=True) / n)) * r
    return rows(y), rows(dx), rows(dz * xh).sum((0, 1)), rows(dz).sum((0, 1))
