"""The operators at the two ends of a language model and between its layers, as cases that can be timed and compared.

==============  =====================================================================================
``embed``       tokens looked up in the table, scaled
``embed_grad``  the lookup and the table's gradient by sorted tokens, as a training step runs them
``norm``        layer norm of a residual stream: the sum with a layer's output and its norm
``norm_grad``   layer norm and its backward: gradients of the rows, the weight and the bias
``norm_packed`` the same with the normalised rows kept for the backward in 8 bits
``pack``        activations into 8 bits with an exponent for each 64 channels, and back
``logprob``     log probabilities of given tokens, entropies and the likeliest alternatives
``logprob_grad`` log probabilities and entropies, and the logits' gradient
==============  =====================================================================================

``run`` computes an operator from elementary torch operations in 32 bits, or, where ``own`` is true, by this
package's kernels; ``exact`` restates the definitions in float64.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_DEV = "cuda"
_GROUP = 64                  # channels that share an exponent in the 8-bit form


# ------------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one token of each of eight sequences on its way into the first layer: the smallest call, latency alone
        dict(name="embed_decode", kind="embed", dtype="bf16", T=8, V=32000, D=2048, idx="int64", pad=False),
        # a training step's two sequences of 4096 tokens through the table of the 1b preset's width
        dict(name="embed_train", kind="embed_grad", dtype="bf16", T=8192, V=32000, D=2048, idx="int64", pad=False),
        # an odd table in 32 bits with a padding token and int32 ids, as a small verification run has it
        dict(name="embed_odd", kind="embed_grad", dtype="fp32", T=1999, V=49999, D=1001, idx="int32", pad=True),
        # one user's prompt of odd length between two layers of the 1b preset's width
        dict(name="norm_prompt", kind="norm", dtype="bf16", wdtype="bf16", R=333, D=2048, res=True),
        # a training step of the residual stream at that width, the weights kept in 32 bits
        dict(name="norm_train", kind="norm_grad", dtype="bf16", wdtype="fp32", R=8192, D=2048, res=True),
        # the norm over each of 16 heads of 128 channels behind the linear attention: many short rows
        dict(name="norm_heads", kind="norm_grad", dtype="bf16", wdtype="bf16", R=131072, D=128, res=False),
        # a residual stream of width 4096 whose rows are kept for the backward in 8 bits
        dict(name="norm_packed", kind="norm_packed", dtype="bf16", wdtype="bf16", R=32768, D=4096, res=True),
        # a layer's input put away in 8 bits and fetched back for the layer's second run
        dict(name="pack_layer", kind="pack", dtype="bf16", R=8192, D=2048),
        # 8192 tokens of documents scored by their log probabilities
        dict(name="score_8k", kind="logprob", dtype="bf16", R=8192, V=32000, top=0, temp=1.0, masked=False),
        # a serving batch's next tokens with 20 alternatives each, sampled at a temperature, a large table
        dict(name="serve_top20", kind="logprob", dtype="fp32", R=24, V=128000, top=20, temp=0.7, masked=True),
        # the loss of a training step, with an entropy term, and the logits' gradient: the largest call
        dict(name="loss_train", kind="logprob_grad", dtype="bf16", R=8192, V=32000, top=0, temp=1.0, masked=False),
        # a policy update on answers of odd length: an odd vocabulary with masked entries, in 32 bits
        dict(name="loss_odd", kind="logprob_grad", dtype="fp32", R=777, V=50001, top=0, temp=0.8, masked=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges around the listed ones: sizes log-uniform, most of them odd."""
    kind = rng.choice(["embed", "embed_grad", "embed_grad", "norm", "norm_grad", "norm_grad", "norm_packed", "pack",
                       "logprob", "logprob", "logprob_grad"])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if kind in ("embed", "embed_grad"):
        D = rng.choice([64, 512, 1000, 1024, 2048, 4096, _log_int(rng, 33, 6000)])
        V = _log_int(rng, 500, min(262144, 120_000_000 // D))
        c.update(T=_log_int(rng, 1, min(65536, 80_000_000 // D)), V=V, D=D, idx=rng.choice(["int64", "int32"]),
                 pad=rng.random() < 0.3)
    elif kind in ("norm", "norm_grad", "norm_packed", "pack"):
        D = rng.choice([64, 128, 1000, 1024, 2048, 4096, 8192, _log_int(rng, 24, 12000)])
        top = 100_000_000 if c["dtype"] == "bf16" else 50_000_000
        c.update(R=_log_int(rng, 1, min(200_000, top // D)), D=D)
        if kind != "pack":
            c.update(wdtype=rng.choice([c["dtype"], "fp32"]), res=rng.random() < 0.5)
    else:
        V = rng.choice([1024, 32000, 65536, 128000, _log_int(rng, 300, 260_000)])
        top = 200_000_000 if c["dtype"] == "bf16" else 100_000_000
        c.update(R=_log_int(rng, 1, min(16384, top // V)), V=V, top=0, temp=rng.choice([1.0, 1.0, 0.7, 1.3]),
                 masked=rng.random() < 0.4)
        if kind == "logprob":
            c["top"] = rng.choice([0, 1, 5, 20])
            if c["top"]:                                 # alternatives are asked for in serving: fewer rows
                c["R"] = min(c["R"], max(1, 30_000_000 // V))
    return c


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=_DEV).mul_(std).to(dtype)

    s = dict(case)
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        T, V, D = case["T"], case["V"], case["D"]
        # word frequencies fall as the inverse of the rank; the table's order is not that of frequency
        u = torch.rand(T, generator=g, device=_DEV, dtype=torch.float64)
        rank = (torch.exp(u * math.log(V + 1)).long() - 1).clamp_(0, V - 1)
        ids = torch.randperm(V, generator=g, device=_DEV)[rank]
        s["pad_id"] = None
        if case["pad"]:
            s["pad_id"] = V - 1
            ids = torch.where(torch.rand(T, generator=g, device=_DEV) < 0.2, V - 1, ids)
        s["ids"] = ids.to(torch.int64 if case["idx"] == "int64" else torch.int32)
        s["scale"] = math.sqrt(D)
        s["weight"] = normal(V, D, std=0.02)
        if kind == "embed_grad":
            s["dy"] = normal(T, D)
    elif kind in ("norm", "norm_grad", "norm_packed"):
        R, D = case["R"], case["D"]
        wd = _DT[case["wdtype"]]
        # a stream whose channels differ in size, a few of them by much
        chan = torch.exp(0.5 * torch.randn(D, generator=g, device=_DEV))
        chan = torch.where(torch.rand(D, generator=g, device=_DEV) < 0.003, 20.0, chan)
        s["x"] = (torch.randn(R, D, generator=g, device=_DEV) * chan + 0.1).to(dt)
        s["residual"] = (torch.randn(R, D, generator=g, device=_DEV) * chan).to(dt) if case["res"] else None
        s["weight"] = (1 + 0.1 * torch.randn(D, generator=g, device=_DEV)).to(wd)
        s["bias"] = (0.1 * torch.randn(D, generator=g, device=_DEV)).to(wd)
        s["eps"] = 1e-5
        if kind != "norm":
            s["dy"] = normal(R, D)
            s["d_h"] = normal(R, D) if case["res"] else None
    elif kind == "pack":
        R, D = case["R"], case["D"]
        chan = torch.exp(0.5 * torch.randn(D, generator=g, device=_DEV))
        s["x"] = (torch.randn(R, D, generator=g, device=_DEV) * chan).to(dt)
    else:
        R, V = case["R"], case["V"]
        targets = torch.randint(V, (R,), generator=g, device=_DEV)
        logits = torch.randn(R, V, generator=g, device=_DEV).mul_(2.5)
        # the given token is often among the likely ones
        logits[torch.arange(R, device=_DEV), targets] += 8 * torch.rand(R, generator=g, device=_DEV)
        if case["masked"]:                               # entries of the table that no answer may hold
            off = torch.rand(V, generator=g, device=_DEV) < 0.05
            off[:64] = False
            logits[:, off] = -math.inf
            targets = torch.where(off[targets], targets % 64, targets)
        ignored = torch.rand(R, generator=g, device=_DEV) < 0.1
        s["targets"] = torch.where(ignored, -100, targets)
        s["logits"] = logits.to(dt)
        if kind == "logprob_grad":
            s["d_lp"] = torch.where(ignored, 0.0, torch.randn(R, generator=g, device=_DEV)) / R
            s["d_ent"] = 0.01 * torch.randn(R, generator=g, device=_DEV) / R
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import mamformer_amd as mh

    kind = s["kind"]
    if kind in ("embed", "embed_grad"):
        out = mh.embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=s["pad_id"])
        if kind == "embed":
            return out
        return out, mh.embedding_bwd(s["dy"], s["ids"], s["V"], scale=s["scale"], padding_idx=s["pad_id"])
    if kind in ("norm", "norm_grad", "norm_packed"):
        res = s["residual"]
        if kind == "norm":
            return mh.layer_norm(s["x"], s["weight"], s["bias"], s["eps"], residual=res)
        packed = kind == "norm_packed"
        out = mh.layer_norm(s["x"], s["weight"], s["bias"], s["eps"], residual=res, packed=packed, return_stats=True)
        kept = out[-2] if packed else out[1] if res is not None else s["x"]
        grads = mh.layer_norm_bwd(s["dy"], kept, out[-1], s["weight"], d_h=s["d_h"])
        return out[0], (out[1] if res is not None else None), *grads
    if kind == "pack":
        return mh.unpack_activations(mh.pack_activations(s["x"]))
    out = mh.token_logprobs(s["logits"], s["targets"], temperature=s["temp"], top=s["top"])
    if kind == "logprob":
        return out.logprobs, out.entropy, out.top_ids, out.top_logprobs
    d = mh.token_logprobs_bwd(s["logits"], s["targets"], out.stats, s["d_lp"], s["d_ent"], temperature=s["temp"])
    return out.logprobs, out.entropy, d


def _run_plain(s):
    kind = s["kind"]
    if kind in ("embed", "embed_grad"):
        ids, w = s["ids"].long(), s["weight"]
        out = (w[ids].float() * s["scale"]).to(w.dtype)
        if kind == "embed":
            return out
        dy = s["dy"].float()
        if s["pad_id"] is not None:
            dy = torch.where((ids == s["pad_id"])[:, None], 0.0, dy)
        dw = torch.zeros(w.shape, device=w.device, dtype=torch.float32).index_add_(0, ids, dy)
        return out, (dw * s["scale"]).to(w.dtype)
    if kind in ("norm", "norm_grad", "norm_packed"):
        dt = s["x"].dtype
        h = s["x"]
        if s["residual"] is not None:
            h = (h.float() + s["residual"].float()).to(dt)
        w, hf = s["weight"].float(), h.float()
        mean = hf.mean(-1, keepdim=True)
        cen = hf - mean
        rstd = (cen.square().mean(-1, keepdim=True) + s["eps"]).rsqrt()
        y = (cen * rstd * w + s["bias"].float()).to(dt)
        hs = h if s["residual"] is not None else None
        if kind == "norm":
            return y if hs is None else (y, hs)
        if kind == "norm_packed":
            hf = _plain_pack(hf)
        c = (hf - mean) * rstd
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - c * (g * c).mean(-1, keepdim=True))
        if s["d_h"] is not None:
            dx = dx + s["d_h"].float()
        return y, hs, dx.to(dt), (dy * c).sum(0).to(s["weight"].dtype), dy.sum(0).to(s["weight"].dtype)
    if kind == "pack":
        return _plain_pack(s["x"].float()).to(s["x"].dtype)
    logits, targets = s["logits"], s["targets"]
    lf = logits.float()
    l = lf / s["temp"]
    l = l - l.amax(-1, keepdim=True)
    e = l.exp()
    S = e.sum(-1, keepdim=True)
    logp = l - S.log()
    p = e / S
    plogp = torch.where(p > 0, p * logp, 0.0)
    ent = -plogp.sum(-1)
    keep = targets >= 0
    at = torch.where(keep, targets, 0)
    lp = torch.where(keep, logp.gather(-1, at[:, None])[:, 0], 0.0)
    if kind == "logprob":
        if not s["top"]:
            return lp, ent, None, None
        ids = torch.sort(lf, dim=-1, descending=True, stable=True)[1][:, :s["top"]]     # equal values: the lowest id first
        return lp, ent, ids, logp.gather(-1, ids)
    d_lp = torch.where(keep, s["d_lp"], 0.0)
    d = -p * d_lp[:, None] - s["d_ent"][:, None] * (plogp + p * ent[:, None])
    d.scatter_add_(-1, at[:, None], d_lp[:, None])
    return lp, ent, (d / s["temp"]).to(logits.dtype)


def _plain_pack(x):
    """x (R, D) fp32 -> the values that its 8-bit codes stand for."""
    R, D = x.shape
    pad = -D % _GROUP
    v = torch.cat([x, x.new_zeros(R, pad)], -1).view(R, -1, _GROUP).double()
    amax = v.abs().amax(-1, keepdim=True)
    man, ex = torch.frexp(amax.clamp_min(2.0 ** -126))                       # amax = man 2^ex, 1/2 <= man < 1
    ex = (ex - 7 + (man > 127 / 128)).long()                                 # least ex with amax <= 127 2^ex
    step = ((ex + 1023) << 52).view(torch.float64)
    v = torch.round(v / step) * step
    return v.view(R, -1)[:, :D].float()


# ------------------------------------------------------------------------------------------------ work and definition

def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        T, V, D = case["T"], case["V"], case["D"]
        ib = 8 if case["idx"] == "int64" else 4
        # distinct tokens of a sample whose frequencies fall as the inverse of the rank
        n = math.log(V + 1)
        distinct = int(sum((1 - math.exp(-T * p)) * w for p, w in
                           ((math.log1p(1 / r) / n, 1 if r < 64 else r // 32) for r in _ranks(V))))
        by = T * ib + max(1, min(distinct, T, V)) * D * es + T * D * es
        if kind == "embed":
            return {"bytes": by, "flops": T * D}
        return {"bytes": by + T * D * es + V * D * es, "flops": 3 * T * D}
    if kind in ("norm", "norm_grad", "norm_packed"):
        R, D = case["R"], case["D"]
        res, n = (1 if case["res"] else 0), R * D * es
        if kind == "norm":
            return {"bytes": n * (2 + 2 * res), "flops": 8 * R * D}
        return {"bytes": n * (2 + 2 * res) + n * (2 + res), "flops": 20 * R * D}
    if kind == "pack":
        return {"bytes": 2 * case["R"] * case["D"] * es, "flops": 4 * case["R"] * case["D"]}
    n = case["R"] * case["V"]
    if kind == "logprob":
        return {"bytes": n * es + 16 * case["R"], "flops": 6 * n}
    return {"bytes": 2 * n * es + 24 * case["R"], "flops": 14 * n}


def _ranks(V):
    """Ranks 1 .. V, one for each 1/32 of its size beyond 64."""
    r = 1
    while r <= V:
        yield r
        r += 1 if r < 64 else r // 32


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        ids, w = s["ids"].long(), s["weight"]
        out = w.double().index_select(0, ids) * s["scale"]
        if kind == "embed":
            return out
        live = torch.ones_like(ids, dtype=torch.bool) if s["pad_id"] is None else ids != s["pad_id"]
        order = torch.argsort(ids[live], stable=True)
        rows, counts = torch.unique_consecutive(ids[live][order], return_counts=True)
        dw = torch.zeros(w.shape, device=w.device, dtype=torch.float64)
        dy, first = s["dy"][live], 0
        for row, n in zip(rows.tolist(), counts.tolist()):
            dw[row] = dy[order[first:first + n]].double().sum(0) * s["scale"]
            first += n
        return out, dw
    if kind in ("norm", "norm_grad", "norm_packed"):
        total = s["x"].double()
        h = total
        if s["residual"] is not None:
            total = total + s["residual"].double()
            h = total.to(s["x"].dtype).double()                              # the stream itself is held in its type
        D = h.shape[1]
        w, b = s["weight"].double(), s["bias"].double()
        mu = h.sum(1) / D
        var = (h * h).sum(1) / D - mu * mu
        r = 1 / torch.sqrt(var + s["eps"])
        y = (h - mu[:, None]) * (r[:, None] * w) + b
        hs = total if s["residual"] is not None else None
        if kind == "norm":
            return y if hs is None else (y, hs)
        if kind == "norm_packed":
            h = _exact_pack(h)
        xh = (h - mu[:, None]) * r[:, None]
        dy = s["dy"].double()
        g = dy * w
        dx = (g - g.sum(1, keepdim=True) / D - xh * ((g * xh).sum(1, keepdim=True) / D)) * r[:, None]
        if s["d_h"] is not None:
            dx += s["d_h"].double()
        return y, hs, dx, torch.einsum("rd,rd->d", dy, xh), dy.sum(0)
    if kind == "pack":
        return _exact_pack(s["x"].double())
    rows = []
    for lo in range(0, case["R"], 1024):                                     # rows at a time: float64 is four times bf16
        z = s["logits"][lo:lo + 1024].double() / s["temp"]
        t = s["targets"][lo:lo + 1024]
        lse = torch.logsumexp(z, 1, keepdim=True)
        logp = z - lse
        p = torch.exp(logp)
        term = torch.special.entr(p)
        ent = term.sum(1)
        keep = t >= 0
        at = t.clamp(min=0)
        lp = torch.where(keep, logp[torch.arange(len(t), device=t.device), at], 0.0)
        if kind == "logprob":
            ids = alt = None
            if case["top"]:
                key = s["logits"][lo:lo + 1024].double()
                ids = torch.empty((len(t), case["top"]), device=t.device, dtype=torch.int64)
                for k in range(case["top"]):
                    best = key.amax(1, keepdim=True)
                    ids[:, k] = _first(key == best)
                    key.scatter_(1, ids[:, k:k + 1], -math.inf)
                alt = torch.take_along_dim(logp, ids, 1)
            rows.append((lp, ent, ids, alt))
            continue
        d_lp = torch.where(keep, s["d_lp"][lo:lo + 1024].double(), 0.0)
        onehot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
        d = d_lp[:, None] * (onehot - p) + s["d_ent"][lo:lo + 1024].double()[:, None] * (term - p * ent[:, None])
        rows.append((lp, ent, d / s["temp"]))
    return tuple(None if parts[0] is None else torch.cat(parts) for parts in zip(*rows))


def _exact_pack(x):
    R, D = x.shape
    out = torch.empty_like(x)
    for lo in range(0, D, _GROUP):
        v = x[:, lo:lo + _GROUP]
        top = v.abs().amax(1).clamp_min(2.0 ** -126)
        e = torch.floor(torch.log2(top)).long() - 7
        for _ in range(3):                                                   # least e with top <= 127 2^e
            e = torch.where(top > 127 * _pow2(e), e + 1, e)
        e = torch.where(top <= 127 * _pow2(e - 1), e - 1, e)
        out[:, lo:lo + _GROUP] = torch.round(v / _pow2(e)[:, None]) * _pow2(e)[:, None]
    return out


def _pow2(e):
    return ((e + 1023) << 52).view(torch.float64)


def _first(hit):
    """Index of the first true value of every row."""
    n = hit.shape[1]
    return torch.where(hit, torch.arange(n, device=hit.device), n).amin(1)
