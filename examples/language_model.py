"""A small language model from this package's operators: trained for some steps, then asked for its next tokens.

Per token: a row of the table (``embedding``), layers of ``layer_norm`` with the residual sum fused and ``Mamba2Layer``, a
last norm, and logits against the table.  Training takes the loss and the logits' gradient from ``token_logprobs`` and can
keep what the norms' backward reads in 8 bits (``--packed``).  Generation takes one token of every sequence at a time
from the layers' caches and shows the likeliest alternatives.

    python -m mamformer_amd.build && python examples/language_model.py --steps 60 --packed
"""

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn as nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import mamformer_amd as mh  # noqa: E402
from mamformer_amd.layers import Mamba2Layer  # noqa: E402


class Norm(nn.Module):
    """The stream h = x + residual and its layer norm; ``packed`` keeps h for the backward in 8 bits."""

    def __init__(self, dim, packed, device, dtype):
        super().__init__()
        self.packed = packed
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype))

    def forward(self, x, residual=None):
        out = mh.layer_norm(x, self.weight, self.bias, residual=residual,
                            packed=self.packed and torch.is_grad_enabled())
        if residual is not None:
            return out[0], out[1]
        return (out[0] if isinstance(out, tuple) else out), x


class LanguageModel(nn.Module):
    def __init__(self, vocab, dim, layers, *, d_state=64, packed=False, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.scale = math.sqrt(dim)
        self.table = nn.Parameter(torch.randn(vocab, dim, device=device).mul_(dim ** -0.5).to(dtype))
        self.norms = nn.ModuleList(Norm(dim, packed, device, dtype) for _ in range(layers + 1))
        self.layers = nn.ModuleList(Mamba2Layer(dim, d_state=d_state, device=device, dtype=dtype) for _ in range(layers))
        for layer in self.layers:                # the step sizes, decays and skips are fp32 whatever the model's type
            for p in (layer.A_log, layer.dt_bias, layer.D):
                p.data = p.data.float()

    def forward(self, ids, caches=None):
        """ids (b, L) -> (logits (b, L, vocab), caches); caches: a list to fill or to go on from, or None."""
        out, h = mh.embedding(ids, self.table, scale=self.scale), None
        new = None if caches is None else []
        for i, (norm, layer) in enumerate(zip(self.norms, self.layers)):
            y, h = norm(out, h)
            out, cache = layer(y, use_cache=caches is not None, cache=caches[i] if caches else None)
            if new is not None:
                new.append(cache)
        y, _ = self.norms[-1](out, h)
        return y @ self.table.t(), new

    def loss(self, ids):
        """Mean negative log probability of every next token, (loss, mean entropy)."""
        logits, _ = self(ids[:, :-1])
        out = mh.token_logprobs(logits, ids[:, 1:].contiguous())
        return -out.logprobs.mean(), out.entropy.mean()

    @torch.no_grad()
    def generate(self, prompt, n, top=3):
        """The likeliest continuation of prompt (b, L) by n tokens: ids (b, n), and for each its ``top`` alternatives with
        their log probabilities, (b, n, top)."""
        logits, caches = self(prompt, [])
        ids, alts, lps = [], [], []
        for _ in range(n):
            last = logits[:, -1]
            out = mh.token_logprobs(last, last.new_zeros(len(last), dtype=torch.int64), top=top)
            ids.append(out.top_ids[:, :1])
            alts.append(out.top_ids)
            lps.append(out.top_logprobs)
            logits, caches = self(ids[-1], caches)
        return torch.cat(ids, 1), torch.stack(alts, 1), torch.stack(lps, 1)


def sequences(vocab, batch, length, device, seed=0):
    """Sequences that a model can learn: each goes through the vocabulary by a step of its own."""
    g = torch.Generator(device=device).manual_seed(seed)
    start = torch.randint(vocab, (batch, 1), generator=g, device=device)
    step = torch.randint(1, 4, (batch, 1), generator=g, device=device)
    return (start + step * torch.arange(length, device=device)) % vocab


def train(model, steps, batch=8, length=128, lr=3e-3):
    """Losses of ``steps`` steps of AdamW."""
    opt = torch.optim.AdamW(model.parameters(), lr=lr, betas=(0.9, 0.95), weight_decay=0.0)
    losses = []
    for i in range(steps):
        ids = sequences(model.table.shape[0], batch, length + 1, model.table.device, seed=i)
        loss, _ = model.loss(ids)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        nn.utils.clip_grad_norm_(model.parameters(), 1.0)
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--vocab", type=int, default=256)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--packed", action="store_true", help="keep the norms' rows for the backward in 8 bits")
    a = ap.parse_args()
    torch.manual_seed(0)
    model = LanguageModel(a.vocab, a.dim, a.layers, packed=a.packed)
    losses = train(model, a.steps)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} (a uniform guess: {math.log(a.vocab):.3f})")
    ids = sequences(a.vocab, 2, 32, "cuda", seed=10 ** 6)
    out, alts, lps = model.generate(ids[:, :24], 8)
    for b in range(2):
        print("prompt ends", ids[b, 20:24].tolist(), "-> continues", out[b].tolist())
        print("  alternatives of the first:", [(int(i), round(float(p), 2)) for i, p in zip(alts[b, 0], lps[b, 0])])


if __name__ == "__main__":
    main()
