"""The example's model: its loss and gradients against the same model from torch's own operators, training, generation."""

import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "language_model.py"
    spec = importlib.util.spec_from_file_location("language_model_example", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def torch_loss(model, ids):
    """The model with torch's lookup, norm and log softmax around the same Mamba layers."""
    D = model.table.shape[1]
    out, h = F.embedding(ids[:, :-1], model.table) * model.scale, None
    for norm, layer in zip(model.norms, [*model.layers, None]):
        h = out if h is None else out + h
        y = F.layer_norm(h, (D,), norm.weight, norm.bias, 1e-5)
        if layer is not None:
            out, _ = layer(y)
    logits = y @ model.table.t()
    return F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(), ids[:, 1:].reshape(-1))


def test_loss_and_gradients_fp32():
    """Both sides are fp32; they differ by the order of their sums (about 2^-24 sqrt(n) a step, some tens of steps deep,
    against gradients that sum over 2 x 96 tokens): 1e-4 of the norm, as for the scans in fp32.  Compared are the gradients
    of these operators' own parameters, table and norms, which all pass through the layers; the layers' parameters have
    tests of their own (a decay's gradient is a sum of two heads' worth of terms that cancel)."""
    ex = example()
    torch.manual_seed(1)
    model = ex.LanguageModel(101, 128, 2, dtype=torch.float32)
    ids = ex.sequences(101, 2, 97, "cuda")
    loss, ent = model.loss(ids)
    own = [model.table, *model.norms.parameters()]
    grads = torch.autograd.grad(loss, own)
    want = torch_loss(model, ids)
    ref = torch.autograd.grad(want, own)
    assert abs(loss.item() - want.item()) <= 1e-4 * want.item() and ent.item() > 0
    for name, g, r in zip(["table", *(n for n, _ in model.norms.named_parameters())], grads, ref):
        err = (g.double() - r.double()).norm() / r.double().norm().clamp_min(1e-30)
        print(f"{name}: {err.item():.2e}", flush=True)
        assert err <= 1e-4, name


@pytest.mark.parametrize("packed", [False, True])
def test_training_and_generation(packed):
    ex = example()
    torch.manual_seed(0)
    model = ex.LanguageModel(64, 128, 2, packed=packed)
    losses = ex.train(model, 60, batch=8, length=96)
    print(f"packed={packed}: loss {losses[0]:.3f} -> {losses[-1]:.3f}", flush=True)
    assert losses[-1] < 0.5 * losses[0]
    ids = ex.sequences(64, 3, 40, "cuda", seed=12345)
    out, alts, lps = model.generate(ids[:, :32], 8)
    assert out.shape == (3, 8) and alts.shape == lps.shape == (3, 8, 3)
    assert torch.equal(alts[:, :, 0], out) and (lps[..., 0] >= lps[..., 1]).all() and (lps <= 0).all()
    with torch.no_grad():                        # the last tokens again from a prompt that holds the others
        logits, _ = model(torch.cat([ids[:, :32], out[:, :-1]], 1))
    again = logits[:, 31:].float().log_softmax(-1).gather(-1, alts)
    # bf16 logits of two ways through the layers: rounding steps of 2^-8 of values up to |lp| and the layers' own
    assert (again - lps).abs().max() <= 0.25
