"""C ABI of the token operators: arguments that an entry point must refuse, before any HIP call (nothing is launched),
and the Python layer's refusals that need no GPU."""

import ctypes as ct

import pytest
import torch

import mamformer_amd as mh
from mamformer_amd import _lib
from tests.test_abi import _rc

P = 1 << 20                                       # an aligned address that nothing reads


def embed():
    return _lib.EmbeddingArgs(10, 100, 64, _lib.MH_BF16, 8, 1.0, P, P, 64, P, 64)


def embed_bwd():
    return _lib.EmbeddingBwdArgs(10, 100, 64, -1, _lib.MH_BF16, 8, _lib.MH_F32, 1.0, P, P, 64, P, P, 1 << 30)


def norm():
    return _lib.LayerNormArgs(10, 64, _lib.MH_BF16, _lib.MH_F32, 1e-5, P, 64, P, 64, P, P, P, 64, P, 64, P, P, P)


def norm_bwd():
    return _lib.LayerNormBwdArgs(10, 64, _lib.MH_BF16, _lib.MH_F32, P, 64, P, 64, P, P, P, P, P, 64, P, 64, P, P, P,
                                 1 << 30)


def pack():
    return _lib.PackArgs(10, 64, _lib.MH_BF16, 0, P, 64, P, P)


def logprob():
    return _lib.LogprobArgs(10, 64, -100, _lib.MH_BF16, 8, 5, 1.0, P, 64, P, P, P, P, P, P, P, 1 << 30)


def logprob_bwd():
    return _lib.LogprobBwdArgs(10, 64, -100, _lib.MH_BF16, 8, 1.0, P, 64, P, P, P, P, P + (1 << 20), 64)


CALLS = {"mh_embedding_fwd": embed, "mh_embedding_bwd": embed_bwd, "mh_layer_norm_fwd": norm,
         "mh_layer_norm_bwd": norm_bwd, "mh_pack_activations": pack, "mh_unpack_activations": pack,
         "mh_token_logprobs_fwd": logprob, "mh_token_logprobs_bwd": logprob_bwd}
INF = float("inf")

REFUSED = [
    ("mh_embedding_fwd", dict(tokens=-1), -2), ("mh_embedding_fwd", dict(dim=0), -2),
    ("mh_embedding_fwd", dict(vocab=0), -2), ("mh_embedding_fwd", dict(tokens=1 << 31), -2),
    ("mh_embedding_fwd", dict(dtype=7), -3), ("mh_embedding_fwd", dict(index_bytes=2), -3),
    ("mh_embedding_fwd", dict(ids=None), -1), ("mh_embedding_fwd", dict(weight=None), -1),
    ("mh_embedding_fwd", dict(out=None), -1), ("mh_embedding_fwd", dict(ids=P + 4), -5),
    ("mh_embedding_fwd", dict(weight=P + 1), -5), ("mh_embedding_fwd", dict(out_stride=63), -4),
    ("mh_embedding_fwd", dict(weight_stride=-64), -4),
    ("mh_embedding_bwd", dict(vocab=1 << 31), -2), ("mh_embedding_bwd", dict(dweight=None), -1),
    ("mh_embedding_bwd", dict(dweight=P + 2), -5), ("mh_embedding_bwd", dict(dweight_dtype=2), -3),
    ("mh_embedding_bwd", dict(dy=None), -1), ("mh_embedding_bwd", dict(workspace=None), -7),
    ("mh_embedding_bwd", dict(workspace_bytes=64), -7), ("mh_embedding_bwd", dict(workspace=P + 8), -7),
    ("mh_layer_norm_fwd", dict(dim=16385), -6), ("mh_layer_norm_fwd", dict(rows=-1), -2),
    ("mh_layer_norm_fwd", dict(eps=-1e-5), -2), ("mh_layer_norm_fwd", dict(eps=float("nan")), -2),
    ("mh_layer_norm_fwd", dict(weight_dtype=3), -3), ("mh_layer_norm_fwd", dict(weight=P + 2), -5),
    ("mh_layer_norm_fwd", dict(h=None), -1), ("mh_layer_norm_fwd", dict(y_stride=32), -4),
    ("mh_layer_norm_fwd", dict(codes=None), -1), ("mh_layer_norm_fwd", dict(codes=P + 4), -5),
    ("mh_layer_norm_bwd", dict(stats=None), -1), ("mh_layer_norm_bwd", dict(h=None, codes=None), -1),
    ("mh_layer_norm_bwd", dict(h=None, codes=P + 4), -5), ("mh_layer_norm_bwd", dict(dx=P + 1), -5),
    ("mh_layer_norm_bwd", dict(dx_stride=0), -4), ("mh_layer_norm_bwd", dict(dweight=P + 2), -5),
    ("mh_layer_norm_bwd", dict(workspace_bytes=0), -7), ("mh_layer_norm_bwd", dict(d_h_stride=-1), -4),
    ("mh_pack_activations", dict(x=None), -1), ("mh_pack_activations", dict(exponents=None), -1),
    ("mh_pack_activations", dict(codes=P + 2), -5), ("mh_pack_activations", dict(x_stride=-1), -4),
    ("mh_unpack_activations", dict(x_stride=63), -4), ("mh_unpack_activations", dict(dtype=5), -3),
    ("mh_token_logprobs_fwd", dict(temperature=0.0), -2), ("mh_token_logprobs_fwd", dict(temperature=-1.0), -2),
    ("mh_token_logprobs_fwd", dict(temperature=INF), -2), ("mh_token_logprobs_fwd", dict(temperature=1e-40), -2),
    ("mh_token_logprobs_fwd", dict(top=65), -6), ("mh_token_logprobs_fwd", dict(top=-1), -6),
    ("mh_token_logprobs_fwd", dict(vocab=4), -6), ("mh_token_logprobs_fwd", dict(targets=None), -1),
    ("mh_token_logprobs_fwd", dict(top_ids=None), -1), ("mh_token_logprobs_fwd", dict(stats=None), -1),
    ("mh_token_logprobs_fwd", dict(top_ids=P + 4), -5), ("mh_token_logprobs_fwd", dict(index_bytes=0), -3),
    ("mh_token_logprobs_bwd", dict(stats=None), -1), ("mh_token_logprobs_bwd", dict(dlogits=P + 2), -4),
    ("mh_token_logprobs_bwd", dict(dlogits=P, dlogits_stride=65), -4),
    ("mh_token_logprobs_bwd", dict(dlogits=P + 64 * 2 * 9 + 2), -4), ("mh_token_logprobs_bwd", dict(dlogits=None), -1),
    ("mh_token_logprobs_bwd", dict(temperature=float("nan")), -2),
]


@pytest.mark.parametrize("fn,fields,code", REFUSED)
def test_refusals(fn, fields, code):
    a = CALLS[fn]()
    for f, v in fields.items():
        setattr(a, f, v)
    assert _rc(fn, ct.byref(a), None) == code
    assert _lib.lib().mh_last_error()


@pytest.mark.parametrize("fn", CALLS)
def test_null_block(fn):
    assert _rc(fn, None, None) == -1


def test_queries():
    n = ct.c_size_t()
    for fn, make in (("mh_embedding_bwd", embed_bwd), ("mh_layer_norm_bwd", norm_bwd), ("mh_token_logprobs", logprob)):
        q = fn + "_workspace_bytes"
        assert _rc(q, ct.byref(make()), ct.byref(n)) == 0
        assert _rc(q, ct.byref(make()), None) == -1
        assert _rc(q, None, ct.byref(n)) == -1
    a = norm_bwd()
    a.dweight = a.dbias = None
    assert _rc("mh_layer_norm_bwd_workspace_bytes", ct.byref(a), ct.byref(n)) == 0 and n.value == 0
    b = embed_bwd()                               # room for the sort's two (id, token) arrays
    b.tokens = 1 << 20
    assert _rc("mh_embedding_bwd_workspace_bytes", ct.byref(b), ct.byref(n)) == 0 and n.value >= 16 << 20


def test_no_rows_launch_nothing():
    for fn, make, rows in (("mh_embedding_fwd", embed, "tokens"), ("mh_layer_norm_fwd", norm, "rows"),
                           ("mh_pack_activations", pack, "rows"), ("mh_unpack_activations", pack, "rows"),
                           ("mh_token_logprobs_fwd", logprob, "rows"), ("mh_token_logprobs_bwd", logprob_bwd, "rows")):
        a = make()
        setattr(a, rows, 0)
        assert _rc(fn, ct.byref(a), None) == 0, fn


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    ids = torch.zeros(3, dtype=torch.int64)
    for call in (lambda: mh.embedding(ids, x), lambda: mh.embedding_bwd(x, ids, 4), lambda: mh.layer_norm(x, w),
                 lambda: mh.layer_norm_bwd(x, x, torch.zeros(3, 2)), lambda: mh.pack_activations(x),
                 lambda: mh.unpack_activations(mh.PackedActivations(torch.zeros(3, 64, dtype=torch.int8),
                                                                    torch.zeros(3, 1, dtype=torch.uint8), 8, x.dtype)),
                 lambda: mh.token_logprobs(x, ids), lambda: mh.token_logprobs_bwd(x, ids, torch.zeros(3, 3))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.parametrize("temperature", [3e-39, 3.5e-39, 4.23e-39])
def test_temperature_whose_scale_leaves_fp32(temperature):
    """1 / temperature is in fp32's range, log2(e) / temperature is not."""
    for fn, make in (("mh_token_logprobs_fwd", logprob), ("mh_token_logprobs_bwd", logprob_bwd)):
        a = make()
        a.temperature = temperature
        assert 1 / a.temperature < 3.4e38 and _rc(fn, ct.byref(a), None) == -2
