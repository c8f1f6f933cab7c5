"""C ABI of the token operators: outputs that share memory with an input or with each other are refused before any HIP call,
except a row tensor that is exactly its input's; rows beside each other in one wider buffer share nothing."""

import ctypes as ct

import pytest

from mamformer_amd import _lib
from tests.test_abi import _rc

BF, F32 = _lib.MH_BF16, _lib.MH_F32
R, D, MB = 10, 64, 1 << 20
STRIDE = -4


def at(i):
    return (16 + i) * MB                          # addresses far apart that nothing reads


def embed():
    return _lib.EmbeddingArgs(R, 100, D, BF, 8, 1.0, at(0), at(1), D, at(2), D)


def embed_bwd():
    return _lib.EmbeddingBwdArgs(R, 100, D, -1, BF, 8, F32, 1.0, at(0), at(1), D, at(2), at(3), 1 << 16)


def norm():
    return _lib.LayerNormArgs(R, D, BF, F32, 1e-5, at(0), D, at(1), D, at(2), at(3), at(4), D, at(5), D, at(6), at(7), at(8))


def norm_bwd():
    return _lib.LayerNormBwdArgs(R, D, BF, F32, at(0), D, at(1), D, None, None, at(2), at(3), at(4), D, at(5), D, at(6), at(7),
                                 at(8), 1 << 16)


def packed_bwd():
    a = norm_bwd()
    a.h, a.codes, a.exponents = None, at(9), at(10)
    return a


def pack():
    return _lib.PackArgs(R, D, BF, 0, at(0), D, at(1), at(2))


def logprob():
    return _lib.LogprobArgs(R, D, -100, BF, 8, 5, 1.0, at(0), D, at(1), at(2), at(3), at(4), at(5), at(6), at(7), 1 << 16)


def logprob_bwd():
    return _lib.LogprobBwdArgs(R, D, -100, BF, 8, 1.0, at(0), D, at(1), at(2), at(3), at(4), at(5), D)


FN = {embed: "mh_embedding_fwd", embed_bwd: "mh_embedding_bwd", norm: "mh_layer_norm_fwd", norm_bwd: "mh_layer_norm_bwd",
      packed_bwd: "mh_layer_norm_bwd", pack: "mh_pack_activations", logprob: "mh_token_logprobs_fwd",
      logprob_bwd: "mh_token_logprobs_bwd"}
ROW = 2 * D                                       # bytes of a bf16 row
LAST = (R - 1) * ROW                              # where the last row begins

REFUSED = [
    # row tensors: a row further, an element further, the last row, another stride in the same place
    (embed, dict(out=at(1))), (embed, dict(out=at(1) + 99 * ROW)), (embed, dict(out=at(0))), (embed, dict(ids=at(2) + LAST)),
    (embed_bwd, dict(dweight=at(1))), (embed_bwd, dict(dy=at(2) + 99 * 4 * D)), (embed_bwd, dict(ids=at(2) + 8)),
    (embed_bwd, dict(workspace=at(2))), (embed_bwd, dict(workspace=at(1) + LAST)),
    (norm, dict(y=at(0) + ROW)), (norm, dict(y=at(0) + 2)), (norm, dict(y=at(0) - LAST)), (norm, dict(y=at(0), y_stride=D + 8)),
    (norm, dict(h=at(1) + 4)), (norm, dict(h=at(4))), (norm, dict(h=at(2))), (norm, dict(y=at(3) - 32)),
    (norm, dict(y=at(0) + ROW, x_stride=2 * D, y_stride=2 * D - 8)),
    (norm, dict(x_stride=0, y=at(0))),            # one row read ten times and written ten times
    (norm, dict(stats=at(0))), (norm, dict(stats=at(4) + LAST)), (norm, dict(codes=at(1) + 8)), (norm, dict(exponents=at(5))),
    (norm, dict(exponents=at(7) + 1)), (norm, dict(stats=at(8) + 8)),
    (norm_bwd, dict(dx=at(0) + ROW)), (norm_bwd, dict(dx=at(1) + 2)), (norm_bwd, dict(dx=at(4), dx_stride=2 * D)),
    (norm_bwd, dict(dx=at(2))), (norm_bwd, dict(dx=at(3) - 2)), (norm_bwd, dict(dweight=at(5))), (norm_bwd, dict(dbias=at(6) + 4)),
    (norm_bwd, dict(dbias=at(0))), (norm_bwd, dict(dweight=at(3))),
    (norm_bwd, dict(workspace=at(0))), (norm_bwd, dict(workspace=at(7))),
    (packed_bwd, dict(dx=at(9))), (packed_bwd, dict(dx=at(10))),
    (pack, dict(codes=at(0) + 8)), (pack, dict(exponents=at(1))), (pack, dict(exponents=at(0) + LAST)),
    (logprob, dict(logprobs=at(0))), (logprob, dict(entropy=at(2) + 4)), (logprob, dict(stats=at(1))),
    (logprob, dict(top_ids=at(3))), (logprob, dict(top_logprobs=at(5) + 8)),
    (logprob, dict(vocab=9000, logits_stride=9000, workspace=at(5))),
    (logprob_bwd, dict(dlogits=at(0) + ROW)), (logprob_bwd, dict(dlogits=at(0) + 2)), (logprob_bwd, dict(dlogits=at(1))),
    (logprob_bwd, dict(dlogits=at(2))), (logprob_bwd, dict(dlogits=at(3))), (logprob_bwd, dict(dlogits=at(4) - 16)),
    (logprob_bwd, dict(logits_stride=2 * D, dlogits_stride=2 * D, dlogits=at(0) + ROW - 2)),
]


@pytest.mark.parametrize("make,fields", REFUSED)
def test_shared_memory_is_refused(make, fields):
    a = make()
    for f, v in fields.items():
        setattr(a, f, v)
    assert _rc(FN[make], ct.byref(a), None) == STRIDE
    assert b"overlap" in _lib.lib().mh_last_error()


def test_unpacking_over_its_codes_is_refused():
    for f, v in (("x", at(1)), ("x", at(2) - LAST)):
        a = pack()
        setattr(a, f, v)
        assert _rc("mh_unpack_activations", ct.byref(a), None) == STRIDE
