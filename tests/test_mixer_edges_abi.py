"""C ABI of the gated delta rule, rotary positions and group norm at the ends of their ranges: refused before any HIP call."""

import ctypes as ct

import pytest

from mamformer_amd import _lib
from tests.test_abi import _rc
from tests.test_mixer_ops_abi import FN, delta, delta_bwd


def heads(a, batch, n):
    """The block for so many heads of one token, a key head each."""
    f = a.fwd if hasattr(a, "fwd") else a
    f.batch, f.heads, f.kheads, f.seqlen = batch, n, n, 1
    return a


@pytest.mark.parametrize("make", [delta, delta_bwd])
def test_heads_beyond_a_grid(make):
    """dv = 48: two workgroups a head, of which 2^23 are a grid's."""
    n = ct.c_size_t()
    query = FN[make].replace("_fwd", "") + "_workspace_bytes"
    assert _rc(query, ct.byref(heads(make(), 1 << 20, 4)), ct.byref(n)) == 0 and n.value > 0
    for fn, last in ((query, ct.byref(n)), (FN[make], None)):
        assert _rc(fn, ct.byref(heads(make(), 1 << 20, 5)), last) == -2
        assert b"32 columns" in _lib.lib().mh_last_error()
