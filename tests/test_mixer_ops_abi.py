"""C ABI of the gated delta rule, rotary positions and group norm: arguments that an entry point must refuse before any HIP
call (nothing is launched), outputs that share memory with what is read, and the Python layer's refusals that need no GPU."""

import ctypes as ct

import pytest
import torch

import mamformer_amd as mh
from mamformer_amd import _lib
from tests.test_abi import _rc

MB = 1 << 20
B, H, HK, L, DK, DV = 2, 4, 2, 100, 32, 48
BF, F32 = _lib.MH_BF16, _lib.MH_F32


def at(i):
    return (64 + i) * MB                          # addresses far apart that nothing reads


def rows(i, heads, d):                            # (b, heads, L, d) contiguous
    return at(i), heads * L * d, L * d, d


def delta():
    a = _lib.DeltaArgs(B, H, HK, L, DK, DV, BF, 0.5, *rows(0, HK, DK), *rows(1, HK, DK), *rows(2, H, DV), *rows(3, H, 1),
                       *rows(4, H, 1), at(5), at(6), *rows(7, H, DV))
    a.workspace, a.workspace_bytes = at(1000), 1 << 40
    return a


def delta_bwd():
    return _lib.DeltaBwdArgs(delta(), *rows(8, H, DV), at(9), *rows(10, HK, DK), *rows(11, HK, DK), *rows(12, H, DV), at(13),
                             at(14), at(15), at(1000), 1 << 40)


def delta_kept():
    a = delta_bwd()
    a.kept, a.kept_bytes = at(500), 256 * MB
    return a


def step():
    return _lib.DeltaStepArgs(B, H, HK, DK, DV, BF, 0.5, at(0), HK * DK, DK, at(1), HK * DK, DK, at(2), H * DV, DV, at(3), H, 1,
                              at(4), H, 1, at(5), at(6), at(7), H * DV, DV)


def rotary():
    return _lib.RotaryArgs(B, H, HK, L, DK, 8, BF, 0, 0, 1, 8, 1.0, at(0), at(1), L, 0, *rows(2, H, DK), *rows(3, HK, DK),
                           *rows(4, H, DK), *rows(5, HK, DK))


C, G, S, N = 96, 4, 50, 3


def norm():
    return _lib.GroupNormArgs(N, S, C, G, BF, F32, 1, 0, 1e-5, at(0), S * C, C, at(1), at(2), at(3), S * C, C, at(4), at(5), MB)


def norm_bwd():
    return _lib.GroupNormBwdArgs(norm(), at(6), S * C, C, at(7), S * C, C, at(8), at(9), at(10), MB)


FN = {delta: "mh_delta_rule_fwd", delta_bwd: "mh_delta_rule_bwd", delta_kept: "mh_delta_rule_bwd", step: "mh_delta_step",
      rotary: "mh_rotary", norm: "mh_group_norm_fwd", norm_bwd: "mh_group_norm_bwd"}


def put(a, fields):
    for f, v in fields.items():
        t = a
        while "." in f:
            head, f = f.split(".", 1)
            t = getattr(t, head)
        setattr(t, f, v)
    return a


REFUSED = [
    (delta, dict(batch=-1), -2), (delta, dict(heads=0), -2), (delta, dict(kheads=3), -2), (delta, dict(seqlen=-1), -2),
    (delta, dict(dk=0), -2), (delta, dict(dk=129), -6), (delta, dict(dv=257), -6), (delta, dict(dtype=9), -3),
    (delta, dict(batch=1 << 22), -2), (delta, dict(seqlen=1 << 40), -2), (delta, dict(heads=1 << 40, kheads=1 << 40), -2),
    (delta, dict(q=None), -1), (delta, dict(k=None), -1), (delta, dict(v=None), -1), (delta, dict(o=None), -1),
    (delta, dict(q=at(0) + 1), -5), (delta, dict(g=at(3) + 2), -5), (delta, dict(beta=at(4) + 1), -5),
    (delta, dict(initial_state=at(5) + 2), -5), (delta, dict(final_state=at(6) + 1), -5),
    (delta, dict(q_stride_l=-1), -4), (delta, dict(o_stride_l=DV - 1), -4), (delta, dict(o_stride_h=DV), -4),
    (delta, dict(g_stride_b=-4), -4), (delta, dict(workspace=None), -7), (delta, dict(workspace_bytes=1000), -7),
    (delta, dict(workspace=at(1000) + 8), -7),
    (delta_bwd, {"fwd.dk": 200}, -6), (delta_bwd, {"fwd.v": None}, -1), (delta_bwd, dict(d_o=None), -1),
    (delta_bwd, dict(dq=None), -1), (delta_bwd, dict(dk=None), -1), (delta_bwd, dict(dv=None), -1),
    (delta_bwd, dict(dg=at(13) + 2), -5), (delta_bwd, dict(d_final_state=at(9) + 1), -5),
    (delta_bwd, dict(dk_stride_l=1), -4), (delta_bwd, dict(workspace=None), -7), (delta_bwd, dict(workspace_bytes=1 << 10), -7),
    (delta_kept, dict(kept_bytes=1 << 10), -7), (delta_kept, dict(kept=at(500) + 4), -7), (delta_kept, dict(workspace=None), -7),
    (step, dict(batch=-1), -2), (step, dict(kheads=3), -2), (step, dict(dk=129), -6), (step, dict(dv=300), -6),
    (step, dict(state_in=None), -1), (step, dict(state_out=None), -1), (step, dict(o=None), -1), (step, dict(q=None), -1),
    (step, dict(state_in=at(5) + 2), -5), (step, dict(dtype=-1), -3), (step, dict(o_stride_h=1), -4),
    (rotary, dict(pairs=17), -2), (rotary, dict(pairs=0), -2), (rotary, dict(dim=0), -2), (rotary, dict(q=None), -1),
    (rotary, dict(k=None), -1), (rotary, dict(q_out=None), -1), (rotary, dict(inv_freq=None), -1),
    (rotary, dict(inv_freq=at(0) + 4), -5), (rotary, dict(positions=at(1) + 4), -5), (rotary, dict(index_bytes=2), -3),
    (rotary, dict(dtype=5), -3), (rotary, dict(k_out_stride_l=3), -4), (rotary, dict(q_stride_b=-8), -4),
    (rotary, dict(positions_stride_b=-1), -4),
    (norm, dict(batch=-1), -2), (norm, dict(groups=5), -2), (norm, dict(channels=0), -2), (norm, dict(channels=65540), -6),
    (norm, dict(eps=-1.0), -2), (norm, dict(eps=float("nan")), -2), (norm, dict(x=None), -1), (norm, dict(y=None), -1),
    (norm, dict(weight=at(1) + 2), -5), (norm, dict(weight_dtype=4), -3), (norm, dict(stats=at(4) + 2), -5),
    (norm, dict(y_stride_s=C - 1), -4), (norm, dict(space=1 << 41), -2), (norm, dict(workspace_bytes=0), -7),
    (norm_bwd, dict(dy=None), -1), (norm_bwd, dict(dx=None), -1), (norm_bwd, {"fwd.stats": None}, -1),
    (norm_bwd, dict(dweight=at(8) + 1), -5), (norm_bwd, dict(dx_stride_s=2), -4), (norm_bwd, dict(workspace=None), -7),
]


@pytest.mark.parametrize("make,fields,code", REFUSED)
def test_refusals(make, fields, code):
    assert _rc(FN[make], ct.byref(put(make(), fields)), None) == code
    assert _lib.lib().mh_last_error()


SHARED = [
    (delta, dict(o=at(2))), (delta, dict(o=at(0) + 2)), (delta, dict(o=at(3))), (delta, dict(final_state=at(5))),
    (delta, dict(final_state=at(1))), (delta, dict(workspace=at(2), workspace_bytes=200 * MB)), (delta, dict(o=at(1000) + 16)),
    (delta_bwd, dict(dq=at(0))), (delta_bwd, dict(dk=at(10) + 64)), (delta_bwd, dict(dv=at(8))), (delta_bwd, dict(dg=at(3))),
    (delta_bwd, dict(dbeta=at(13) + 4)), (delta_bwd, dict(d_initial_state=at(9))), (delta_bwd, dict(d_initial_state=at(5))),
    (delta_kept, dict(workspace=at(500), workspace_bytes=256 * MB)), (delta_kept, dict(dv=at(500))),
    (step, dict(o=at(2))), (step, dict(state_out=at(5) + 4)), (step, dict(o=at(6))), (step, dict(state_out=at(1))),
    (rotary, dict(q_out=at(2) + 2)), (rotary, dict(k_out=at(4))), (rotary, dict(q_out=at(1))), (rotary, dict(k_out=at(0))),
    (rotary, dict(q_out=at(3))), (rotary, dict(q_out=at(2), q_out_stride_l=DK + 1, q_out_stride_h=L * (DK + 1),
                                               q_out_stride_b=H * L * (DK + 1))),
    (norm, dict(y=at(0) + 2)), (norm, dict(stats=at(3))), (norm, dict(y=at(1))),
    (norm_bwd, dict(dx=at(0) + 2)), (norm_bwd, dict(dx=at(6) + 2)), (norm_bwd, dict(dbias=at(8))), (norm_bwd, dict(dx=at(4))),
    (norm_bwd, dict(dweight=at(1))),
]


@pytest.mark.parametrize("make,fields", SHARED)
def test_shared_memory_is_refused(make, fields):
    assert _rc(FN[make], ct.byref(put(make(), fields)), None) == -4
    assert b"overlap" in _lib.lib().mh_last_error()


@pytest.mark.parametrize("fn", sorted(set(FN.values())))
def test_null_block(fn):
    assert _rc(fn, None, None) == -1


def test_queries():
    n = ct.c_size_t()
    for q, make in (("mh_delta_rule_workspace_bytes", delta), ("mh_delta_rule_bwd_workspace_bytes", delta_bwd),
                    ("mh_group_norm_workspace_bytes", norm), ("mh_group_norm_bwd_workspace_bytes", norm_bwd)):
        assert _rc(q, ct.byref(make()), ct.byref(n)) == 0 and n.value > 0
        assert _rc(q, ct.byref(make()), None) == -1
        assert _rc(q, None, ct.byref(n)) == -1

    def size(a, q="mh_delta_rule_workspace_bytes"):
        assert _rc(q, ct.byref(a), ct.byref(n)) == 0
        return n.value
    plain, keep = size(delta()), size(put(delta(), dict(keep=1)))
    bwd = "mh_delta_rule_bwd_workspace_bytes"
    # what a forward keeps and what a backward needs beside it are what a backward alone needs
    assert plain < keep and size(delta_bwd(), bwd) == keep + size(delta_kept(), bwd)
    assert size(put(delta(), dict(seqlen=0))) == 0 and size(put(delta(), dict(batch=0))) == 0


def test_no_rows_launch_nothing():
    for make, fields in ((delta, dict(batch=0)), (delta_bwd, {"fwd.batch": 0}), (step, dict(batch=0)), (rotary, dict(batch=0)),
                         (rotary, dict(seqlen=0)), (norm, dict(batch=0)),
                         (delta, dict(seqlen=0, final_state=None, q=None, k=None, v=None, o=None))):
        assert _rc(FN[make], ct.byref(put(make(), fields)), None) == 0, (make, fields)


def test_cpu_tensors_are_refused():
    q, v, s = torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 8, 8)
    x, st = torch.zeros(2, 3, 8), torch.zeros(2, 2, 2)
    for call in (lambda: mh.gated_delta_rule(q, q, v), lambda: mh.gated_delta_rule_bwd(v, q, q, v),
                 lambda: mh.gated_delta_step(s, q[:, :, 0], q[:, :, 0], v[:, :, 0]), lambda: mh.rotary(q, q, torch.zeros(4)),
                 lambda: mh.group_norm(x, 2), lambda: mh.group_norm_bwd(x, x, st, 2)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
