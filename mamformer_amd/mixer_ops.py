"""Operators around and beside the linear-attention scans of ``ops``: what a token mixer runs before, as and behind its scan.

=====================================  ====================================================================
``rotary_frequencies``, ``rotary``      rotary positions of queries and keys, whole or part of the head, in both pair
                                        layouts, scaled for long contexts (R/mamformer/layers/rope.py:36-392, applied
                                        at R/mamformer/layers/kda_diff.py:276-280)
``gated_delta_rule``,                   the scan that corrects its state: each token replaces what the decayed state
``gated_delta_rule_bwd``,               answers to its key instead of adding to it; over sequences, with its gradients,
``gated_delta_step``                    and for one token
``group_norm``, ``group_norm_bwd``      group norm, channels last, with its affine part and an activation fused (the
                                        norm behind the scan, R/mamformer/layers/kda_diff.py:345-348), and its backward
=====================================  ====================================================================

``rotary``, ``gated_delta_rule`` and ``group_norm`` are differentiable (a tensor with a forward-mode tangent is refused); the
``_bwd`` functions give the gradients explicitly.  bf16 and fp32 tensors of any strides (a last dimension that is not
contiguous is copied).  As in ``ops``, every call launches kernels of ``libmamformer_hip.so`` on the current torch stream,
does not synchronise, and has no CPU path.  All results are the same bits at every call with the same inputs.
"""

from __future__ import annotations

import ctypes as ct
import math

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import (DeltaArgs, DeltaBwdArgs, DeltaStepArgs, GroupNormArgs, GroupNormBwdArgs, RotaryArgs)
from .ops import _DT, _ptr, _require_cuda, _stream
from .token_ops import _INDEX_BYTES, _dtype, _like, _norm_params, _optional_workspace, _vec

__all__ = ["rotary_frequencies", "rotary", "gated_delta_rule", "gated_delta_rule_bwd", "gated_delta_step", "group_norm",
           "group_norm_bwd"]


def _through_autograd(*ts):
    """Whether a call goes through its autograd function (as in ``token_ops``: a forward-mode level counts, and raises there)."""
    if _forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _channels(t):
    """t with contiguous channels (a copy where they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _result(t):
    """(a new tensor of t's layout, its strides), with contiguous channels: torch may order dimensions of equal strides the
    other way."""
    out = torch.empty_like(t)
    st = out.stride()
    if st[-1] != 1 and t.shape[-1] != 1:
        out = torch.empty(t.shape, device=t.device, dtype=t.dtype)
        st = out.stride()
    return out, st


def _f32(t):
    return t if t is None or t.dtype is torch.float32 else t.to(torch.float32)


def _strides3(t):
    return (None, 0, 0, 0) if t is None else (t.data_ptr(), *t.stride()[:3])


def _strides2(t):
    return (None, 0, 0) if t is None else (t.data_ptr(), *t.stride()[:2])


# ------------------------------------------------------------------------------------------------ rotary positions

def rotary_frequencies(dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0,
                       device="cuda"):
    """(inv_freq, scale) for ``rotary``: the angles per position of ``dim / 2`` pairs, float64 on ``device``, and the factor
    for the turned channels.

    scaling=None: ``base ** (-2 i / dim)``.  For contexts ``factor`` times as long as those trained on: ``"linear"`` divides
    the frequencies by factor; ``"ntk"`` raises the base to ``base * factor ** (dim / (dim - 2))``; ``"yarn"`` divides those
    whose wave turns less than ``beta_slow`` times in ``original_length``, keeps those that turn more than ``beta_fast``
    times, ramps between, and scales by ``0.1 ln(factor) + 1``.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary_frequencies: dim must be even and positive, got {dim}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r} (linear, ntk, yarn)")
    if not base > 0 or not factor >= 1:
        raise ValueError(f"rotary_frequencies: base must be positive and factor at least 1, got {base}, {factor}")
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    scale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if not original_length or not beta_fast > beta_slow > 0:
            raise ValueError("rotary_frequencies: yarn needs original_length and beta_fast > beta_slow > 0")

        def pair(turns):                         # the pair whose wave turns so many times in original_length
            return dim * math.log(original_length / (2 * math.pi * turns)) / (2 * math.log(base))

        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    return freq.to(device), scale


def rotary(q, k, inv_freq, positions=None, *, offset=0, interleaved=False, scale=1.0, inverse=False):
    """Rotary positions of queries and keys: (q', k'), or q' alone where ``k`` is None; new tensors of their layouts.

    q (B, H, L, D) and k (B, HK, L, D) of one dtype; inv_freq (n,) float32 or float64 with 2 n <= D.  Of the first 2 n
    channels the pairs (i, n + i), or with ``interleaved`` (2 i, 2 i + 1), are turned by the angle
    (positions + offset) * inv_freq[i] and multiplied by ``scale``; the others are copied.  ``positions``: int32 or int64
    (L,) or (B, L), None for 0 .. L - 1.  Angles are reduced in 64 bits: one of x radians
    is off by x 2^-51 at most, less than fp32's own rounding up to 2^27.  ``inverse`` turns back, which with the same ``scale`` is the gradient.  Differentiable in q and k (an inv_freq that requires
    a gradient is refused).
    """
    name = "rotary"
    _require_cuda(name, q, k, inv_freq, positions)
    qs, ks = q.shape, None if k is None else k.shape
    if len(qs) != 4 or k is not None and (len(ks) != 4 or ks[0] != qs[0] or ks[2] != qs[2] or ks[3] != qs[3]
                                          or k.dtype is not q.dtype):
        raise ValueError(f"{name}: q and k must be (B, H, L, D) and (B, HK, L, D) of one dtype, got {tuple(q.shape)} and "
                         f"{None if k is None else tuple(k.shape)}")
    _dtype(name, "q", q)
    if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float32, torch.float64) or not 2 <= 2 * inv_freq.shape[0] <= qs[3]:
        raise ValueError(f"{name}: inv_freq must be (n,) float32 or float64 with 2 <= 2 n <= {q.shape[3]}, got "
                         f"{tuple(inv_freq.shape)} {inv_freq.dtype}")
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name}: has no gradient for inv_freq; detach it")
    if positions is not None:
        if positions.dtype not in _INDEX_BYTES:
            raise TypeError(f"{name}: positions must be int32 or int64, got {positions.dtype}")
        if positions.shape not in ((qs[2],), (qs[0], qs[2])):
            raise ValueError(f"{name}: positions must be (L,) or (B, L), got {tuple(positions.shape)} for q {tuple(q.shape)}")
    offset = int(offset)
    if not -1 << 63 <= offset < 1 << 63:
        raise ValueError(f"{name}: offset {offset} outside 64 bits")
    cfg = (offset, bool(interleaved), float(scale), bool(inverse))
    if _through_autograd(q, k):
        out = _RotaryFn.apply(q, k, inv_freq, positions, cfg)
    else:
        out = _rotary(q, k, inv_freq, positions, cfg)
    return out if k is not None else out[0]


def _rotary(q, k, inv_freq, positions, cfg):
    offset, interleaved, scale, inverse = cfg
    q = _channels(q)
    B, H, L, D = q.shape
    if not H and k is not None:                  # keys alone
        return torch.empty_like(q), _rotary(k, None, inv_freq, positions, cfg)[0]
    inv_freq = _vec(inv_freq)
    pos_sb = 0
    if positions is not None:
        if positions.stride(-1) != 1 and L != 1:
            positions = positions.contiguous()
        pos_sb = positions.stride(0) if positions.dim() == 2 else 0
    (qo, (ob, oh, ol, _)), ko, HK = _result(q), None, 0
    if k is not None:
        k = _channels(k)
        (ko, ks), HK = _result(k), k.shape[1]
    qb, qh, ql, _ = q.stride()
    a = RotaryArgs(B, H, HK, L, D, inv_freq.shape[0], _DT[q.dtype], interleaved, inverse, inv_freq.dtype is torch.float64,
                   0 if positions is None else _INDEX_BYTES[positions.dtype], scale, inv_freq.data_ptr(), _ptr(positions), pos_sb,
                   offset, q.data_ptr(), qb, qh, ql)
    a.q_out, a.q_out_stride_b, a.q_out_stride_h, a.q_out_stride_l = qo.data_ptr(), ob, oh, ol
    if HK:
        a.k, a.k_stride_b, a.k_stride_h, a.k_stride_l = _strides3(k)
        a.k_out, a.k_out_stride_b, a.k_out_stride_h, a.k_out_stride_l = ko.data_ptr(), *ks[:3]
    if H:
        _lib.call("mh_rotary", ct.byref(a), _stream(q.device))
    return qo, ko


class _RotaryFn(torch.autograd.Function):
    """Autograd node of ``rotary``: its backward is the turn by the negative angles."""

    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, cfg):
        ctx.save_for_backward(inv_freq, positions)
        ctx.cfg = (cfg[0], cfg[1], cfg[2], not cfg[3])
        ctx.set_materialize_grads(False)
        return _rotary(q, k, inv_freq, positions, cfg)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        inv_freq, positions = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        if dq is None and dk is None:
            return (None,) * 5
        if dq is None:
            return None, _rotary(dk, None, inv_freq, positions, ctx.cfg)[0], None, None, None
        return *_rotary(dq, dk, inv_freq, positions, ctx.cfg), None, None, None


# ------------------------------------------------------------------------------------------------ gated delta rule

def gated_delta_rule(q, k, v, g=None, beta=None, *, scale=None, initial_state=None, return_final_state=False,
                     recompute=False):
    """Gated delta rule over sequences: o (B, H, L, dv) like v, or (o, final state (B, H, dk, dv) float32).

    With a state S (dk, dv) in fp32 for each (batch, head), zero or ``initial_state``:
        S_t = e^{g_t} S_{t-1} + beta_t k_t (v_t - e^{g_t} S_{t-1}^T k_t)^T,   o_t = scale S_t^T q_t
    q, k (B, HK, L, dk) and v (B, H, L, dv) of one dtype, dk <= 128, dv <= 256, H a multiple of HK (value head h reads key
    head h // (H // HK)); g (log decay, None: 0; -inf clears the state) and beta (None: 1) (B, H, L); scale: None is
    dk ** -0.5.  Keys are taken as they are: for a stable state beta |k|^2 <= 2, so normalise them before.

    Operands of the products keep 22 bits of the largest value of their column or piece, sums are fp32: results are exact to
    about 2^-20 of the norms that enter them, before the one rounding to bf16.

    A token with beta = 0 and g = 0 changes nothing, which is what padding behind a sequence takes, with finite q, k and v: a
    NaN or infinity, a padding token's too, may reach every result of its head from the 64-token piece that holds it on.
    With L = 0 the state goes through.
    Differentiable in all tensors: a call that records a gradient keeps the states and systems of its pieces for it, about
    3 KB a token and head of 128 x 128 (bf16); with ``recompute`` it keeps its inputs alone, and the gradients' pass computes
    the rest again (a fifth more time for a training step).  The gradients are the same bits.
    """
    name = "gated_delta_rule"
    _require_cuda(name, q, k, v, g, beta, initial_state)
    _delta_shapes(name, q, k, v, g, beta, initial_state, 4)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if _through_autograd(q, k, v, g, beta, initial_state):
        o, final = _GatedDeltaFn.apply(q, k, v, g, beta, initial_state, scale, return_final_state, recompute)
    else:
        o, final, _ = _delta_fwd(q, k, v, g, beta, initial_state, scale, return_final_state, False)
    return (o, final) if return_final_state else o


def _delta_shapes(name, q, k, v, g, beta, state, dims):
    qs, vs = q.shape, v.shape
    if len(qs) != dims or len(vs) != dims or qs != k.shape or qs[0] != vs[0] or dims == 4 and qs[2] != vs[2]:
        t = ", L" if dims == 4 else ""
        raise ValueError(f"{name}: q and k must be (B, HK{t}, dk) and v (B, H{t}, dv), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    _dtype(name, "q", q)
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise TypeError(f"{name}: q, k and v must have one dtype, got {q.dtype}, {k.dtype} and {v.dtype}")
    gates = vs[:-1]
    for what, t in (("g", g), ("beta", beta)):
        if t is not None and (t.shape != gates or t.dtype not in _DT):
            raise ValueError(f"{name}: {what} must be {tuple(gates)} float32 or bfloat16, got {tuple(t.shape)} {t.dtype}")
    if state is not None:
        _like(name, "state" if dims == 3 else "initial_state", state, (vs[0], vs[1], qs[-1], vs[-1]), torch.float32)


def _delta_args(q, k, v, g, beta, state, scale):
    (B, HK, L, dk), (H, dv) = q.shape, v.shape[1::2]
    return DeltaArgs(B, H, HK, L, dk, dv, _DT[q.dtype], scale, *_strides3(q), *_strides3(k), *_strides3(v), *_strides3(g),
                     *_strides3(beta), _ptr(state))


def _delta_fwd(q, k, v, g, beta, state, scale, want_final, keep):
    q, k, v, g, beta, state = _channels(q), _channels(k), _channels(v), _f32(g), _f32(beta), _vec(state)
    o, (ob, oh, ol, _) = _result(v)
    final = None
    if want_final:
        final = torch.empty((*v.shape[:2], q.shape[-1], v.shape[-1]), device=v.device, dtype=torch.float32)
    a = _delta_args(q, k, v, g, beta, state, scale)
    a.final_state, a.keep = _ptr(final), keep
    a.o, a.o_stride_b, a.o_stride_h, a.o_stride_l = o.data_ptr(), ob, oh, ol
    ws = _optional_workspace("mh_delta_rule_workspace_bytes", a, v.device)
    _lib.call("mh_delta_rule_fwd", ct.byref(a), _stream(v.device))
    return o, final, ws if keep else None


def gated_delta_rule_bwd(do, q, k, v, g=None, beta=None, *, scale=None, initial_state=None, d_final_state=None):
    """Gradients of ``gated_delta_rule``: (dq, dk, dv, dg, dbeta, d_initial_state).

    do (B, H, L, dv) like v; d_final_state (B, H, dk, dv) float32 or None.  dq, dk, dv are like q, k, v, the value heads
    that share a key head summed in their order; dg and dbeta (B, H, L) and d_initial_state (B, H, dk, dv) float32, each
    None where its input is.
    """
    name = "gated_delta_rule_bwd"
    _require_cuda(name, do, q, k, v, g, beta, initial_state, d_final_state)
    _delta_shapes(name, q, k, v, g, beta, initial_state, 4)
    _like(name, "do", do, v.shape, v.dtype)
    if d_final_state is not None:
        _like(name, "d_final_state", d_final_state, (*v.shape[:2], q.shape[-1], v.shape[-1]), torch.float32)
    return _delta_bwd(do, q, k, v, g, beta, initial_state, d_final_state, q.shape[-1] ** -0.5 if scale is None else float(scale))


def _delta_bwd(do, q, k, v, g, beta, initial_state, d_final_state, scale, kept=None):
    q, k, v, do = _channels(q), _channels(k), _channels(v), _channels(do)
    g, beta, initial_state, d_final_state = _f32(g), _f32(beta), _vec(initial_state), _vec(d_final_state)
    dq, dk, dv = _result(q)[0], _result(k)[0], _result(v)[0]
    dg, dbeta = (None if t is None else torch.empty(v.shape[:-1], device=v.device, dtype=torch.float32) for t in (g, beta))
    d_state = None if initial_state is None else torch.empty_like(initial_state)
    a = DeltaBwdArgs(_delta_args(q, k, v, g, beta, initial_state, scale), *_strides3(do), _ptr(d_final_state), *_strides3(dq),
                     *_strides3(dk), *_strides3(dv), _ptr(dg), _ptr(dbeta), _ptr(d_state))
    if kept is not None:
        a.kept, a.kept_bytes = kept.data_ptr(), kept.numel()
    ws = _optional_workspace("mh_delta_rule_bwd_workspace_bytes", a, v.device)
    _lib.call("mh_delta_rule_bwd", ct.byref(a), _stream(v.device))
    return dq, dk, dv, dg, dbeta, d_state


class _GatedDeltaFn(torch.autograd.Function):
    """Autograd node of the gated delta rule: forward = ``mh_delta_rule_fwd``, backward = ``mh_delta_rule_bwd``."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, scale, want_final, recompute):
        o, final, kept = _delta_fwd(q, k, v, g, beta, state, scale, want_final, not recompute)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, g, beta, state, kept)
        ctx.scale = scale
        return o, final

    @staticmethod
    @once_differentiable
    def backward(ctx, do, d_final):
        q, k, v, g, beta, state, kept = ctx.saved_tensors
        if do is None and d_final is None:
            return (None,) * 9
        if do is None:
            do = torch.zeros_like(v)
        grads = _delta_bwd(do, q, k, v, g, beta, state, d_final, ctx.scale, kept)
        grads = [d if need else None for d, need in zip(grads, ctx.needs_input_grad)]
        for i, t in ((3, g), (4, beta)):
            if grads[i] is not None and t.dtype is not torch.float32:
                grads[i] = grads[i].to(t.dtype)
        return *grads, None, None, None


def gated_delta_step(state, q, k, v, g=None, beta=None, *, scale=None, state_out=None):
    """One token of the gated delta rule for every sequence: o (B, H, dv) like v.

    state (B, H, dk, dv) float32 contiguous, updated in place, or into ``state_out`` (like state) where that is given; q, k
    (B, HK, dk), v (B, H, dv), g and beta (B, H) as ``gated_delta_rule`` takes them for a sequence.  For decoding: it records
    no gradient.
    """
    name = "gated_delta_step"
    _require_cuda(name, state, q, k, v, g, beta, state_out)
    _delta_shapes(name, q, k, v, g, beta, state, 3)
    if not state.is_contiguous():
        raise ValueError(f"{name}: state must be contiguous")
    if state_out is None:
        state_out = state
    else:
        _like(name, "state_out", state_out, state.shape, torch.float32)
        if not state_out.is_contiguous():
            raise ValueError(f"{name}: state_out must be contiguous")
    if _through_autograd(state, q, k, v, g, beta, state_out):
        raise RuntimeError(f"{name}: has no backward; call it under torch.no_grad(), or gated_delta_rule with L = 1")
    q, k, v, g, beta = _channels(q), _channels(k), _channels(v), _f32(g), _f32(beta)
    o, (ob, oh, _) = _result(v)
    (B, HK, dk), (_, H, dv) = q.shape, v.shape
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    a = DeltaStepArgs(B, H, HK, dk, dv, _DT[q.dtype], dk ** -0.5 if scale is None else scale, q.data_ptr(), qb, qh,
                      k.data_ptr(), kb, kh, v.data_ptr(), vb, vh, *_strides2(g), *_strides2(beta), state.data_ptr(),
                      state_out.data_ptr(), o.data_ptr(), ob, oh)
    _lib.call("mh_delta_step", ct.byref(a), _stream(v.device))
    torch.autograd.graph.increment_version(state_out)    # the kernel writes where torch does not see it
    return o


# ------------------------------------------------------------------------------------------------ group norm

_ACTIVATIONS = (None, "silu")


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, *, activation=None, return_stats=False):
    """Group norm of a channels-last tensor, with its affine part and an activation: y like x.

    x (N, ..., C), C up to 65536 and a multiple of ``num_groups``; mean and variance of each (batch entry, group of
    neighbouring channels) over the group's channels and all positions between.  A norm of each head of each token, as a
    linear-attention scan is followed by, is that of (tokens, C) with a group a head.  weight, bias (C,) fp32 or bf16 of
    one dtype, each optional; activation: None or "silu".  Sums are fp64 over positions, fp32 (of centred values) within one;
    values are centred by the mean before its rounding, in the gradients by the fp32 mean.  A group whose squares leave fp32's
    range (values beyond about 1e19) is NaN throughout.

    ``return_stats``: (y, stats), the groups' fp32 (mean, 1 / sqrt(var + eps)), shaped (N, num_groups, 2).
    Differentiable in x, weight and bias.
    """
    name = "group_norm"
    _require_cuda(name, x, weight, bias)
    _group_shapes(name, x, num_groups, weight, bias, activation)
    if _through_autograd(x, weight, bias):
        y, stats = _GroupNormFn.apply(x, weight, bias, num_groups, eps, activation)
    else:
        y, stats = _group_norm_fwd(x, weight, bias, num_groups, eps, activation, return_stats)
    return (y, stats) if return_stats else y


def _group_shapes(name, x, num_groups, weight, bias, activation):
    _dtype(name, "x", x)
    if x.dim() < 2 or x.shape[-1] < 1 or num_groups < 1 or x.shape[-1] % num_groups:
        raise ValueError(f"{name}: x must be (N, ..., C) with C a multiple of num_groups, got {tuple(x.shape)} and {num_groups}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{name}: unknown activation {activation!r} (None, 'silu')")
    _norm_params(name, weight, bias, x.shape[-1])


def _space(t):
    """t (N, ..., C) as (N, positions, C) with contiguous channels (a copy where no view of it is)."""
    if t.dim() != 3:
        n = 1
        for d in t.shape[1:-1]:
            n *= d
        t = t.reshape(t.shape[0], n, t.shape[-1])
    return _channels(t)


def _group_args(x3, weight, bias, num_groups, eps, activation, stats, dtype):
    par = weight if weight is not None else bias
    pd = x3.dtype if dtype is None else dtype
    return GroupNormArgs(*x3.shape, num_groups, _DT[x3.dtype], _DT[pd] if par is None else _DT[par.dtype],
                         activation is not None, 0, eps, *_strides2(x3), _ptr(weight), _ptr(bias), None, 0, 0, _ptr(stats))


def _group_norm_fwd(x, weight, bias, num_groups, eps, activation, want_stats):
    x3, weight, bias = _space(x), _vec(weight), _vec(bias)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    y3 = _space(y)
    stats = torch.empty((x3.shape[0], num_groups, 2), device=x.device, dtype=torch.float32) if want_stats else None
    if want_stats and not x3.shape[1]:
        stats.fill_(math.nan)                    # the mean of no values; no kernel runs
    a = _group_args(x3, weight, bias, num_groups, eps, activation, stats, None)
    a.y, a.y_stride_b, a.y_stride_s = _strides2(y3)
    ws = _optional_workspace("mh_group_norm_workspace_bytes", a, x.device)
    _lib.call("mh_group_norm_fwd", ct.byref(a), _stream(x.device))
    return y, stats


def group_norm_bwd(dy, x, stats, num_groups, weight=None, bias=None, *, activation=None, need_bias=True, dtype=None):
    """Gradients of ``group_norm``: (dx, dweight, dbias).

    dy like x; stats as ``group_norm`` returns them; weight and bias as it took them (the activation's slope needs both).
    dx like x; dweight (None without ``weight``) and dbias (None unless ``need_bias``) have the parameters' dtype (without
    them ``dtype``, None: that of dy), fp32 sums in a fixed order, rounded once.
    """
    name = "group_norm_bwd"
    _require_cuda(name, dy, x, stats, weight, bias)
    _group_shapes(name, x, num_groups, weight, bias, activation)
    _like(name, "dy", dy, x.shape, x.dtype)
    _like(name, "stats", stats, (x.shape[0], num_groups, 2), torch.float32)
    if dtype is not None and dtype not in _DT:
        raise TypeError(f"{name}: dtype {dtype} not supported (float32, bfloat16)")
    x3, dy3, weight, bias, stats = _space(x), _space(dy), _vec(weight), _vec(bias), _vec(stats)
    C, dev = x.shape[-1], x.device
    par = weight if weight is not None else bias
    par_dtype = par.dtype if par is not None else dy.dtype if dtype is None else dtype
    dx = torch.empty(x.shape, device=dev, dtype=x.dtype)
    dw = torch.empty((C,), device=dev, dtype=par_dtype) if weight is not None else None
    db = torch.empty((C,), device=dev, dtype=par_dtype) if need_bias else None
    a = GroupNormBwdArgs(_group_args(x3, weight, bias, num_groups, 0.0, activation, stats, par_dtype), *_strides2(dy3),
                         *_strides2(_space(dx)), _ptr(dw), _ptr(db))
    ws = _optional_workspace("mh_group_norm_bwd_workspace_bytes", a, dev)
    _lib.call("mh_group_norm_bwd", ct.byref(a), _stream(dev))
    return dx, dw, db


class _GroupNormFn(torch.autograd.Function):
    """Autograd node of ``group_norm``: forward = ``mh_group_norm_fwd``, backward = ``mh_group_norm_bwd``."""

    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, activation):
        y, stats = _group_norm_fwd(x, weight, bias, num_groups, eps, activation, True)
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.cfg = num_groups, activation
        return y, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _):
        if dy is None:
            return (None,) * 6
        x, weight, bias, stats = ctx.saved_tensors
        num_groups, activation = ctx.cfg
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dx, dw, db = group_norm_bwd(dy, x, stats, num_groups, weight, bias, activation=activation, need_bias=need_b)
        return dx if need_x else None, dw if need_w else None, db, None, None, None
