"""Operators at the two ends of a language model and between its layers, beside the scans of ``ops``.

=====================================  ====================================================================
``embedding``, ``embedding_bwd``        scaled token lookup, and the table's gradient
``layer_norm``, ``layer_norm_bwd``      layer norm of the residual stream (the sum with a layer's output fused),
                                        and its backward with the weight's and bias's gradients
``pack_activations``,                   activations in 8 bits with an exponent for each 64 channels, for what a
``unpack_activations``                  backward pass reads; ``layer_norm`` can keep its input so
``token_logprobs``,                     log probabilities of given tokens with entropies and the likeliest
``token_logprobs_bwd``                  alternatives, and the logits' gradient
=====================================  ====================================================================

``embedding``, ``layer_norm`` and ``token_logprobs`` are differentiable (a tensor with a forward-mode tangent is refused);
the ``_bwd`` functions give their gradients explicitly, and results of those and of packing carry none.  bf16 and fp32
tensors of any width and row stride (a last dimension that is not contiguous is copied).  As in ``ops``, every call
launches kernels of ``libmamformer_hip.so`` on the current torch stream, does not synchronise, and has no CPU path.  All
results are the same bits at every call with the same inputs.
"""

from __future__ import annotations

import ctypes as ct
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import (EmbeddingArgs, EmbeddingBwdArgs, LayerNormArgs, LayerNormBwdArgs, LogprobArgs, LogprobBwdArgs,
                   PackArgs)
from .ops import _DT, _ptr, _require_cuda, _stream, _workspace

__all__ = ["embedding", "embedding_bwd", "layer_norm", "layer_norm_bwd", "PackedActivations", "pack_activations",
           "unpack_activations", "TokenLogprobs", "token_logprobs", "token_logprobs_bwd"]

_INDEX_BYTES = {torch.int32: 4, torch.int64: 8}
_GROUP = 64                                      # channels that share an exponent in the 8-bit form


def _dtype(name, what, t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"{name}: {what} dtype {t.dtype} not supported (float32, bfloat16)") from None


def _indices(name, what, t):
    if t.dtype not in _INDEX_BYTES:
        raise TypeError(f"{name}: {what} must be int32 or int64, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(t, D):
    """t as (rows, D) with contiguous rows (a copy where no view of it is)."""
    t = t if t.dim() == 2 else t.reshape(-1, D)
    return t if t.stride(1) == 1 or D == 1 else t.contiguous()


def _empty(t):
    """A contiguous tensor of the shape and dtype of t (for a contiguous t by the shorter way)."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _optional_workspace(query, a, dev):
    """The workspace that ``query`` asks for, entered in the arguments; None where it asks for none."""
    n = ct.c_size_t()
    _lib.call(query, ct.byref(a), ct.byref(n))
    if not n.value:
        return None
    ws = torch.empty((n.value,), device=dev, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
    return ws


def _through_autograd(a, b=None, c=None, d=None):
    """Whether a call goes through its autograd function: one of its tensors requires a gradient, or a forward-mode level is
    open.  A tensor with a tangent does not require a gradient; the functions have no forward-mode rule, so that autograd
    raises for it rather than take a lost tangent as zero."""
    return _forward_ad._current_level >= 0 or (
        a.requires_grad or b is not None and b.requires_grad or c is not None and c.requires_grad
        or d is not None and d.requires_grad) and torch.is_grad_enabled()


def _like(name, what, t, shape, dtype):
    if t.shape != shape or t.dtype is not dtype:
        raise ValueError(f"{name}: {what} must be {tuple(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")


# ------------------------------------------------------------------------------------------------ token table

def embedding(ids, weight, *, scale=1.0, padding_idx=None):
    """Rows of a token table: ``scale * weight[ids]``, shaped (*ids.shape, D), in the dtype of the table.

    ids int32 or int64 of any shape; weight (V, D).  An id outside [0, V) gives zeros and no gradient (nothing can be
    raised from the GPU without waiting for it).  ``padding_idx``: its row takes no gradient; it is looked up as any
    other.  Differentiable in ``weight`` (``embedding_bwd``).
    """
    _require_cuda("embedding", ids, weight)
    if weight.dim() != 2:
        raise ValueError(f"embedding: weight must be (V, D), got {tuple(weight.shape)}")
    if padding_idx is not None:
        padding_idx = _padding(padding_idx, weight.shape[0])
    if _through_autograd(weight):
        return _EmbeddingFn.apply(weight, ids, scale, padding_idx)
    return _embedding_fwd(weight, ids, scale)


def _padding(padding_idx, V):
    if padding_idx is None:
        return -1                                # no row has it
    if not -V <= padding_idx < V:
        raise ValueError(f"embedding: padding_idx {padding_idx} outside a table of {V} rows")
    return padding_idx % V


def _embedding_fwd(weight, ids, scale):
    dt = _dtype("embedding", "weight", weight)
    ids = _indices("embedding", "ids", ids)
    V, D = weight.shape
    w = _rows(weight, D)
    out = w.new_empty((*ids.shape, D))
    n = ids.numel()
    if n and D:
        a = EmbeddingArgs(n, V, D, dt, ids.element_size(), scale, ids.data_ptr(), w.data_ptr(), w.stride(0),
                          out.data_ptr(), D)
        _lib.call("mh_embedding_fwd", ct.byref(a), _stream(w.device))
    return out


def embedding_bwd(dy, ids, num_embeddings, *, scale=1.0, padding_idx=None, dtype=None):
    """Gradient of ``embedding`` with respect to its table, (num_embeddings, D) in ``dtype`` (float32 or bfloat16; None:
    that of dy).

    dy (*ids.shape, D).  Each row is the fp32 sum over its tokens in their order (of many tokens: of equal shares of them,
    joined in order), times ``scale``, rounded once; rows without tokens are zero.
    """
    name = "embedding_bwd"
    _require_cuda(name, dy, ids)
    dt = _dtype(name, "dy", dy)
    ids = _indices(name, "ids", ids)
    V = int(num_embeddings)
    if V < 1:
        raise ValueError(f"{name}: num_embeddings must be positive, got {V}")
    if dy.dim() < 1 or dy.shape[:-1] != ids.shape or dy.shape[-1] < 1:
        raise ValueError(f"{name}: dy must be (*ids.shape, D), got {tuple(dy.shape)} for ids {tuple(ids.shape)}")
    out_dtype = dy.dtype if dtype is None else dtype
    if out_dtype not in _DT:
        raise TypeError(f"{name}: dtype {out_dtype} not supported (float32, bfloat16)")
    D = dy.shape[-1]
    dy = _rows(dy, D)
    dw = torch.empty((V, D), device=dy.device, dtype=out_dtype)
    a = EmbeddingBwdArgs(ids.numel(), V, D, _padding(padding_idx, V), dt, ids.element_size(), _DT[out_dtype], scale,
                         ids.data_ptr(), dy.data_ptr(), dy.stride(0), dw.data_ptr())
    ws, a.workspace_bytes = _workspace("mh_embedding_bwd_workspace_bytes", a, dy.device)
    a.workspace = ws.data_ptr()
    _lib.call("mh_embedding_bwd", ct.byref(a), _stream(dy.device))
    return dw


class _EmbeddingFn(torch.autograd.Function):
    """Autograd node of the lookup: forward = ``mh_embedding_fwd``, backward = ``mh_embedding_bwd``."""

    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.cfg = weight.shape[0], weight.dtype, scale, padding_idx
        return _embedding_fwd(weight, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        V, dtype, scale, pad = ctx.cfg
        dw = embedding_bwd(dy, ctx.saved_tensors[0], V, scale=scale, padding_idx=pad, dtype=dtype)
        return dw, None, None, None


# ------------------------------------------------------------------------------------------------ 8-bit activations

class PackedActivations(NamedTuple):
    """Activations (*shape, dim) in 8 bits: int8 ``codes`` (*shape, dp) and a uint8 exponent byte for each 64 channels,
    ``exponents`` (*shape, dp / 64), where dp is ``dim`` up to a multiple of 64; ``dtype`` is what they were packed from.
    Channel c stands for codes[c] * 2 ** (exponents[c // 64] - 132), and for NaN where the byte is 255."""
    codes: torch.Tensor
    exponents: torch.Tensor
    dim: int
    dtype: torch.dtype


def _packed_buffers(shape, D, dev):
    dp = (D + _GROUP - 1) // _GROUP * _GROUP
    return (torch.empty((*shape, dp), device=dev, dtype=torch.int8),
            torch.empty((*shape, dp // _GROUP), device=dev, dtype=torch.uint8))


def _packed_rows(name, p):
    """Rows of a PackedActivations whose tensors are what the kernels read."""
    dp = (p.dim + _GROUP - 1) // _GROUP * _GROUP
    lead = p.codes.shape[:-1]
    if p.dim < 1 or p.codes.dtype is not torch.int8 or p.exponents.dtype is not torch.uint8 \
            or p.codes.shape[-1] != dp or p.exponents.shape != (*lead, dp // _GROUP):
        raise ValueError(f"{name}: codes {tuple(p.codes.shape)} {p.codes.dtype} and exponents "
                         f"{tuple(p.exponents.shape)} {p.exponents.dtype} do not hold {p.dim} channels")
    if not p.codes.is_contiguous() or not p.exponents.is_contiguous():
        raise ValueError(f"{name}: codes and exponents must be contiguous")
    return p.exponents.numel() // (dp // _GROUP)


def pack_activations(x):
    """x (..., D) as ``PackedActivations``: about half a bf16 tensor's memory.

    Each 64 channels of a row share the exponent e of the least power of two with max|x| <= 127 * 2**e; a code is
    x * 2**-e rounded to nearest even, so |error| <= 2**(e - 1), less than 1/127 of the group's largest value where that is
    a normal number (e is at least -132: smaller groups keep an absolute error of 2**-133).  A group that holds an infinity
    or a NaN reads back as NaN.  Not differentiable: it is for what a backward pass keeps.
    """
    _require_cuda("pack_activations", x)
    dt = _dtype("pack_activations", "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"pack_activations: x must be (..., D), got {tuple(x.shape)}")
    D = x.shape[-1]
    codes, exps = _packed_buffers(x.shape[:-1], D, x.device)
    x2 = _rows(x.detach(), D)
    a = PackArgs(x2.shape[0], D, dt, 0, x2.data_ptr(), x2.stride(0), codes.data_ptr(), exps.data_ptr())
    _lib.call("mh_pack_activations", ct.byref(a), _stream(x.device))
    return PackedActivations(codes, exps, D, x.dtype)


def unpack_activations(packed, dtype=None):
    """The values of a ``PackedActivations``, in ``dtype`` (None: what they were packed from); every value is exact."""
    name = "unpack_activations"
    _require_cuda(name, packed.codes, packed.exponents)
    rows = _packed_rows(name, packed)
    out = torch.empty((*packed.codes.shape[:-1], packed.dim), device=packed.codes.device,
                      dtype=packed.dtype if dtype is None else dtype)
    a = PackArgs(rows, packed.dim, _dtype(name, "output", out), 0, out.data_ptr(), packed.dim, packed.codes.data_ptr(),
                 packed.exponents.data_ptr())
    _lib.call("mh_unpack_activations", ct.byref(a), _stream(out.device))
    return out


# ------------------------------------------------------------------------------------------------ layer norm

def layer_norm(x, weight=None, bias=None, eps=1e-5, *, residual=None, packed=False, return_stats=False):
    """Layer norm over the last dimension, with the residual stream's sum and its 8-bit form fused.

    x (..., D), D <= 16384; weight, bias (D,) fp32 or bf16 of one dtype, each optional.  With ``residual`` (like x) what
    is normalised is h = x + residual, rounded to the dtype of x, and h is returned too: the stream that goes on.  Mean
    and variance are fp32, the variance that of the centred values; a row whose sum or squares leave fp32's range (values
    beyond about 1e19) is NaN throughout.

    Returns y (like x), or a tuple of y, then h (with ``residual``), then h as ``PackedActivations`` (``packed``), then
    the rows' fp32 (mean, 1 / sqrt(var + eps)), shaped (..., 2) (``return_stats``).

    Differentiable in x, residual, weight and bias.  With ``packed`` the backward reads h from its 8-bit form, so that
    neither x nor h is kept for it: the statistics are those of h itself, only the normalised values that enter dx and
    dweight carry the 8-bit rounding.
    """
    name = "layer_norm"
    _require_cuda(name, x, weight, bias, residual)
    _dtype(name, "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x must be (..., D), got {tuple(x.shape)}")
    D = x.shape[-1]
    if residual is not None:
        _like(name, "residual", residual, x.shape, x.dtype)
    _norm_params(name, weight, bias, D)
    if _through_autograd(x, weight, bias, residual):
        y, h, codes, exps, stats = _LayerNormFn.apply(x, residual, weight, bias, eps, packed)
    else:
        y, h, codes, exps, stats = _layer_norm_fwd(x, residual, weight, bias, eps, packed, return_stats)
    out = [y]
    if residual is not None:
        out.append(h)
    if packed:
        out.append(PackedActivations(codes, exps, D, x.dtype))
    if return_stats:
        out.append(stats)
    return y if len(out) == 1 else tuple(out)


def _norm_params(name, weight, bias, D):
    if weight is not None and (weight.shape != (D,) or weight.dtype not in _DT):
        raise ValueError(f"{name}: weight must be ({D},) float32 or bfloat16, got {tuple(weight.shape)} {weight.dtype}")
    if bias is not None and (bias.shape != (D,) or bias.dtype not in _DT):
        raise ValueError(f"{name}: bias must be ({D},) float32 or bfloat16, got {tuple(bias.shape)} {bias.dtype}")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise TypeError(f"{name}: weight and bias must have one dtype, got {weight.dtype} and {bias.dtype}")


def _vec(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _layer_norm_fwd(x, residual, weight, bias, eps, packed, stats):
    D, dev = x.shape[-1], x.device
    x2 = _rows(x, D)
    weight, bias = _vec(weight), _vec(bias)
    y = _empty(x)
    h = codes = exps = st = res = None
    if residual is not None:
        res = _rows(residual, D)
        h = _empty(x)
    if packed:
        codes, exps = _packed_buffers(x.shape[:-1], D, dev)
    if stats:
        st = torch.empty((*x.shape[:-1], 2), device=dev, dtype=torch.float32)
    par = weight if weight is not None else bias
    a = LayerNormArgs(x2.shape[0], D, _DT[x.dtype], 0 if par is None else _DT[par.dtype], eps, x2.data_ptr(),
                      x2.stride(0), _ptr(res), 0 if res is None else res.stride(0), _ptr(weight), _ptr(bias),
                      y.data_ptr(), D, _ptr(h), D, _ptr(st), _ptr(codes), _ptr(exps))
    _lib.call("mh_layer_norm_fwd", ct.byref(a), _stream(dev))
    return y, h, codes, exps, st


def layer_norm_bwd(dy, h, stats, weight=None, *, d_h=None, bias=True, dtype=None):
    """Gradients of ``layer_norm``: (dx, dweight, dbias).

    dy (..., D); h: what was normalised (x, or the sum with the residual), a tensor like dy or ``PackedActivations``;
    stats (..., 2) as ``layer_norm`` returns them; ``d_h``: the gradient that reaches the stream h by its other uses,
    added into dx.  dx (like dy) is the gradient of x and of residual alike.  dweight (None without ``weight``) and dbias
    (None unless ``bias``) have the weight's dtype (without one ``dtype``, None: that of dy); both are fp32 sums over the
    rows in a fixed order, rounded once.
    """
    name = "layer_norm_bwd"
    is_packed = isinstance(h, PackedActivations)
    src = h.codes if is_packed else h
    _require_cuda(name, dy, src, stats, weight, d_h)
    dt = _dtype(name, "dy", dy)
    if dy.dim() < 1 or dy.shape[-1] < 1:
        raise ValueError(f"{name}: dy must be (..., D), got {tuple(dy.shape)}")
    shape, D, dev = dy.shape, dy.shape[-1], dy.device
    if is_packed:
        _require_cuda(name, dy, h.exponents)
        _packed_rows(name, h)
        if h.dim != D or h.codes.shape[:-1] != shape[:-1]:
            raise ValueError(f"{name}: {tuple(h.codes.shape[:-1])} rows of {h.dim} packed channels do not match dy "
                             f"{tuple(shape)}")
    else:
        _like(name, "h", h, shape, dy.dtype)
        src = _rows(h, D)
    _like(name, "stats", stats, (*shape[:-1], 2), torch.float32)
    if d_h is not None:
        _like(name, "d_h", d_h, shape, dy.dtype)
        d_h = _rows(d_h, D)
    _norm_params(name, weight, None, D)
    dx = _empty(dy)
    weight, stats, dy = _vec(weight), _vec(stats), _rows(dy, D)
    par_dtype = weight.dtype if weight is not None else dy.dtype if dtype is None else dtype
    if par_dtype not in _DT:
        raise TypeError(f"{name}: dtype {par_dtype} not supported (float32, bfloat16)")
    dw = torch.empty((D,), device=dev, dtype=par_dtype) if weight is not None else None
    db = torch.empty((D,), device=dev, dtype=par_dtype) if bias else None
    a = LayerNormBwdArgs(dy.shape[0], D, dt, _DT[par_dtype], dy.data_ptr(), dy.stride(0),
                         None if is_packed else src.data_ptr(), 0 if is_packed else src.stride(0),
                         src.data_ptr() if is_packed else None, h.exponents.data_ptr() if is_packed else None,
                         stats.data_ptr(), _ptr(weight), _ptr(d_h), 0 if d_h is None else d_h.stride(0),
                         dx.data_ptr(), D, _ptr(dw), _ptr(db))
    ws = _optional_workspace("mh_layer_norm_bwd_workspace_bytes", a, dev)
    _lib.call("mh_layer_norm_bwd", ct.byref(a), _stream(dev))
    return dx, dw, db


class _LayerNormFn(torch.autograd.Function):
    """Autograd node of ``layer_norm``: forward = ``mh_layer_norm_fwd``, backward = ``mh_layer_norm_bwd``."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, packed):
        y, h, codes, exps, stats = _layer_norm_fwd(x, residual, weight, bias, eps, packed, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (codes, exps, stats) if t is not None))
        kept = codes if packed else x if h is None else h
        ctx.save_for_backward(kept, exps, stats, weight)
        ctx.packed = (x.shape[-1], x.dtype) if packed else None
        ctx.par_dtype = None if bias is None else bias.dtype
        return y, h, codes, exps, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, d_h, *_):
        kept, exps, stats, weight = ctx.saved_tensors
        need_x, need_res, need_w, need_b = ctx.needs_input_grad[:4]
        if dy is None:                           # only the stream was used
            return d_h if need_x else None, d_h if need_res else None, None, None, None, None
        h = PackedActivations(kept, exps, *ctx.packed) if ctx.packed else kept
        dx, dw, db = layer_norm_bwd(dy, h, stats, weight, d_h=d_h, bias=need_b, dtype=ctx.par_dtype)
        return dx if need_x else None, dx if need_res else None, dw if need_w else None, db, None, None


# ------------------------------------------------------------------------------------------------ log probabilities

class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``, each shaped like its targets (with a last dimension of their own: the
    alternatives, and the 3 values a row that ``token_logprobs_bwd`` takes as ``stats``)."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    stats: torch.Tensor


def token_logprobs(logits, targets, *, temperature=1.0, top=0, ignore_index=-100):
    """Log probabilities of given tokens, the distributions' entropies and their likeliest tokens, as ``TokenLogprobs``.

    logits (..., V); targets (...) int32 or int64.  With l = logits / temperature: logprobs = l[target] - ln sum exp l
    (0 where the target is ``ignore_index`` or outside [0, V)), entropy = -sum p ln p, and with ``top`` (up to 64)
    top_ids (..., top) int64 and top_logprobs (..., top), largest first, equal logits by the lowest id, NaN first.
    Results are fp32 sums over one reading of the row.

    Entries of -inf have no weight; a row of nothing else gives logprobs and top_logprobs of -inf and an entropy of 0.
    A NaN or +inf makes its row's results NaN.  Differentiable in ``logits`` through logprobs and entropy
    (``token_logprobs_bwd``); top_logprobs carries no gradient.
    """
    name = "token_logprobs"
    _require_cuda(name, logits, targets)
    _logprob_shapes(name, logits, targets)
    if _through_autograd(logits):
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, targets, temperature, top, ignore_index))
    return TokenLogprobs(*_token_logprobs_fwd(logits, targets, temperature, top, ignore_index))


def _logprob_shapes(name, logits, targets):
    _dtype(name, "logits", logits)
    if logits.dim() < 1 or logits.shape[-1] < 1 or targets.shape != logits.shape[:-1]:
        raise ValueError(f"{name}: logits must be (..., V) and targets (...), got {tuple(logits.shape)} and "
                         f"{tuple(targets.shape)}")


def _token_logprobs_fwd(logits, targets, temperature, top, ignore_index):
    tgt = _indices("token_logprobs", "targets", targets)
    V, dev, lead = logits.shape[-1], logits.device, tgt.shape
    l2 = _rows(logits, V)
    rows = l2.shape[0]
    # tensors of their own, not views of one: either may be changed in place without the other
    # (made from others, which is the shorter way)
    lp = torch.empty_like(tgt, dtype=torch.float32)
    ent = torch.empty_like(lp)
    stats = lp.new_empty((*lead, 3))
    ids = alt = None
    if top:
        ids = torch.empty((*lead, top), device=dev, dtype=torch.int64)
        alt = torch.empty((*lead, top), device=dev, dtype=torch.float32)
    a = LogprobArgs(rows, V, ignore_index, _DT[l2.dtype], tgt.element_size(), top, temperature, l2.data_ptr(),
                    l2.stride(0), tgt.data_ptr(), lp.data_ptr(), ent.data_ptr(), stats.data_ptr(), _ptr(ids), _ptr(alt))
    ws = _optional_workspace("mh_token_logprobs_workspace_bytes", a, dev)
    _lib.call("mh_token_logprobs_fwd", ct.byref(a), _stream(dev))
    return lp, ent, ids, alt, stats


def token_logprobs_bwd(logits, targets, stats, d_logprobs=None, d_entropy=None, *, temperature=1.0, ignore_index=-100,
                       out=None):
    """Gradient of ``token_logprobs`` with respect to the logits, (..., V) in their dtype.

    stats: the forward's; d_logprobs, d_entropy (...): the gradients of the two results, each optional.  ``out``: where
    to write it, which may be ``logits`` itself (a loss that needs its logits no more saves their size so).  To autograd
    that is an in-place change like torch's own: a backward pass that still has to read the tensor raises, and ``out`` may
    not be a leaf that requires a gradient, nor a view of one, where gradients are recorded.  A row whose gradients are
    both zero, or that has only -inf, gets zeros whatever its logits are.
    """
    name = "token_logprobs_bwd"
    _require_cuda(name, logits, targets, stats, d_logprobs, d_entropy, out)
    _logprob_shapes(name, logits, targets)
    tgt = _indices(name, "targets", targets)
    V, dev, lead = logits.shape[-1], logits.device, tgt.shape
    _like(name, "stats", stats, (*lead, 3), torch.float32)
    grads = []
    for what, t in (("d_logprobs", d_logprobs), ("d_entropy", d_entropy)):
        if t is not None:
            if t.shape != lead:
                raise ValueError(f"{name}: {what} must be {tuple(lead)}, got {tuple(t.shape)}")
            t = t.to(torch.float32).contiguous()
        grads.append(t)
    l2 = _rows(logits, V)
    given = out is not None
    if not given:
        out = _empty(logits)
        o2 = out if out.dim() == 2 else out.view(-1, V)
    else:
        _like(name, "out", out, logits.shape, logits.dtype)
        owner = out if out._base is None else out._base
        if owner.requires_grad and owner.is_leaf and torch.is_grad_enabled():
            raise RuntimeError(f"{name}: out is a leaf that requires a gradient, or a view of one")
        o2 = out if out.dim() == 2 else out.view(-1, V)      # raises where no rows can be written in place
        if o2.stride(1) != 1 and V > 1:
            raise ValueError(f"{name}: out must have contiguous rows")
    stats = _vec(stats)
    a = LogprobBwdArgs(l2.shape[0], V, ignore_index, _DT[l2.dtype], tgt.element_size(), temperature, l2.data_ptr(),
                       l2.stride(0), tgt.data_ptr(), stats.data_ptr(), _ptr(grads[0]), _ptr(grads[1]), o2.data_ptr(),
                       o2.stride(0))
    _lib.call("mh_token_logprobs_bwd", ct.byref(a), _stream(dev))
    if given:
        torch.autograd.graph.increment_version(out)      # the kernel writes where torch does not see it
    return out


class _TokenLogprobsFn(torch.autograd.Function):
    """Autograd node of the log probabilities: forward = ``mh_token_logprobs_fwd``, backward =
    ``mh_token_logprobs_bwd``."""

    @staticmethod
    def forward(ctx, logits, targets, temperature, top, ignore_index):
        lp, ent, ids, alt, stats = _token_logprobs_fwd(logits, targets, temperature, top, ignore_index)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (ids, alt, stats) if t is not None))
        ctx.save_for_backward(logits, targets, stats)
        ctx.cfg = temperature, ignore_index
        return lp, ent, ids, alt, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, d_lp, d_ent, *_):
        logits, targets, stats = ctx.saved_tensors
        if d_lp is None and d_ent is None:
            return (None,) * 5
        temperature, ignore_index = ctx.cfg
        d = token_logprobs_bwd(logits, targets, stats, d_lp, d_ent, temperature=temperature, ignore_index=ignore_index)
        return d, None, None, None, None
