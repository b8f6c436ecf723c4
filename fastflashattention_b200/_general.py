"""Attention whose keys are not the queries' own: cross attention, and attention with a
learned relative position bias.

Both run the kernels of general attention (``csrc/ffa_gen_*.cuh``) through the torch
operators ``torch.ops.ffa_b200.general*`` (``csrc/ffa_torch_gen.cpp``).  The checks follow
the package's strict policy: an input outside the contract raises ``UnsupportedConfig``
with the violated constraint, and nothing falls back.
"""
from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib

_MAX_LEN = 1 << 29
_MAX_DISTANCE = 1024
_MAX_BUCKETS = 256


def _rows_problem(name, t, batch, device):
    """Why ``t`` is not a per-sequence int32 vector, or ``None``."""
    if not isinstance(t, torch.Tensor):
        return f"{name} is not a torch.Tensor"
    if t.device != device:
        return f"{name} is on device '{t.device}'; it must be on '{device}' with the query"
    if t.dtype is not torch.int32:
        return f"{name} dtype is {t.dtype}; only int32 is supported"
    if tuple(t.shape) != (batch,) or not t.is_contiguous():
        return f"{name} must be a contiguous tensor of shape ({batch},), one entry for each sequence"
    return None


def _tangent_problem(*tensors):
    """Why forward-mode derivatives rule out the tensors, or ``None``: the kernels know none, and
    a tangent that is dropped would be a derivative of zero."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        return "forward-mode derivatives (dual tensors, torch.func.jvp) are not supported"
    return None


def _inside(query, key, value, enable_gqa):
    """Whether the three tensors meet the contract: the checks of ``_shape_reason`` without its
    messages, for calls whose kernels take less time than the checks' bookkeeping."""
    t, bf16 = torch.Tensor, torch.bfloat16
    if not (isinstance(query, t) and isinstance(key, t) and isinstance(value, t)):
        return False
    qs, ks = query.shape, key.shape
    if len(qs) != 4 or len(ks) != 4 or value.shape != ks:
        return False
    batch, heads, rows, dim = qs
    kv_heads, keys = ks[1], ks[2]
    return (batch == ks[0] and dim == ks[3] and dim % 8 == 0 and 8 <= dim <= 128
            and (heads == kv_heads or (enable_gqa and kv_heads > 0 and heads % kv_heads == 0))
            and rows < _MAX_LEN and keys < _MAX_LEN
            and query.dtype is bf16 and key.dtype is bf16 and value.dtype is bf16
            and query.is_cuda and key.is_cuda and value.is_cuda
            and query.get_device() == key.get_device() == value.get_device())


def _shape_reason(query, key, value, key_lengths, scale, enable_gqa):
    """Why the tensors are outside the contract of general attention, or ``None``."""
    if not _inside(query, key, value, enable_gqa):
        from . import _tensor_problem
        for name, t in (("query", query), ("key", key), ("value", value)):
            problem = _tensor_problem(name, t)
            if problem is not None:
                return problem
            if t.device != query.device:
                return f"{name} is on device '{t.device}'; it must be on '{query.device}' with the query"
        qs, ks, vs = (tuple(t.shape) for t in (query, key, value))
        if ks != vs:
            return f"shapes of key {ks} and value {vs} differ"
        if qs[0] != ks[0] or qs[3] != ks[3]:
            return f"query {qs} and key {ks} must have the same batch and head_dim"
        if qs[3] % 8 != 0 or not 8 <= qs[3] <= 128:
            return f"head_dim={qs[3]}; must be a multiple of 8, at most 128"
        if qs[1] != ks[1]:
            if not enable_gqa:
                return f"query has {qs[1]} heads and key {ks[1]}; pass enable_gqa=True to share key heads"
            if ks[1] == 0 or qs[1] % ks[1] != 0:
                return f"query heads ({qs[1]}) must be a multiple of key heads ({ks[1]})"
        if max(qs[2], ks[2]) >= _MAX_LEN:
            return f"lengths {qs[2]} and {ks[2]}; must be below 2^29"
    if scale is not None and not math.isfinite(scale):
        return f"scale={scale}; must be finite"
    if key_lengths is not None:
        problem = _rows_problem("key_lengths", key_lengths, query.shape[0], query.device)
        if problem is not None:
            return problem
    return _tangent_problem(query, key, value)


def _bias_reason(query, bias, max_distance, bidirectional, is_causal, query_offset):
    """Why the position bias or the offset is outside the contract, or ``None``."""
    if not isinstance(bias, torch.Tensor):
        return "bias is not a torch.Tensor"
    if bias.device != query.device:
        return f"bias is on device '{bias.device}'; it must be on '{query.device}' with the query"
    if bias.dtype is not torch.bfloat16:
        return f"bias dtype is {bias.dtype}; only bfloat16 is supported"
    if bias.dim() != 2 or bias.shape[1] != query.shape[1]:
        return f"bias has shape {tuple(bias.shape)}; expected [buckets, {query.shape[1]}], a column for each query head"
    both = (not is_causal) if bidirectional is None else bool(bidirectional)
    buckets = bias.shape[0]
    if not (4 if both else 2) <= buckets <= _MAX_BUCKETS or (both and buckets % 2):
        return (f"bias has {buckets} buckets; must be between {4 if both else 2} and {_MAX_BUCKETS}"
                + (", and even for both directions" if both else ""))
    first = (buckets // 2 if both else buckets) // 2
    if isinstance(max_distance, bool) or not isinstance(max_distance, int) or not first < max_distance <= _MAX_DISTANCE:
        return (f"max_distance={max_distance}; must be an integer above the {first} distances that have a bucket of "
                f"their own, at most {_MAX_DISTANCE}")
    if isinstance(query_offset, torch.Tensor):
        problem = _rows_problem("query_offset", query_offset, query.shape[0], query.device)
        if problem is not None:
            return problem
    elif isinstance(query_offset, bool) or not isinstance(query_offset, int):
        return "query_offset is neither an integer nor a torch.Tensor"
    elif abs(query_offset) > _MAX_LEN:
        return f"query_offset={query_offset}; must be within +-2^29"
    return _tangent_problem(bias)


@functools.lru_cache(maxsize=64)
def bucket_borders(side: int, max_distance: int) -> tuple:
    """Smallest distance of each of the ``side`` buckets of one direction.

    The first half, ``m = side // 2`` buckets, hold the distances 0 .. m-1.  A distance
    r >= m falls into bucket ``m + floor((side - m) * log(r / m) / log(max_distance / m))``,
    at most ``side - 1``: bucket m + j starts at the least r with
    ``(r / m) ** (side - m) >= (max_distance / m) ** j``.  That is decided in integers, so a
    distance on a border is on its upper side whatever the logarithms' last bits say.
    """
    m = side // 2
    out = list(range(m))
    r = m
    for j in range(side - m):
        while r ** (side - m) * m ** j < max_distance ** j * m ** (side - m):
            r += 1
        out.append(r)
    return tuple(out)


_operators = None


def _op(wants_grad):
    """The operator of ``torch.ops.ffa_b200`` for a call with or without gradients (the
    overload itself: finding it by name costs a microsecond a call)."""
    global _operators
    if _operators is None:
        ops = _lib.ops()
        _operators = (ops.general.default, ops.general_attention.default)
    return _operators[wants_grad]


def _refuse(reason):
    from . import UnsupportedConfig
    raise UnsupportedConfig(reason)


def cross_attention(query, key, value, key_lengths=None, scale=None, enable_gqa=False):
    """Exact bf16 attention over keys of another length.

    ``query`` is ``[B, Hq, Sq, D]``, ``key`` and ``value`` are ``[B, Hkv, Sk, D]``, bfloat16
    CUDA tensors with D a multiple of 8 up to 128; returns ``[B, Hq, Sq, D]`` bfloat16.  Any
    strides do; a layout whose strides are multiples of 8 elements, with D contiguous, is
    read in place.

    ``key_lengths`` (int32 ``[B]`` on the device, clamped to [0, Sk]): sequence b has only its
    first ``key_lengths[b]`` keys.  What lies behind them is never used, whatever it holds,
    and gets zero gradients.  A query without any key returns zeros and passes no gradient.
    ``enable_gqa``: Hq may be a multiple of Hkv; query head h reads key head h // (Hq / Hkv).
    ``scale`` defaults to ``1/sqrt(D)``.

    The backward is deterministic; second and forward-mode derivatives are refused.  A few
    queries (Hq / Hkv * Sq up to 64, a decoding step) take one pass over the keys that is
    split over the SMs.
    """
    reason = _shape_reason(query, key, value, key_lengths, scale, enable_gqa)
    if reason is not None:
        _refuse(reason)
    grad = torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad)
    return _op(grad)(query, key, value, None, key_lengths, None, 0, (), False, False, scale)


def relative_attention(query, key, value, bias, max_distance=128, bidirectional=None, is_causal=False,
                       query_offset=0, key_lengths=None, scale=None, enable_gqa=False):
    """Exact bf16 attention with a bias learned by relative position.

    ``softmax(scale * q_i . k_j + bias[bucket(j - p_i), h])`` with ``p_i = i + query_offset``.
    ``query``, ``key``, ``value``, ``key_lengths``, ``scale`` and ``enable_gqa`` are those of
    :func:`cross_attention`.

    ``bias`` is the learned table, bfloat16 ``[buckets, Hq]``; its gradient is computed with
    the others.  Half of the buckets hold one distance each, the others grow with the
    logarithm of the distance up to ``max_distance`` (at most 1024), from where the last one
    holds all (:func:`bucket_borders`).  ``bidirectional`` (default: ``not is_causal``) gives
    keys behind the query's position a half of the buckets of their own; otherwise they count
    as distance 0.  Finite entries and +inf act as if clamped to [-2^14, 2^14]; -inf masks its
    bucket.

    A call whose ``bias`` wants a gradient (``bias.requires_grad`` with gradients enabled) computes
    its output with probabilities in 16 bits instead of 8, which the gradient's cancelling sums
    need: its values differ in the last bits from those of other calls, its forward is a fifth to a
    third slower, and a few queries do not take the single pass of a decoding step.  Decode
    under ``torch.no_grad()``.

    ``is_causal``: key j is visible to query i iff ``j <= p_i``.  ``query_offset`` is an
    integer or an int32 ``[B]`` device tensor: the position of the first query among the keys,
    0 for a sequence that attends to itself, ``length - Sq`` for the newest Sq tokens over a
    cache of ``length`` keys.  A tensor may change between the replays of a captured graph.
    """
    reason = _shape_reason(query, key, value, key_lengths, scale, enable_gqa)
    if reason is None:
        reason = _bias_reason(query, bias, max_distance, bidirectional, is_causal, query_offset)
    if reason is not None:
        _refuse(reason)
    both = (not is_causal) if bidirectional is None else bool(bidirectional)
    borders = bucket_borders(bias.shape[0] // 2 if both else bias.shape[0], max_distance)
    offsets, offset = (query_offset, 0) if isinstance(query_offset, torch.Tensor) else (None, query_offset)
    grad = torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad
                                        or bias.requires_grad)
    return _op(grad)(query, key, value, bias, key_lengths, offsets, offset, borders, both, bool(is_causal), scale)
