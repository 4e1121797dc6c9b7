"""Sequence mixing over long records: attention to the states of another
length, with a learned position bias, and a gated linear recurrence.

GPU: fused HIP kernels from ``seist_amd._C`` (cross_attention.hip,
gated_scan.hip). CPU, and on any device while torch traces: plain fp32
PyTorch composites with identical semantics. Layouts are channels-first:
(N, H, E, L) and (N, C, L).
"""

import functools
import math
from typing import Optional, Tuple

import torch

from . import ext, use_native

# the kernels' limits
_MAX_DEPTH = 128
_MAX_BUCKETS = 64
_MAX_DISTANCE = 1024
# a bias at or under this takes its pair out of the softmax
_OUT = -1e30

_DTYPES = (torch.float32, torch.bfloat16)


def _refuse(op: str, what: str):
    raise ValueError(f"{op}: {what}")


def _check_lengths(op: str, name: str, lengths, like: torch.Tensor):
    if lengths is not None and (
            lengths.dim() != 1 or lengths.size(0) != like.size(0)
            or lengths.dtype not in (torch.int32, torch.int64)
            or lengths.device != like.device):
        _refuse(op, f"{name} has to be ({like.size(0)},) int32 or int64 on "
                    f"{like.device}, got {tuple(lengths.shape)} "
                    f"{lengths.dtype} on {lengths.device}")


# ---------------------------------------------------------------------------
# learned relative position bias: distances to buckets
# ---------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _bucket_thresholds(num_buckets: int, max_distance: int) -> list:
    """Distances at which a side's buckets after the exact ones begin: the
    m-th at exact * (max_distance / exact) ** (m / wide), rounded up, in
    whole numbers so that no distance is ever off by a rounding."""
    exact = num_buckets // 4
    wide = num_buckets // 2 - exact
    found = []
    for m in range(1, wide):
        least = exact ** (wide - m) * max_distance ** m
        low, high = exact, max_distance
        while low < high:
            mid = (low + high) // 2
            if mid ** wide >= least:
                high = mid
            else:
                low = mid + 1
        found.append(low)
    return found


def _check_buckets(op: str, num_buckets: int, max_distance: int):
    if num_buckets % 2 or not 4 <= num_buckets <= _MAX_BUCKETS:
        _refuse(op, f"an even number of buckets from 4 to {_MAX_BUCKETS} is "
                    f"needed, got {num_buckets}")
    if not num_buckets // 4 < max_distance <= _MAX_DISTANCE:
        _refuse(op, f"max_distance has to be over {num_buckets // 4} and at "
                    f"most {_MAX_DISTANCE}, got {max_distance}")


def relative_position_buckets(distance: torch.Tensor, num_buckets: int,
                              max_distance: int) -> torch.Tensor:
    """Bucket of each signed distance (key position - query position).

    Half of the buckets are for keys at or before the query, half for keys
    after it. Of a half, the first ``num_buckets // 4`` stand for one distance
    each; the rest widen geometrically up to ``max_distance``, and the last
    holds everything from there on. Buckets come in ``distance``'s type.
    """
    _check_buckets("relative_position_buckets", num_buckets, max_distance)
    exact = num_buckets // 4
    # 64 bits hold every threshold, and the size of the lowest 32-bit distance
    n = (distance if distance.is_floating_point() else distance.long()).abs()
    steps = torch.tensor(_bucket_thresholds(num_buckets, max_distance),
                         dtype=n.dtype, device=n.device)
    at = torch.where(n < exact, n,
                     exact + torch.bucketize(n, steps, right=True).to(n.dtype))
    return (at + (distance > 0) * (num_buckets // 2)).to(distance.dtype)


# ---------------------------------------------------------------------------
# attention to keys and values of another length
# ---------------------------------------------------------------------------


def _check_cross_attention(q, k, v, kv_lengths, bias_table, scale, key_step,
                           query_start):
    op = "cross_attention"
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape \
            or k.size(0) != q.size(0) or k.size(2) != q.size(2):
        _refuse(op, "q (N, H, E, Lq) and k, v (N, Hkv, E, Lk) are needed, "
                    f"got {tuple(q.shape)}, {tuple(k.shape)}, "
                    f"{tuple(v.shape)}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        _refuse(op, "q, k and v have to be all float32 or all bfloat16, got "
                    f"{q.dtype}, {k.dtype}, {v.dtype}")
    if k.device != q.device or v.device != q.device:
        _refuse(op, "q, k and v have to be on one device")
    H, E = q.size(1), q.size(2)
    if k.size(1) == 0 or H % k.size(1):
        _refuse(op, f"{H} query heads cannot share {k.size(1)} key heads")
    if not 1 <= E <= _MAX_DEPTH:
        _refuse(op, f"heads of 1 to {_MAX_DEPTH} channels are needed, got "
                    f"{E}")
    if scale is not None and not 0 < scale < math.inf:
        _refuse(op, f"scale has to be positive, got {scale}")
    _check_lengths(op, "kv_lengths", kv_lengths, q)
    if bias_table is not None:
        if bias_table.dim() != 2 or bias_table.size(0) != H \
                or bias_table.dtype != q.dtype \
                or bias_table.device != q.device:
            _refuse(op, f"bias_table has to be ({H}, buckets) {q.dtype} on "
                        f"{q.device}, got {tuple(bias_table.shape)} "
                        f"{bias_table.dtype} on {bias_table.device}")
        if key_step < 1:
            _refuse(op, f"key_step has to be 1 or more, got {key_step}")
        if key_step * (k.size(3) + 128) >= 2 ** 27 \
                or abs(query_start) + q.size(3) + 256 >= 2 ** 27:
            _refuse(op, "positions have to stay under 2**27")


def _cross_attention_plain(q, k, v, lengths, table, scale, key_step,
                           query_start, max_distance):
    N, H, E, Lq = q.shape
    Hkv, Lk = k.size(1), k.size(3)
    G = H // Hkv
    qf = q.float().reshape(N, Hkv, G, E, Lq).transpose(-1, -2)
    kf = k.float().unsqueeze(2)
    vf = v.float().unsqueeze(2)
    if lengths is not None:
        hidden = torch.arange(Lk, device=q.device) >= lengths[:, None]
        # before any product: a gradient of zero times NaN is NaN
        kf = kf.masked_fill(hidden[:, None, None, None, :], 0.0)
        vf = vf.masked_fill(hidden[:, None, None, None, :], 0.0)
    s = torch.matmul(qf, kf).reshape(N, H, Lq, Lk) * scale
    if table is not None:
        d = (torch.arange(Lk, device=q.device)[None, :] * key_step
             - torch.arange(Lq, device=q.device)[:, None] - query_start)
        bias = table.float()[:, relative_position_buckets(
            d, table.size(1), max_distance)]
        s = (s + bias).masked_fill(bias <= _OUT, -math.inf)
    if lengths is not None:
        s = s.masked_fill(hidden[:, None, None, :], -math.inf)
    # a query with no key left has no weights: zeros, and no gradient
    none = (s == -math.inf).all(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
    out = torch.matmul(p.reshape(N, Hkv, G, Lq, Lk), vf.transpose(-1, -2))
    return out.transpose(-1, -2).reshape(N, H, E, Lq).to(q.dtype)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    kv_lengths: Optional[torch.Tensor] = None,
                    bias_table: Optional[torch.Tensor] = None, *,
                    key_step: int = 1, query_start: int = 0,
                    max_distance: int = 128,
                    scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale * q^T k + bias) v^T to keys of any other length.

    q: (N, H, E, Lq); k, v: (N, Hkv, E, Lk) with H a multiple of Hkv, query
    head h reading key head h // (H // Hkv); E up to 128; all bf16 or all
    fp32. Any strides; a copy is made only where the last axis is not
    contiguous or a head's channels lie further apart than 4 GiB, which a
    head has to fit into. Returns (N, H, E, Lq) in q's type. ``scale``
    defaults to 1 / sqrt(E). Differentiable in q, k, v and ``bias_table``,
    once and in reverse mode; the kernels refuse other derivatives.

    Scores, weights' sums and gradients are summed in 32 bits. In bf16 the
    weights, and in the gradients their slopes, are rounded to bf16 where they
    meet the values, keys and queries.

    ``kv_lengths``: (N,), the keys of each record that count, from 0 to Lk;
    nothing behind them is read into the result, NaN included.

    ``bias_table``: (H, buckets) in q's type, added to the scores by the
    bucket (:func:`relative_position_buckets`) of
    ``j * key_step - (query_start + i)`` for key j and query i. ``key_step``
    is the number of query positions a key stands for (the pooling ratio of
    pooled keys), ``query_start`` the position of the first query (for queries
    that come one at a time); positions stay under 2**27. An entry at or under
    -1e30, such as -inf or the type's lowest value, takes its pairs out of the
    softmax whatever their scores are, NaN and infinities included. Their
    weights are zeros, which still meet the values, and in the gradients the
    keys and queries: only what is behind ``kv_lengths`` may hold anything
    there.

    A query with no key left gives zeros and no gradient.
    """
    thresholds = []
    if bias_table is not None and bias_table.dim() == 2:
        _check_buckets("cross_attention", bias_table.size(1), max_distance)
        thresholds = _bucket_thresholds(bias_table.size(1), max_distance)
    if use_native(q):
        # with its own checks, the same as those below; nothing where torch
        # traces, which the plain steps can be followed by
        out = ext().cross_attention(q, k, v, kv_lengths, bias_table, scale,
                                    key_step, query_start, max_distance,
                                    thresholds)
        if out is not None:
            return out
    _check_cross_attention(q, k, v, kv_lengths, bias_table, scale, key_step,
                           query_start)
    if scale is None:
        scale = 1.0 / math.sqrt(q.size(2))
    return _cross_attention_plain(q, k, v, kv_lengths, bias_table, scale,
                                  key_step, query_start, max_distance)


# ---------------------------------------------------------------------------
# gated linear recurrence
# ---------------------------------------------------------------------------


def _check_gated_scan(x, gate, state, lengths):
    op = "gated_scan"
    if x.dim() != 3 or gate.shape != x.shape or x.size(2) < 1:
        _refuse(op, "x and gate of one shape (N, C, L), L at least 1, are "
                    f"needed, got {tuple(x.shape)} and {tuple(gate.shape)}")
    if x.dtype not in _DTYPES or gate.dtype != x.dtype:
        _refuse(op, "x and gate have to be both float32 or both bfloat16, "
                    f"got {x.dtype} and {gate.dtype}")
    if gate.device != x.device:
        _refuse(op, "x and gate have to be on one device")
    if state is not None and (state.shape != x.shape[:2]
                              or state.dtype != torch.float32
                              or state.device != x.device):
        _refuse(op, f"state has to be {tuple(x.shape[:2])} float32 on "
                    f"{x.device}, got {tuple(state.shape)} {state.dtype} on "
                    f"{state.device}")
    _check_lengths(op, "lengths", lengths, x)


def _gated_scan_plain(x, gate, state, lengths, reverse):
    N, C, L = x.shape
    gate, x32 = gate.float(), x.float()
    valid = None
    if lengths is not None:
        valid = torch.arange(L, device=x.device) < lengths[:, None, None]
        # before any product: a gradient of zero times NaN is NaN
        gate = torch.where(valid, gate, 0.0)
        x32 = torch.where(valid, x32, 0.0)
    a, b = torch.sigmoid(gate), torch.sigmoid(-gate) * x32
    if valid is not None:
        a = torch.where(valid, a, 1.0)
    if reverse:
        a, b = a.flip(-1), b.flip(-1)
    h = x.new_zeros(N, C, dtype=torch.float32) if state is None else state
    out = []
    for t in range(L):
        h = a[..., t] * h + b[..., t]
        out.append(h)
    hs = torch.stack(out, -1)
    if reverse:
        hs = hs.flip(-1)
    if valid is not None:
        hs = torch.where(valid, hs, 0.0)
    return hs.to(x.dtype), h.clone()


def gated_scan(x: torch.Tensor, gate: torch.Tensor,
               state: Optional[torch.Tensor] = None,
               lengths: Optional[torch.Tensor] = None,
               reverse: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """h_t = sigmoid(gate_t) * h_{t-1} + (1 - sigmoid(gate_t)) * x_t.

    x, gate: (N, C, L), both bf16 or both fp32, L at least 1; any strides, a
    copy is made only where the last axis is not contiguous (so the two halves
    of one projection can be given as they are). ``state``: the fp32 (N, C)
    state before the first sample, zeros by default. Returns h (N, C, L) in
    x's type and the fp32 state (N, C) after the last sample, which continues
    a record that comes in pieces, down to one sample a call. Differentiable
    in x, gate and state, once and in reverse mode; the kernels refuse other
    derivatives, 2**24 rows and more, and 2**30 samples and more.

    ``lengths``: (N,), the samples of each record that count; behind them h is
    zero, the state stays, and nothing is read into the result. ``reverse``
    runs from the last sample that counts to the first.
    """
    if use_native(x):
        # with its own checks, the same as those below; nothing where torch
        # traces, which the plain steps can be followed by
        found = ext().gated_scan(x, gate, state, lengths, reverse)
        if found:
            h, last = found
            return h, last
    _check_gated_scan(x, gate, state, lengths)
    return _gated_scan_plain(x, gate, state, lengths, reverse)
