"""Attention over long user-behaviour histories.

What follows ``sequence_embedding_lookup`` in a ranker: its ``[B, T, dim]``
rows and ``[B, T]`` mask, projected to heads, attend to each other.

* :func:`history_attention` -- causal attention with a sliding window, a few
  first tokens that stay visible, heads that share keys, the lookup's mask and
  a learned relative position bias; differentiable.
* :class:`HistoryCache` -- the keys and values of histories that grow: prompts
  written at once, then one new token a row, which attends to what it sees.
* :class:`RelativeBuckets` -- which distances share a learned bias, and
  :func:`relative_position_bias`, that bias made whole for an attention that
  takes it as a tensor; differentiable.

The operators are ``mdl_hip::history_attention`` (differentiable) over
``history_attention_forward`` and ``history_attention_backward``,
``history_cache_step``, ``history_cache_write_`` and
``relative_position_bias`` (over its ``_forward`` and ``_backward``): ROCm
kernels in ``libmdl_torch.so`` over the C ABI, CPU kernels (PyTorch operations,
for parameters on the CPU) and fake kernels registered here.  The differentiable
ones have first gradients only: a dual input is refused, and so is what would
differentiate a gradient.

The mask marks a row's real columns.  A masked column is neither read as a key
nor answered as a query: its output and gradients are zeros whatever its rows
hold.  Softmax, sums and gradients of the bias are taken in fp32; weights and
their gradients are rounded to bfloat16 for the products of bfloat16 inputs.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor

from . import library  # noqa: F401  (loads libmdl_torch.so and its schemas)
from .embeddings import _deferred_counter, index_check_mode
from .library import _cpu_kernel, _fake_kernel

# the operators' overloads, looked up once
_ATTENTION = torch.ops.mdl_hip.history_attention.default
_BIAS = torch.ops.mdl_hip.relative_position_bias.default
_STEP = torch.ops.mdl_hip.history_cache_step.default
_WRITE = torch.ops.mdl_hip.history_cache_write_.default

MAX_BUCKET_START = 2048
MAX_BUCKETS = 1024


class RelativeBuckets:
    """Distances that share a learned bias.

    Half of a direction's buckets hold one distance each; the others widen
    with the logarithm of the distance up to ``max_distance``, from which on
    all share the last one.  Causal by default: a key after its query counts as distance 0.
    ``bidirectional`` gives each direction half of the buckets, the keys after
    the query the second half.
    """

    def __init__(self, num_buckets: int, max_distance: int, bidirectional: bool = False) -> None:
        per_side = num_buckets // 2 if bidirectional else num_buckets
        if per_side < 2 or (bidirectional and num_buckets % 2):
            raise ValueError("relative buckets need at least two a direction, and an even number for two directions")
        if num_buckets > MAX_BUCKETS:
            raise ValueError(f"at most {MAX_BUCKETS} relative buckets")
        if max_distance <= per_side // 2:
            raise ValueError("max_distance must lie past the distances that have a bucket of their own")
        self.num_buckets = num_buckets
        self.max_distance = max_distance
        self.bidirectional = bidirectional
        # the distances at which buckets 1, 2, ... of one direction begin
        self.starts = tuple(_bucket_starts(per_side, max_distance))
        self._on_device: dict[torch.device, Tensor] = {}

    def __repr__(self) -> str:
        return f"RelativeBuckets({self.num_buckets}, {self.max_distance}, bidirectional={self.bidirectional})"

    @torch.compiler.assume_constant_result  # a compiled graph takes the kept tensor
    def starts_on(self, device: torch.device) -> Tensor:
        """The starts as a tensor, kept for later calls.  What is kept serves
        any of them: never an inference tensor, and nothing made under a
        dispatch mode (fake tensors, tracing) or a functional transform, where
        each call makes its own."""

        moded = torch._C._len_torch_dispatch_stack() > 0  # a kept tensor is foreign to fake ones
        t = None if moded else self._on_device.get(device)
        if t is None:
            with torch.inference_mode(False):
                t = torch.tensor(self.starts, dtype=torch.int32, device=device)
            if not moded and torch._C._functorch.peek_interpreter_stack() is None:
                self._on_device[device] = t
        return t

    @property
    def distances(self) -> int:
        """Distances told apart: from the last bucket's start on all are alike."""

        return self.starts[-1] + 1

    def of(self, distance: Tensor) -> Tensor:
        """Bucket of each ``query column - key column``."""

        starts = torch.tensor(self.starts, device=distance.device)
        side = torch.bucketize(distance.abs() if self.bidirectional else distance.clamp(min=0), starts, right=True)
        return torch.where(distance < 0, side + self.num_buckets // 2, side) if self.bidirectional else side


def _bucket_starts(count: int, max_distance: int) -> list[int]:
    """Bucket E + b (E = count // 2, n = count - E) begins at the smallest d
    with (d / E)^n >= (max_distance / E)^b, in whole numbers (where several
    share it, all but the last are empty)."""

    single = count // 2
    steps = count - single
    starts = list(range(1, single + 1))
    for b in range(1, steps):
        bound = max_distance ** b * single ** (steps - b)  # d^n >= bound
        lo, hi = starts[-1], max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid ** steps >= bound:
                hi = mid
            else:
                lo = mid + 1
        starts.append(lo)
    return starts


# ----------------------------------------------------------- CPU and fakes --


def _visible(mask: Optional[Tensor], q_len: int, k_len: int, window: int, sinks: int, device) -> Tensor:
    """[B or 1, q_len, k_len]: which columns each query sees."""

    column = torch.arange(k_len, device=device)
    distance = column[k_len - q_len:, None] - column
    near = distance >= 0
    if mask is None:
        if window:
            near = near & ((distance < window) | (column < sinks))
        return near[None]
    first = mask.int().argmax(1)[:, None, None]
    seen = near & mask[:, None, :] & mask[:, k_len - q_len:, None]
    if window:
        seen = seen & ((distance < window) | (column < first + sinks))
    return seen


def _check_attention(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale) -> None:
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("attention takes q [B, Lq, Hq, D], k and v [B, Lk, Hkv, D]")
    if k.shape != v.shape or k.size(0) != q.size(0) or k.size(3) != q.size(3):
        raise ValueError("attention queries, keys and values are misaligned")
    if q.size(2) <= 0 or k.size(2) <= 0 or q.size(2) % k.size(2):
        raise ValueError("attention query heads must be a multiple of the key heads")
    if q.size(1) > k.size(1):
        raise ValueError("attention queries are the last rows of the keys: more queries than keys")
    if not 1 <= q.size(3) <= 128:
        raise ValueError("attention head dimension must be 1 to 128")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError("attention queries, keys and values must have one dtype")
    if q.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported attention dtype {q.dtype}; expected float32 or bfloat16")
    if window < 0 or sinks < 0:
        raise ValueError("attention window must be positive and sinks not negative")
    if not 0 < scale < 1e30:
        raise ValueError("attention scale must be positive")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError("attention mask must be torch.bool")
        if mask.shape != k.shape[:2]:
            raise ValueError("attention mask must be [B, Lk]")
    if bias_table is not None:
        _check_bias(bias_table, bucket_starts, distances, q.size(2))


def _check_bias(bias_table, bucket_starts, distances, heads) -> None:
    if bucket_starts is None:
        raise ValueError("a bias table needs its buckets")
    if bias_table.ndim != 2 or bias_table.size(1) != heads or bucket_starts.numel() != bias_table.size(0) - 1:
        raise ValueError(f"bias_table must be [buckets, {heads}]")
    if not 1 <= distances <= MAX_BUCKET_START + 1:
        raise ValueError("bias buckets must begin at distances up to 2048")


def _weights_cpu(q, k, mask, bias_table, bucket_starts, window, sinks, scale):
    """(fp32 q, k by head, softmax weights [B, Hkv, G, Lq, Lk], buckets)."""

    B, Lq, H, D = q.shape
    Lk, K = k.size(1), k.size(2)
    keep_q = keep_k = None
    if mask is not None:
        keep_q, keep_k = mask[:, Lk - Lq:, None, None], mask[:, :, None, None]
    qf = (q.float() if keep_q is None else torch.where(keep_q, q.float(), 0.0)).reshape(B, Lq, K, H // K, D)
    kf = k.float() if keep_k is None else torch.where(keep_k, k.float(), 0.0)
    qf = qf.permute(0, 2, 3, 1, 4)
    kf = kf.permute(0, 2, 1, 3)[:, :, None]
    scores = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    bucket = None
    if bias_table is not None:
        column = torch.arange(Lk)
        distance = (column[Lk - Lq:, None] - column).clamp(min=0)
        bucket = torch.bucketize(distance, bucket_starts.long(), right=True)
        scores = scores + bias_table.float()[bucket].permute(2, 0, 1).reshape(K, H // K, Lq, Lk)
    seen = _visible(mask, Lq, Lk, window, sinks, q.device)[:, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return qf, kf, e / torch.where(total == 0, 1.0, total), bucket


def _values_cpu(v, mask):
    vf = v.float() if mask is None else torch.where(mask[:, :, None, None], v.float(), 0.0)
    return vf.permute(0, 2, 1, 3)[:, :, None]


@_cpu_kernel("history_attention_forward")
def _attention_forward_cpu(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale, need_backward):
    _check_attention(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale)
    if q.numel() == 0:
        out = torch.empty(q.shape, dtype=q.dtype)
    else:
        _, _, p, _ = _weights_cpu(q, k, mask, bias_table, bucket_starts, window, sinks, scale)
        out = torch.matmul(p, _values_cpu(v, mask)).permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype)
    stats = q.new_zeros(_stats_shape(q, need_backward), dtype=torch.float32)
    return out.contiguous(), stats, q.new_empty(0, dtype=torch.uint8)


def _stats_shape(q, need_backward):
    return (q.size(0), q.size(2), q.size(1), 2) if need_backward else (0,)


@_fake_kernel("history_attention_forward")
def _attention_forward_fake(q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale, need_backward):
    words = 0
    if q.device.type != "cpu":
        # the call's prepared buffer: mask bits, first columns, bias by distance
        def part(n):
            return (n + 255) // 256 * 256

        if mask is not None:
            words += part(k.size(0) * ((k.size(1) + 63) // 64 + 1) * 8) + part(k.size(0) * 8)
        if bias_table is not None:
            words += part(q.size(2) * (distances + 512) * 4)
    return (q.new_empty(q.shape), q.new_empty(_stats_shape(q, need_backward), dtype=torch.float32),
            q.new_empty(words, dtype=torch.uint8))


@_cpu_kernel("history_attention_backward")
def _attention_backward_cpu(grad_out, q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale, out,
                            stats, prepared, need_table):
    B, Lq, H, D = q.shape
    Lk, K = k.size(1), k.size(2)
    need_table = need_table and bias_table is not None
    if q.numel() == 0:
        return (torch.zeros(q.shape, dtype=q.dtype), torch.zeros(k.shape, dtype=k.dtype),
                torch.zeros(v.shape, dtype=v.dtype),
                torch.zeros(bias_table.shape, dtype=bias_table.dtype) if need_table else q.new_empty(0))
    qf, kf, p, bucket = _weights_cpu(q, k, mask, bias_table, bucket_starts, window, sinks, scale)
    go = grad_out.float()
    if mask is not None:
        go = torch.where(mask[:, Lk - Lq:, None, None], go, 0.0)
    go = go.reshape(B, Lq, K, H // K, D).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), go).sum(2)
    dp = torch.matmul(go, _values_cpu(v, mask).transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = torch.matmul(ds, kf) * scale
    dk = (torch.matmul(ds.transpose(-1, -2), qf) * scale).sum(2)
    dtable = q.new_empty(0)
    if need_table:
        flat = torch.zeros(bias_table.size(0), H)
        flat.index_add_(0, bucket.reshape(-1), ds.sum(0).reshape(H, -1).t())
        dtable = flat.to(bias_table.dtype)
    return (dq.permute(0, 3, 1, 2, 4).reshape(q.shape).to(q.dtype).contiguous(),
            dk.permute(0, 2, 1, 3).to(k.dtype).contiguous(), dv.permute(0, 2, 1, 3).to(v.dtype).contiguous(), dtable)


@_fake_kernel("history_attention_backward")
def _attention_backward_fake(grad_out, q, k, v, mask, bias_table, bucket_starts, distances, window, sinks, scale, out,
                             stats, prepared, need_table):
    table = bias_table.new_empty(bias_table.shape) if need_table and bias_table is not None else q.new_empty(0)
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), table


def _cache_rows_cpu(positions, capacity, sinks):
    """(position held by each slot once position n is stored, negative: none;
    the new token's slot) of every row."""

    ring = capacity - sinks
    slot = torch.arange(capacity)
    n = positions[:, None]
    held = torch.where(slot < sinks, slot, n - torch.remainder(n - slot, ring))
    held = torch.where((slot >= sinks) & (held < sinks), -1, held)
    at = torch.where(positions < sinks, positions, sinks + torch.remainder(positions - sinks, ring))
    return torch.where(held > n, -1, held), at


def _check_cache(k, v, cache_k, cache_v, sinks) -> None:
    if cache_k.ndim != 4 or cache_k.shape != cache_v.shape:
        raise ValueError("history cache keys and values must be [B, capacity, Hkv, D]")
    if not cache_k.dtype == cache_v.dtype == k.dtype == v.dtype:
        raise TypeError("history cache, keys and values must have one dtype")
    if cache_k.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported attention dtype {cache_k.dtype}; expected float32 or bfloat16")
    if sinks < 0 or cache_k.size(1) <= sinks:
        raise ValueError("history cache capacity must exceed its sinks")
    if not 1 <= cache_k.size(3) <= 128:
        raise ValueError("attention head dimension must be 1 to 128")


def _check_positions(t, cache, what) -> None:
    if t.dtype != torch.long:
        raise TypeError(f"{what} must be torch.long")
    if t.ndim != 1 or t.size(0) != cache.size(0):
        raise ValueError(f"{what} must hold one entry per row of the cache")


@_cpu_kernel("history_cache_step")
def _cache_step_cpu(q, k, v, cache_k, cache_v, positions, bias_table, bucket_starts, distances, window, sinks, scale):
    _check_cache(k, v, cache_k, cache_v, sinks)
    B, capacity, K, D = cache_k.shape
    if q.ndim != 3 or k.shape != (B, K, D) or v.shape != k.shape or q.size(0) != B or q.size(2) != D:
        raise ValueError("a step takes q [B, Hq, D], k and v [B, Hkv, D] of the cache's rows")
    if q.size(1) == 0 or q.size(1) % K:
        raise ValueError("attention query heads must be a multiple of the key heads")
    if not 0 <= window <= capacity - sinks:
        raise ValueError("attention window must fit the cache beside its sinks")
    if not 0 < scale < 1e30:
        raise ValueError("attention scale must be positive")
    _check_positions(positions, cache_k, "positions")
    if bias_table is not None:
        _check_bias(bias_table, bucket_starts, distances, q.size(1))
    if B == 0:
        return torch.empty_like(q)
    with torch._C._AutoDispatchBelowAutograd():  # operations of PyTorch, of which nothing is recorded
        return _stored_and_answered_cpu(q, k, v, cache_k, cache_v, positions, bias_table, bucket_starts, window, sinks,
                                        scale)


def _stored_and_answered_cpu(q, k, v, cache_k, cache_v, positions, bias_table, bucket_starts, window, sinks, scale):
    B, capacity, K, D = cache_k.shape
    held, at = _cache_rows_cpu(positions, capacity, sinks)
    row = (positions >= 0).nonzero().flatten()
    cache_k[row, at[row]] = k[row]
    cache_v[row, at[row]] = v[row]
    distance = positions[:, None] - held
    seen = (held >= 0) & (positions >= 0)[:, None]
    if window:
        seen = seen & ((distance < window) | (held < sinks))
    kf = torch.where(seen[:, :, None, None], cache_k.float(), 0.0)
    vf = torch.where(seen[:, :, None, None], cache_v.float(), 0.0)
    qf = q.float().reshape(B, K, -1, D)
    scores = torch.matmul(qf, kf.permute(0, 2, 3, 1)) * scale
    if bias_table is not None:
        bucket = torch.bucketize(distance.clamp(min=0), bucket_starts.long(), right=True)
        scores = scores + bias_table.float()[bucket].reshape(B, capacity, K, -1).permute(0, 2, 3, 1)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e / torch.where(total == 0, 1.0, total), vf.permute(0, 2, 1, 3))
    return out.reshape(q.shape).to(q.dtype)


@_fake_kernel("history_cache_step")
def _cache_step_fake(q, k, v, cache_k, cache_v, positions, bias_table, bucket_starts, distances, window, sinks, scale):
    return q.new_empty(q.shape)


@_cpu_kernel("history_cache_write_")
def _cache_write_cpu(k, v, cache_k, cache_v, lengths, sinks, right_aligned):
    _check_cache(k, v, cache_k, cache_v, sinks)
    B, capacity, K, D = cache_k.shape
    if k.ndim != 4 or k.shape != v.shape or k.size(0) != B or k.shape[2:] != (K, D):
        raise ValueError("a prompt's k and v must be [B, L, Hkv, D] of the cache's rows")
    _check_positions(lengths, cache_k, "lengths")
    ring, L = capacity - sinks, k.size(1)
    if bool((lengths > L).any()):
        raise ValueError(f"history cache lengths must not exceed the prompt's {L} rows")
    with torch._C._AutoDispatchBelowAutograd():  # as for a step
        for b in range(B):
            n = int(lengths[b])
            p = torch.arange(max(n, 0))
            p = p[(p < sinks) | (p >= n - ring)]
            slots = torch.where(p < sinks, p, sinks + (p - sinks) % ring)
            rows = p + (L - n if right_aligned else 0)
            cache_k[b, slots], cache_v[b, slots] = k[b, rows], v[b, rows]


@_fake_kernel("history_cache_write_")
def _cache_write_fake(k, v, cache_k, cache_v, lengths, sinks, right_aligned):
    return None


def _bias_buckets_cpu(bucket_starts, bidirectional, side, q_len, k_len):
    column = torch.arange(k_len)
    distance = column[k_len - q_len:, None] - column
    near = distance.abs() if bidirectional else distance.clamp(min=0)
    bucket = torch.bucketize(near, bucket_starts.long(), right=True)
    return torch.where(distance < 0, bucket + side, bucket) if bidirectional else bucket


def _check_relative_bias(table, bucket_starts, bidirectional, q_len, k_len) -> None:
    if table.ndim != 2 or table.size(0) < 1 or table.size(1) < 1:
        raise ValueError("bias table must be [buckets, heads]")
    if table.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported bias dtype {table.dtype}; expected float32 or bfloat16")
    side = table.size(0) // 2 if bidirectional else table.size(0)
    if bucket_starts.numel() != side - 1 or side * (2 if bidirectional else 1) != table.size(0):
        raise ValueError("bucket_starts must have one entry fewer than a direction has buckets")
    if not 0 <= q_len <= k_len:
        raise ValueError("a relative bias has 0 <= q_len <= k_len")


@_cpu_kernel("relative_position_bias_forward")
def _relative_bias_cpu(table, bucket_starts, bidirectional, q_len, k_len):
    _check_relative_bias(table, bucket_starts, bidirectional, q_len, k_len)
    bucket = _bias_buckets_cpu(bucket_starts, bidirectional, table.size(0) // 2, q_len, k_len)
    return table.t()[:, bucket].contiguous()


@_fake_kernel("relative_position_bias_forward")
def _relative_bias_fake(table, bucket_starts, bidirectional, q_len, k_len):
    return table.new_empty((table.size(1), q_len, k_len))


@_cpu_kernel("relative_position_bias_backward")
def _relative_bias_backward_cpu(grad, bucket_starts, num_buckets, bidirectional):
    heads, q_len, k_len = grad.shape
    bucket = _bias_buckets_cpu(bucket_starts, bidirectional, num_buckets // 2, q_len, k_len)
    sums = torch.zeros(num_buckets, heads)
    sums.index_add_(0, bucket.reshape(-1), grad.float().reshape(heads, -1).t())
    return sums.to(grad.dtype)


@_fake_kernel("relative_position_bias_backward")
def _relative_bias_backward_fake(grad, bucket_starts, num_buckets, bidirectional):
    return grad.new_empty((num_buckets, grad.size(0)))


# ------------------------------------------------------------- attention --


def _bias_arguments(bias_table: Optional[Tensor], buckets: Optional[RelativeBuckets]) -> tuple[Optional[Tensor], int]:
    """(starts on the table's device, distances told apart) of a causal bias."""

    if bias_table is None:
        if buckets is not None:
            raise ValueError("relative buckets without a bias table")
        return None, 0
    if buckets is None:
        raise ValueError("a bias table needs its buckets")
    if buckets.bidirectional:
        raise ValueError("history attention is causal: its buckets are not bidirectional")
    if bias_table.ndim != 2 or bias_table.size(0) != buckets.num_buckets:
        raise ValueError(f"bias_table must have one row for each of the {buckets.num_buckets} buckets")
    if buckets.starts[-1] > MAX_BUCKET_START:
        raise ValueError(f"the last bucket of an attention bias must begin at {MAX_BUCKET_START} or before")
    return buckets.starts_on(bias_table.device), buckets.distances


def _window_argument(window: Optional[int]) -> int:
    if window is None:
        return 0
    if window <= 0:
        raise ValueError("attention window must be positive (None: every earlier column)")
    return int(window)


def history_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    *,
    mask: Optional[Tensor] = None,
    window: Optional[int] = None,
    sinks: int = 0,
    bias_table: Optional[Tensor] = None,
    buckets: Optional[RelativeBuckets] = None,
    scale: Optional[float] = None,
) -> Tensor:
    """Causal attention of ``q [B, Lq, Hq, D]`` over ``k, v [B, Lk, Hkv, D]``.

    The queries are the last ``Lq`` of the ``Lk`` columns; query head ``h``
    reads key head ``h // (Hq // Hkv)``.  Column ``j`` is visible to column
    ``c`` when both are unmasked in ``mask [B, Lk]``, ``j <= c``, and
    ``c - j < window`` or ``j`` is among the ``sinks`` columns from the row's
    first unmasked one on.  Scores are ``scale * q.k`` (``D ** -0.5`` by
    default) plus ``bias_table[buckets.of(c - j), h]``.  A query that sees
    nothing gets zeros.  ``D`` is 1 to 128; fp32 or bf16.
    """

    starts, distances = _bias_arguments(bias_table, buckets)
    if scale is None:
        scale = q.size(-1) ** -0.5 if q.ndim else 1.0
    return _ATTENTION(q, k, v, mask, bias_table, starts, distances, _window_argument(window), int(sinks), float(scale))


def relative_position_bias(table: Tensor, q_len: int, k_len: int, buckets: RelativeBuckets) -> Tensor:
    """``[heads, q_len, k_len]`` bias of ``table [buckets, heads]``: the value of
    ``buckets.of(i + k_len - q_len - j)`` at ``[h, i, j]``, in the table's
    dtype; its gradient sums over each bucket's places."""

    if table.ndim != 2 or table.size(0) != buckets.num_buckets:
        raise ValueError(f"bias table must have one row for each of the {buckets.num_buckets} buckets")
    return _BIAS(table, buckets.starts_on(table.device), buckets.bidirectional, int(q_len), int(k_len))


def _check_lengths(lengths: Tensor, rows: int) -> None:
    message = f"history cache lengths must not exceed the prompt's {rows} rows"
    mode = index_check_mode()
    if mode == "sync":
        if bool((lengths > rows).any()):
            raise ValueError(message)
    elif mode == "deferred":
        _deferred_counter(lengths.device).add_((lengths > rows).sum())
    else:
        torch._assert_async((lengths <= rows).all(), message)


class HistoryCache:
    """Keys and values of histories that grow, one row per user.

    ``k`` and ``v`` are ``[B, capacity, Hkv, D]``.  Position ``p`` of a row's
    history lies in slot ``p`` while the capacity lasts; from then on new
    positions replace the oldest ones, the first ``sinks`` excepted.  With
    ``capacity == sinks + window`` a row keeps just what its next token sees,
    however long its history.

    Inference only: nothing here is differentiable, and nothing is recorded.
    Steps and writes change ``k`` and ``v`` in place, which autograd learns of.
    """

    def __init__(self, k: Tensor, v: Tensor, *, window: Optional[int] = None, sinks: int = 0) -> None:
        _check_cache(k, v, k, v, sinks)
        self._window = _window_argument(window)
        if self._window > k.size(1) - sinks:
            raise ValueError("attention window must fit the cache beside its sinks")
        self.k = k
        self.v = v
        self.sinks = int(sinks)

    @classmethod
    def empty(cls, batch: int, capacity: int, kv_heads: int, head_dim: int, *, window: Optional[int] = None,
              sinks: int = 0, dtype: torch.dtype = torch.float32, device=None) -> "HistoryCache":
        shape = (batch, capacity, kv_heads, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   window=window, sinks=sinks)

    @property
    def window(self) -> Optional[int]:
        return self._window or None

    @property
    def capacity(self) -> int:
        return self.k.size(1)

    def write(self, k: Tensor, v: Tensor, lengths: Tensor, *, right_aligned: bool = False) -> None:
        """Store prompts: ``k, v [B, L, Hkv, D]`` hold positions ``0 ..
        lengths[b] - 1`` of each row in their first rows, or in their last
        ones (``sequence_embedding_lookup``'s window) with ``right_aligned``.
        A length above ``L`` is refused, on a ROCm device as out-of-range ids
        are (``embeddings.set_index_check_mode``): the rows it misses would be
        answered from all the same.  A negative one stores nothing."""

        if lengths.is_cuda and k.ndim == 4:
            _check_lengths(lengths, k.size(1))
        _WRITE(k, v, self.k, self.v, lengths, self.sinks, right_aligned)

    def step(self, q: Tensor, k: Tensor, v: Tensor, positions: Tensor, *, bias_table: Optional[Tensor] = None,
             buckets: Optional[RelativeBuckets] = None, scale: Optional[float] = None) -> Tensor:
        """Store one new token a row and attend from it.

        ``k, v [B, Hkv, D]`` are stored as position ``positions[b]``; the answer
        to ``q [B, Hq, D]`` runs over the positions up to it that lie within
        the window or among the sinks, as :func:`history_attention` would give
        it.  A negative position stores nothing and is answered with zeros.
        """

        starts, distances = _bias_arguments(bias_table, buckets)
        if scale is None:
            scale = q.size(-1) ** -0.5
        return _STEP(q, k, v, self.k, self.v, positions, bias_table, starts, distances, self._window, self.sinks,
                     float(scale))
