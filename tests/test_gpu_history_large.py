"""Rows whose largest score is a bias of mask size, on a GPU: outputs, every
gradient and steps against 64-bit values.

Such a bias swallows the scores beside it (fp32: 1e10 / scale has steps of
4096), so the weights are known: uniform over a row's visible keys of the
largest bias, 0 elsewhere.  Rows that see no such bias keep their softmax."""

import math

import pytest
import torch

from mdl_amd.history import HistoryCache, RelativeBuckets, history_attention
from tests import history_reference as R
from tests.test_gpu_history import announce, holes, make

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def reference(q, k, v, mask, window, sinks, table, rule, do, swallow=True):
    """out, dq, dk, dv, dtable in float64; scores beside a row's largest bias
    of 1e9 or more in size are left out with ``swallow``."""

    (B, Lq, H, D), (Lk, K) = q.shape, k.shape[1:3]
    mask = torch.ones(B, Lk, dtype=torch.bool) if mask is None else mask
    seen = R.visible(mask, Lq, window or 0, sinks)
    column = torch.arange(Lk)
    which = rule.of(column[Lk - Lq:, None] - column)
    q, k, v, do, table = (t.double() for t in (q, k, v, do, table))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dtable = torch.zeros_like(table)
    for h in range(H):
        g = h // (H // K)
        s = torch.einsum("bid,bjd->bij", q[:, :, h], k[:, :, g]) * D ** -0.5
        bias = table[which, h].expand(B, -1, -1)
        top = bias.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
        large = (top.abs() >= 1e9) if swallow else torch.zeros_like(top, dtype=torch.bool)
        x = torch.where(large, torch.where(bias == top, 0.0, -math.inf), s + bias).masked_fill(~seen, -math.inf)
        p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        out[:, :, h] = torch.einsum("bij,bjd->bid", p, v[:, :, g])
        go = torch.where(seen.any(-1)[..., None], do[:, :, h], 0.0)
        dv[:, :, g] += torch.einsum("bij,bid->bjd", p, go)
        dp = torch.einsum("bid,bjd->bij", go, v[:, :, g])
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        dq[:, :, h] = torch.einsum("bij,bjd->bid", ds, k[:, :, g]) * D ** -0.5
        dk[:, :, g] += torch.einsum("bij,bid->bjd", ds, q[:, :, h]) * D ** -0.5
        dtable[:, h] = torch.bincount(which.flatten(), ds.sum(0).flatten(), table.size(0))
    return out, dq, dk, dv, dtable


def check(device, dtype, B, L, H, K, D, mask, window, sinks, table, rule, fp32=1e-5, swallow=True):
    announce("large", dtype, B, L, H, K, D, window, sinks, rule, table[:, 0].tolist())
    q, k, v = (make(i, dtype, B, L, h, D, std=3.0 if i < 2 else 1.0) for i, h in ((0, H), (1, K), (2, K)))
    do = make(3, dtype, B, L, H, D)
    leaves = [t.to(device).requires_grad_() for t in (q, k, v, table)]
    out = history_attention(*leaves[:3], mask=None if mask is None else mask.to(device), window=window, sinks=sinks,
                            bias_table=leaves[3], buckets=rule)
    got = [out.detach(), *torch.autograd.grad(out, leaves, do.to(device))]
    want = reference(q, k, v, mask, window, sinks, table, rule, do, swallow)
    for name, g, w in zip(("out", "dq", "dk", "dv", "dtable"), got, want):
        R.close(g, w, dtype, name, fp32=fp32)


def values(dtype):
    return [-1e10, -1e20, torch.finfo(dtype).min, 1e10, torch.finfo(dtype).max]


# (rows, heads, key heads, head dimension, window, first tokens): without a window; the far part with
# every pair in the last bucket; the far part with buckets told apart
SHAPES = [(150, 2, 2, 32, None, 0), (600, 4, 2, 64, 40, 3), (600, 2, 1, 128, 33, 40), (300, 2, 1, 24, 7, 5)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n", range(5))
def test_one_large_bias_everywhere(device, dtype, shape, n):
    L, H, K, D, window, sinks = shape
    rule = RelativeBuckets(32, 128)
    table = torch.full((32, H), values(dtype)[n], dtype=dtype)
    check(device, dtype, 2, L, H, K, D, holes(5, 2, L, "holes"), window, sinks, table, rule)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n", range(5))
def test_large_biases_among_others(device, dtype, shape, n):
    """One head of two with the large value in some buckets only, near and far:
    tiles then hold rows of both kinds."""

    L, H, K, D, window, sinks = shape
    rule = RelativeBuckets(32, 128)
    table = make(7, dtype, 32, H)
    table[5, ::2] = table[6, ::2] = table[20, ::2] = table[31, ::2] = values(dtype)[n]
    check(device, dtype, 2, L, H, K, D, holes(6, 2, L, "holes"), window, sinks, table, rule)


@pytest.mark.parametrize("shape", SHAPES)
def test_a_bias_that_costs_digits(device, shape):
    """-1e4 keeps the scores, at steps of 2^-7 or less where a score is divided by
    the scale (1e4 D^0.5 < 2^17): up to D roundings of half of that move a
    weight by 2^-8 scale sqrt(D / 3) of itself, 2.3e-3, and a gradient takes it
    from p and from delta, so within 2^-7."""

    L, H, K, D, window, sinks = shape
    table = torch.full((32, H), -1e4)
    check(device, F32, 2, L, H, K, D, None, window, sinks, table, RelativeBuckets(32, 128), fp32=2.0 ** -7,
          swallow=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,K,D", [(2, 2, 32), (8, 1, 128)])
@pytest.mark.parametrize("lengths,capacity,window,sinks", [([40, 3, 0], 64, None, 0), ([300, 41], 28, 24, 4),
                                                           ([1500], 2000, None, 0)])
@pytest.mark.parametrize("n", range(5))
@pytest.mark.parametrize("everywhere", [True, False])
def test_steps_with_large_biases(device, dtype, H, K, D, lengths, capacity, window, sinks, n, everywhere):
    announce("large step", dtype, H, K, D, lengths, capacity, window, sinks, values(dtype)[n], everywhere)
    rule = RelativeBuckets(32, 128)
    table = make(7, dtype, 32, H)
    if everywhere:
        table[:] = values(dtype)[n]
    else:
        table[5, ::2] = table[31, ::2] = values(dtype)[n]
    B, top = len(lengths), max(lengths) + 1
    k, v, q = make(0, dtype, B, top, K, D, std=3.0), make(1, dtype, B, top, K, D), make(2, dtype, B, H, D, std=3.0)
    at, row = torch.tensor(lengths), torch.arange(B)
    cache = HistoryCache.empty(B, capacity, K, D, window=window, sinks=sinks, dtype=dtype, device=device)
    cache.write(k.to(device), v.to(device), at.to(device))
    got = cache.step(q.to(device), k[row, at].to(device), v[row, at].to(device), at.to(device),
                     bias_table=table.to(device), buckets=rule)
    for b, n in enumerate(lengths):
        wide = torch.zeros(1, n + 1, H, D, dtype=dtype)
        wide[0, -1] = q[b]
        want = reference(wide[:, -1:], k[b:b + 1, :n + 1], v[b:b + 1, :n + 1], None, window, sinks, table, rule,
                         torch.zeros(1, 1, H, D))[0]
        R.close(got[b], want[0, 0], dtype, b)
