"""Plain 64-bit forms of the operators over histories, written from their
definitions: what the tests of the CPU and ROCm kernels compare with."""

import math

import torch


def bucket(distance, count, max_distance, bidirectional=False):
    """Bucket of (query column - key column), one pair at a time: half of a
    direction's buckets hold one distance, the others equal steps of the
    logarithm up to max_distance (whole numbers decide)."""

    side = count // 2 if bidirectional else count
    single, steps = side // 2, side - side // 2

    def one(d):
        base = side if bidirectional and d < 0 else 0
        d = abs(d) if bidirectional else max(d, 0)
        if d < single:
            return base + d
        b = 0
        while b + 1 < steps and d ** steps * single ** (b + 1) >= max_distance ** (b + 1) * single ** steps:
            b += 1
        return base + single + b

    values = {int(d): one(int(d)) for d in distance.unique()}
    return torch.tensor([values[int(d)] for d in distance.flatten()]).reshape(distance.shape)


def visible(mask, q_len, window, sinks):
    """[B, q_len, k_len] of a [B, k_len] mask, column by column."""

    B, k_len = mask.shape
    seen = torch.zeros(B, q_len, k_len, dtype=torch.bool)
    for b in range(B):
        live = mask[b].nonzero().flatten().tolist()
        if not live:
            continue
        j = torch.arange(k_len)
        for i in range(q_len):
            c = i + k_len - q_len
            if not mask[b, c]:
                continue
            near = (c - j < window) | (j < live[0] + sinks) if window else torch.ones(k_len, dtype=torch.bool)
            seen[b, i] = mask[b] & (j <= c) & near
    return seen


def attention(q, k, v, mask, window, sinks, table, buckets, scale=None, grad=None):
    """out, and with ``grad`` also dq, dk, dv and dtable, in float64."""

    q, k, v = q.double(), k.double(), v.double()
    B, Lq, H, D = q.shape
    Lk, K = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    if mask is None:
        mask = torch.ones(B, Lk, dtype=torch.bool)
    seen = visible(mask, Lq, window, sinks)
    which = None
    if table is not None:
        column = torch.arange(Lk)
        which = bucket(column[Lk - Lq:, None] - column, *buckets)
    k, v = (torch.where(mask[:, :, None, None], t, 0.0) for t in (k, v))
    q = torch.where(mask[:, Lk - Lq:, None, None], q, 0.0)
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    dtable = None if table is None else torch.zeros(table.shape, dtype=torch.float64)
    for h in range(H):
        g = h // (H // K)
        x = torch.einsum("bid,bjd->bij", q[:, :, h], k[:, :, g]) * scale
        if table is not None:
            x = x + table.double()[which, h]
        x = x.masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total == 0, 1.0, total)
        out[:, :, h] = torch.einsum("bij,bjd->bid", p, v[:, :, g])
        if grad is None:
            continue
        go = torch.where(mask[:, Lk - Lq:, None], grad[:, :, h].double(), 0.0)
        dv[:, :, g] += torch.einsum("bij,bid->bjd", p, go)
        dp = torch.einsum("bid,bjd->bij", go, v[:, :, g])
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        dq[:, :, h] = torch.einsum("bij,bjd->bid", ds, k[:, :, g]) * scale
        dk[:, :, g] += torch.einsum("bij,bid->bjd", ds, q[:, :, h]) * scale
        if table is not None:
            dtable[:, h] = torch.bincount(which.flatten(), ds.sum(0).flatten(), table.size(0))
    return out if grad is None else (out, dq, dk, dv, dtable)


def step(q, histories_k, histories_v, window, sinks, table, buckets, scale=None):
    """Answers of the last positions of whole histories (lists of [n, Hkv, D])."""

    out = []
    for b, (k, v) in enumerate(zip(histories_k, histories_v)):
        n = k.size(0)
        row = torch.zeros(1, n, q.size(1), q.size(2))
        row[0, -1] = q[b].float()
        out.append(attention(row[:, -1:], k[None], v[None], None, window, sinks, table, buckets, scale)[0, 0])
    return torch.stack(out)


def norm(x, o, w_post, w_next, gate, scale, eps, dy=None, dh=None):
    """(y, h), and with gradients (y, h, dx, do, dgate, dscale, dpost, dnext)."""

    x = x.double()
    one = torch.ones(x.size(-1), dtype=torch.float64)
    w_next = w_next.double()
    y = x
    if o is not None:
        o = o.double()
        sg = torch.ones_like(o) if gate is None else 1 / (1 + torch.exp(-gate.double()))
        sc = one if scale is None else scale.double()
        wp = one if w_post is None else w_post.double()
        inv_o = (o.square().mean(-1, keepdim=True) + eps).rsqrt()
        y = x + sg * sc * wp * o * inv_o
    inv_y = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = y * inv_y * w_next
    if dy is None and dh is None:
        return y, h
    rows = tuple(range(x.ndim - 1))
    dx = torch.zeros_like(y) if dy is None else dy.double()
    dnext = torch.zeros_like(one)
    if dh is not None:
        a, n = dh.double() * w_next, y * inv_y
        dnext = (dh.double() * n).sum(rows)
        dx = dx + inv_y * (a - n * (a * n).mean(-1, keepdim=True))
    if o is None:
        return y, h, dx, None, None, None, None, dnext
    n = o * inv_o
    b = dx * sg * sc * wp
    return (y, h, dx, inv_o * (b - n * (b * n).mean(-1, keepdim=True)), dx * n * sc * wp * sg * (1 - sg),
            (dx * sg * wp * n).sum(rows), (dx * sg * sc * n).sum(rows), dnext)


def close(got, want, dtype, what="", fp32=1e-5):
    """Norm-wise comparison.  A bfloat16 rounding moves a value by at most 2^-9
    of itself, and a result passes at most four of them (inputs of its last
    product and of the one before, a statistic, the result), so it is within
    4 x 2^-9 of the norm.  fp32 sums of a few thousand products of unit size
    stay within 2^-24 sqrt(n) of theirs, below 1e-5.  The norm counts at least as
    0.1 an element: results whose unit terms cancel keep the terms' errors."""

    tol = 4 * 2.0 ** -9 if dtype == torch.bfloat16 else fp32
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    error = float((got - want).norm())
    assert error <= tol * (float(want.norm()) + 0.1 * math.sqrt(want.numel())), (what, error, float(want.norm()))
