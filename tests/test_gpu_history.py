"""The operators over histories on a GPU, against plain 64-bit forms.

Tolerances are those of history_reference.close: shares of the norm that follow
from the number of bfloat16 roundings, 1e-5 for fp32.
"""

import math

import pytest
import torch

from mdl_amd.block_norm import gated_residual_norm
from mdl_amd.history import HistoryCache, RelativeBuckets, history_attention, relative_position_bias
from tests import history_reference as R
from tests.test_history import _encoder

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def announce(*what):
    print("CASE", *what, flush=True)


def make(seed, dtype, *shape, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def holes(seed, B, L, kind):
    """[B, L] masks: full, right-aligned ragged rows (one of them empty, one of
    one column), or columns left out anywhere."""

    if kind == "full":
        return None
    mask = torch.ones(B, L, dtype=torch.bool)
    g = torch.Generator().manual_seed(seed)
    if kind == "ragged":
        for b in range(B):
            n = (0, 1, L)[b] if b < min(3, B) else int(torch.randint(0, L + 1, (1,), generator=g))
            mask[b, : L - n] = False
    else:
        mask = torch.rand(B, L, generator=g) < 0.6
    return mask


def run_attention(device, dtype, B, Lq, Lk, H, K, D, mask, window, sinks, rule, seed=0, std=1.0, fp32=1e-5):
    announce("attention", dtype, B, Lq, Lk, H, K, D, window, sinks, rule)
    q, do = make(seed, dtype, B, Lq, H, D, std=std), make(seed + 1, dtype, B, Lq, H, D)
    k, v = make(seed + 2, dtype, B, Lk, K, D, std=std), make(seed + 3, dtype, B, Lk, K, D)
    table = None if rule is None else make(seed + 4, dtype, rule[0], H)
    leaves = [None if t is None else t.to(device).requires_grad_() for t in (q, k, v, table)]
    out = history_attention(*leaves[:3], mask=None if mask is None else mask.to(device), window=window, sinks=sinks,
                            bias_table=leaves[3], buckets=None if rule is None else RelativeBuckets(*rule))
    out.backward(do.to(device))
    want = R.attention(q, k, v, mask, window or 0, sinks, table, rule, grad=do)
    got = [out.detach()] + [None if t is None else t.grad for t in leaves]
    for name, g, w in zip(("out", "dq", "dk", "dv", "dtable"), got, want):
        if g is not None:
            R.close(g, w, dtype, name, fp32=fp32)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [1, 7, 24, 32, 33, 64, 80, 96, 128])
def test_attention_head_dims(device, dtype, D):
    run_attention(device, dtype, 2, 70, 70, 4, 2, D, holes(1, 2, 70, "holes"), 40, 3, (10, 40))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (2, 2), (31, 31), (32, 32), (33, 65), (64, 64), (1, 129), (127, 128),
                                   (129, 129), (257, 300)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (33, 2), (64, 100)])
def test_attention_lengths(device, dtype, Lq, Lk, window, sinks):
    run_attention(device, dtype, 2, Lq, Lk, 2, 1, 32, None, window, sinks, (8, 24))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["ragged", "holes"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 0), (70, 5), (64, 64)])
@pytest.mark.parametrize("rule", [None, (32, 128)])
def test_attention_masks(device, dtype, kind, window, sinks, rule):
    run_attention(device, dtype, 5, 200, 200, 4, 4, 64, holes(3, 5, 200, kind), window, sinks, rule)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,K,D", [(8, 1, 64), (6, 3, 40), (3, 3, 16), (16, 2, 128)])
def test_attention_shared_heads(device, dtype, H, K, D):
    run_attention(device, dtype, 2, 150, 170, H, K, D, holes(5, 2, 170, "holes"), 60, 4, (16, 64))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_sinks_far_beyond_the_window(device, dtype):
    # many queries see the first tokens only across a gap longer than one block of rows
    run_attention(device, dtype, 2, 1100, 1100, 2, 1, 64, holes(6, 2, 1100, "ragged"), 64, 40, (32, 1024))
    run_attention(device, dtype, 1, 900, 900, 2, 2, 128, None, 33, 300, (32, 1024))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_many_units(device, dtype):
    run_attention(device, dtype, 40, 65, 65, 4, 2, 32, holes(7, 40, 65, "ragged"), 30, 2, (8, 24))
    run_attention(device, dtype, 0, 8, 8, 4, 2, 32, None, 4, 0, None)


def test_attention_large_scores(device):
    # Scores of up to 1000: the running maximum moves often and most weights
    # vanish.  fp32 scores are off by 1000 x 2^-24 or so, 6e-5, and the weights by
    # as much of themselves; the gradients take that six times (k is of size 6).
    run_attention(device, F32, 2, 130, 130, 2, 1, 64, None, None, 0, (8, 24), std=6.0, fp32=4e-4)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_places_do_not_matter(device, dtype):
    announce("masked places", dtype)
    q, k, v = (make(i, dtype, 3, 90, 2, 64) for i in range(3))
    do = make(4, dtype, 3, 90, 2, 64)
    mask = holes(9, 3, 90, "holes")
    mask[1] = False

    def run():
        leaves = [t.to(device).requires_grad_() for t in (q, k, v)]
        out = history_attention(*leaves, mask=mask.to(device), window=30, sinks=2)
        return [out.detach(), *torch.autograd.grad(out, leaves, do.to(device))]

    want = run()
    for value in (math.nan, math.inf, -math.inf):
        q[~mask], k[~mask], v[~mask], do[~mask] = value, value, -value, value
        for a, b in zip(run(), want):
            assert torch.equal(a, b)
    assert not any(t[~mask.to(device)].any() for t in want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-math.inf, "lowest", -1e4])
def test_bias_shuts_distances_out(device, dtype, low):
    announce("low bias", dtype, low)
    low = torch.finfo(dtype).min if low == "lowest" else low
    q, k, v, do = (make(i, dtype, 2, 70, 2, 32) for i in range(4))
    table = make(5, dtype, 8, 2)
    table[3:] = low  # only the three nearest are seen
    leaves = [t.to(device).requires_grad_() for t in (q, k, v, table)]
    out = history_attention(*leaves[:3], bias_table=leaves[3], buckets=RelativeBuckets(8, 24))
    out.backward(do.to(device))
    want = R.attention(q, k, v, None, 3, 0, table[:3].float().new_zeros(8, 2).copy_(table.float().clamp(-1e4)), (8, 24),
                       grad=do)
    for name, g, w in zip(("out", "dq", "dk", "dv", "dtable"), [out.detach()] + [t.grad for t in leaves], want):
        R.close(g, w, dtype, name)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [-1e4, -3e6, -1e10, -1e20, "lowest"])
def test_bias_of_mask_size_everywhere(device, dtype, low):
    """Rows that see only biases meant as masks still answer an average of
    their values: scores are added to the bias in fp32, where a bias of 1e10 or
    more swallows them all (the mean), and one of 1e4 none of 0.01."""

    announce("mask-size bias", dtype, low)
    value = torch.finfo(dtype).min if low == "lowest" else low
    q, k, v = (make(i, dtype, 2, 150, 2, 32, std=3.0 if i < 2 else 1.0) for i in range(3))
    table = torch.full((8, 2), value, dtype=dtype)
    leaves = [t.to(device).requires_grad_() for t in (q, k, v, table)]
    out = history_attention(*leaves[:3], bias_table=leaves[3], buckets=RelativeBuckets(8, 24))
    out.square().sum().backward()
    assert all(torch.isfinite(t.grad).all() for t in leaves)
    got = out.detach().double().cpu()
    span = v.double().abs().cummax(1).values * (1 + 2.0 ** -8)
    assert torch.isfinite(got).all() and (got.abs() <= span).all()
    if low not in (-1e4, -3e6):
        mean = v.double().cumsum(1) / torch.arange(1, 151)[:, None, None]
        R.close(got, mean, dtype)
    elif low == -1e4 and dtype == F32:
        # scores next to 5.7e4 (the bias divided by the scale) are off by 2^-9, the weights by 2^-9 scale
        want = R.attention(q, k, v, None, 0, 0, torch.zeros(8, 2), (8, 24))
        R.close(got, want, dtype, fp32=2.0 ** -9)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("how", ["fused", "offset", "expanded", "heads_first", "grad"])
def test_attention_strides(device, dtype, how):
    announce("strides", dtype, how)
    B, L, H, K, D = 2, 75, 4, 2, 64
    q, k, v = make(0, dtype, B, L, H, D), make(1, dtype, B, L, K, D), make(2, dtype, B, L, K, D)
    do = make(3, dtype, B, L, H, D)
    dq, dk, dv, ddo = (t.to(device) for t in (q, k, v, do))
    if how == "fused":
        whole = torch.cat([dq, dk, dv], 2)
        dq, dk, dv = whole.split([H, K, K], 2)
    elif how == "offset":  # rows that start at an odd element
        dq, dk, dv = (torch.cat([t.new_zeros(B, L, t.size(2), 3), t], -1)[..., 3:] for t in (dq, dk, dv))
    elif how == "expanded":
        k, v = k[:1].expand(B, -1, -1, -1), v[:, :, :1].expand(-1, -1, K, -1)
        dk, dv = dk[:1].expand(B, -1, -1, -1), dv[:, :, :1].expand(-1, -1, K, -1)
    elif how == "heads_first":
        dq, dk, dv = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (dq, dk, dv))
    else:
        do = do[:1, :, :, :1].expand(B, L, H, D)
        ddo = ddo[:1, :, :, :1].expand(B, L, H, D)
    leaves = [t.detach().requires_grad_() for t in (dq, dk, dv)]
    out = history_attention(*leaves, window=20, sinks=2)
    grads = torch.autograd.grad(out, leaves, ddo)
    want = R.attention(q, k, v, None, 20, 2, None, None, grad=do)
    for g, w in zip((out.detach(), *grads), want):
        R.close(g, w, dtype, how)


def test_attention_repeats_itself_and_follows_its_stream(device):
    announce("stream")
    mask = holes(2, 6, 300, "ragged")
    a = run_attention(device, BF16, 6, 300, 300, 4, 2, 64, mask, 100, 4, (32, 128))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = run_attention(device, BF16, 6, 300, 300, 4, 2, 64, mask, 100, 4, (32, 128))
    side.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq,Lk,window,D", [(1, 1, None, 64), (150, 150, 1, 64), (90, 100, 1, 24), (70, 70, 1, 128)])
def test_one_visible_key_gives_no_score_gradient(device, dtype, Lq, Lk, window, D):
    """p is 1 whatever the score: dq, dk and the bias's gradient are 0 to the bit."""

    announce("one key", dtype, Lq, Lk, window, D)
    got = run_attention(device, dtype, 2, Lq, Lk, 4, 2, D, None if Lq == 1 else holes(4, 2, Lk, "holes"), window, 0,
                        (8, 24))
    for g in (got[1], got[2], got[4]):
        assert not g.any()


def test_attention_against_differences(device):
    # fp32: the loss moves by step^2 of its third derivative (about 1e-4 here)
    # and by its own rounding, 1e-6 / step, of a directional derivative of order 10
    announce("differences")
    q, k, v = (make(i, F32, 2, 40, h, 32) for i, h in ((0, 4), (1, 2), (2, 2)))
    table, do = make(3, F32, 8, 4), make(4, F32, 2, 40, 4, 32)
    inputs = [t.to(device) for t in (q, k, v, table)]
    rule = RelativeBuckets(8, 24)

    def loss(ts):
        out = history_attention(*ts[:3], window=12, sinks=2, bias_table=ts[3], buckets=rule)
        return (out.double() * do.to(device).double()).sum()

    leaves = [t.clone().requires_grad_() for t in inputs]
    grads = torch.autograd.grad(loss(leaves), leaves)
    for n in range(4):
        way = make(20 + n, F32, *inputs[n].shape).to(device)
        ends = [float(loss([t + s * way if i == n else t for i, t in enumerate(inputs)])) for s in (1e-2, -1e-2)]
        slope = float((grads[n].double() * way).sum())
        size = float(grads[n].norm() * way.norm())
        assert abs((ends[0] - ends[1]) / 2e-2 - slope) < 1e-2 * size, n


# -------------------------------------------------------------------- step --


def run_steps(device, dtype, lengths, capacity, window, sinks, H, K, D, rule, steps=3, chunk_offset=0):
    announce("step", dtype, lengths, capacity, window, sinks, H, K, D, rule)
    B, top = len(lengths), max(lengths) + steps
    k, v = make(0, dtype, B, top, K, D), make(1, dtype, B, top, K, D)
    q = make(2, dtype, steps, B, H, D)
    table = None if rule is None else make(3, dtype, rule[0], H)
    cache = HistoryCache.empty(B, capacity, K, D, window=window, sinks=sinks, dtype=dtype, device=device)
    if max(lengths):
        cache.write(k[:, :max(lengths)].to(device), v[:, :max(lengths)].to(device), torch.tensor(lengths).to(device))
    for t in range(steps):
        at = torch.tensor(lengths) + t
        row = torch.arange(B)
        got = cache.step(q[t].to(device), k[row, at].to(device), v[row, at].to(device), at.to(device),
                         bias_table=None if table is None else table.to(device),
                         buckets=None if rule is None else RelativeBuckets(*rule))
        want = R.step(q[t], [k[b, : at[b] + 1] for b in range(B)], [v[b, : at[b] + 1] for b in range(B)],
                      window or 0, sinks, table, rule)
        R.close(got, want, dtype, f"step {t}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,K,D", [(1, 1, 1), (4, 1, 24), (8, 2, 64), (6, 2, 33), (16, 1, 128), (12, 1, 80), (20, 1, 32)])
def test_step_heads(device, dtype, H, K, D):
    run_steps(device, dtype, [0, 1, 30, 99], 36, 32, 3, H, K, D, (8, 24))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths,capacity,window,sinks", [([0], 1, 1, 0), ([5], 8, None, 0), ([0, 7, 8], 16, None, 0),
                                                           ([63, 64, 65], 64, 64, 0), ([2, 40], 6, 4, 2),
                                                           ([900, 17], 700, 640, 60), ([3000], 3004, None, 0),
                                                           ([2500], 2304, 2048, 256), ([500, 1], 2000, 100, 7)])
def test_step_lengths(device, dtype, lengths, capacity, window, sinks):
    run_steps(device, dtype, lengths, capacity, window, sinks, 4, 2, 64, (32, 128))
    run_steps(device, dtype, lengths, capacity, window, sinks, 2, 2, 40, None, steps=2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_step_strided_cache_and_inactive_rows(device, dtype):
    announce("strided cache", dtype)
    B, C, K, D, H = 3, 20, 2, 24, 4
    store = torch.full((C, B, 2, K, D + 1), math.nan, dtype=dtype, device=device)
    k, v = store[:, :, 0, :, :D].transpose(0, 1), store[:, :, 1, :, :D].transpose(0, 1)
    cache = HistoryCache(k, v, window=18, sinks=2)
    hk, hv = make(0, dtype, B, 30, K, D), make(1, dtype, B, 30, K, D)
    cache.write(hk[:, :25].to(device), hv[:, :25].to(device), torch.tensor([25, 6, 9]).to(device))
    at = torch.tensor([25, -3, 9])
    before = store.clone()
    q = make(2, dtype, B, H, D)
    row = torch.arange(B)
    got = cache.step(q.to(device), hk[row, at].to(device), hv[row, at].to(device), at.to(device))
    want = R.step(q, [hk[b, : max(at[b] + 1, 1)] for b in range(B)], [hv[b, : max(at[b] + 1, 1)] for b in range(B)],
                  18, 2, None, None)
    want[1] = 0
    R.close(got, want, dtype)
    changed = (store.nan_to_num(7.0) != before.nan_to_num(7.0)).flatten(2).any(-1)  # [C, B]
    slots = [2 + (25 - 2) % 18, 9]
    assert changed.nonzero().tolist() == sorted([[slots[0], 0], [slots[1], 2]])


def test_step_far_into_a_large_cache(device):
    announce("offsets past 32 bits")
    # 34 users of 2^20 slots of 128 values: the last user's rows lie past 2^32 elements
    B, C, K, D, H = 34, 1 << 20, 1, 128, 2
    store = torch.empty(B, C, 1, D, dtype=BF16, device=device)  # 9.1 GB, k and v share it
    cache = HistoryCache(store, torch.empty_like(store), window=None, sinks=0)
    n = 400
    hk, hv = make(0, BF16, B, n + 1, K, D), make(1, BF16, B, n + 1, K, D)
    lengths = torch.full((B,), -1)
    lengths[B - 1] = n
    cache.write(hk[:, :n].to(device), hv[:, :n].to(device), lengths.clamp(min=0).to(device))
    q = make(2, BF16, B, H, D)
    got = cache.step(q.to(device), hk[:, n].to(device), hv[:, n].to(device), lengths.to(device))
    want = R.step(q[-1:], [hk[-1]], [hv[-1]], 0, 0, None, None)
    R.close(got[-1:], want, BF16)
    assert not got[:-1].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("right", [False, True])
@pytest.mark.parametrize("D", [5, 64])
def test_cache_write_places_rows(device, dtype, right, D):
    announce("write", dtype, right, D)
    B, T, K, capacity, sinks = 4, 40, 2, 19, 3
    k, v = make(0, dtype, B, T, K, D), make(1, dtype, B, T, K, D)
    lengths = torch.tensor([0, 7, 22, 40])
    cache = HistoryCache.empty(B, capacity, K, D, window=16, sinks=sinks, dtype=dtype, device=device)
    cache.k.fill_(9.0)
    cache.v.fill_(9.0)
    cache.write(k.to(device), v.to(device), lengths.to(device), right_aligned=right)
    want_k, want_v = torch.full_like(cache.k, 9.0).cpu(), torch.full_like(cache.v, 9.0).cpu()
    for b in range(B):
        n = int(lengths[b])
        for p in range(n):
            slot = p if p < sinks else sinks + (p - sinks) % (capacity - sinks)
            want_k[b, slot], want_v[b, slot] = (t[b, T - n + p if right else p] for t in (k, v))
    assert torch.equal(cache.k.cpu(), want_k) and torch.equal(cache.v.cpu(), want_v)


# -------------------------------------------------------------------- bias --


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_len,k_len,heads", [(1, 1, 1), (1, 700, 3), (33, 65, 2), (130, 130, 5), (300, 517, 4)])
@pytest.mark.parametrize("rule", [(32, 128, False), (8, 24, True), (2, 5, False)])
def test_relative_bias(device, dtype, q_len, k_len, heads, rule):
    announce("bias", dtype, q_len, k_len, heads, rule)
    table = make(0, dtype, rule[0], heads)
    leaf = table.to(device).requires_grad_()
    out = relative_position_bias(leaf, q_len, k_len, RelativeBuckets(*rule))
    column = torch.arange(k_len)
    which = R.bucket(column[k_len - q_len:, None] - column, *rule)
    assert torch.equal(out.detach().cpu(), table.t()[:, which])
    for g in (make(1, dtype, heads, q_len, k_len), make(1, dtype, heads, 1, 1).expand(heads, q_len, k_len),
              make(2, dtype, heads, k_len, q_len).transpose(1, 2)):
        got = torch.autograd.grad(out, leaf, g.to(device), retain_graph=True)[0]
        want = torch.stack([torch.bincount(which.flatten(), g[h].double().flatten(), rule[0]) for h in range(heads)], 1)
        R.close(got, want, dtype)


# -------------------------------------------------------------------- norm --


@pytest.mark.parametrize("dtype,shape", [(d, s) for d in (F32, BF16)
                                         for s in [(1, 1), (3, 7), (2, 5, 64), (130, 96), (1000, 128), (40, 250),
                                                   (17, 512), (9, 1000), (600, 256), (33, 2048), (5, 4096)]]
                         + [(BF16, (3, 8192)), (BF16, (2, 5001)), (F32, (2, 4001))])
def test_norm(device, dtype, shape):
    announce("norm", dtype, shape)
    D = shape[-1]
    x, o, g, dy, dh = (make(i, dtype, *shape) for i in range(5))
    s, wp, wn = (make(5 + i, dtype, D) for i in range(3))
    for gate, scale, post in ((True, True, True), (False, True, False), (True, False, True), (False, False, False)):
        ins = [x, o, g if gate else None, s if scale else None, wp if post else None, wn]
        leaves = [None if t is None else t.to(device).requires_grad_() for t in ins]
        y, h = gated_residual_norm(leaves[0], leaves[1], leaves[4], leaves[5], gate=leaves[2], residual_scale=leaves[3])
        torch.autograd.backward([y, h], [dy.to(device), dh.to(device)])
        want = R.norm(ins[0], ins[1], ins[4], ins[5], ins[2], ins[3], 1e-6, dy, dh)
        got = [y.detach(), h.detach()] + [None if t is None else t.grad for t in leaves]
        for name, a, w in zip(("y", "h", "x", "o", "gate", "scale", "post", "next"), got, want):
            if a is not None:
                R.close(a, w, dtype, name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_parts(device, dtype):
    announce("norm parts", dtype)
    x, o, g, d = (make(i, dtype, 50, 4, 96) for i in range(4))
    wp, wn = make(4, dtype, 96), make(5, dtype, 96)
    dx, do, dg = (t.to(device) for t in (x, o, g))
    # one of the two results used, or an upstream gradient of one value
    for use in ("y", "h", "expanded"):
        leaves = [t.clone().requires_grad_() for t in (dx, do, dg, wp.to(device), wn.to(device))]
        y, h = gated_residual_norm(leaves[0], leaves[1], leaves[3], leaves[4], gate=leaves[2])
        up = d.to(device) if use != "expanded" else torch.ones((), dtype=dtype, device=device).expand(50, 4, 96)
        grads = torch.autograd.grad(y if use == "y" else h, leaves, up, allow_unused=True)
        want = R.norm(x, o, wp, wn, g, None, 1e-6, d if use == "y" else None,
                      None if use == "y" else up.cpu().expand(50, 4, 96))
        for a, w in zip(grads, (want[2], want[3], want[4], want[6], want[7])):
            if a is None:
                assert not w.any()
            else:
                R.close(a, w, dtype, use)
    # strided inputs, no block before the norm, no rows at all
    t = torch.cat([dx, do, dg], -1)
    y, h = gated_residual_norm(t[..., 1:97], t[..., 96:192], wp.to(device), wn.to(device), gate=t[..., 192:])
    ty = t.cpu()
    for a, w in zip((y, h), R.norm(ty[..., 1:97], ty[..., 96:192], wp, wn, ty[..., 192:], None, 1e-6)):
        R.close(a, w, dtype)
    first, h = gated_residual_norm(dx, None, None, wn.to(device))
    assert first is dx
    R.close(h, R.norm(x, None, None, wn, None, None, 1e-6)[1], dtype)
    assert gated_residual_norm(dx[:0], do[:0], None, wn.to(device))[1].shape == (0, 4, 96)


def test_norm_against_differences(device):
    # as for attention: fp32 rounding over the step, and its square
    announce("norm differences")
    ins = [make(i, F32, 30, 128).to(device) for i in range(3)] + [make(3 + i, F32, 128).to(device) for i in range(3)]
    dy, dh = make(8, F32, 30, 128).to(device).double(), make(9, F32, 30, 128).to(device).double()

    def loss(t):
        y, h = gated_residual_norm(t[0], t[1], t[3], t[4], gate=t[2], residual_scale=t[5])
        return (y.double() * dy).sum() + (h.double() * dh).sum()

    leaves = [t.clone().requires_grad_() for t in ins]
    grads = torch.autograd.grad(loss(leaves), leaves)
    for n in range(6):
        way = make(20 + n, F32, *ins[n].shape).to(device)
        ends = [float(loss([t + s * way if i == n else t for i, t in enumerate(ins)])) for s in (1e-2, -1e-2)]
        slope, size = float((grads[n].double() * way).sum()), float(grads[n].norm() * way.norm())
        assert abs((ends[0] - ends[1]) / 2e-2 - slope) < 1e-2 * size, n


# ------------------------------------------------------------------ others --


def test_device_refusals(device):
    announce("refusals")
    q = torch.zeros(1, 4, 2, 136, device=device)
    with pytest.raises(ValueError):
        history_attention(q, q, q)
    a = q[..., :8].contiguous()
    with pytest.raises((ValueError, RuntimeError)):
        history_attention(a, a.cpu(), a)
    with pytest.raises((ValueError, RuntimeError)):
        history_attention(a, a, a, mask=torch.ones(1, 4, dtype=torch.bool))
    with pytest.raises((ValueError, RuntimeError)):
        HistoryCache(a, a).step(a[:, 0], a[:, 0], a[:, 0], torch.tensor([0]))
    with pytest.raises(ValueError):
        wide = torch.zeros(2, 4104, device=device)
        gated_residual_norm(wide, wide, None, wide[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_step_and_norm_in_a_graph(device, dtype):
    announce("graph", dtype)
    B, H, K, D, C = 4, 4, 2, 32, 640
    k0, v0 = (make(i, dtype, B, C, K, D).to(device) for i in (0, 1))
    q, k, v = make(2, dtype, B, H, D).to(device), make(3, dtype, B, K, D).to(device), make(4, dtype, B, K, D).to(device)
    x, w = make(5, dtype, B, H * D).to(device), make(6, dtype, H * D).to(device)
    at = torch.tensor([600, 3, -1, 300], device=device)
    cache = HistoryCache(k0.clone(), v0.clone(), window=600, sinks=8)

    def both(c):
        a = c.step(q, k, v, at)
        return a, gated_residual_norm(x, a.flatten(1), None, w)[1]

    both(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(cache)
    for n in range(4):
        at += 1
        q.copy_(make(30 + n, dtype, B, H, D))
        eager = both(HistoryCache(cache.k.clone(), cache.v.clone(), window=600, sinks=8))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b), n


def test_encoder_on_the_gpu(device):
    announce("encoder")
    host, enc = _encoder(), _encoder().to(device)
    g = torch.Generator().manual_seed(0)
    lengths = torch.tensor([4, 9, 1])
    ids = torch.where(torch.arange(14) < lengths[:, None] + 5, torch.randint(1, 50, (3, 14), generator=g), 0)
    # the same weights on both sides: products and norms of 16 values in fp32
    for a, b in zip(enc.parameters(), host.parameters()):
        assert torch.equal(a.detach().cpu(), b.detach())
    (want, _), (got, mask) = host(ids, lengths + 5), enc(ids.to(device), (lengths + 5).to(device))
    torch.testing.assert_close(got.cpu(), want, rtol=1e-4, atol=1e-4)
    got.square().sum().backward()
    want.square().sum().backward()
    for (name, a), b in zip(enc.named_parameters(), host.parameters()):
        if not a.grad.is_sparse:
            torch.testing.assert_close(a.grad.cpu(), b.grad, rtol=1e-3, atol=1e-3, msg=name)
    caches = enc.caches(3)
    seen = torch.where(torch.arange(14) < lengths[:, None], ids, 0)
    enc.prefill(seen.to(device), lengths.to(device), caches)
    for t in range(5):
        at = lengths + t
        h = enc.step(ids[torch.arange(3), at].to(device), at.to(device), caches)
    torch.testing.assert_close(h, got[:, -1].detach(), rtol=1e-4, atol=1e-4)
