"""The operators over histories on a GPU where callers and limits meet: state
that autograd watches, arguments that disagree, the largest rules, scores that
biases swallow."""

import pytest
import torch

from mdl_amd.embeddings import check_index_errors, index_check_mode, set_index_check_mode
from mdl_amd.history import HistoryCache, RelativeBuckets, history_attention
from tests import history_reference as R
from tests.test_gpu_history import announce, holes, make, run_attention, run_steps

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("how", ["step", "write"])
def test_a_cache_written_before_its_backward_raises(device, how):
    """Steps and writes change the cache in place: autograd is told, so that a
    backward over what it held before raises instead of reading the new rows."""

    announce("version", how)
    k, v, q = (make(i, F32, 2, 8, 2, 16).to(device) for i in range(3))
    cache = HistoryCache(k, v, window=4)
    leaf = q.clone().requires_grad_()
    out = history_attention(leaf, cache.k, cache.v)
    before = cache.k._version, cache.v._version
    if how == "step":
        cache.step(q[:, 0], q[:, 1], q[:, 2], torch.tensor([3, 9], device=device))
    else:
        cache.write(q[:, :3], q[:, 3:6], torch.tensor([3, 2], device=device))
    assert cache.k._version > before[0] and cache.v._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_a_cache_of_inference_tensors_takes_steps(device):
    announce("inference cache")
    q = make(0, F32, 2, 4, 2, 16).to(device)
    with torch.inference_mode():
        cache = HistoryCache.empty(2, 8, 2, 16, device=device)
        cache.write(q[:, :3], q[:, 1:], torch.tensor([3, 2], device=device))
    outside = HistoryCache.empty(2, 8, 2, 16, device=device)
    outside.write(q[:, :3], q[:, 1:], torch.tensor([3, 2], device=device))
    at = torch.tensor([3, 2], device=device)
    assert torch.equal(cache.step(q[:, 0], q[:, 1], q[:, 2], at), outside.step(q[:, 0], q[:, 1], q[:, 2], at))
    assert torch.equal(cache.k, outside.k)


def test_a_length_past_the_prompt_is_refused(device):
    # "async", the default, would trap the device: only lengths that pass are written under it
    announce("long lengths")
    k = make(0, F32, 2, 5, 2, 16).to(device)
    cache = HistoryCache.empty(2, 16, 2, 16, device=device)
    good, bad = torch.tensor([5, -1], device=device), torch.tensor([5, 6], device=device)
    mode = index_check_mode()
    try:
        set_index_check_mode("sync")
        with pytest.raises(ValueError, match="5 rows"):
            cache.write(k, k, bad)
        assert not cache.k.any()
        cache.write(k, k, good)
        set_index_check_mode("deferred")
        cache.write(k, k, good)
        check_index_errors()
        cache.write(k, k, bad)
        with pytest.raises(IndexError, match="^1 .*history prompts"):
            check_index_errors()
        set_index_check_mode("async")
        cache.write(k, k, good)
        torch.cuda.synchronize()
    finally:
        set_index_check_mode(mode)
    assert torch.equal(cache.k[0, :5], k[0])


def _raw(device, dtype, starts, distances, D=32, H=8):
    """Outputs and gradients of the operators themselves, whose starts and
    number of distances are separate arguments."""

    q, k, v = (make(i, dtype, 2, 90, h, D).to(device) for i, h in ((0, H), (1, 1), (2, 1)))
    table = make(3, dtype, len(starts) + 1, H).to(device)
    starts = torch.tensor(starts, dtype=torch.int32, device=device)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = torch.ops.mdl_hip.history_attention(*leaves[:3], None, table, starts, distances, 20, 3, 0.2)
    got = [out.detach(), *torch.autograd.grad(out.float().square().sum(), leaves)]
    with torch.no_grad():
        cache = HistoryCache.empty(2, 128, 1, D, dtype=dtype, device=device)
        cache.write(k, v, torch.tensor([90, 60], device=device))
        got.append(torch.ops.mdl_hip.history_cache_step(
            q[:, 0], k[:, 0], v[:, 0], cache.k, cache.v, torch.tensor([90, 60], device=device), table, starts, distances,
            100, 0, 0.2))
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_starts_past_the_distances_stay_in_bounds(device, dtype):
    """Starts that do not fit the distances told apart make no promise for the
    bias, but nothing outside the kernels' sums and buckets is touched: what
    runs after them is as if they had not."""

    announce("starts past distances", dtype)
    rule = list(RelativeBuckets(8, 24).starts)
    want = _raw(device, dtype, rule, rule[-1] + 1)
    for starts, distances in (([5, 300, 2000, 30000, 2**31 - 1, 2**31 - 1, 2**31 - 1], 3), (rule, 1),
                              ([-2**31, -40000, -7, 0, 1, 2, 3], 4)):
        for t in _raw(device, dtype, starts, distances):
            assert torch.isfinite(t).all(), (starts, distances)
    for a, b in zip(_raw(device, dtype, rule, rule[-1] + 1), want):
        assert torch.equal(a, b)


# the most buckets and distances that an attention takes: 1024 of them, the last from 2048 on
LARGEST = RelativeBuckets(1024, 2053)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_attention_with_the_largest_rule(device, monkeypatch, dtype, D):
    """The keys' and the far part's kernels at the most LDS that they take."""

    assert LARGEST.starts[-1] == 2048
    monkeypatch.setattr(R, "bucket", lambda distance, *_: LARGEST.of(distance))
    run_attention(device, dtype, 1, 2200, 2200, 2, 1, D, None, 700, 40, (1024, 2053))
    run_attention(device, dtype, 1, 300, 2200, 2, 2, D, holes(4, 1, 2200, "holes"), None, 0, (1024, 2053))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("max_distance", [798, 804, 806, 807, 810])
def test_attention_around_64_kb_of_lds(device, monkeypatch, dtype, max_distance):
    # rules of 660 to 680 distances at head dimension 32: the far part's LDS passes 64 KB among them
    rule = RelativeBuckets(40, max_distance)
    monkeypatch.setattr(R, "bucket", lambda distance, *_: rule.of(distance))
    run_attention(device, dtype, 1, 800, 800, 1, 1, 32, None, 200, 5, (40, max_distance))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("H,D", [(8, 128), (8, 64), (2, 128), (12, 128)])
@pytest.mark.parametrize("B", [1, 300])
def test_step_with_the_largest_rule(device, monkeypatch, dtype, H, D, B):
    monkeypatch.setattr(R, "bucket", lambda distance, *_: LARGEST.of(distance))
    lengths = [2250] if B == 1 else [3 * (i % 20) for i in range(B)]
    run_steps(device, dtype, lengths, 2304 if B == 1 else 64, None, 0, H, 1, D, (1024, 2053), steps=1)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_more_users_than_a_grid_is_high(device, dtype):
    """A write takes the batches that a step takes: 70,000 rows, of two blocks each."""

    announce("many users", dtype)
    B, L, D = 70000, 66, 4
    k = torch.arange(B * L, dtype=torch.float32).remainder(251).reshape(B, L, 1, 1).expand(B, L, 1, D).to(dtype).to(device)
    lengths = torch.arange(B, device=device) % (L + 1)
    cache = HistoryCache.empty(B, L + 1, 1, D, dtype=dtype, device=device)
    cache.write(k, -k, lengths, right_aligned=True)
    column = torch.arange(L, device=device)
    rows = (column + L - lengths[:, None]).clamp(max=L - 1)
    want = torch.where((column < lengths[:, None])[..., None], k[:, :, 0].gather(1, rows[..., None].expand(B, L, D)), 0.0)
    assert torch.equal(cache.k[:, :L, 0], want.to(dtype)) and torch.equal(cache.v, -cache.k)
    one = torch.ones(B, 1, D, dtype=dtype, device=device)
    assert cache.step(one, one, one, lengths).shape == (B, 1, D)


@pytest.mark.parametrize("name", ["attention", "attention_forward", "step", "write", "bias", "norm"])
def test_opcheck(device, name):
    announce("opcheck", name)
    ops = torch.ops.mdl_hip
    grad = name not in ("step", "write", "attention_forward")
    q, k, v = (make(i, F32, 2, 9, h, 8).to(device).requires_grad_(grad) for i, h in ((0, 4), (1, 2), (2, 2)))
    table = make(3, F32, 6, 4).to(device).requires_grad_(grad)
    rule = RelativeBuckets(6, 8)
    starts, mask = rule.starts_on(q.device), holes(1, 2, 9, "holes").to(device)
    bias = (table, starts, rule.distances)
    if name == "attention":
        torch.library.opcheck(ops.history_attention.default, (q, k, v, mask, *bias, 3, 1, 0.5))
    elif name == "attention_forward":
        # its third result is the call's prepared buffer, whose padding holds anything: values are not compared
        torch.library.opcheck(ops.history_attention_forward.default, (q, k, v, mask, *bias, 3, 1, 0.5, True),
                              test_utils=("test_schema", "test_faketensor"))
    elif name == "step":
        torch.library.opcheck(ops.history_cache_step.default,
                              (q[:, 0], k[:, 0], v[:, 0], k.clone(), v.clone(), torch.tensor([1, 5], device=device), *bias,
                               3, 1, 0.5), test_utils=("test_schema", "test_faketensor"))
    elif name == "write":
        torch.library.opcheck(ops.history_cache_write_.default,
                              (k, v, k.clone(), v.clone(), torch.tensor([2, 9], device=device), 1, True),
                              test_utils=("test_schema", "test_faketensor"))
    elif name == "bias":
        torch.library.opcheck(ops.relative_position_bias.default, (table, starts, False, 4, 9))
    else:
        x, o, gate = (make(i, F32, 3, 8).to(device).requires_grad_() for i in range(3))
        w = [make(4 + i, F32, 8).to(device).requires_grad_() for i in range(3)]
        torch.library.opcheck(ops.gated_residual_norm.default, (x, o, w[0], w[1], gate, w[2], 1e-6))


def test_a_rule_first_compiled_under_inference_trains(device):
    announce("compiled rule")
    rule = RelativeBuckets(6, 8)

    def attend(q, table):
        return history_attention(q, q[:, :, :2], q[:, :, 2:], window=3, bias_table=table, buckets=rule)

    compiled = torch.compile(attend, backend="aot_eager", fullgraph=True)
    q, table = make(0, F32, 2, 5, 4, 8).to(device), make(1, F32, 6, 4).to(device)
    with torch.inference_mode():
        first = compiled(q, table)
    leaves = [t.clone().requires_grad_() for t in (q, table)]
    for call in (attend, compiled):
        out = call(*leaves)
        assert torch.equal(out, first)
        grads = torch.autograd.grad(out.square().sum(), leaves)
        assert all(torch.isfinite(g).all() and g.any() for g in grads)
