"""The operators over histories on a GPU where callers and limits meet: state
that autograd watches, arguments that disagree, the largest rules, scores that
biases swallow."""

import pytest
import torch

from mdl_amd.embeddings import check_index_errors, index_check_mode, set_index_check_mode
from mdl_amd.history import HistoryCache, RelativeBuckets, history_attention
from tests import history_reference as R
from tests.test_gpu_history import announce, make

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
