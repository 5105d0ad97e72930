"""The cache of histories on the CPU: what its steps leave behind and what its
writes refuse."""

import pytest
import torch

from mdl_amd.history import HistoryCache
from tests.test_history import _encoder


def rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape)))


def test_steps_and_writes_record_nothing():
    """Nothing of a cache is differentiable, with parameters upstream too: no
    graph hangs on it, and none grows from step to step."""

    cache = HistoryCache.empty(2, 8, 2, 4)
    q, k, v = (rand(2, 3, 2, 4).requires_grad_() for _ in range(3))
    cache.write(k, v, torch.tensor([2, 3]))
    for t in range(2):
        out = cache.step(q[:, t], k[:, t], v[:, t], torch.tensor([2 + t, 3 + t]))
        for x in (out, cache.k, cache.v):
            assert not x.requires_grad and x.grad_fn is None
    held = cache.k.clone()
    before = cache.k._version
    cache.step(q[:, 0], k[:, 0], v[:, 0], torch.tensor([5, 6]))
    assert cache.k._version > before  # autograd still learns of the change
    with torch.no_grad():
        other = HistoryCache(held, torch.zeros_like(held))
        other.step(q[:, 0], k[:, 0], v[:, 0], torch.tensor([5, 6]))
    assert torch.equal(other.k, cache.k)


def test_blocks_step_without_no_grad():
    enc = _encoder()
    caches = enc.caches(2)
    x = rand(2, 16)
    for t in range(3):
        for block, cache in zip(enc.blocks, caches):
            block.step(x, x, torch.tensor([t, t]), cache)
            assert cache.k.grad_fn is None and cache.v.grad_fn is None


@pytest.mark.parametrize("right", [False, True])
def test_a_length_past_the_prompt_is_refused(right):
    """Nothing is stored: a step at the true length would answer from rows that
    were never written."""

    cache = HistoryCache.empty(3, 16, 2, 4)
    k, v = rand(3, 5, 2, 4), rand(3, 5, 2, 4)
    with pytest.raises(ValueError, match="5 rows"):
        cache.write(k, v, torch.tensor([2, 6, 1]), right_aligned=right)
    assert not cache.k.any() and not cache.v.any()
    cache.write(k, v, torch.tensor([5, 0, -2]), right_aligned=right)
    assert cache.k[0, :5].ne(0).all() and not cache.k[1:].any()


def test_prefill_refuses_lengths_past_its_columns():
    enc = _encoder()
    with pytest.raises(ValueError, match="9 rows"):
        enc.prefill(torch.ones(2, 9, dtype=torch.long), torch.tensor([4, 11]), enc.caches(2))
