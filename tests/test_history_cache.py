"""The cache of histories on the CPU: what its steps leave behind."""

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
