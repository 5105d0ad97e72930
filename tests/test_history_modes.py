"""A bucket rule used under one mode (inference, fake tensors, functional
transforms, compilation) serves every other one afterwards."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mdl_amd.history import RelativeBuckets, history_attention, relative_position_bias
from tests.test_history import _encoder


def rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape)))


def attend(rule, q, table):
    return history_attention(q, q[:, :, :2], q[:, :, 2:], window=3, bias_table=table, buckets=rule)


def train(rule):
    """A training pass with the rule, as a fresh rule of the same distances gives it."""

    results = []
    for r in (rule, RelativeBuckets(6, 8)):
        q, table = rand(2, 5, 4, 3).requires_grad_(), rand(6, 4).requires_grad_()
        loss = attend(r, q, table).square().sum() + relative_position_bias(table, 4, 5, r).square().sum()
        loss.backward()
        results.append((loss.detach(), q.grad, table.grad))
    for a, b in zip(*results):
        assert type(a) is torch.Tensor and torch.equal(a, b)


def test_a_rule_first_used_in_inference_mode_trains():
    rule = RelativeBuckets(6, 8)
    with torch.inference_mode():
        attend(rule, rand(2, 5, 4, 3), rand(6, 4))
        relative_position_bias(rand(6, 4), 4, 5, rule)
    train(rule)
    with torch.inference_mode():
        attend(rule, rand(2, 5, 4, 3), rand(6, 4))
    train(rule)


def test_a_rule_first_used_on_fake_tensors_works_on_real_ones():
    rule = RelativeBuckets(6, 8)
    for _ in range(2):  # before and after the rule holds a real tensor
        with FakeTensorMode():
            out = attend(rule, torch.randn(2, 5, 4, 3), torch.randn(6, 4))
            assert out.shape == (2, 5, 4, 3)
            assert relative_position_bias(torch.randn(6, 4), 4, 5, rule).shape == (4, 4, 5)
        train(rule)


@pytest.mark.parametrize("transform", ["jvp", "grad", "vmap", "functionalize"])
def test_a_rule_first_used_under_a_transform_works_outside(transform):
    rule = RelativeBuckets(6, 8)
    table = rand(6, 4)
    call = lambda t: relative_position_bias(t, 4, 5, rule).sum()  # noqa: E731
    try:
        if transform == "jvp":
            torch.func.jvp(call, (table,), (table,))
        elif transform == "grad":
            torch.func.grad(call)(table)
        elif transform == "vmap":
            torch.func.vmap(call)(table[None])
        else:
            torch.func.functionalize(call)(table)
    except RuntimeError:
        pass  # what the transform makes of the operator does not matter here
    train(rule)


def test_a_rule_first_used_in_a_compiled_function_works_outside():
    rule = RelativeBuckets(6, 8)
    compiled = torch.compile(lambda q, t: attend(rule, q, t), backend="aot_eager", fullgraph=True)
    for inference in (True, False, False):
        q, table = rand(2, 5, 4, 3), rand(6, 4)
        with torch.inference_mode(inference):
            compiled(q, table)
        # the graph holds the kept tensor and makes none of its own
        kept = rule._on_device[q.device]
        assert type(kept) is torch.Tensor and not kept.is_inference() and kept.tolist() == list(rule.starts)
        torch.testing.assert_close(compiled(q, table), attend(RelativeBuckets(6, 8), q, table))
        train(rule)


def test_an_encoder_that_answered_first_trains_afterwards():
    enc, other = _encoder(), _encoder()
    ids, lengths = torch.randint(1, 50, (3, 9), generator=torch.Generator().manual_seed(1)), torch.tensor([4, 9, 1])
    ids = torch.where(torch.arange(9) < lengths[:, None], ids, 0)
    with torch.inference_mode():
        caches = enc.caches(3)
        enc.prefill(ids, lengths, caches)
        enc.step(ids[:, 0], lengths, caches)
        enc(ids, lengths)
    for e in (enc, other):
        e(ids, lengths)[0].sum().backward()
    for a, b in zip(enc.parameters(), other.parameters()):
        assert torch.equal(a.grad.to_dense(), b.grad.to_dense())


def test_the_deferred_counter_first_used_in_inference_mode_counts_outside(monkeypatch):
    """Lookups and prompt writes of an evaluation make it; a later step outside
    inference mode adds to it and resets it."""

    from mdl_amd import embeddings

    monkeypatch.setattr(embeddings, "_DEFERRED_COUNTERS", {})
    with torch.inference_mode():
        embeddings._deferred_counter(torch.device("cpu")).add_(1)
    embeddings._deferred_counter(torch.device("cpu")).add_(1)
    with pytest.raises(IndexError, match="^2 "):
        embeddings.check_index_errors()
    embeddings.check_index_errors()
