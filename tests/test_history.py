"""Operators over histories without a GPU: their CPU kernels against plain
64-bit forms, gradients against differences, refusals, schemas and the C ABI's
checks."""

import math
import re
import subprocess

import numpy as np
import pytest
import torch
from torch.library import opcheck

from mdl_amd import _lib
from mdl_amd.block_norm import gated_residual_norm
from mdl_amd.embeddings import EmbeddingShardSpec, ShardedEmbedding
from mdl_amd.history import HistoryCache, RelativeBuckets, history_attention, relative_position_bias
from mdl_amd.history_encoder import HistoryEncoder
from tests import history_reference as R
from tests.conftest import ROOT

OPS = torch.ops.mdl_hip
HEADER = ROOT / "include" / "mdl_hip.h"


@pytest.mark.parametrize("count,max_distance,two", [(32, 128, False), (8, 24, False), (2, 5, False), (30, 31, False),
                                                    (64, 1024, False), (32, 128, True), (4, 9, True)])
def test_buckets_follow_their_definition(count, max_distance, two):
    d = torch.arange(-300, 2100, 7)
    assert torch.equal(RelativeBuckets(count, max_distance, two).of(d), R.bucket(d, count, max_distance, two))


def _inputs(dtype, B=2, Lq=7, Lk=9, H=4, K=2, D=6, buckets=(6, 8), seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).to(dtype)  # noqa: E731
    mask = torch.rand(B, Lk, generator=g) < 0.8
    mask[0, :3] = False
    return r(B, Lq, H, D), r(B, Lk, K, D), r(B, Lk, K, D), r(B, Lq, H, D), mask, r(buckets[0], H), buckets


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (3, 0), (3, 2), (1, 0), (2, 50)])
def test_attention_cpu(dtype, window, sinks):
    q, k, v, do, mask, table, rule = _inputs(dtype)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    out = history_attention(*leaves[:3], mask=mask, window=window, sinks=sinks, bias_table=leaves[3],
                            buckets=RelativeBuckets(*rule))
    out.backward(do)
    want = R.attention(q, k, v, mask, window or 0, sinks, table, rule, grad=do)
    for name, got, w in zip(("out", "dq", "dk", "dv", "dtable"), [out.detach()] + [t.grad for t in leaves], want):
        assert got.dtype == dtype
        R.close(got, w, dtype, name)


def test_reference_gradients_against_differences():
    """The formulas the tests compare with: central differences of the 64-bit
    forms (step 1e-5: off by 1e-10 of the third derivative and 1e-11 / 1e-5 of
    the value)."""

    q, k, v, do, mask, table, rule = [t.double() if torch.is_tensor(t) and t.is_floating_point() else t
                                      for t in _inputs(torch.float32, B=1, Lq=4, Lk=5, H=2, K=1, D=3)]
    grads = R.attention(q, k, v, mask, 2, 1, table, rule, grad=do)[1:]
    inputs = [q, k, v, table]
    for n, g in enumerate(grads):
        for at in np.ndindex(*inputs[n].shape):
            vals = []
            for s in (1e-5, -1e-5):
                moved = [t.clone() for t in inputs]
                moved[n][at] += s
                vals.append(float((R.attention(*moved[:3], mask, 2, 1, moved[3], rule) * do).sum()))
            assert abs((vals[0] - vals[1]) / 2e-5 - float(g[at])) < 1e-6
    torch.manual_seed(1)
    args = [torch.randn(3, 5, dtype=torch.float64) for _ in range(2)]
    wp, wn, sc = (torch.rand(5, dtype=torch.float64) + 0.5 for _ in range(3))
    gate, dy, dh = (torch.randn(3, 5, dtype=torch.float64) for _ in range(3))
    all_in = [args[0], args[1], gate, sc, wp, wn]
    form = lambda t: R.norm(t[0], t[1], t[4], t[5], t[2], t[3], 1e-6)  # noqa: E731
    got = R.norm(args[0], args[1], wp, wn, gate, sc, 1e-6, dy, dh)[2:]
    for n, g in enumerate(got):
        for at in np.ndindex(*all_in[n].shape):
            vals = []
            for s in (1e-5, -1e-5):
                moved = [t.clone() for t in all_in]
                moved[n][at] += s
                y, h = form(moved)
                vals.append(float((y * dy).sum() + (h * dh).sum()))
            assert abs((vals[0] - vals[1]) / 2e-5 - float(g[at])) < 1e-6, n


def test_what_is_masked_does_not_matter():
    q, k, v, do, mask, table, rule = _inputs(torch.float32, Lq=9)
    want = history_attention(q, k, v, mask=mask, window=4, sinks=1)
    q[~mask], k[~mask], v[~mask] = math.nan, math.inf, math.nan
    assert torch.equal(history_attention(q, k, v, mask=mask, window=4, sinks=1), want)
    assert not want[~mask].any()
    none = torch.zeros_like(mask)
    assert not history_attention(q, k, v, mask=none).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("capacity,window,sinks", [(12, None, 0), (7, 5, 2), (6, 4, 1)])
def test_cache_steps_are_the_whole_attention(dtype, capacity, window, sinks):
    q, k, v, _, _, table, rule = _inputs(dtype, Lq=12, Lk=12)
    start = torch.tensor([3, 5])
    cache = HistoryCache.empty(2, capacity, 2, 6, window=window, sinks=sinks, dtype=dtype)
    aligned = torch.stack([torch.cat([k[b, 12 - 5:12 - 5 + 5 - s], k[b, :s]]) for b, s in enumerate((3, 5))])
    aligned_v = torch.stack([torch.cat([v[b, 12 - 5:12 - 5 + 5 - s], v[b, :s]]) for b, s in enumerate((3, 5))])
    cache.write(aligned, aligned_v, start, right_aligned=True)
    for t in range(6):
        at = start + t
        row = torch.arange(2)
        got = cache.step(q[row, at], k[row, at], v[row, at], at, bias_table=table, buckets=RelativeBuckets(*rule))
        want = R.step(q[row, at], [k[b, : at[b] + 1] for b in range(2)], [v[b, : at[b] + 1] for b in range(2)],
                      window or 0, sinks, table, rule)
        R.close(got, want, dtype)
    before = cache.k.clone()
    assert not cache.step(q[:, 0], k[:, 0], v[:, 0], torch.tensor([-1, -1])).any()
    assert torch.equal(cache.k, before)


@pytest.mark.parametrize("two", [False, True])
def test_relative_bias_cpu(two):
    table = torch.randn(8, 3, requires_grad=True)
    rule = RelativeBuckets(8, 20, two)
    out = relative_position_bias(table, 5, 30, rule)
    column = torch.arange(30)
    which = R.bucket(column[25:, None] - column, 8, 20, two)
    assert torch.equal(out, table.detach().t()[:, which])
    g = torch.randn(3, 5, 30)
    out.backward(g)
    want = torch.stack([torch.bincount(which.flatten(), g[h].double().flatten(), 8) for h in range(3)], 1)
    R.close(table.grad, want, torch.float32)


@pytest.mark.parametrize("gate,scale,post", [(True, True, True), (False, False, False), (True, False, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_cpu(dtype, gate, scale, post):
    torch.manual_seed(2)
    r = lambda *s: torch.randn(*s).to(dtype).requires_grad_()  # noqa: E731
    x, o, wn = r(4, 3, 10), r(4, 3, 10), r(10)
    g, s, wp = r(4, 3, 10) if gate else None, r(10) if scale else None, r(10) if post else None
    dy, dh = torch.randn(4, 3, 10).to(dtype), torch.randn(4, 3, 10).to(dtype)
    y, h = gated_residual_norm(x, o, wp, wn, gate=g, residual_scale=s)
    torch.autograd.backward([y, h], [dy, dh])
    want = R.norm(*[None if t is None else t.detach() for t in (x, o, wp, wn, g, s)], 1e-6, dy, dh)
    for name, got, w in zip(("y", "h", "x", "o", "gate", "scale", "post", "next"),
                            (y.detach(), h.detach()) + tuple(None if t is None else t.grad for t in (x, o, g, s, wp, wn)),
                            want):
        if got is not None:
            R.close(got, w, dtype, name)


def test_first_norm_passes_the_stream_through():
    x, w = torch.randn(3, 4, requires_grad=True), torch.rand(4, requires_grad=True)
    y, h = gated_residual_norm(x, None, None, w)
    assert y is x
    h.sum().backward()
    R.close(x.grad, R.norm(x.detach(), None, None, w.detach(), None, None, 1e-6, None, torch.ones(3, 4))[2],
            torch.float32)


@pytest.mark.parametrize("name", ["attention", "attention_forward", "step", "write", "bias", "norm"])
def test_opcheck_cpu(name):
    q, k, v, _, mask, table, rule = _inputs(torch.float32)
    r = RelativeBuckets(*rule)
    starts = r.starts_on(q.device)
    if name.startswith("attention"):
        grad = name == "attention"
        leaves = [t.requires_grad_(grad) for t in (q, k, v, table)]
        args = (*leaves[:3], mask, leaves[3], starts, r.distances, 3, 1, 0.5)
        if grad:
            opcheck(OPS.history_attention.default, args)
        else:
            opcheck(OPS.history_attention_forward.default, (*args, True))
    elif name == "step":
        opcheck(OPS.history_cache_step.default,
                (q[:, 0], k[:, 0], v[:, 0], k.clone(), v.clone(), torch.tensor([1, 5]), table, starts, r.distances, 3,
                 1, 0.5), test_utils=("test_schema", "test_faketensor"))
    elif name == "write":
        opcheck(OPS.history_cache_write_.default, (k, v, k.clone(), v.clone(), torch.tensor([2, 9]), 1, True),
                test_utils=("test_schema", "test_faketensor"))
    elif name == "bias":
        opcheck(OPS.relative_position_bias.default, (table.requires_grad_(), starts, False, 4, 9))
    else:
        x, o, g = (torch.randn(3, 8, requires_grad=True) for _ in range(3))
        w = [torch.rand(8, requires_grad=True) for _ in range(3)]
        opcheck(OPS.gated_residual_norm.default, (x, o, w[0], w[1], g, w[2], 1e-6))


def test_refusals():
    q, k, v, do, mask, table, rule = _inputs(torch.float32)
    r = RelativeBuckets(*rule)
    bad = [
        (ValueError, lambda: history_attention(q[0], k, v)),
        (ValueError, lambda: history_attention(q, k[:1], v[:1])),
        (ValueError, lambda: history_attention(k, q[:, :, :1], q[:, :, :1])),  # more queries than keys
        (ValueError, lambda: history_attention(q[:, :, :3], k, v)),
        (TypeError, lambda: history_attention(q, k.bfloat16(), v)),
        (TypeError, lambda: history_attention(q.double(), k.double(), v.double())),
        (ValueError, lambda: history_attention(q, k, v, window=0)),
        (ValueError, lambda: history_attention(q, k, v, sinks=-1)),
        (ValueError, lambda: history_attention(q, k, v, scale=-1.0)),
        (ValueError, lambda: history_attention(q, k, v, scale=math.nan)),
        (TypeError, lambda: history_attention(q, k, v, mask=mask.int())),
        (ValueError, lambda: history_attention(q, k, v, mask=mask[:, :4])),
        (ValueError, lambda: history_attention(q, k, v, bias_table=table)),
        (ValueError, lambda: history_attention(q, k, v, buckets=r)),
        (ValueError, lambda: history_attention(q, k, v, bias_table=table[:3], buckets=r)),
        (ValueError, lambda: history_attention(q, k, v, bias_table=table[:, :3], buckets=r)),
        (ValueError, lambda: history_attention(q, k, v, bias_table=table, buckets=RelativeBuckets(6, 9, True))),
        (ValueError, lambda: history_attention(q, k, v, bias_table=table, buckets=RelativeBuckets(6, 10**6))),
        (ValueError, lambda: RelativeBuckets(1, 5)),
        (ValueError, lambda: RelativeBuckets(9, 5, True)),
        (ValueError, lambda: RelativeBuckets(8, 4)),
        (ValueError, lambda: RelativeBuckets(2048, 9000)),
        (ValueError, lambda: HistoryCache.empty(1, 4, 1, 8, window=4, sinks=1)),
        (ValueError, lambda: HistoryCache.empty(1, 2, 1, 8, sinks=2)),
        (TypeError, lambda: HistoryCache(k, v.bfloat16())),
        (TypeError, lambda: HistoryCache(k, v).step(q[:, 0], k[:, 0], v[:, 0], torch.tensor([1, 2]).int())),
        (ValueError, lambda: HistoryCache(k, v).step(q[:, 0], k[:, 0], v[:, 0], torch.tensor([1]))),
        (ValueError, lambda: HistoryCache(k, v).step(q[:, 0], k[:, 0, :1], v[:, 0, :1], torch.tensor([1, 2]))),
        (ValueError, lambda: HistoryCache(k, v).write(k[:, :, :1], v[:, :, :1], torch.tensor([1, 2]))),
        (ValueError, lambda: relative_position_bias(table, 9, 4, r)),
        (ValueError, lambda: relative_position_bias(table[:3], 4, 9, r)),
        (ValueError, lambda: gated_residual_norm(q, q[:1], None, torch.ones(6))),
        (ValueError, lambda: gated_residual_norm(q, q, None, torch.ones(5))),
        (ValueError, lambda: gated_residual_norm(q, None, None, torch.ones(6), gate=q)),
        (TypeError, lambda: gated_residual_norm(q, q.bfloat16(), None, torch.ones(6))),
        (TypeError, lambda: gated_residual_norm(q, q, torch.ones(6).bfloat16(), torch.ones(6))),
        (ValueError, lambda: gated_residual_norm(q, q, None, torch.ones(6), eps=-1.0)),
    ]
    for n, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            pytest.fail(f"call {n} was taken")


def _encoder(dtype=torch.float32, device="cpu", depth=2, window=5, sinks=2):
    torch.manual_seed(5)
    spec = EmbeddingShardSpec(table_name="events", strategy="table_wise", world_size=1, table_owner=0)
    events = ShardedEmbedding(50, 16, table_name="events", shard_spec=spec, dtype=dtype, init_std=1.0)
    enc = HistoryEncoder(events, depth, 4, kv_heads=2, head_dim=8, window=window, sinks=sinks,
                         buckets=RelativeBuckets(6, 8)).to(device)
    with torch.no_grad():
        for block in enc.blocks:
            block.bias_table.normal_()
    return enc


def test_encoder_steps_are_the_whole_history():
    enc = _encoder()
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(1, 50, (3, 14), generator=g)
    lengths = torch.tensor([4, 9, 1])
    caches = enc.caches(3)
    col = torch.arange(14)
    h = enc.prefill(torch.where(col < lengths[:, None], ids, 0), lengths, caches)
    whole, mask = enc(torch.where(col < lengths[:, None], ids, 0), lengths)
    torch.testing.assert_close(h[mask], whole[mask].detach())
    for t in range(5):
        at = lengths + t
        h = enc.step(ids[torch.arange(3), at], at, caches)
        whole, _ = enc(torch.where(col < at[:, None] + 1, ids, 0), at + 1)
        torch.testing.assert_close(h, whole[:, -1].detach(), rtol=1e-4, atol=1e-5)


def test_encoder_trains_its_table_and_its_blocks():
    from mdl_amd.optim import ShardedRowWiseAdagrad

    enc = _encoder()
    dense = [p for n, p in enc.named_parameters() if not n.startswith("events")]
    sparse = ShardedRowWiseAdagrad([enc.events.weight], lr=0.3)
    opt = torch.optim.SGD(dense, lr=0.05)
    ids, lengths = torch.randint(1, 50, (8, 12)), torch.randint(1, 13, (8,))
    ids = torch.where(torch.arange(12) < lengths[:, None], ids, 0)
    target = torch.randn(8, 16)
    losses = []
    for _ in range(12):
        h, _ = enc(ids, lengths)
        loss = (h[:, -1] - target).square().mean()
        loss.backward()
        assert all(p.grad is not None for p in dense)
        sparse.step()
        opt.step()
        sparse.zero_grad(set_to_none=True)
        opt.zero_grad(set_to_none=True)
        losses.append(float(loss))
    assert losses[-1] < 0.7 * losses[0]


# ----------------------------------------------------------------- C ABI --


def test_struct_layouts_match_header(tmp_path):
    fields = {"mdl_attention": _lib.ATTENTION_DTYPE, "mdl_attention_grads": _lib.ATTENTION_GRADS_DTYPE,
              "mdl_attention_step": _lib.ATTENTION_STEP_DTYPE, "mdl_block_norm": _lib.BLOCK_NORM_DTYPE,
              "mdl_block_norm_grads": _lib.BLOCK_NORM_GRADS_DTYPE}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){"]
    for st, dt in fields.items():
        lines.append(f'printf("{st} size %zu\\n", sizeof({st}));')
        lines += [f'printf("{st} {n} %zu\\n", offsetof({st}, {n}));' for n in dt.names]
    probe = tmp_path / "probe.c"
    probe.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", str(probe), "-o", str(tmp_path / "probe")], check=True)
    got = {}
    for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split("\n"):
        if line:
            st, name, value = line.split()
            got[st, name] = int(value)
    for st, dt in fields.items():
        assert got[st, "size"] == dt.itemsize
        assert all(got[st, n] == dt.fields[n][1] for n in dt.names)
    assert re.search(r"mdl_attention_forward", HEADER.read_text())


def test_bad_descriptors_fail_before_any_launch():
    lib = _lib.lib()
    good = np.zeros(1, dtype=_lib.ATTENTION_DTYPE)
    good[0]["batch"], good[0]["q_len"], good[0]["k_len"] = 1, 4, 4
    good[0]["q_heads"], good[0]["kv_heads"], good[0]["head_dim"], good[0]["scale"] = 4, 2, 8, 0.5
    for name in ("q", "k", "v"):
        good[0][name] = 4096  # never dereferenced

    def forward(**changes):
        a = good.copy()
        for name, value in changes.items():
            a[0][name] = value
        return lib.mdl_attention_forward(a.ctypes.data, None, 4096, None, None), lib.mdl_last_error()

    assert lib.mdl_attention_forward(None, None, None, None, None) == -1
    for changes, code in (({"q_len": 5}, -1), ({"q_heads": 3}, -1), ({"head_dim": 129}, -4), ({"dtype": 7}, -1),
                          ({"scale": 0.0}, -1), ({"scale": np.nan}, -1), ({"sinks": -1}, -1), ({"q": 0}, -1),
                          ({"mask": 4096}, -1),
                          ({"bias_table": 4096, "num_buckets": 4, "distances": 9}, -1),
                          ({"bias_table": 4096, "bucket_starts": 4096, "num_buckets": 4, "distances": 4000}, -4)):
        assert forward(**changes)[0] == code, changes
    assert forward(batch=0)[0] == 0
    assert lib.mdl_attention_backward(good.ctypes.data, None, None, None, 0, None) == -1
    step = np.zeros(1, dtype=_lib.ATTENTION_STEP_DTYPE)
    step[0]["batch"], step[0]["capacity"], step[0]["sinks"] = 1, 4, 4
    assert lib.mdl_attention_step_forward(step.ctypes.data, None, None, 0, None) == -1
    assert b"capacity" in lib.mdl_last_error()
    assert lib.mdl_relative_bias(None, None, 4, 0, 2, 3, 2, 0, None, None) == -1
    assert lib.mdl_relative_bias_grad(4096, 4096, 4, 0, 2, 3, 3, 0, 4096, None, 0, None) == -3
    norm = np.zeros(1, dtype=_lib.BLOCK_NORM_DTYPE)
    norm[0]["rows"], norm[0]["dim"] = 2, 9000
    assert lib.mdl_block_norm_forward(norm.ctypes.data, None, None, None) == -4
    norm[0]["dim"], norm[0]["gate"] = 8, 4096
    assert lib.mdl_block_norm_forward(norm.ctypes.data, None, None, None) == -1
