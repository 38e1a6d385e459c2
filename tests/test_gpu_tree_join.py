"""Split calls of many rows, whose records are joined by one wave per four rows (past 16384 rows of a call), by four (up to that),
or by more (few rows of many records): sampled rows against 64 bits."""

from __future__ import annotations

import pytest
import torch

from tests.serving_util import assert_rows, tree_oracle
from tests.test_gpu_tree_attention import Call

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
BF16, F16 = torch.bfloat16, torch.float16


def check_rows(call, out, tokens, heads):
    """Token j of a chain sees what the one token of a request whose context is j longer does."""

    starts = call.starts.tolist()
    owner = [max(b for b in range(len(starts) - 1) if starts[b] <= t) for t in tokens]
    context = [int(call.context[b]) + t - starts[b] for b, t in zip(owner, tokens)]
    q, got, per = call.q[tokens], out.cpu()[tokens], call.q.shape[1] // call.k.shape[1]
    for h in heads:  # of keys, with all their query heads
        part = slice(h * per, (h + 1) * per)
        one = lambda x: None if x is None else x[:, h : h + 1]  # noqa: E731
        expected, allowed = tree_oracle(q[:, part], one(call.k), one(call.v), one(call.ks), one(call.vs), call.table[owner], context,
                                        list(range(len(tokens) + 1)), None, call.scale, call.out[tokens][:, part])
        assert_rows(got[:, part], expected, allowed, f"head {h}")


def edges(call, block):
    """First and last tokens of requests and of blocks of rows, and some between."""

    starts, group = call.starts.tolist(), call.q.shape[1] // call.k.shape[1]
    step, picked = max(block // group, 1), set()
    for first, end in zip(starts, starts[1:]):
        for t in (first, first + 1, first + step - 1, first + step, first + 3 * step - 1, first + 3 * step, (first + end) // 2, end - 2, end - 1):
            if first <= t < end:
                picked.add(t)
    return sorted(picked)


@pytest.mark.parametrize("model,cache", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, torch.int8)])
@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("context,counts,heads,group", [
    ([700, 650], [520, 520], 8, 4),  # more than 16384 rows: one wave
    ([1100, 900], [520, 33], 4, 4),  # fewer: four waves
])
def test_joined_rows(device, d, model, cache, context, counts, heads, group):
    call = Call(context, counts, heads, group, d, 16, model, cache, masks=None)
    out = call.run(device)
    assert torch.isfinite(out).all() and (sum(counts) * heads * group > 16384) == (heads == 8)
    check_rows(call, out, edges(call, 64 if d == 256 else 128), [0, heads // 2, heads - 1])
    for _ in range(2):
        assert torch.equal(call.run(device), out)


@pytest.mark.parametrize("model,cache", [(BF16, BF16), (BF16, E4M3)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_requests_past_the_border(device, d, model, cache):
    """Requests of unequal length, some without tokens, whose items lie across ranges."""

    counts = [0, 300, 1, 17, 128, 0, 129, 300, 64, 190] * 2
    context = [10, 0, 900, 333, 64, 5, 1, 700, 2000, 128] * 2
    call = Call(context, counts, 2, 4, d, 16, model, cache, masks=None)
    out = call.run(device)
    assert sum(counts) * 8 > 16384
    check_rows(call, out, edges(call, 64 if d == 256 else 128), [0, 1])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_few_rows_of_many_records(device, d):
    call = Call([9000], [2], 1, 2, d, 16, BF16, BF16, masks=None)
    check_rows(call, call.run(device), [0, 1], [0])
