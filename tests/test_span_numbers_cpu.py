"""Numbers of the windowed, shared-prefix and log-probability calls that are not
whole: refused where a whole number is meant, on the CPU with the launch
replaced by one that records its numbers."""

import numpy as np
import pytest
import torch

from foundry_b200 import ops
from foundry_b200.ops import _rt


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    got = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)  # what get_device() says of a CPU tensor
    monkeypatch.setattr(_rt, "sm_count", lambda: 148)
    monkeypatch.setattr(_rt, "launch_mapped", lambda *a, **k: got.append(a))
    return got


def _decode(window, sinks):
    bf = dict(dtype=torch.bfloat16)
    cache = torch.zeros(10, 2, 64, 128, **bf)
    q, lens = torch.zeros(3, 8, 128, **bf), torch.ones(3, dtype=torch.int32)
    ops.window_decode_attention(q, cache, cache, torch.zeros(3, 4, dtype=torch.int32), lens, torch.zeros_like(q),
                                window, sinks, ops.SpanWorkspace(device="cpu"))


def _prefill(window, sinks):
    q, kv = torch.zeros(200, 512, dtype=torch.bfloat16), torch.zeros(200, 256, dtype=torch.bfloat16)
    tiles = torch.tensor([0, 128], dtype=torch.int32)
    ops.window_prefill_attention(q, kv, kv, torch.zeros_like(q), torch.tensor([0, 200], dtype=torch.int32),
                                 torch.zeros_like(tiles), tiles, 4, 2, window, sinks)


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_window_and_sinks_are_whole_numbers(launches, call):
    """As a float they would reach the kernel's integers as their bits: a window over everything."""
    for window, sinks in ((1024.0, 4), (64.5, 4), (64, 4.0), (np.float32(64), 0), ("64", 0), (None, 0), (64, None)):
        with pytest.raises(ValueError, match="window"):
            call(window, sinks)
    assert not launches
    for window, sinks in ((64, 4), (np.int64(64), np.int32(4)), (torch.tensor(64), torch.tensor(4))):
        call(window, sinks)
        numbers = launches.pop()[2:]
        assert sum(isinstance(x, float) for x in numbers) == 1  # the scale
        assert all(type(x) in (int, float) for x in numbers) and {64, 4} <= set(numbers)


def test_plan_takes_whole_rows_and_pages():
    """2.5 pages would be 160 tokens that the rows leave out, of which the shared kernel reads 128."""
    for sizes, pages in (([3], [2.5]), ([3], [2.0]), ([3.0], [2]), ([1.5, 1.5], [2, 2]), ([3], ["2"]), ([None], [2])):
        with pytest.raises(ValueError, match="whole numbers"):
            ops.PrefixPlan(sizes, pages, 8, 2, 4, device="cpu", share=True)
    want = ops.PrefixPlan([3, 2], [2, 4], 8, 2, 4, device="cpu", share=True)
    for sizes, pages in ((np.array([3, 2]), np.array([2, 4])), (torch.tensor([3, 2]), torch.tensor([2, 4]))):
        plan = ops.PrefixPlan(sizes, pages, 8, 2, 4, device="cpu", share=True)
        assert plan.rows == 5 and torch.equal(plan.items, want.items) and torch.equal(plan.row_prefix, want.row_prefix)


@pytest.mark.parametrize("scale", [1e-45, 1e-38, 1e38, 1e300, float("inf"), float("nan"), 0.0, -0.1])
def test_scale_that_fp32_does_not_hold(launches, scale):
    """Times log2(e) it would be zero (masked scores: -inf * 0), infinite or subnormal in the kernel."""
    q, cache = torch.zeros(3, 8, 128, dtype=torch.bfloat16), torch.zeros(10, 2, 64, 128, dtype=torch.bfloat16)
    kv, tiles = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    args = q, cache, cache, torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.zeros_like(q)
    plan = ops.PrefixPlan([3], [2], 8, 2, 4, device="cpu", share=True)
    ws = ops.SpanWorkspace(plan.partials, device="cpu")

    def calls(scale):
        yield lambda: ops.window_decode_attention(*args, 64, 0, ws, scale=scale)
        yield lambda: ops.prefix_decode_attention(*args, plan, ws, scale=scale)
        yield lambda: ops.window_prefill_attention(q.view(3, 1024), kv, kv, torch.zeros(3, 1024, dtype=torch.bfloat16),
                                                   torch.tensor([0, 3], dtype=torch.int32), tiles, tiles, 8, 2, 64, 0,
                                                   scale=scale)

    for call in calls(scale):
        with pytest.raises(ValueError, match="scale"):
            call()
    assert not launches
    for fine in (None, 1, 0.0883, 1e-30, 1e30):
        for call in calls(fine):
            call()
