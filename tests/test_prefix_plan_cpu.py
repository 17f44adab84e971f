"""Which groups of a mixed batch a PrefixPlan shares: each for itself."""

import random

import pytest
import torch

from foundry_b200 import ops
from foundry_b200.ops import _rt
from foundry_b200.ops import span_attention as S


@pytest.fixture(autouse=True)
def _sms(monkeypatch):
    monkeypatch.setattr(_rt, "sm_count", lambda: 148)


def _plan(groups, n_q=32, n_kv=8, **kw):
    sizes, pages = [n for n, _ in groups], [p for _, p in groups]
    return ops.PrefixPlan(sizes, pages, n_q, n_kv, max(pages, default=0), device="cpu", **kw)


def _shared(plan, groups):
    """For each group, whether its rows leave their prefix to the shared kernel."""
    got, row = [], 0
    for n, p in groups:
        tokens = set(plan.row_prefix[row:row + n].tolist())
        assert tokens in ({0}, {p * 64})
        got.append(tokens == {p * 64} and p > 0)
        row += n
    return got


@pytest.mark.parametrize("rows", [16, 64, 256])
@pytest.mark.parametrize("pairs", [1, 60, 96, 400])
@pytest.mark.parametrize("at", ["first", "last"])
def test_small_groups_do_not_decide_for_a_large_one(rows, pairs, at):
    alone = _plan([(rows, 512)])
    assert alone.items_n
    small = [(2, 1)] * pairs
    groups = [(rows, 512)] + small if at == "first" else small + [(rows, 512)]
    plan = _plan(groups)
    # the large one as if it were alone, the others row by row
    large = 0 if at == "first" else pairs
    assert _shared(plan, groups) == [i == large for i in range(len(groups))]
    assert (plan.tiles, plan.cluster, plan.parts, plan.items_n) == (alone.tiles, alone.cluster, alone.parts, alone.items_n)
    first = 0 if at == "first" else 2 * pairs
    moved = alone.items.clone()
    moved[:, 0] += first
    assert torch.equal(plan.items, moved)


def test_every_group_that_pays_is_shared():
    """Two prompts of very different lengths, both worth it, and one row that shares nothing."""
    groups = [(100, 300), (1, 500), (200, 40)]
    assert _shared(_plan(groups), groups) == [True, False, True]
    assert _shared(_plan(groups, share=True), groups) == [True, True, True]
    assert not _plan(groups, share=False).items_n




def test_estimate_of_equal_clusters():
    """Whole waves of what the SMs hold, each as long as one cluster."""
    assert S._prefix_us([(100, 32)], 2, 4, 1, 148) == 25 * 2.1 + 7
    assert S._prefix_us([(100, 33)], 2, 4, 1, 148) == 2 * (25 * 2.1 + 7)
    assert S._prefix_us([(100, 16)], 2, 4, 2, 148) == 13 * 2.1 + 7 + 0.7
    assert S._prefix_us([(100, 1)], 1, 1, 1, 148) == 100 * 1.8 + 7
    # a wave is as long as its longest cluster, the rest of a wave costs nothing more; further ones start late
    assert S._prefix_us([(100, 30), (10, 2)], 2, 4, 1, 148) == pytest.approx(25 * 2.1 + 7)
    assert S._prefix_us([(100, 30), (10, 3)], 2, 4, 1, 148) == pytest.approx((25 * 2.1 + 7) + (3 * 2.1 + 7) + 12)
    assert S._prefix_us([(100, 8), (10, 8)], 2, 4, 2, 148) == pytest.approx(13 * 2.1 + 7 + 8)


def test_no_mixture_is_estimated_worse_than_all_or_nothing():
    """Random mixtures: the choice is at least as good, by the estimate, as sharing none and as sharing all."""
    rng = random.Random(1)
    for _ in range(30):
        groups = [(rng.choice([1, 2, 3, 8, 40, 150]), rng.choice([0, 1, 2, 9, 64, 300])) for _ in range(rng.randint(1, 40))]
        n_q, n_kv = rng.choice([(32, 8), (32, 4), (8, 8), (16, 1)])
        plan, everything = _plan(groups, n_q, n_kv), _plan(groups, n_q, n_kv, share=True)
        again = [n * p * 64 * n_kv * 512 / 5.5e6 if n > 1 else 0.0 for n, p in groups]

        def us(plan):
            shared = _shared(plan, groups)
            kinds = [((p + 1) // 2, n_kv * -(-n // (S.prefix_rows(n_q // n_kv) * plan.tiles)))
                     for (n, p), s in zip(groups, shared) if s]
            kernel = S._prefix_us(sorted(kinds, reverse=True), plan.tiles, plan.cluster, plan.parts, 148) if kinds else 0.0
            return kernel + sum(a for a, s in zip(again, shared) if not s)

        assert us(plan) <= sum(again) + 1e-6
        assert us(plan) <= us(everything) + 1e-6 or any(n == 1 and p for n, p in groups)


def test_many_different_groups_are_planned_at_once():
    """Prompts of every length: the search does not grow with their number squared."""
    import time

    rng = random.Random(2)
    groups = [(rng.randint(2, 60), rng.randint(1, 4000)) for _ in range(2000)]
    t = time.perf_counter()
    plan = _plan(groups)
    assert plan.items_n and time.perf_counter() - t < 2.0  # 0.1 s here


def test_share_is_a_truth_value_or_none():
    groups = [(100, 300)]
    for no in (False, 0, torch.tensor(False)):
        assert not _plan(groups, share=no).items_n
    for yes in (True, 1, torch.tensor(True)):
        assert _plan([(2, 1)], share=yes).items_n
