"""Token log probabilities of rows with many equal logits: constrained decoding,
where all but a few tokens are masked, constant rows, quantised logits. Their
alternatives come from the pass that every row takes, not from a pass for each
alternative: seen from the time against that of rows without ties."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

V = 128256


@pytest.fixture(autouse=True)
def _status_clean():
    from foundry_b200 import ops

    yield
    if "logprobs" in ops._rt.loaded_images():
        assert ops.status("logprobs") == 0


def _rows(kind, rows, vocab, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    low = -math.inf if kind.endswith("inf") else torch.finfo(dtype).min
    if kind == "random":
        return x
    if kind == "constant":
        return torch.full_like(x, 1.5)
    if kind.startswith("three"):
        keep = torch.tensor([7, vocab // 3, vocab - 5], device="cuda")
    elif kind.startswith("block"):
        keep = torch.arange(vocab // 2, vocab // 2 + 40, device="cuda")
    elif kind.startswith("none"):
        keep = torch.arange(0, device="cuda")
    elif kind == "levels":  # five values, the largest in many places
        return (torch.randint(0, 5, (rows, vocab), generator=g, device="cuda") - 2).to(dtype)
    y = torch.full_like(x, low)
    y[:, keep] = x[:, keep]
    return y


KINDS = ["constant", "three-inf", "three-lowest", "block-inf", "levels"]


@pytest.mark.parametrize("kind", KINDS + ["none-lowest"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,k", [(1, V, 20), (3, 5001, 32), (256, 50257, 5), (500, 9001, 20), (2, 40_003, 1)])
def test_order_is_exact(kind, dtype, rows, vocab, k):
    from foundry_b200 import ops

    x = _rows(kind, rows, vocab, dtype, seed=rows)
    top, ids = torch.empty(rows, k, device="cuda"), torch.empty(rows, k, dtype=torch.int32, device="cuda")
    ws = ops.LogprobWorkspace()
    ops.token_logprobs(x, None, None, None, top, ids, ws=ws)
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids.long(), order)
    want = x.double().log_softmax(-1).gather(1, order)
    assert torch.equal(torch.isinf(top), torch.isinf(want))
    # values next to ln V: an fp32 sum of V terms and its logarithm (the bound of the plain comparison, at its largest)
    off = torch.where(torch.isinf(want), 0.0, top - want).abs()
    assert (off <= 2.0**-20 + (V / 256 + 40) * 2.0**-24 + 2.0**-23 * want.nan_to_num(0.0, 0.0, 0.0).abs()
            + 2.0**-23 * 20).all()
    assert not ws.tickets.any()


@pytest.mark.parametrize("rows,k", [(1, 20), (256, 1), (256, 5), (256, 32), (1000, 5)])
def test_ties_cost_no_pass_per_alternative(rows, k):
    """Rows with ties within 4 times the time of rows without (a pass for each
    alternative made it 10 to 60 times at these sizes)."""
    from foundry_b200 import ops

    top, ids = torch.empty(rows, k, device="cuda"), torch.empty(rows, k, dtype=torch.int32, device="cuda")
    ws = ops.LogprobWorkspace()

    def us(x):
        best = math.inf
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(5):
                ops.token_logprobs(x, None, None, None, top, ids, ws=ws)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 200)
        return best

    base = us(_rows("random", rows, V, torch.bfloat16))
    times = {kind: us(_rows(kind, rows, V, torch.bfloat16)) for kind in KINDS}
    assert all(t <= 4 * base for t in times.values()), (base, times)
