"""Token log probabilities against the definition in 64 bits.

Tolerance: Z is an fp32 sum of 2^y: each term is off by 2^-22 (2^x) and by
2^-23 |y| ln 2 <= 2^-23 * |x - max| (y's two roundings), weighted by p; the
sums add at most N + 24 roundings of 2^-24, N the terms of one thread. That
moves ln Z by the same absolute amount, and a log probability is rounded once
more (2^-24 |lp|). H's second term is a sum of the same kind, |U / Z| as large
as sum p |x - max|.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    from foundry_b200 import ops

    yield
    if "logprobs" in ops._rt.loaded_images():
        assert ops.status("logprobs") == 0, "logprobs reported a device-side error"


def _run(x, ids, k, ws=None):
    from foundry_b200 import ops

    t = x.shape[0]
    lp, h = torch.full((t,), 7.0, device="cuda"), torch.full((t,), 7.0, device="cuda")
    tlp = torch.full((t, k), 7.0, device="cuda") if k else None
    tid = torch.full((t, k), -7, dtype=torch.int32, device="cuda") if k else None
    ws = ws or ops.LogprobWorkspace()
    ops.token_logprobs(x, ids, lp, h, tlp, tid, ws=ws)
    assert not ws.tickets.any()
    return lp, h, tlp, tid


def _check(x, ids, k, ws=None):
    from foundry_b200.ops import logprobs as L

    t, v = x.shape
    lp, h, tlp, tid = _run(x, ids, k, ws)
    y = x.double() - x.double().amax(-1, keepdim=True)
    z = y.exp().sum(-1, keepdim=True)
    ref = y - z.log()
    p = ref.exp()
    far = torch.where(p > 0, -y, 0.0)
    share = min(v, L.share_of(t, v, L.CTAS_PER_SM * torch.cuda.get_device_properties(0).multi_processor_count)[0])
    rel = (share / 256 + 16 + 24) * 2.0**-24 + 2.0**-22 + (p * far).sum(-1) * 2.0**-23
    at = ids.long().clamp_min(0)
    want = ref.gather(1, at[:, None])[:, 0]
    want = torch.where(ids < 0, 0.0, want)
    assert torch.equal(torch.isinf(lp), torch.isinf(want))
    fine = ~torch.isinf(want)
    assert ((lp - want).abs() <= rel + 2.0**-23 * want.abs())[fine].all(), (lp - want).abs().max()
    ent = -torch.where(p > 0, p * ref, 0.0).sum(-1)
    size = (p * far).sum(-1)
    assert ((h - ent).abs() <= rel + 2 * rel * size + 2.0**-23 * ent).all(), (h - ent).abs().max()
    if k:
        order = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(tid.long(), order)
        want = ref.gather(1, order)
        assert torch.equal(torch.isinf(tlp), torch.isinf(want))
        off = torch.where(torch.isinf(want), 0.0, tlp - want).abs()
        assert (off <= rel[:, None] + 2.0**-23 * torch.where(torch.isinf(want), 0.0, want.abs())).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,v,k", [
    (1, 1, 1), (1, 7, 3), (3, 33, 32), (2, 257, 8), (5, 1000, 5), (1, 128256, 20), (37, 4099, 0), (300, 2048, 1),
    (64, 50257, 20), (700, 1111, 32), (9, 151936, 5),
])
def test_against_64_bits(dtype, t, v, k):
    g = torch.Generator(device="cuda").manual_seed(t + v)
    x = (torch.randn(t, v, generator=g, device="cuda") * 3).to(dtype)
    ids = torch.randint(-1, v, (t,), generator=g, device="cuda").to(torch.int32)
    _check(x, ids, k)


@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_strided_rows_of_any_alignment(offset):
    g = torch.Generator(device="cuda").manual_seed(offset)
    wide = torch.randn(20, 9001, generator=g, device="cuda").to(torch.bfloat16)
    x = wide[:, offset:offset + 8200 + offset]
    _check(x, torch.arange(20, dtype=torch.int32, device="cuda"), 20)


@pytest.mark.parametrize("k", [1, 20, 32])
def test_ties_and_masks(k):
    """Constant rows, few distinct values, rows in rising and falling order, the
    largest logits all in one thread's part, masks of -inf and of the type's
    lowest value, all but a few masked, one certain token."""
    v = 20_000
    g = torch.Generator(device="cuda").manual_seed(k)
    rows = [torch.zeros(v), torch.full((v,), -3.0), torch.arange(v) / 64.0, -torch.arange(v) / 64.0]
    rows.append(torch.randint(0, 3, (v,), generator=g, device="cuda").float().cpu())
    one = torch.randn(v)
    one[torch.arange(8 * 17, v, 2048)] = 50.0 + torch.arange(len(range(8 * 17, v, 2048)))
    rows.append(one)
    clustered = torch.randn(v)  # whole vectors of one thread above all else
    for j in range(8 * 5, v - 8, 2048):
        clustered[j:j + 8] = 40.0
    rows.append(clustered)
    for low in (-math.inf, torch.finfo(torch.bfloat16).min):
        few = torch.full((v,), low)
        few[torch.tensor([3, 77, 19_999])] = torch.tensor([1.0, -2.0, 1.0])
        half = torch.randn(v)
        half[::2] = low
        rows += [few, half]
    rows.append(torch.full((v,), torch.finfo(torch.bfloat16).min))
    certain = torch.randn(v)
    certain[1234] = 60.0
    rows.append(certain)
    x = torch.stack(rows).cuda().to(torch.bfloat16)
    ids = torch.full((len(rows),), 3, dtype=torch.int32, device="cuda")
    ids[-1] = 1234
    _check(x, ids, k)
    _check(x.float(), ids, k)
    _check(x.repeat(40, 1), ids.repeat(40), k)


def test_many_above_the_bound():
    """One thread's part holds more of the largest logits than the candidate list."""
    v = 1 << 19
    x = torch.zeros(300, v, dtype=torch.bfloat16, device="cuda")  # a share is several thousand vectors
    x[:, :] = torch.linspace(-1, 0, v, device="cuda").to(torch.bfloat16)
    base = torch.arange(0, v, 2048, device="cuda")
    for e in range(8):
        x[:, base + e] = 5.0 + e / 8 + (torch.arange(len(base), device="cuda") / 32).to(torch.bfloat16)
    got = _run(x, torch.zeros(300, dtype=torch.int32, device="cuda"), 32)
    order = torch.sort(x[:1].float(), dim=-1, descending=True, stable=True).indices[:, :32]
    assert torch.equal(got[3].long(), order.expand(300, -1))


def test_rows_without_a_distribution():
    """-inf throughout, +inf or NaN somewhere: NaN, and the other rows are not touched by it."""
    x = torch.randn(4, 5000, device="cuda")
    x[1] = -math.inf
    x[2, 17] = math.inf
    x[3, 4000] = math.nan
    ids = torch.tensor([5, 5, 5, 5], dtype=torch.int32, device="cuda")
    lp, h, tlp, tid = _run(x, ids, 4)
    assert torch.isfinite(lp[0]) and torch.isfinite(h[0]) and torch.isfinite(tlp[0]).all()
    assert torch.isnan(lp[1:]).all() and torch.isnan(h[1:]).all() and torch.isnan(tlp[1:]).all()
    assert tid[1].tolist() == [0, 1, 2, 3] and tid[2, 0] == 17


def test_outputs_left_out_and_replayed():
    from foundry_b200 import ops

    x = torch.randn(50, 30_000, device="cuda").to(torch.bfloat16)
    ids = torch.randint(0, 30_000, (50,), device="cuda", dtype=torch.int32)
    ws = ops.LogprobWorkspace()
    lp, h, tlp, tid = _run(x, ids, 7, ws)
    only_h = torch.empty(50, device="cuda")
    ops.token_logprobs(x, None, None, only_h, ws=ws)
    only_lp = torch.empty(50, device="cuda")
    ops.token_logprobs(x, ids, only_lp, None, ws=ws)
    assert torch.equal(only_h, h) and torch.equal(only_lp, lp)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    a, b = torch.empty(50, 7, device="cuda"), torch.empty(50, 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side), ops._rt.pdl():
        ops.token_logprobs(x, None, None, None, a, b, ws=ws)
        ops.token_logprobs(x, ids, only_lp, None, ws=ws)
    x.copy_(x.roll(3, 1))
    graph.replay()
    torch.cuda.synchronize()
    # the same logits in other places: the same values, but for the order of the sums
    torch.testing.assert_close(a, tlp, atol=1e-4, rtol=0)
