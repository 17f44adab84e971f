"""NaN and infinite scores in full tiles of a prefill and of a shared prefix:
every row that sees such a key is NaN (inf - inf, and NaN, in the softmax of the
formula), at whatever place of its tile the key lies and whatever comes after
it; no other row is touched."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, PAGE = 128, 64


@pytest.fixture(autouse=True)
def _status_clean():
    from foundry_b200 import ops

    yield
    for img in ("attention_span", "attention_tile"):
        if img in ops._rt.loaded_images():
            assert ops.status(img) == 0, f"{img} reported a device-side error"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _spoil(key, bad):
    """A key whose score with a query of positive first dimension is ``bad``."""
    key.zero_()
    key[0] = bad


# The scores behind the bad key are as before, or so much larger that the running
# maximum moves and what has been summed is scaled down.
@pytest.mark.parametrize("louder", [1, 12])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n_q,n_kv", [(4, 2), (3, 1)])
def test_prefill(n_q, n_kv, bad, louder):
    from foundry_b200 import ops

    t, first, window = 1000, 256, 400
    cu, (ts, tst) = _i32([0, t]), map(_i32, ops.prefill_tiles([t]))

    def run(qkv):
        q, k, v = qkv.split([n_q * D, n_kv * D, n_kv * D], 1)
        out = torch.full((t, n_q * D), 7.0, dtype=torch.bfloat16, device="cuda")
        return ops.window_prefill_attention(q, k, v, out, cu, ts, tst, n_q, n_kv, window, 0).view(t, n_q, D)

    good = _randn(t, (n_q + 2 * n_kv) * D, seed=1)
    good[:, :n_q * D:D] = good[:, :n_q * D:D].abs() + 0.125
    good[first + 128:, n_q * D:(n_q + n_kv) * D] *= louder
    want = run(good)
    assert torch.isfinite(want).all()
    for at in range(first, first + 9):
        qkv = good.clone()
        _spoil(qkv[at, n_q * D:(n_q + 1) * D], bad)
        got = run(qkv)
        sees = torch.zeros(t, n_q, dtype=torch.bool, device="cuda")
        sees[at:at + window, :n_q // n_kv] = True
        assert torch.isnan(got[sees]).all(), at
        assert torch.equal(got[~sees], want[~sees]), at


@pytest.mark.parametrize("louder", [1, 12])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("rows,shared", [(16, 24), (100, 24), (64, 512)])  # one query tile; two; two in several parts
def test_shared_prefix(rows, shared, bad, louder):
    from foundry_b200 import ops

    n_q, n_kv = 16, 4
    pages = shared + 1
    kc, vc = _randn(shared + rows, n_kv, PAGE, D, seed=1), _randn(shared + rows, n_kv, PAGE, D, seed=2)
    kc[4:shared] *= louder
    table = torch.arange(shared, dtype=torch.int32, device="cuda").repeat(rows, 1)
    table = torch.cat([table, torch.arange(shared, shared + rows, dtype=torch.int32, device="cuda")[:, None]], 1)
    table, lens = table.contiguous(), _i32([shared * PAGE + 1 + i % 60 for i in range(rows)])
    q = _randn(rows, n_q, D, seed=3)
    q[..., 0] = q[..., 0].abs() + 0.125
    plan = ops.PrefixPlan([rows], [shared], n_q, n_kv, pages, share=True)
    assert plan.cluster * plan.parts > 1 and plan.tiles == (1 if rows == 16 else 2)
    ws = ops.SpanWorkspace(plan.partials)

    def run(kc):
        out = torch.full_like(q, 7.0)
        return ops.prefix_decode_attention(q, kc, vc, table, lens, out, plan, ws)

    want = run(kc)
    assert torch.isfinite(want).all()
    for at in range(9):
        spoilt = kc.clone()
        _spoil(spoilt[2, 1, at], bad)
        got = run(spoilt)
        sees = torch.zeros(rows, n_q, dtype=torch.bool, device="cuda")
        sees[:, 4:8] = True
        assert torch.isnan(got[sees]).all(), at
        assert torch.equal(got[~sees], want[~sees]), at
