"""Windowed and shared-prefix attention and token log probabilities where a call
is at the edge of what it may be: NaN in what a row sees and in what no row
sees, device data that contradicts the call, two calls at a time, the same page
twice, a cache beyond 4 GB. Tolerances are those of the plain comparison of
each operator (bf16 probabilities and output: 2^-8 of sum p|v| and of the
output; scores 128 roundings of 2^-23)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, PAGE = 128, 64
BAD_ARG = 16  # FB_KERR_BAD_ARG


@pytest.fixture(autouse=True)
def _status_clean():
    from foundry_b200 import ops

    yield
    for img in ("attention_span", "attention_tile", "logprobs"):
        if img in ops._rt.loaded_images():
            assert ops.status(img) == 0, f"{img} reported a device-side error"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _randn(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _batch(lens, n_q=8, n_kv=2, shared=0, extra=0):
    """q, caches, table and lengths; the first ``shared`` pages are the same for all rows."""
    b, pages = len(lens), max(1, max(math.ceil(n / PAGE) for n in lens), shared) + extra
    table = torch.arange(b * pages, dtype=torch.int32, device="cuda").view(b, pages)
    table[:, :shared] = table[0, :shared].clone()
    shape = (b * pages, n_kv, PAGE, D)
    return _randn(b, n_q, D, seed=1), _randn(*shape, seed=2), _randn(*shape, seed=3), table.contiguous(), _i32(lens)


def _reference(q, kc, vc, table, n, lo=0, sinks=0):
    """One row over its tokens t < n with t >= lo or t < sinks -> (o, tolerance)."""
    at = torch.arange(n, device="cuda")
    at = at[(at >= lo) | (at < sinks)]
    page = table.long()[at // PAGE]
    n_kv = kc.shape[1]
    k, v = (c[page, :, at % PAGE].transpose(0, 1).double() for c in (kc, vc))
    q = q.view(n_kv, -1, D).double()
    s = q @ k.transpose(1, 2) / math.sqrt(D)
    p = s.softmax(-1)
    o, a = p @ v, p @ v.abs()
    worst = (q.abs() @ k.abs().transpose(1, 2) / math.sqrt(D)).amax(-1, keepdim=True)
    tol = 2.0**-8 * (a + o.abs()) + (2 * 128 * 2.0**-23 * worst + 2.0**-20) * a
    return o.reshape(-1, D), tol.reshape(-1, D)


def _close(got, ref):
    o, tol = ref
    assert torch.isfinite(got).all()
    assert ((got.double() - o).abs() <= tol + 1e-30).all()


@pytest.mark.parametrize("op", ["window", "prefix"])
def test_nan_in_what_a_row_sees_stays_with_the_row(op):
    from foundry_b200 import ops

    lens = [400, 300, 401, 260]
    q, kc, vc, table, lens_t = _batch(lens, shared=4)
    plan = ops.PrefixPlan([4], [4], 8, 2, table.shape[1], share=True)
    ws = ops.SpanWorkspace(plan.partials)

    def run():
        out = torch.empty_like(q)
        if op == "window":
            return ops.window_decode_attention(q, kc, vc, table, lens_t, out, 150, 4, ws)
        return ops.prefix_decode_attention(q, kc, vc, table, lens_t, out, plan, ws)

    want = run().clone()
    q[1, 5] = math.nan  # a head's query
    kc[table[2, 5].long(), 1, 10] = math.nan  # a token of the third row's own part
    got = run()
    assert torch.isnan(got[1, 5]).all() and torch.isnan(got[2, 4:]).all()
    keep = torch.ones(4, 8, dtype=torch.bool, device="cuda")
    keep[1, 5] = False
    keep[2, 4:] = False
    assert torch.equal(got[keep], want[keep])
    vc[table[0, 0].long(), 0, 2, 7] = math.nan  # what all rows see (a sink, the shared prompt)
    assert torch.isnan(run()[:, :4, 7]).all()


def test_nan_query_of_a_prefill_stays_with_its_row():
    from foundry_b200 import ops

    for n_q, n_kv in ((4, 2), (3, 1)):
        lens = [200, 333]
        qkv = _randn(533, (n_q + 2 * n_kv) * D)
        q, k, v = qkv.split([n_q * D, n_kv * D, n_kv * D], 1)
        cu, (ts, tst) = _i32([0, 200, 533]), map(_i32, ops.prefill_tiles(lens))
        outs = []
        for _ in range(2):
            out = torch.empty(533, n_q * D, dtype=torch.bfloat16, device="cuda")
            ops.window_prefill_attention(q, k, v, out, cu, ts, tst, n_q, n_kv, 64, 2)
            outs.append(out.view(533, n_q, D))
            q[77, D:2 * D] = math.nan
        keep = torch.ones(533, n_q, dtype=torch.bool, device="cuda")
        keep[77, 1] = False
        assert torch.isnan(outs[1][77, 1]).all() and torch.equal(outs[0][keep], outs[1][keep])


@pytest.mark.parametrize("lens", [[100, 37, 1], [100, 0, 0], [0, 0, 0], [129, 300, 5], [512, 511, 65]])
@pytest.mark.parametrize("n_q,n_kv", [(8, 2), (32, 2), (3, 3)])
def test_prefix_longer_than_every_row(lens, n_q, n_kv):
    """Padding rows, and rows shorter than their prefix: what no row sees of the
    shared pages has never been written (NaN)."""
    from foundry_b200 import ops

    q, kc, vc, table, lens_t = _batch(lens, n_q, n_kv, shared=8)
    ref = [_reference(q[r], kc, vc, table[r], n) if n else None for r, n in enumerate(lens)]
    longest = max(lens)
    for c in (kc, vc):
        flat = c[table[0, :8].long()].transpose(1, 2).reshape(8 * PAGE, n_kv, D)
        flat[longest:] = math.nan
        c[table[0, :8].long()] = flat.view(8, PAGE, n_kv, D).transpose(1, 2)
    plan = ops.PrefixPlan([3], [8], n_q, n_kv, table.shape[1], share=True)
    out = torch.full_like(q, 7.0)
    ops.prefix_decode_attention(q, kc, vc, table, lens_t, out, plan, ops.SpanWorkspace(plan.partials))
    for r, n in enumerate(lens):
        if n:
            _close(out[r], ref[r])
        else:
            assert (out[r] == 0).all()


def test_bad_device_data_is_reported_and_touches_nothing():
    """Page numbers outside the cache, lengths beyond the table, tokens beyond the
    vocabulary: a status bit; the other rows are right."""
    from foundry_b200 import ops

    def reported(img):
        assert ops.status(img) == BAD_ARG
        ops.clear_status(img)

    q, kc, vc, table, lens_t = _batch([300, 200, 150], shared=2)
    ws = ops.SpanWorkspace(1 << 10)
    good, out = torch.empty_like(q), torch.empty_like(q)
    ops.window_decode_attention(q, kc, vc, table, lens_t, good, 1000, 0, ws)
    for bad in (-1, kc.shape[0], 1 << 30, -(1 << 31)):
        broken = table.clone()
        broken[1, 2] = bad
        ops.window_decode_attention(q, kc, vc, broken, lens_t, out, 1000, 0, ws)
        reported("attention_span")
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    long = lens_t.clone()
    long[2], long[0] = table.shape[1] * PAGE + 1, -5
    ops.window_decode_attention(q, kc, vc, table, long, out, 100, 0, ws)
    reported("attention_span")
    assert (out[0] == 0).all() and torch.isfinite(out).all()
    plan = ops.PrefixPlan([3], [2], 8, 2, table.shape[1], share=True)
    for bad in (-1, kc.shape[0], 1 << 30):
        broken = table.clone()
        broken[0, 1] = bad
        ops.prefix_decode_attention(q, kc, vc, broken, lens_t, out, plan, ws)
        reported("attention_tile")
    x, ids = _randn(4, 1000), _i32([3, 1000, 1 << 30, -1])
    lp, lws = torch.empty(4, device="cuda"), ops.LogprobWorkspace()
    ops.token_logprobs(x, ids, lp, None, ws=lws)
    reported("logprobs")
    assert torch.isfinite(lp[[0, 3]]).all() and torch.isnan(lp[1:3]).all()
    # and afterwards all is as before
    ops.prefix_decode_attention(q, kc, vc, table, lens_t, out, plan, ws)
    torch.testing.assert_close(out, good, atol=0.02, rtol=0.02)
    assert not ws.tickets.any() and not lws.tickets.any()


def test_prefill_tables_padded_with_tiles_behind_the_end():
    from foundry_b200 import ops

    lens = [200, 130]
    qkv = _randn(330, 4 * D)
    q, k, v = qkv.split([2 * D, D, D], 1)
    ts, tst = ops.prefill_tiles(lens)
    outs = []
    for pad in (0, 5):
        out = torch.full((330, 2 * D), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.window_prefill_attention(q, k, v, out, _i32([0, 200, 330]), _i32(ts + [0] * pad), _i32(tst + [1 << 20] * pad),
                                     2, 1, 100, 4)
        outs.append(out)
    assert torch.equal(*outs)


def test_two_calls_at_a_time():
    """Workspaces of their own on two streams: neither disturbs the other."""
    from foundry_b200 import ops

    lens = [700 + 91 * i for i in range(24)]
    q, kc, vc, table, lens_t = _batch(lens, 32, 8, shared=10)
    plan = ops.PrefixPlan([24], [10], 32, 8, table.shape[1], share=True)
    x = _randn(100, 30_000)
    ids = torch.arange(100, dtype=torch.int32, device="cuda")
    qkv = _randn(2000, 48 * D, seed=5)
    pq, pk, pv = qkv.split([32 * D, 8 * D, 8 * D], 1)
    plens = [1500, 500]
    cu, (ts, tst) = _i32([0, 1500, 2000]), map(_i32, ops.prefill_tiles(plens))
    streams = [torch.cuda.Stream() for _ in range(2)]
    state = []
    for _ in streams:
        state.append(dict(ws=ops.SpanWorkspace(plan.partials), lws=ops.LogprobWorkspace(), a=torch.empty_like(q),
                          b=torch.empty_like(q), c=torch.empty(2000, 32 * D, dtype=torch.bfloat16, device="cuda"),
                          lp=torch.empty(100, device="cuda"), top=torch.empty(100, 8, device="cuda"),
                          tid=torch.empty(100, 8, dtype=torch.int32, device="cuda")))

    def step(s):
        ops.prefix_decode_attention(q, kc, vc, table, lens_t, s["a"], plan, s["ws"])
        ops.window_decode_attention(q, kc, vc, table, lens_t, s["b"], 300, 4, s["ws"])
        ops.window_prefill_attention(pq, pk, pv, s["c"], cu, ts, tst, 32, 8, 256, 4)
        ops.token_logprobs(x, ids, s["lp"], None, s["top"], s["tid"], ws=s["lws"])

    step(state[0])
    torch.cuda.synchronize()
    names = ("a", "b", "c", "lp", "top", "tid")
    want = [state[0][n].clone() for n in names]
    for s in state:
        for n in names:
            s[n].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for st, s in zip(streams, state):
            with torch.cuda.stream(st):
                step(s)
    torch.cuda.synchronize()
    for s in state:
        for n, w in zip(names, want):
            assert torch.equal(s[n], w), n


def test_one_page_everywhere_and_output_over_the_query():
    """The same page at every place of every table; out in q's memory."""
    from foundry_b200 import ops

    q, kc, vc, table, lens_t = _batch([1000, 64, 65, 999])
    table[:] = 3
    ref = [_reference(q[r], kc, vc, table[r], n, max(n - 300, 0), 5) for r, n in enumerate(lens_t.tolist())]
    ops.window_decode_attention(q, kc, vc, table, lens_t, q, 300, 5, ops.SpanWorkspace())
    for r in range(4):
        _close(q[r], ref[r])


def test_a_cache_beyond_32_bit_offsets():
    """Pages whose elements lie past 2^31 (8.6 GB a cache, of which little is written)."""
    from foundry_b200 import ops

    blocks, n_kv, n_q = 1 << 17, 4, 16
    kc = torch.empty(blocks, n_kv, PAGE, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    assert kc.numel() > 1 << 31
    ids = [blocks - 1 - 3 * i for i in range(6)]
    kc[ids], vc[ids] = _randn(6, n_kv, PAGE, D, seed=1), _randn(6, n_kv, PAGE, D, seed=2)
    q, lens = _randn(2, n_q, D, seed=3), [6 * PAGE - 9, 5 * PAGE]
    table, out = _i32([ids, ids]), torch.empty(2, n_q, D, dtype=torch.bfloat16, device="cuda")
    plan = ops.PrefixPlan([2], [4], n_q, n_kv, 6, share=True)
    ws = ops.SpanWorkspace(plan.partials)
    ref = [_reference(q[r], kc, vc, table[r], n) for r, n in enumerate(lens)]
    ops.prefix_decode_attention(q, kc, vc, table, _i32(lens), out, plan, ws)
    for r in range(2):
        _close(out[r], ref[r])
    ops.window_decode_attention(q, kc, vc, table, _i32(lens), out, 1 << 20, 0, ws)
    for r in range(2):
        _close(out[r], ref[r])


def test_logits_beyond_32_bit_offsets():
    from foundry_b200 import ops

    t, v = 20_000, 151_936  # 6 GB
    x = torch.zeros(t, v, dtype=torch.bfloat16, device="cuda")
    hot = (torch.arange(t, device="cuda") * 7) % v
    x[torch.arange(t, device="cuda"), hot] = 20.0
    lp, tid = torch.empty(t, device="cuda"), torch.empty(t, 2, dtype=torch.int32, device="cuda")
    ops.token_logprobs(x, hot.to(torch.int32), lp, None, torch.empty(t, 2, device="cuda"), tid, ws=ops.LogprobWorkspace())
    # ln p = -ln Z, Z = 1 + (v - 1) e^-20 in [1, 2): each fp32 addition to Z is off by
    # 2^-24 at most. Of the hot logit's thread these are: 17 within its 32 logits, one
    # for each further 32 of its v / 256, and at most 24 in the join of threads and
    # pieces; the terms e^-20 are off by 2^-22 (2^x) and 20 * 2^-23 (x) of themselves.
    z1 = (v - 1) * math.exp(-20.0)
    want = -math.log1p(z1)
    tol = (17 + v / 256 / 32 + 24) * 2.0**-24 + z1 * (2.0**-22 + 20 * 2.0**-23) + 2.0**-24 * abs(want)
    assert ((lp - want).abs() <= tol).all(), (lp - want).abs().max()
    assert torch.equal(tid[:, 0].long(), hot)
    assert torch.equal(tid[:, 1].long(), torch.where(hot == 0, 1, 0))
