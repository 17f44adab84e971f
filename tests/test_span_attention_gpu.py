"""Shared-prefix and windowed attention against the definition in 64 bits.

Tolerance, per output element (A = sum p|v| / l from the 64-bit reference):
p is rounded to bf16 before P V (relative 2^-8 of each term: 2^-8 A), the
output once more (2^-8 |o|); scores are fp32 sums of 128 exact products, off
by at most 128 * 2^-23 * sum |q k| * scale, which moves p and l by that much
each, and 2^x by 2^-21: (2 * 128 * 2^-23 * S + 2^-20) A.
"""

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


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, g, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(torch.bfloat16)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _attend(q, k, v, seen, scale):
    """q [.., m, d], k, v [.., n, d], seen [.., m, n] -> (o, tolerance) in 64 bits."""
    q, k, v = q.double(), k.double(), v.double()
    s = torch.where(seen, q @ k.transpose(-1, -2) * scale, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = (s - torch.where(m == -math.inf, 0.0, m)).exp()
    l = p.sum(-1, keepdim=True).clamp_min(1e-300)
    o, a = p @ v / l, p @ v.abs() / l
    worst = torch.where(seen, q.abs() @ k.abs().transpose(-1, -2) * scale, 0.0).amax(-1, keepdim=True)
    tol = 2.0**-8 * (a + o.abs()) + (2 * 128 * 2.0**-23 * worst + 2.0**-20) * a
    return o, tol


def _close(got, o, tol):
    off = (got.double() - o).abs()
    assert torch.isfinite(got).all(), "not finite"
    assert (off <= tol + 1e-30).all(), f"off by {(off / (tol + 1e-30)).max().item():.2f} tolerances"


def _paged(lens, n_q, n_kv, seed, shared=None, extra=0, keep=None):
    """A paged cache whose every value is NaN but for the tokens of the rows
    that ``keep(row, position)`` names (all by default). ``shared``: list of
    (first row, rows, pages)."""
    g = _gen(seed)
    b = len(lens)
    pages = max(1, max(math.ceil(n / PAGE) for n in lens)) + extra
    nblocks = b * pages + 3
    order = torch.randperm(nblocks, generator=g, device="cuda").tolist()
    table = [[order[r * pages + p] for p in range(pages)] for r in range(b)]
    for r0, rows, n in shared or []:
        for r in range(r0, r0 + rows):
            table[r][:n] = table[r0][:n]
    kc = torch.full((nblocks, n_kv, PAGE, D), math.nan, dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    for r, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        if keep is not None:
            at = at[keep(r, at)]
        page, off = _i32(table[r]).long()[at // PAGE], at % PAGE
        kc[page, :, off] = _randn(len(at), n_kv, D, g=g)
        vc[page, :, off] = _randn(len(at), n_kv, D, g=g)
        if keep is not None:
            live = set((at // PAGE).tolist())
            table[r] = [id if p in live else -1 for p, id in enumerate(table[r])]
    q = _randn(b, n_q, D, g=g, scale=2.0)
    return q, kc, vc, _i32(table), _i32(lens)


def _paged_reference(q, kc, vc, table, lens, seen_of, scale):
    b, n_q, _ = q.shape
    n_kv = kc.shape[1]
    o, tol = torch.zeros(b, n_q, D, dtype=torch.float64, device="cuda"), torch.zeros(b, n_q, D, dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens.tolist()):
        at = torch.arange(n, device="cuda")
        at = at[seen_of(r, at)]
        if not len(at):
            continue
        page = table[r].long()[at // PAGE]
        k, v = (c[page, :, at % PAGE].transpose(0, 1) for c in (kc, vc))
        seen = torch.ones(n_kv, n_q // n_kv, len(at), dtype=torch.bool, device="cuda")
        oo, tt = _attend(q[r].view(n_kv, -1, D), k, v, seen, scale)
        o[r], tol[r] = oo.reshape(n_q, D), tt.reshape(n_q, D)
    return o, tol


LENS = [0, 1, 5, 63, 64, 65, 127, 128, 129, 200, 700, 1311]


@pytest.mark.parametrize("n_q,n_kv", [(4, 1), (8, 8), (6, 2), (32, 8), (10, 2), (32, 4), (16, 1), (24, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (64, 1), (100, 4), (129, 64), (300, 70), (5000, 4), (640, 130)])
def test_window_decode(n_q, n_kv, window, sinks):
    """Every head layout, windows and sinks that end inside pages, empty rows; all
    that no query sees is NaN, and its pages are gone from the table."""
    from foundry_b200 import ops

    def seen(n):
        return lambda _r, at: (at >= n - window) | (at < sinks)

    def seen_of(r, at):
        return seen(LENS[r])(r, at)

    q, kc, vc, table, lens = _paged(LENS, n_q, n_kv, seed=window + sinks, keep=seen_of)
    out = torch.full_like(q, 7.0)
    ops.window_decode_attention(q, kc, vc, table, lens, out, window, sinks, ops.SpanWorkspace())
    o, tol = _paged_reference(q, kc, vc, table, lens, seen_of, 1 / math.sqrt(D))
    _close(out, o, tol)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("n", [1, 64, 1000, 40_000])
def test_window_decode_one_row(n):
    """A single sequence: cut over as many CTAs as it has chunks; twice, bit for bit the same."""
    from foundry_b200 import ops

    q, kc, vc, table, lens = _paged([n], 32, 8, seed=n)
    ws, outs = ops.SpanWorkspace(), []
    for _ in range(3):
        out = torch.empty_like(q)
        ops.window_decode_attention(q, kc, vc, table, lens, out, 1 << 20, 0, ws, scale=0.05)
        outs.append(out)
    o, tol = _paged_reference(q, kc, vc, table, lens, lambda r, at: at >= 0, 0.05)
    _close(outs[0], o, tol)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert not ws.tickets.any()


def test_window_decode_many_rows_strided():
    """More rows than threads and CTAs, q and out as slices of wider rows; the rest of out stays."""
    from foundry_b200 import ops

    lens = [(37 * i) % 500 for i in range(700)]
    q, kc, vc, table, lens_t = _paged(lens, 8, 2, seed=3, extra=1)
    wide_q = torch.zeros(700, 1536, dtype=torch.bfloat16, device="cuda")
    wide_q[:, :1024] = q.view(700, 1024)
    wide_o = torch.full((700, 2048), 3.0, dtype=torch.bfloat16, device="cuda")
    out = wide_o[:, 512:1536].unflatten(1, (8, D))
    ops.window_decode_attention(wide_q[:, :1024].unflatten(1, (8, D)), kc, vc, table, lens_t, out, 200, 10, ops.SpanWorkspace())
    o, tol = _paged_reference(q, kc, vc, table, lens_t, lambda r, at: (at >= lens[r] - 200) | (at < 10), 1 / math.sqrt(D))
    _close(out, o, tol)
    assert (wide_o[:, :512] == 3).all() and (wide_o[:, 1536:] == 3).all()


GROUPS = [
    ([1], [1], [70]),
    ([3], [2], [128, 129, 400]),
    ([5, 1, 2], [3, 0, 1], [192, 200, 0, 150, 321, 90, 64, 130]),  # an empty row, one shorter than its prefix
    ([40, 33], [7, 4], [448 + i for i in range(40)] + [256 + 9 * i for i in range(33)]),
    ([70], [21], [21 * 64 + (i * 7) % 90 for i in range(70)]),
    ([3, 2], [301, 120], [301 * 64 + 5, 301 * 64, 19_000, 120 * 64 + 64, 1]),  # cut into many parts
]


@pytest.mark.parametrize("n_q,n_kv", [(4, 1), (8, 8), (6, 2), (32, 8), (10, 2), (32, 4), (16, 1), (28, 2)])
@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("sizes,pages,lens", GROUPS)
def test_prefix_decode(n_q, n_kv, sizes, pages, lens, share):
    from foundry_b200 import ops

    shared, r = [], 0
    for n, p in zip(sizes, pages):
        shared.append((r, n, p))
        r += n
    q, kc, vc, table, lens_t = _paged(lens, n_q, n_kv, seed=len(lens), shared=shared, extra=1)
    # a row shorter than the prefix left its part of the shared pages to the others
    for r0, n, p in shared:
        ids = table[r0, :p].long()
        kc[ids], vc[ids] = torch.nan_to_num(kc[ids]), torch.nan_to_num(vc[ids])
    plan = ops.PrefixPlan(sizes, pages, n_q, n_kv, table.shape[1], share=share)
    assert bool(plan.items_n) == share
    ws = ops.SpanWorkspace(plan.partials)
    out = torch.full_like(q, 7.0)
    ops.prefix_decode_attention(q, kc, vc, table, lens_t, out, plan, ws)
    o, tol = _paged_reference(q, kc, vc, table, lens_t, lambda r, at: at >= 0, 1 / math.sqrt(D))
    _close(out, o, tol)
    again = torch.empty_like(q)
    ops.prefix_decode_attention(q, kc, vc, table, lens_t, again, plan, ws)
    assert torch.equal(out, again) and not ws.tickets.any()


def test_prefix_decode_agrees_with_decode_attention_in_a_captured_graph():
    """Replayed while the sequences grow: lengths are read on the device."""
    from foundry_b200 import ops

    n, pages = 24, 5
    lens = [pages * PAGE + 3 * i for i in range(n)]
    q, kc, vc, table, lens_t = _paged([m + 64 for m in lens], 32, 8, seed=9, shared=[(0, n, pages)])
    lens_t = _i32(lens)
    kc, vc = torch.nan_to_num(kc), torch.nan_to_num(vc)
    plan = ops.PrefixPlan([n], [pages], 32, 8, table.shape[1], share=True)
    ws = ops.SpanWorkspace(plan.partials)
    out, ref = torch.empty_like(q), torch.empty_like(q)
    dws = ops.DecodeWorkspace(n, 32, 64)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    ops.prefix_decode_attention(q, kc, vc, table, lens_t, out, plan, ws)  # loads the kernels
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side), ops._rt.pdl():
        ops.prefix_decode_attention(q, kc, vc, table, lens_t, out, plan, ws)
        ops.window_decode_attention(q, kc, vc, table, lens_t, ref, 1 << 20, 0, ws)
    for _ in range(3):
        lens_t += 17
        graph.replay()
        torch.cuda.synchronize()
        o, tol = _paged_reference(q, kc, vc, table, lens_t, lambda r, at: at >= 0, 1 / math.sqrt(D))
        _close(out, o, tol)
        _close(ref, o, tol)
        ops.decode_attention(q, kc, vc, table, lens_t, ref, table.shape[1], dws)
        _close(ref, o, tol)


@pytest.mark.parametrize("n_q,n_kv", [(2, 1), (3, 1), (4, 4), (32, 8), (16, 1)])
@pytest.mark.parametrize("lens,window,sinks", [
    ([1], 1, 0), ([1, 2, 0, 127, 128, 129], 64, 4), ([300, 5, 700], 128, 1), ([513], 1000, 4), ([900, 130], 200, 130),
    ([1100], 1, 300), ([640], 257, 0),
    # many items for every CTA, of one key tile, of few, of both in turn
    ([(37 * i) % 128 + 1 for i in range(250)], 64, 4), ([(531 * i) % 900 for i in range(40)], 128, 4),
])
def test_window_prefill(n_q, n_kv, lens, window, sinks):
    """Packed prompts as slices of one matrix, NaN behind the last one."""
    from foundry_b200 import ops

    t, pad = sum(lens), 40
    g = _gen(t + window)
    qkv = _randn(t + pad, (n_q + 2 * n_kv) * D, g=g)
    qkv[:, : n_q * D] *= 2
    qkv[t:] = math.nan
    q, k, v = qkv.split([n_q * D, n_kv * D, n_kv * D], 1)
    out = torch.full((t + pad, n_q * D), 7.0, dtype=torch.bfloat16, device="cuda")
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    ts, tst = ops.prefill_tiles(lens)
    ops.window_prefill_attention(q, k, v, out, _i32(cu), _i32(ts), _i32(tst), n_q, n_kv, window, sinks)
    assert (out[t:] == 7).all()
    assert ops.status("attention_tile") == 0
    for a, b in zip(cu, cu[1:]):
        if a == b:
            continue
        i = torch.arange(b - a, device="cuda")
        back = i[:, None] - i[None]
        seen = (back >= 0) & ((back < window) | (i[None] < sinks))
        heads = lambda x, n: x[a:b].unflatten(1, (n, D)).transpose(0, 1)  # noqa: E731
        rep = n_q // n_kv
        o, tol = _attend(heads(q, n_q), heads(k, n_kv).repeat_interleave(rep, 0),
                         heads(v, n_kv).repeat_interleave(rep, 0), seen, 1 / math.sqrt(D))
        _close(heads(out, n_q), o, tol)
