"""What the windowed, shared-prefix and log-probability ops refuse, and how a
prefix plan and the shares of a launch are laid out: on the CPU, with the
launch replaced by one that records its numbers."""

import math

import pytest
import torch

from foundry_b200 import ops
from foundry_b200.ops import _rt
from foundry_b200.ops import logprobs as L
from foundry_b200.ops import span_attention as S


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    """CPU tensors pass as those of the current device; launches are recorded."""
    got = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)  # what get_device() says of a CPU tensor
    monkeypatch.setattr(_rt, "sm_count", lambda: 148)
    monkeypatch.setattr(_rt, "launch_mapped", lambda *a, **k: got.append((a, k)))
    return got


def _decode(b=3, n_q=8, n_kv=2, blocks=10, pages=4):
    bf = dict(dtype=torch.bfloat16)
    return dict(q=torch.zeros(b, n_q, 128, **bf), k_cache=torch.zeros(blocks, n_kv, 64, 128, **bf),
                v_cache=torch.zeros(blocks, n_kv, 64, 128, **bf),
                block_tables=torch.zeros(b, pages, dtype=torch.int32), seq_lens=torch.ones(b, dtype=torch.int32),
                out=torch.zeros(b, n_q, 128, **bf))


def _ws(**kw):
    return ops.SpanWorkspace(device="cpu", **kw)


def _window(a, window=64, sinks=0, ws=None, **kw):
    return ops.window_decode_attention(*a.values(), window, sinks, ws or _ws(), **kw)


def test_decode_launches(launches):
    _window(_decode())
    (image, kernel, grid, _, threads, smem, maps, *numbers), kw = launches.pop()
    assert (image, kernel, threads, maps) == ("attention_span", "fb_span_attn_g4", 192, 5)
    assert grid == 3 * 2 * 4 and not kw["after_own"]
    for n_q, n_kv, want in ((8, 8, "g4"), (16, 2, "g8"), (10, 2, "g8"), (16, 1, "g16"), (9, 1, "g16")):
        _window(_decode(n_q=n_q, n_kv=n_kv))
        assert launches.pop()[0][1] == "fb_span_attn_" + want
    _window(_decode(b=0))
    assert not launches


@pytest.mark.parametrize("change,what", [
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.bfloat16)), "q must be"),
    (dict(q=torch.zeros(3, 8, 128)), "q must be"),
    (dict(out=torch.zeros(3, 8, 128)), "out must be"),
    (dict(out=torch.zeros(2, 8, 128, dtype=torch.bfloat16)), "out must be"),
    (dict(out=torch.zeros(1, 8, 128, dtype=torch.bfloat16).expand(3, -1, -1)), "overlap"),
    (dict(q=torch.zeros(1, 8, 128, dtype=torch.bfloat16).expand(3, -1, -1)), "stride"),
    (dict(q=torch.zeros(3, 8, 256, dtype=torch.bfloat16)[:, :, ::2]), "next to each other"),
    (dict(q=torch.zeros(3, 8 * 128 + 4, dtype=torch.bfloat16)[:, 4:].unflatten(1, (8, 128))), "next to each other"),
    (dict(k_cache=torch.zeros(10, 2, 32, 128, dtype=torch.bfloat16)), "caches must be"),
    (dict(v_cache=torch.zeros(9, 2, 64, 128, dtype=torch.bfloat16)), "caches must be"),
    (dict(k_cache=torch.zeros(10, 2, 64, 256, dtype=torch.bfloat16)[..., :128]), "contiguous"),
    (dict(k_cache=torch.zeros(0, 2, 64, 128, dtype=torch.bfloat16),
          v_cache=torch.zeros(0, 2, 64, 128, dtype=torch.bfloat16)), "cache of no"),
    (dict(block_tables=torch.zeros(3, 4, dtype=torch.int64)), "block_tables"),
    (dict(block_tables=torch.zeros(3, 8, dtype=torch.int32)[:, ::2]), "block_tables"),
    (dict(block_tables=torch.zeros(3, 0, dtype=torch.int32)), "block_tables"),
    (dict(seq_lens=torch.ones(4, dtype=torch.int32)), "seq_lens"),
    (dict(seq_lens=torch.ones(3)), "seq_lens"),
])
def test_decode_refuses_tensors(launches, change, what):
    with pytest.raises(ValueError, match=what):
        _window({**_decode(), **change})
    assert not launches


def test_decode_refuses_numbers(launches):
    for kw, what in ((dict(window=0), "window"), (dict(window=-3), "window"), (dict(sinks=-1), "sinks"),
                     (dict(window=1 << 30), "window"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                     (dict(scale=math.nan), "scale")):
        with pytest.raises(ValueError, match=what):
            _window(_decode(), **kw)
    for n_q, n_kv in ((7, 2), (34, 2), (17, 1)):
        with pytest.raises(ValueError, match="query heads"):
            _window(_decode(n_q=n_q, n_kv=n_kv))
    assert not launches


def test_another_device_is_refused(launches, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="current CUDA device"):
        _window(_decode())
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.token_logprobs(torch.zeros(2, 5), None, None, None, ws=ops.LogprobWorkspace(device="cpu"))
    assert not launches


def test_prefix_refusals(launches):
    a = _decode()
    plan = ops.PrefixPlan([3], [2], 8, 2, 4, device="cpu", share=True)
    ok = _ws(partials=plan.partials)
    ops.prefix_decode_attention(*a.values(), plan, ok)
    (first, kw1), (second, kw2) = launches
    assert first[1].startswith("fb_prefix_attn_q") and kw1["cluster"] == plan.cluster
    assert second[1].startswith("fb_span_attn") and kw2["after_own"]
    launches.clear()
    with pytest.raises(ValueError, match="workspace of 0"):
        ops.prefix_decode_attention(*a.values(), plan, _ws())
    for other in (ops.PrefixPlan([2], [2], 8, 2, 4, device="cpu"), ops.PrefixPlan([3], [2], 16, 2, 4, device="cpu"),
                  ops.PrefixPlan([3], [2], 8, 2, 5, device="cpu")):
        with pytest.raises(ValueError, match="plan for"):
            ops.prefix_decode_attention(*a.values(), other, ok)
    for sizes, pages in (([1, 2], [1]), ([-1], [1]), ([3], [5]), ([3], [-1])):
        with pytest.raises(ValueError):
            ops.PrefixPlan(sizes, pages, 8, 2, 4, device="cpu")
    assert not launches


@pytest.mark.parametrize("sizes,pages,n_q,n_kv", [
    ([1], [1], 4, 1), ([5, 1, 2], [3, 0, 1], 6, 2), ([256], [32], 32, 8), ([37] * 4, [101] * 4, 32, 4),
    ([128], [512], 64, 8), ([3, 40], [301, 7], 16, 1), ([], [], 8, 8), ([0, 4], [3, 2], 8, 8),
])
def test_prefix_plan_covers_every_row_and_page_once(sizes, pages, n_q, n_kv):
    p = ops.PrefixPlan(sizes, pages, n_q, n_kv, 512, device="cpu", share=True)
    group = n_q // n_kv
    seen = {}
    assert p.items_n % max(1, p.cluster * p.parts) == 0 and 1 <= p.cluster <= 8
    for i, (row0, rows, page0, n, part, *_) in enumerate(p.items.tolist() if p.items_n else []):
        assert page0 % 2 == 0 and 0 <= part < p.parts and rows <= p.tiles * S.prefix_rows(group)
        first = p.items[i - i % p.cluster].tolist()
        assert first[:2] == [row0, rows] and first[4] == part  # a cluster has the same rows and part
        for r in range(row0, row0 + rows):
            for page in range(page0, page0 + n):
                assert (r, page) not in seen
                seen[r, page] = part
    want, row = set(), 0
    for n, pg in zip(sizes, pages):
        want |= {(r, page) for r in range(row, row + n) for page in range(pg)}
        assert all(v == (pg * 64 if pg else 0) for v in p.row_prefix[row:row + n].tolist())
        row += n
    assert set(seen) == want
    assert p.partials == (sum(sizes) * n_q * p.parts if p.items_n else 0)


def test_prefix_plan_reads_row_by_row_what_is_not_worth_sharing():
    assert not ops.PrefixPlan([1], [400], 32, 8, 512, device="cpu").items_n  # nobody to share with
    assert not ops.PrefixPlan([4], [8], 32, 8, 64, device="cpu").items_n
    assert ops.PrefixPlan([256], [32], 32, 8, 64, device="cpu").items_n
    assert ops.PrefixPlan([1, 256], [32, 32], 32, 8, 64, device="cpu").row_prefix[0] == 0


def _prefill(t=200, n_q=4, n_kv=2):
    bf = dict(dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32)
    return dict(q=torch.zeros(t, n_q * 128, **bf), k=torch.zeros(t, n_kv * 128, **bf),
                v=torch.zeros(t, n_kv * 128, **bf), out=torch.zeros(t, n_q * 128, **bf),
                cu_seqlens=torch.tensor([0, t], **i32), tile_seq=torch.zeros(2, **i32),
                tile_start=torch.tensor([0, 128], **i32))


def test_prefill_launches_and_refusals(launches):
    ops.window_prefill_attention(*_prefill().values(), 4, 2, 64, 4)
    assert launches.pop()[0][1] == "fb_window_prefill_q2"
    ops.window_prefill_attention(*_prefill(n_q=6).values(), 6, 2, 64, 4)
    assert launches.pop()[0][1] == "fb_window_prefill_q1"
    empty = _prefill()
    empty.update(tile_seq=torch.zeros(0, dtype=torch.int32), tile_start=torch.zeros(0, dtype=torch.int32))
    ops.window_prefill_attention(*empty.values(), 4, 2, 64, 4)
    bad = [
        dict(q=torch.zeros(200, 4 * 128)), dict(k=torch.zeros(200, 128, dtype=torch.bfloat16)),
        dict(v=torch.zeros(199, 2 * 128, dtype=torch.bfloat16)),
        dict(out=torch.zeros(200, 4 * 128 + 4, dtype=torch.bfloat16)[:, :512]),
        dict(q=torch.zeros(200, 1024, dtype=torch.bfloat16)[:, ::2]),
        dict(q=torch.zeros(1, 512, dtype=torch.bfloat16).expand(200, -1)),
        dict(cu_seqlens=torch.tensor([0, 200])), dict(tile_seq=torch.zeros(3, dtype=torch.int32)),
        dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), dict(tile_start=torch.zeros(2)),
    ]
    for change in bad:
        with pytest.raises(ValueError):
            ops.window_prefill_attention(*{**_prefill(), **change}.values(), 4, 2, 64, 4)
    for n_q, n_kv, window, sinks in ((4, 3, 64, 4), (34, 2, 64, 4), (4, 2, 0, 4), (4, 2, 64, -1)):
        with pytest.raises(ValueError):
            ops.window_prefill_attention(*_prefill().values(), n_q, n_kv, window, sinks)
    assert not launches


def test_logprobs_refusals(launches):
    ws = ops.LogprobWorkspace(device="cpu")
    x, ids, f = torch.zeros(3, 50), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    top, top_ids = torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int32)
    ops.token_logprobs(x, ids, f, f.clone(), top, top_ids, ws=ws)
    ops.token_logprobs(x.to(torch.bfloat16)[:, 1:], None, None, f, ws=ws)
    ops.token_logprobs(x[:0], ids[:0], f[:0], None, ws=ws)
    assert [a[1] for a, _ in launches] == ["fb_logprobs_f32", "fb_logprobs_bf16"]
    launches.clear()
    for args in (
        (x.double(), ids, f, None), (x[0], ids, f, None), (torch.zeros(3, 100)[:, ::2], ids, f, None),
        (x, ids.long(), f, None), (x, ids[:2], f, None), (x, ids, f[:2], None), (x, ids, f.double(), None),
        (x, ids, None, f), (x, None, f, f), (x, ids, f, None, top, None), (x, ids, f, None, None, top_ids),
        (x, ids, f, None, top, top_ids.long()), (x, ids, f, None, top.t().contiguous().t(), top_ids),
        (x, ids, f, None, torch.zeros(3, 33), torch.zeros(3, 33, dtype=torch.int32)),
        (x[:, :3], ids, f, None, top, top_ids), (x[:, :0], ids, f, None),
    ):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args, ws=ws)
    assert not launches


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 128256), (3, 4095), (100, 50257), (444, 151936), (445, 151936),
                                        (4096, 1000), (256, 128256), (20_000, 17)])
def test_logprob_shares_cover_every_logit_once(rows, vocab):
    """The kernel's walk over a CTA's flat positions, and the pieces that it counts for a row."""
    ctas = L.CTAS_PER_SM * 148
    share, pitch = L.share_of(rows, vocab, ctas)
    grid = min(ctas, math.ceil(rows * pitch / share))
    assert grid * share >= rows * pitch and share % 64 == 0 and pitch >= vocab
    pieces = {}
    for cta in range(grid):
        at, end, count = cta * share, min((cta + 1) * share, rows * pitch), 0
        while at < end:
            row, c0 = divmod(at, pitch)
            n = min(vocab - c0, end - at)
            if n <= 0:
                break
            pieces.setdefault(row, []).append((cta, c0, n, at == cta * share))
            at, count = at + n, count + 1
    assert len(pieces) == rows
    for row, got in pieces.items():
        assert [c for _, c, _, _ in got] == [sum(n for _, _, n, _ in got[:i]) for i in range(len(got))]
        assert sum(n for _, _, n, _ in got) == vocab
        first = row * pitch // share
        assert [c for c, *_ in got] == list(range(first, (row * pitch + vocab - 1) // share + 1))
        assert len(got) <= 1024  # MAX_PIECES of the kernel
        # slots: a CTA's first piece has the first one, a cut row's first piece inside a share the second
        if len(got) > 1:
            for i, (_, _, _, is_first) in enumerate(got):
                assert is_first == (not (i == 0 and row * pitch % share))


def test_sizes_that_indices_do_not_hold_are_refused(launches):
    """On tensors without that memory behind them (expanded ones, or none at all)."""
    bf = dict(dtype=torch.bfloat16, device="meta")
    a = {k: v.to("meta") for k, v in _decode().items()}
    a["block_tables"] = torch.empty(3, (1 << 24) + 1, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="too many pages"):
        S._decode_dims(*a.values())
    a["block_tables"] = torch.empty(1 << 22, 1 << 9, dtype=torch.int32, device="meta")
    a["q"] = a["out"] = torch.empty(1 << 22, 8, 128, **bf)
    a["seq_lens"] = torch.empty(1 << 22, dtype=torch.int32, device="meta")
    with pytest.raises(ValueError, match="too many pages"):
        S._decode_dims(*a.values())
    a = {k: v.to("meta") for k, v in _decode().items()}
    a["k_cache"] = a["v_cache"] = torch.empty(1 << 24, 2, 64, 128, **bf)
    with pytest.raises(ValueError, match="too many blocks"):
        S._decode_dims(*a.values())
    with pytest.raises(ValueError, match="rows of a vocabulary"):
        ops.token_logprobs(torch.zeros(1, 1).expand(1 << 30, 1), None, None, None, ws=ops.LogprobWorkspace(device="cpu"))
    far = torch.empty(1, dtype=torch.bfloat16, device="meta").as_strided((200, 512), (1 << 31, 1))
    with pytest.raises(ValueError, match="do not overlap"):
        ops.window_prefill_attention(*{**_prefill(), "out": far}.values(), 4, 2, 64, 4)
    assert not launches


def test_a_plan_of_many_groups_is_made_at_once():
    n = 20_000
    p = ops.PrefixPlan([2] * n, [4] * n, 8, 2, 8, device="cpu", share=True)
    assert p.items_n == n * p.cluster * p.parts


class _NoTensors:
    """The detailed checks alone."""

    decode = rows = staticmethod(lambda *a: None)


def test_native_checks_agree_with_the_detailed_ones(launches, monkeypatch):
    a, ws, lws = _decode(b=5, n_q=24, n_kv=3), _ws(partials=1 << 12), ops.LogprobWorkspace(device="cpu")
    plan = ops.PrefixPlan([5], [2], 24, 3, 4, device="cpu", share=True)
    x, f, i = torch.zeros(5, 90), torch.zeros(5), torch.zeros(5, dtype=torch.int32)
    top, top_ids = torch.zeros(5, 7), torch.zeros(5, 7, dtype=torch.int32)

    def calls():
        launches.clear()
        _window(a, ws=ws)
        ops.prefix_decode_attention(*a.values(), plan, ws)
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            ops.token_logprobs(x.to(dtype), i, f, f, top, top_ids, ws=lws)
        ops.token_logprobs(x[:, 3:80], None, None, f, ws=lws)
        ops.token_logprobs(x[:, :1], i, f, None, ws=lws)
        # without the address of a temporary
        return [(args[:7] if args[0] == "logprobs" else args, kw, args[8:]) for args, kw in launches]

    got = calls()
    assert len(got) == 8
    monkeypatch.setattr(S.native, "tensors", lambda: _NoTensors)
    assert calls() == got


def test_native_checks_leave_other_calls_to_the_detailed_ones():
    n = S.native.tensors()
    a = list(_decode().values())
    assert n.decode(*a, -1, 64)[:5] == (3, 8, 2, 10, 4) and n.decode(*a, 0, 64) is None
    for at, other in ((0, torch.zeros(3, 8, 136, dtype=torch.bfloat16)[..., :128]), (0, None), (1, a[1][:, :1]),
                      (1, a[1].float()), (3, a[3].long()), (4, a[4][:2]), (5, a[5].unsqueeze(0)), (4, 7)):
        assert n.decode(*a[:at], other, *a[at + 1:], -1, 64) is None
    assert n.decode(*a, -1, 32) is None
    x, f, i = torch.zeros(3, 9), torch.zeros(3), torch.zeros(3, dtype=torch.int32)
    assert n.rows(x, i, f, None, None, None, -1)[:5] == (2, 3, 9, 0, 9)
    for args in ((None, i, f, f, None, None), (x.t(), None, None, f, None, None), (x, i, None, f, None, None),
                 (x, i.long(), f, f, None, None), (x, i, f, f, f, i), (x.double(), i, f, f, None, None)):
        assert n.rows(*args, -1) is None
    for bad in ((), (1, 2), tuple(a)):
        with pytest.raises(TypeError):
            n.decode(*bad)


def test_workspace_or_plan_of_another_device_is_refused(launches):
    a, ws, lws = _decode(), _ws(partials=1 << 10), ops.LogprobWorkspace(device="cpu")
    plan = ops.PrefixPlan([3], [2], 8, 2, 4, device="cpu", share=True)
    ws.device = 1
    with pytest.raises(ValueError, match="another device"):
        _window(a, ws=ws)
    with pytest.raises(ValueError, match="another device"):
        ops.prefix_decode_attention(*a.values(), plan, ws)
    ws.device, plan.device = -1, 1
    with pytest.raises(ValueError, match="another device"):
        ops.prefix_decode_attention(*a.values(), plan, ws)
    lws.device = 1
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.token_logprobs(torch.zeros(2, 5), None, None, torch.zeros(2), ws=lws)
    assert not launches
