"""Attention over part of the context (csrc/kernels/attention_span.cu,
attention_tile.cu): decode for a batch whose sequences share a long prompt,
and a sliding window with sinks for decode and prefill. head_dim is 128, the
KV page 64 tokens, tensors bf16, 1 to 16 query heads per KV head.

Window and sinks: the query at position i sees key j iff ``j <= i`` and
(``j > i - window`` or ``j < sinks``).

A decode call is one launch (two with a shared prefix) that needs no plan of
the lengths: it reads them on the device, so a captured graph stays valid as
sequences grow.
"""

from __future__ import annotations

import math
import operator

import torch

from .. import _native as native
from . import _rt
from .attention import LOG2E, PAGE

_SPAN, _TILE = "attention_span", "attention_tile"
MAX_GROUP = 16
SPAN_SMEM = 74 * 1024
TILE_SMEM = {1: 108 * 1024, 2: 227 * 1024}
PREFIX_THREADS = {1: 192, 2: 384}  # by query tiles per CTA
PREFILL_THREADS = {1: 192, 2: 512}
TILE = 128  # queries (and keys) of a tile
_BF16, _I32 = torch.bfloat16, torch.int32


def _check(cond: bool, what: str) -> None:
    if not cond:
        raise ValueError(what)


def _check_device(*tensors: torch.Tensor) -> int:
    cur = torch.cuda.current_device()
    for t in tensors:
        if t.get_device() != cur:
            raise ValueError(f"tensors must be on the current CUDA device {cur}, got one on {t.device}")
    return cur


def _check_scale(scale: float | None) -> float:
    if scale is None:
        return 1.0 / math.sqrt(128)
    if not 2.0**-120 <= scale <= 2.0**120:  # (NaN is neither; beyond, fp32 holds it as zero or not at all)
        raise ValueError(f"scale must be positive and in fp32's range, got {scale}")
    return float(scale)


def _check_window(window: int, sinks: int) -> tuple[int, int]:
    """As plain integers: a float among a launch's numbers reaches the kernel as its bits."""
    try:
        window, sinks = operator.index(window), operator.index(sinks)
    except TypeError:
        raise ValueError(f"window and sinks must be whole numbers, got {window!r}, {sinks!r}") from None
    if not (0 < window < 1 << 30 and 0 <= sinks < 1 << 30):
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window}, {sinks}")
    return window, sinks


def _check_group(n_q: int, n_kv: int) -> int:
    if not (n_kv > 0 and n_q % n_kv == 0 and 1 <= n_q // n_kv <= MAX_GROUP):
        raise ValueError(f"{n_q} query heads for {n_kv} KV heads: a whole number from 1 to {MAX_GROUP} per KV head")
    return n_q // n_kv


def _decode_dims(q, k_cache, v_cache, block_tables, seq_lens, out) -> tuple[int, ...]:
    """(batch, n_q, n_kv, blocks, max_blocks, the tensors' addresses, row strides
    of q and out, device) of a decode call, or a ValueError."""
    cur = torch.cuda.current_device()
    numbers = native.tensors().decode(q, k_cache, v_cache, block_tables, seq_lens, out, cur, PAGE)
    if numbers is not None:  # what almost every call is; anything else is looked at one by one
        return *numbers, cur
    _check(q.dim() == 3 and q.shape[2] == 128 and q.dtype == _BF16, "q must be bf16 [batch, heads, 128]")
    b, n_q, _ = q.shape
    _check(out.shape == q.shape and out.dtype == _BF16, "out must be bf16 of q's shape")
    for t in (q, out):
        _check(t.stride(2) == 1 and t.stride(1) == 128 and (t.stride(0) % 8 == 0 or b == 1) and t.data_ptr() % 16 == 0,
               "q and out must hold a row's heads next to each other, rows at multiples of 16 bytes")
    _check(b <= 1 or out.stride(0) >= n_q * 128, "out's rows overlap")
    _check(b <= 1 or q.stride(0) > 0, "q's row stride must be positive")
    _check(k_cache.dim() == 4 and tuple(k_cache.shape[2:]) == (PAGE, 128) and k_cache.shape == v_cache.shape
           and k_cache.dtype == _BF16 and v_cache.dtype == _BF16, f"caches must be bf16 [blocks, kv heads, {PAGE}, 128]")
    _check(k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.data_ptr() % 16 == 0
           and v_cache.data_ptr() % 16 == 0, "caches must be contiguous and 16-byte aligned")
    blocks, n_kv = k_cache.shape[:2]
    _check(blocks > 0 and (blocks + 1) * n_kv * PAGE < 1 << 31, "cache of no or too many blocks")
    _check(block_tables.dtype == _I32 and block_tables.dim() == 2 and block_tables.shape[0] == b
           and block_tables.is_contiguous(), "block_tables must be contiguous int32 [batch, max_blocks]")
    _check(seq_lens.dtype == _I32 and tuple(seq_lens.shape) == (b,) and seq_lens.is_contiguous(),
           "seq_lens must be contiguous int32 [batch]")
    max_blocks = block_tables.shape[1]
    _check(0 < max_blocks <= 1 << 24 and b * n_kv * (max_blocks // 2 + 2) < 1 << 30, "block_tables of no or too many pages")
    _check_device(q, k_cache, v_cache, block_tables, seq_lens, out)
    ld = n_q * 128
    return (b, n_q, n_kv, blocks, max_blocks, *(t.data_ptr() for t in (q, k_cache, v_cache, block_tables, seq_lens, out)),
            *(t.stride(0) if b > 1 else ld for t in (q, out)), cur)


def span_ctas(group: int, sms: int) -> int:
    """CTAs of a decode launch: all that are resident at once."""
    return sms * (3 if group <= 8 else 2)


class SpanWorkspace:
    """Partial results of the decode calls: two pieces per CTA (the same for
    every batch and length), and the results of shared prefixes for
    ``partials`` (row, head, part) results (``PrefixPlan.partials``). With
    ``arena`` the buffers come from it (a runner whose graphs are saved).

    Calls that may run at the same time need a workspace each; calls in stream
    order, captured graphs among them, may share one. Every call leaves
    ``tickets`` zeroed; ``clear()`` puts that right after a device-side error."""

    def __init__(self, partials: int = 0, arena=None, device=None):
        if arena is not None:
            empty, zeros = arena.empty, arena.zeros
        else:
            device = device or torch.device("cuda", torch.cuda.current_device())
            empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
            zeros = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device=device)  # noqa: E731
        self.sms = _rt.sm_count()
        self.ctas = [span_ctas(g, self.sms) for g in range(MAX_GROUP + 1)]  # of a launch, by heads per KV head
        pieces = max(2 * span_ctas(g, self.sms) * p for g, p in ((8, 8), (16, 16)))  # (piece, head) pairs
        self.o = empty((pieces * 128,), torch.float32)
        self.ml = empty((pieces * 2,), torch.float32)
        self.tickets = zeros((span_ctas(1, self.sms),), torch.int32)
        self.partials = partials
        self.prefix_o = empty((max(partials, 1) * 128,), torch.float32)
        self.prefix_ml = empty((max(partials, 1) * 2,), torch.float32)
        self.o_ptr, self.ml_ptr, self.tickets_ptr = self.o.data_ptr(), self.ml.data_ptr(), self.tickets.data_ptr()
        self.prefix_o_ptr, self.prefix_ml_ptr = self.prefix_o.data_ptr(), self.prefix_ml.data_ptr()
        self.device = self.tickets.get_device()

    def clear(self) -> None:
        self.tickets.zero_()


def _span(dims, ws: SpanWorkspace, window: int, sinks: int, scale: float, plan: "PrefixPlan | None" = None) -> None:
    b, n_q, n_kv, blocks, max_blocks, q, k, v, tables, lens, out, ld_q, ld_out, device = dims
    g, rows = n_q // n_kv, blocks * n_kv * PAGE
    if ws.device != device:
        raise ValueError("the workspace is on another device")
    _rt.launch_mapped(
        _SPAN, "fb_span_attn_g4" if g <= 4 else "fb_span_attn_g8" if g <= 8 else "fb_span_attn_g16",
        min(ws.ctas[g], b * n_kv * (max_blocks // 2 + 2)), 1, 192, SPAN_SMEM, 5,
        k, 128, rows, 256, PAGE, 0, 0, v, 128, rows, 256, PAGE, 0, 0, k, 128, rows, 256, 16, 0, 0,
        v, 128, rows, 256, 16, 0, 0,
        # q's heads are a dimension of their own: one box holds a KV head's heads of one row
        q, 128, n_q, 256, g, b, ld_q * 2,
        tables, max_blocks, blocks, lens, out, ld_out, b, n_kv, g,
        window, sinks, plan.row_prefix_ptr if plan else 0, ws.prefix_o_ptr, ws.prefix_ml_ptr,
        plan.parts if plan else 0, ws.o_ptr, ws.ml_ptr, ws.tickets_ptr, scale * LOG2E, device=device,
        after_own=plan is not None)


def window_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                            seq_lens: torch.Tensor, out: torch.Tensor, window: int, sinks: int, ws: SpanWorkspace,
                            scale: float | None = None) -> torch.Tensor:
    """Decode attention over the last ``window`` tokens (the current one among
    them) and the first ``sinks`` ones. Arguments as for ``decode_attention``;
    q and out [B, Hq, 128] may have any row stride that is a multiple of 8.

    Block-table entries of pages without a visible token are never read: their
    pages may have been freed. Rows of length 0 get zeros."""
    dims = _decode_dims(q, k_cache, v_cache, block_tables, seq_lens, out)
    _check_group(dims[1], dims[2])
    window, sinks = _check_window(window, sinks)
    scale = _check_scale(scale)
    if dims[0]:
        _span(dims, ws, window, sinks, scale)
    return out


def prefix_rows(group: int) -> int:
    """Sequences of a 128-row query tile: whole groups of 8 rows per head."""
    return (128 // group) & ~7


# Clusters of c CTAs of fb_prefix_attn_q2 that 148 SMs hold at a time (measured by
# the second wave's appearance: a cluster lies in one GPC, so not every SM is in
# one); of fb_prefix_attn_q1, two CTAs per SM, twice as many.
_CLUSTERS = {1: 148, 2: 72, 3: 44, 4: 32, 5: 24, 6: 16, 7: 14, 8: 13}


_PREFIX_LEAST_US = 7.0  # of the prefix kernel: start, end and join


def _prefix_us(kinds: list[tuple[int, int]], tiles: int, cluster: int, parts: int, sms: int) -> float:
    """Estimated microseconds of the prefix kernel for ``kinds`` of (key tiles,
    query tiles x KV heads), the longest first: ``parts`` clusters of ``cluster``
    CTAs for each query tile, which have an equal part of the keys each. Measured
    on 148 SMs: 2.1 us per key tile with two query tiles per CTA, 2.2 with two
    CTAs per SM, 1.8 with one, and 7 us for start, end and join; 0.7 us per further
    part in the kernel that goes on from them. Clusters run in waves of as many as
    the SMs hold, a wave as long as its longest cluster.

    Clusters of different lengths are not started longest first, KV head by KV
    head: 12 us per further wave and 8 per further part came closest to the best
    of all shapes in 12 measured mixtures (6% above it on average, at most 22%; 15%
    and 43% with every cluster taken for as long as the longest)."""
    held, splits = _clusters_held(tiles, cluster, sms), cluster * parts
    step = _step_us(tiles, sum(n for _, n in kinds) * splits, sms)
    wave, part = (12.0, 8.0) if kinds[0][0] != kinds[-1][0] else (0.0, 0.7)
    us, clusters, waves = part * (parts - 1) - wave, 0, 0
    for keys, n in kinds:
        clusters += n * parts
        begun = -(-clusters // held)
        if begun > waves:
            us += (begun - waves) * (-(-keys // splits) * step + _PREFIX_LEAST_US + wave)
            waves = begun
    return us


def _clusters_held(tiles: int, cluster: int, sms: int) -> int:
    return max(1, _CLUSTERS[cluster] * (3 - tiles) * sms // 148)


def _step_us(tiles: int, ctas: int, sms: int) -> float:
    return 2.1 if tiles == 2 else 2.2 if ctas > sms else 1.8


def _few_bits(x: int) -> int:
    """x rounded up to three significant bits."""
    low = max(0, x.bit_length() - 3)
    return -(-x >> low) << low


def _share(groups: list[tuple[int, int]], group: int, n_kv: int, share: bool | None) -> tuple[set, int, int, int]:
    """(the (rows, pages) to share, query tiles per CTA, cluster size, parts) with
    the least estimated time of the prefix kernel and of reading the other groups'
    prefixes row by row. ``share`` True: all of them, None: those that are worth it."""
    nb, sms, longest = prefix_rows(group), _rt.sm_count(), max((p + 1) // 2 for _, p in groups)
    # kinds of groups: (rows, key tiles) -> [groups, us to read them row by row at 85% of the HBM rate, (rows, pages)]
    kinds: dict = {}
    coarse = len(set(groups)) > 64  # many different ones: alike to a few bits are alike, so that the search stays short
    for n, p in groups:
        keys = (p + 1) // 2
        kind = kinds.setdefault((_few_bits(n), _few_bits(keys)) if coarse else (n, keys), [0, 0.0, set()])
        kind[0] += 1
        kind[1] += n * p * PAGE * n_kv * 512 / 5.5e6
        kind[2].add((n, p))
    kinds = sorted(((keys, n, count, us, which) for (n, keys), (count, us, which) in kinds.items()),
                   key=lambda kind: -kind[0])
    again = sum(kind[3] for kind in kinds)
    if not share and again <= _PREFIX_LEAST_US:
        return set(), 1, 1, 1
    best, mixed = (math.inf if share else again, 1, 1, 1, []), not share and len(kinds) > 1
    for t in (1, 2):
        work = [(keys, n_kv * count * -(-n // (nb * t))) for keys, n, count, _, _ in kinds]
        step = _step_us(t, sms + 1, sms)
        for c in _CLUSTERS:
            held = _clusters_held(t, c, sms)
            for p in (1, 2, 4, 8):
                if c * p > max(1, longest):
                    break
                us = _prefix_us(work, t, c, p, sms)
                if us < best[0]:
                    best = us, t, c, p, kinds
                if not mixed:
                    continue
                # without the kinds that save less than their part of the SMs' time
                paid = [i for i, (keys, n) in enumerate(work) if kinds[i][3] > n * p * (
                    -(-keys // (c * p)) * step + _PREFIX_LEAST_US) / held]
                if 0 < len(paid) < len(kinds):
                    us = _prefix_us([work[i] for i in paid], t, c, p, sms) + again - sum(kinds[i][3] for i in paid)
                    if us < best[0]:
                        best = us, t, c, p, [kinds[i] for i in paid]
    return {g for kind in best[4] for g in kind[4]}, *best[1:4]


class PrefixPlan:
    """Which rows of a decode batch share how many leading pages.

    Group g holds the next ``group_sizes[g]`` rows; the first
    ``prefix_pages[g]`` entries of their block tables are the same pages
    (0: nothing shared). The lengths need not be known, only that; a row may
    even be shorter than its prefix (a padding row of length 0). The plan
    holds until the batch's composition changes: captured graphs read it, so
    it has to outlive them.

    Groups that are too small, or prefixes too short, for the shared pages'
    extra kernel to pay are read row by row (``share=None``: each group by an
    estimate of both; True and False decide for all)."""

    def __init__(self, group_sizes: list[int], prefix_pages: list[int], n_q: int, n_kv: int, max_blocks: int,
                 arena=None, device=None, share: bool | None = None):
        group = _check_group(n_q, n_kv)
        try:
            group_sizes, prefix_pages = ([operator.index(x) for x in v] for v in (group_sizes, prefix_pages))
        except TypeError:
            raise ValueError(f"group sizes and prefix pages must be whole numbers, got {group_sizes}, {prefix_pages}") from None
        _check(len(group_sizes) == len(prefix_pages), "one number of prefix pages for each group")
        _check(all(n >= 0 for n in group_sizes) and all(0 <= p <= max_blocks for p in prefix_pages),
               f"group sizes must not be negative, prefixes 0 to {max_blocks} pages")
        self.n_q, self.n_kv, self.max_blocks = n_q, n_kv, max_blocks
        self.rows = sum(group_sizes)
        least = 1 if share else 2  # rows that can share anything
        groups = [(n, p) for n, p in zip(group_sizes, prefix_pages) if n >= least and p]
        shared, self.tiles, self.cluster, self.parts = set(), 1, 1, 1
        if groups and (share is None or share):
            shared, self.tiles, self.cluster, self.parts = _share(groups, group, n_kv, share)
        nb, splits = prefix_rows(group), self.cluster * self.parts
        items, info, row = [], [], 0
        for n, pages in zip(group_sizes, prefix_pages):
            is_shared = n >= least and (n, pages) in shared
            if is_shared:
                keys = math.ceil(pages / 2)
                cuts = [min(2 * (keys * s // splits), pages) for s in range(splits + 1)]
                for r0 in range(0, n, nb * self.tiles):
                    items += [[row + r0, min(nb * self.tiles, n - r0), a, e - a, s // self.cluster, 0, 0, 0]
                              for s, (a, e) in enumerate(zip(cuts, cuts[1:]))]
            info += [pages * PAGE if is_shared else 0] * n
            row += n
        self.kernel = f"fb_prefix_attn_q{self.tiles}"
        self.items_n = len(items)
        # (row, head, part) results that a SpanWorkspace has to hold
        self.partials = self.rows * n_q * self.parts if items else 0
        host = torch.tensor([x for item in items or [[0] * 8] for x in item] + (info or [0]), dtype=_I32)
        if arena is not None:
            on_device = arena.empty(tuple(host.shape), _I32)
            on_device.copy_(host)
        else:
            on_device = host.to(device or torch.device("cuda", torch.cuda.current_device()))
        n = 8 * max(1, len(items))
        self.items, self.row_prefix = on_device[:n].view(-1, 8), on_device[n:]
        self.items_ptr, self.row_prefix_ptr = self.items.data_ptr(), self.row_prefix.data_ptr()
        self.device = on_device.get_device()


def prefix_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                            seq_lens: torch.Tensor, out: torch.Tensor, plan: PrefixPlan, ws: SpanWorkspace,
                            scale: float | None = None) -> torch.Tensor:
    """Decode attention for a batch whose rows share leading pages by groups
    (``plan``): each group's shared pages are read once, for all its rows. The
    result and the arguments are those of ``decode_attention`` (``seq_lens``
    counts all tokens, ``block_tables`` begin with the shared pages). Rows of
    length 0 get zeros. A row that is shorter than its group's prefix needs the
    values that the longer ones see of it to be finite (it takes them times zero)."""
    dims = _decode_dims(q, k_cache, v_cache, block_tables, seq_lens, out)
    b, n_q, n_kv, blocks, max_blocks, q_ptr, k, v, tables, lens, _, ld_q, _, device = dims
    if (plan.rows, plan.n_q, plan.n_kv, plan.max_blocks) != (b, n_q, n_kv, max_blocks):
        raise ValueError(f"plan for {plan.rows} rows, {plan.n_q} / {plan.n_kv} heads and {plan.max_blocks} pages, "
                         f"got {b}, {n_q} / {n_kv} and {max_blocks}")
    if plan.partials > ws.partials:
        raise ValueError(f"workspace of {ws.partials} partial results, {plan.partials} needed")
    scale = _check_scale(scale)
    if not b:
        return out
    if plan.device != device or ws.device != device:
        raise ValueError("the plan or the workspace is on another device")
    if plan.items_n:
        g, rows = n_q // n_kv, blocks * n_kv * PAGE
        _rt.launch_mapped(
            _TILE, plan.kernel, plan.items_n, n_kv, PREFIX_THREADS[plan.tiles], TILE_SMEM[plan.tiles], 3,
            q_ptr, n_q * 128, b, ld_q * 2, prefix_rows(g), 0, 0,
            k, 128, rows, 256, PAGE, 0, 0, v, 128, rows, 256, PAGE, 0, 0,
            plan.items_ptr, tables, max_blocks, lens, ws.prefix_o_ptr,
            ws.prefix_ml_ptr, g, n_q, n_kv, plan.parts, blocks, scale * LOG2E, device=device, cluster=plan.cluster)
    _span(dims, ws, 0, 0, scale, plan if plan.items_n else None)
    return out


def window_prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                             cu_seqlens: torch.Tensor, tile_seq: torch.Tensor, tile_start: torch.Tensor,
                             n_q: int, n_kv: int, window: int, sinks: int,
                             scale: float | None = None) -> torch.Tensor:
    """Causal attention over packed prompts with a sliding window and sinks.
    q: [T, *] with head h at columns h * 128 (row stride q.stride(0)); k, v
    likewise with n_kv heads; out [T, n_q * 128]. The tile tables come from
    ``prefill_tiles(seqlens)``; a tile that starts behind its prompt's end is
    skipped (padding). Rows outside every prompt are neither used (they may hold
    anything) nor written. All of a prompt's k and v must be finite: a query takes
    what it does not see times zero where other queries of its 128 see it or where
    the tile of 128 keys reaches over its window."""
    group = _check_group(n_q, n_kv)
    window, sinks = _check_window(window, sinks)
    scale = _check_scale(scale)
    maps = []
    t = q.shape[0]
    for x, heads in ((q, n_q), (k, n_kv), (v, n_kv), (out, n_q)):
        if not (x.dim() == 2 and x.dtype is _BF16 and x.shape[0] == t and x.shape[1] >= heads * 128):
            raise ValueError(f"q, k, v and out must be bf16 [T, heads * 128] or wider, got {x.dtype} {tuple(x.shape)} for {heads} heads")
        ld, inner = x.stride()
        if t == 1:
            ld = heads * 128
        if inner != 1 or ld % 8 or not heads * 128 <= ld < 1 << 30 or x.data_ptr() % 16:
            raise ValueError("q, k, v and out must be row-contiguous with 16-byte aligned rows that do not overlap")
        maps += x.data_ptr(), heads * 128, t, ld * 2, TILE, 0, 0
    for x in (cu_seqlens, tile_seq, tile_start):
        if not (x.dtype is _I32 and x.dim() == 1 and x.is_contiguous()):
            raise ValueError("cu_seqlens and the tile tables must be contiguous int32")
    n_tiles, n_seqs = tile_seq.shape[0], cu_seqlens.shape[0] - 1
    if tile_start.shape[0] != n_tiles or n_seqs < 0:
        raise ValueError("tile tables of different lengths, or no cu_seqlens")
    if n_tiles * n_q >= 1 << 30:
        raise ValueError(f"{n_tiles} tiles of {n_q} heads are too many")
    _check_device(q, k, v, out, cu_seqlens, tile_seq, tile_start)
    if not n_tiles or not n_seqs or not t:
        return out
    # Two heads of one KV head share its K/V tiles (8192 tokens, 32 / 8 heads: 154 us, a head at a time 216).
    qt = 2 if group % 2 == 0 else 1
    _rt.launch_mapped(
        _TILE, "fb_window_prefill_q2" if qt == 2 else "fb_window_prefill_q1",
        min(n_tiles * (n_q // qt), _rt.sm_count() * (3 - qt)), 1, PREFILL_THREADS[qt], TILE_SMEM[qt], 3, *maps[:21],
        out.data_ptr(), ld, t, n_seqs, cu_seqlens.data_ptr(), tile_seq.data_ptr(), tile_start.data_ptr(),
        n_tiles, n_q, n_kv, window, sinks, scale * LOG2E)
    return out
