"""The cases by which the shared-prefix, windowed and log-probability operators are measured.

Three operators of a decode step and of prefill:

``prefix``   decode attention of a batch whose sequences share a long prompt, read once per group
``decode``   decode attention over the last ``window`` tokens and the first ``sinks`` ones of a paged cache
``prefill``  causal attention of packed prompts with the same window and sinks
``logprobs`` log probability of given tokens, entropy and the most probable alternatives

Each in its plain form (elementary torch operations in 32 bits) and, with ``own`` set, as a user calls it.
"""

from __future__ import annotations

import math

import torch

own = False

D = 128  # head dimension
PAGE = 64  # tokens of a cache page


def listed():
    return [
        # a few requests on a short system prompt: the smallest call, latency counts
        dict(name="prefix-small", op="prefix", groups=1, rows=4, n_q=32, n_kv=8, prefix_pages=8, lo=1, hi=100),
        # a full decode batch on one system prompt, Llama-3-8B heads, the bench's private lengths
        dict(name="prefix-chat", op="prefix", groups=1, rows=256, n_q=32, n_kv=8, prefix_pages=32, lo=1, hi=640),
        # four documents, each asked many questions; Qwen3-30B-A3B heads
        dict(name="prefix-documents", op="prefix", groups=4, rows=37, n_q=32, n_kv=4, prefix_pages=101, lo=17, hi=300),
        # one long context (code base, book) behind every request, Llama-3-70B heads
        dict(name="prefix-long", op="prefix", groups=1, rows=128, n_q=64, n_kv=8, prefix_pages=512, lo=50, hi=1000),
        # one stream of an endless generation: latency
        dict(name="decode-single", op="decode", batch=1, n_q=32, n_kv=8, window=1024, sinks=4, lo=5000, hi=5000),
        # a full batch of chats, many past the window, some shorter than it
        dict(name="decode-batch", op="decode", batch=256, n_q=32, n_kv=8, window=1000, sinks=4, lo=1, hi=8000),
        # long windows, a sink of one page, Qwen3-30B-A3B heads
        dict(name="decode-wide", op="decode", batch=61, n_q=32, n_kv=4, window=4096, sinks=64, lo=2000, hi=32000),
        # a chunk of short prompts of every length
        dict(name="prefill-short", op="prefill", seqs=13, n_q=32, n_kv=8, window=128, sinks=4, lo=1, hi=700),
        # one prompt of the runner's largest chunk
        dict(name="prefill-long", op="prefill", seqs=1, n_q=32, n_kv=8, window=1024, sinks=4, lo=8192, hi=8192),
        # one decoded token with five alternatives: latency
        dict(name="logprobs-single", op="logprobs", rows=1, vocab=128256, k=5, dtype="bfloat16"),
        # a decode batch with the most alternatives that serving APIs give
        dict(name="logprobs-batch", op="logprobs", rows=256, vocab=128256, k=20, dtype="bfloat16"),
        # scoring a long prompt, logits in 32 bits
        dict(name="logprobs-prompt", op="logprobs", rows=2000, vocab=151936, k=1, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["prefix", "decode", "prefill", "logprobs"])
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 200000)
        rows = _log_int(rng, 1, max(1, min(4096, 300_000_000 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, k=rng.choice([0, 1, 3, 5, 8, 20, 32]),
                    dtype=rng.choice(["bfloat16", "float32"]))
    n_kv = rng.choice([1, 2, 4, 8])
    n_q = n_kv * rng.choice([1, 2, 4, 5, 8, 16] if n_kv < 8 else [1, 3, 4, 8])
    if op == "prefix":
        groups, pages = rng.choice([1, 1, 2, 5]), _log_int(rng, 1, 512)
        rows = _log_int(rng, 1, max(1, min(256 // groups, 4_000_000 // (groups * n_q * pages))))
        lo = _log_int(rng, 1, 300)
        return dict(op=op, groups=groups, rows=rows, n_q=n_q, n_kv=n_kv, prefix_pages=pages, lo=lo,
                    hi=lo + _log_int(rng, 1, 700))
    window, sinks = _log_int(rng, 1, 4096), rng.choice([0, 1, 4, 16, 64, 100])
    if op == "decode":
        batch = _log_int(rng, 1, max(1, min(256, 2_000_000 // (n_kv * (window + sinks)))))
        lo = _log_int(rng, 1, 8000)
        return dict(op=op, batch=batch, n_q=n_q, n_kv=n_kv, window=window, sinks=sinks, lo=lo,
                    hi=lo + _log_int(rng, 1, 8000))
    seqs = _log_int(rng, 1, 30)
    lo = _log_int(rng, 1, 4000 // seqs)
    window = min(window, 900 if n_q <= 32 else 450)
    return dict(op=op, seqs=seqs, n_q=n_q, n_kv=n_kv, window=window, sinks=sinks, lo=lo,
                hi=lo + _log_int(rng, 1, 4000 // seqs))


def _lengths(case):
    """The lengths of a case's sequences: spread over [lo, hi], in no order."""
    n = {"prefix": case.get("groups", 1) * case.get("rows", 1), "decode": case.get("batch"),
         "prefill": case.get("seqs")}[case["op"]]
    span = case["hi"] - case["lo"] + 1
    return [case["lo"] + int((0.5 + 0.6180339887498949 * i) % 1.0 * span) for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16) * scale

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    st = dict(case)
    if case["op"] == "logprobs":
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        logits = torch.randn(rows, vocab, generator=g, device="cuda")
        logits = logits.mul_(2.5).to(getattr(torch, case["dtype"]))
        # the token that was sampled: a likely one in most rows
        likely = logits[:, : min(vocab, 4096)].argmax(-1)
        anyone = torch.randint(vocab, (rows,), generator=g, device="cuda")
        st["logits"], st["ids"] = logits, torch.where(anyone % 3 == 0, anyone, likely).to(torch.int32)
        f32 = dict(dtype=torch.float32, device="cuda")
        st["logprobs"], st["entropy"] = torch.empty(rows, **f32), torch.empty(rows, **f32)
        st["top_logprobs"] = torch.empty(rows, k, **f32)
        st["top_ids"] = torch.empty(rows, k, dtype=torch.int32, device="cuda")
        if own:
            from foundry_b200 import ops

            st["ws"] = ops.LogprobWorkspace()
        return st
    n_q, n_kv, lens = case["n_q"], case["n_kv"], _lengths(case)
    if case["op"] == "prefill":
        t = sum(lens)
        qkv = normal(t, (n_q + 2 * n_kv) * D)  # one matrix, as the projection leaves it
        qkv[:, : n_q * D] *= 1.5
        st["q"], st["k"], st["v"] = qkv.split([n_q * D, n_kv * D, n_kv * D], dim=1)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st["cu_seqlens"], st["out"] = i32(cu), torch.empty(t, n_q * D, dtype=torch.bfloat16, device="cuda")
        st["seq_of"] = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), i32(lens).long())
        tiles = [(i, s) for i, n in enumerate(lens) for s in range(0, n, 128)]
        st["tile_seq"], st["tile_start"] = i32([i for i, _ in tiles]), i32([s for _, s in tiles])
        return st
    # a paged cache with its pages in random order; pages that hold no visible token have been freed
    b = len(lens)
    if case["op"] == "prefix":
        shared = case["prefix_pages"]
        lens = [shared * PAGE + n for n in lens]
        tail = math.ceil(max(lens) / PAGE) - shared
        blocks = case["groups"] * shared + b * tail
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        front = order[: case["groups"] * shared].view(case["groups"], 1, shared).expand(-1, case["rows"], -1)
        st["block_tables"] = torch.cat([front.reshape(b, shared), order[case["groups"] * shared:].view(b, tail)], 1)
    else:
        pages = math.ceil(max(lens) / PAGE)
        live = [(i, p) for i, n in enumerate(lens) for p in range(math.ceil(n / PAGE))
                if p * PAGE < case["sinks"] or p * PAGE + PAGE > n - case["window"]]
        blocks = len(live)
        table = torch.zeros(b, pages, dtype=torch.int32)
        table[[i for i, _ in live], [p for _, p in live]] = torch.arange(blocks, dtype=torch.int32)
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        st["block_tables"] = order[table.cuda().long()].contiguous()
    st["block_tables"] = st["block_tables"].contiguous()
    st["seq_lens"] = i32(lens)
    st["k_cache"], st["v_cache"] = normal(blocks, n_kv, PAGE, D), normal(blocks, n_kv, PAGE, D)
    st["q"] = normal(b, n_q, D, scale=1.5)
    st["out"] = torch.empty(b, n_q, D, dtype=torch.bfloat16, device="cuda")
    if own:  # what a serving loop keeps between steps: the batch's plan and a workspace
        from foundry_b200 import ops

        partials = 0
        if case["op"] == "prefix":
            st["plan"] = ops.PrefixPlan([case["rows"]] * case["groups"], [case["prefix_pages"]] * case["groups"],
                                        n_q, n_kv, st["block_tables"].shape[1])
            partials = st["plan"].partials
        st["ws"] = ops.SpanWorkspace(partials)
    return st


def _attend(scores, visible, values):
    """softmax of the visible scores [..., g, k] times values [..., k, d]; zero where nothing is visible."""
    scores = scores.masked_fill(~visible, -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = (scores - m.masked_fill(m == -math.inf, 0.0)).exp()
    return (p @ values) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _prefix(st):
    """Shared keys in one product for the whole group, private ones per sequence, one softmax over both."""
    ng, r, p, hk = st["groups"], st["rows"], st["prefix_pages"], st["n_kv"]
    q = st["q"].float().view(ng, r, hk, -1, D) / math.sqrt(D)
    tables = st["block_tables"].long().view(ng, r, -1)

    def shared(cache):  # [groups, Hkv, tokens, D]
        return cache[tables[:, 0, :p]].float().transpose(1, 2).reshape(ng, hk, p * PAGE, D)

    def private(cache):  # [groups, rows, Hkv, tokens, D]
        return cache[tables[:, :, p:]].float().transpose(2, 3).reshape(ng, r, hk, -1, D)

    k, v = shared(st["k_cache"]), shared(st["v_cache"])
    s1 = torch.einsum("nrhgd,nhkd->nrhgk", q, k)
    s2 = q @ private(st["k_cache"]).transpose(-1, -2)
    pos = p * PAGE + torch.arange(s2.shape[-1], device=q.device)
    s2 = s2.masked_fill((pos >= st["seq_lens"].view(ng, r, 1))[:, :, None, None], -math.inf)
    m = torch.maximum(s1.amax(-1, keepdim=True), s2.amax(-1, keepdim=True))
    p1, p2 = (s1 - m).exp_(), (s2 - m).exp_()
    o = torch.einsum("nrhgk,nhkd->nrhgd", p1, v) + p2 @ private(st["v_cache"])
    o = o / (p1.sum(-1, keepdim=True) + p2.sum(-1, keepdim=True))
    return o.reshape(st["out"].shape).to(torch.bfloat16)


def _decode(st):
    """The sinks' and the window's tokens of every sequence, gathered."""
    b, hk, w, n = st["batch"], st["n_kv"], st["window"], st["seq_lens"].long()[:, None]
    sink = torch.arange(st["sinks"], device="cuda").expand(b, -1)
    recent = n - w + torch.arange(w, device="cuda")
    pos = torch.cat([sink, recent], 1)
    visible = torch.cat([sink < n, recent >= st["sinks"]], 1)
    at = pos.clamp_min(0) * visible
    page = st["block_tables"].long().gather(1, at // PAGE)
    k, v = (st[c][page, :, at % PAGE].float().transpose(1, 2) for c in ("k_cache", "v_cache"))
    q = st["q"].float().view(b, hk, -1, D) / math.sqrt(D)
    o = _attend(q @ k.transpose(-1, -2), visible[:, None, None], v)
    return o.reshape(st["out"].shape).to(torch.bfloat16)


def _prefill(st):
    """All tokens against all, masked to the same prompt, the past, and the window or the sinks."""
    t, hk = st["q"].shape[0], st["n_kv"]
    seq = st["seq_of"]
    pos = torch.arange(t, device="cuda") - st["cu_seqlens"].long()[seq]
    i, j = pos[:, None], pos[None]
    visible = (seq[:, None] == seq[None]) & (j <= i) & ((j > i - st["window"]) | (j < st["sinks"]))
    q = st["q"].float().view(t, hk, -1, D).permute(1, 2, 0, 3) / math.sqrt(D)
    k, v = (st[c].float().view(t, hk, 1, D).permute(1, 2, 0, 3) for c in ("k", "v"))
    o = _attend(q @ k.transpose(-1, -2), visible, v)
    return o.permute(2, 0, 1, 3).reshape(t, -1).to(torch.bfloat16)


def _logprobs(st):
    x = st["logits"].float()
    y = x - x.amax(-1, keepdim=True)
    e = y.exp()
    z = e.sum(-1, keepdim=True)
    lse = z.log()
    entropy = lse[:, 0] - (e * y).sum(-1) / z[:, 0]
    logprobs = y.gather(1, st["ids"].long()[:, None])[:, 0] - lse[:, 0]
    if not st["k"]:
        return [logprobs, entropy]
    value, index = torch.sort(y, dim=-1, descending=True, stable=True)  # equal logits: the lowest token first
    return [logprobs, entropy, value[:, : st["k"]] - lse, index[:, : st["k"]].to(torch.int32)]


def run(st):
    if not own:
        return {"prefix": _prefix, "decode": _decode, "prefill": _prefill, "logprobs": _logprobs}[st["op"]](st)
    from foundry_b200 import ops

    if st["op"] == "prefix":
        return ops.prefix_decode_attention(st["q"], st["k_cache"], st["v_cache"], st["block_tables"], st["seq_lens"],
                                           st["out"], st["plan"], st["ws"])
    if st["op"] == "decode":
        return ops.window_decode_attention(st["q"], st["k_cache"], st["v_cache"], st["block_tables"], st["seq_lens"],
                                           st["out"], st["window"], st["sinks"], st["ws"])
    if st["op"] == "prefill":
        return ops.window_prefill_attention(st["q"], st["k"], st["v"], st["out"], st["cu_seqlens"], st["tile_seq"],
                                            st["tile_start"], st["n_q"], st["n_kv"], st["window"], st["sinks"])
    if not st["k"]:
        ops.token_logprobs(st["logits"], st["ids"], st["logprobs"], st["entropy"], ws=st["ws"])
        return [st["logprobs"], st["entropy"]]
    ops.token_logprobs(st["logits"], st["ids"], st["logprobs"], st["entropy"], st["top_logprobs"], st["top_ids"],
                       ws=st["ws"])
    return [st["logprobs"], st["entropy"], st["top_logprobs"], st["top_ids"]]


def work(case):
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        size = {"bfloat16": 2, "float32": 4}[case["dtype"]]
        return {"bytes": rows * (vocab * size + 4 + 8 + 8 * case["k"]), "flops": rows * vocab * 6}
    lens, n_q, n_kv = _lengths(case), case["n_q"], case["n_kv"]
    kv, qo = 2 * n_kv * D * 2, 2 * n_q * D * 2  # bytes of a cached token; of a query and its output
    if case["op"] == "prefix":
        shared = case["prefix_pages"] * PAGE
        return {"bytes": (case["groups"] * shared + sum(lens)) * kv + len(lens) * (qo + 4),
                "flops": 4 * D * n_q * sum(shared + n for n in lens)}
    w, s = case["window"], case["sinks"]
    if case["op"] == "decode":
        seen = sum(min(n, w + min(s, max(0, n - w))) for n in lens)
        return {"bytes": seen * kv + len(lens) * (qo + 4), "flops": 4 * D * n_q * seen}
    pairs = sum(min(i + 1, w + min(s, max(0, i + 1 - w))) for n in lens for i in range(n))
    return {"bytes": sum(lens) * (kv + qo), "flops": 4 * D * n_q * pairs}


def exact(case, seed):
    """From the definitions in 64 bits, one sequence (and one head, one block of rows) after another."""
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        got = []
        for x, ids in zip(st["logits"].split(256), st["ids"].split(256)):
            lp = torch.log_softmax(x.double(), -1)
            entropy = -torch.special.xlogy(lp.exp(), lp.exp()).sum(-1)
            got.append([lp.gather(1, ids.long()[:, None])[:, 0], entropy])
            if case["k"]:
                # only what reaches the k-th value is put in order: equal logits by their index
                kth = x.double().topk(min(case["k"], x.shape[1]), -1).values[:, -1:]
                rest = torch.where(x.double() >= kth, x.double(), -math.inf)
                order = torch.argsort(rest, dim=-1, descending=True, stable=True)[:, : case["k"]]
                got[-1] += [lp.gather(1, order), order.to(torch.int32)]
        return [torch.cat(v) for v in zip(*got)]
    n_q, n_kv = case["n_q"], case["n_kv"]
    group, out = n_q // n_kv, torch.empty(st["out"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "prefill":
        cu = st["cu_seqlens"].tolist()
        for a, b in zip(cu, cu[1:]):
            i = torch.arange(b - a, device="cuda")
            back = i[:, None] - i[None]
            seen = (back >= 0) & ((back < case["window"]) | (i[None] < case["sinks"]))
            for h in range(n_q):
                c = slice(h // group * D, h // group * D + D)
                s = st["q"][a:b, h * D:h * D + D].double() @ st["k"][a:b, c].double().T / math.sqrt(D)
                p = torch.softmax(torch.where(seen, s, -math.inf), -1)
                out[a:b, h * D:h * D + D] = p @ st["v"][a:b, c].double()
        return out
    for r, n in enumerate(st["seq_lens"].tolist()):
        at = torch.arange(n, device="cuda")
        if case["op"] == "decode":
            at = at[(at >= n - case["window"]) | (at < case["sinks"])]
        page = st["block_tables"][r].long()[at // PAGE]
        k, v = st["k_cache"][page, :, at % PAGE].double(), st["v_cache"][page, :, at % PAGE].double()
        s = torch.einsum("hgd,thd->hgt", st["q"][r].double().view(n_kv, group, D), k) / math.sqrt(D)
        out[r] = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), v).reshape(n_q, D)
    return out
