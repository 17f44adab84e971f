"""The runner with windowed attention and log probabilities: prefill, decode
(eager and captured) and the answer's probabilities, against the fp32 reference."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _engine(window=0, sinks=0, **kw):
    from foundry_b200.models.llama import tiny
    from foundry_b200.runner.engine import EngineConfig, LLMEngine

    cfg = tiny(layers=2, vocab=4096)
    cfg.window, cfg.sinks = window, sinks
    kw.setdefault("region_base", None)
    return LLMEngine(EngineConfig(model=cfg, max_batch=8, max_seq_len=512, max_prefill_tokens=1024,
                                  max_prefill_seqs=8, graph_sizes=[1, 2, 4, 8], **kw))


def _prompts(lens):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("window,sinks", [(0, 0), (32, 4), (100, 0)])
def test_generate_logprobs(window, sinks):
    """Tokens, their log probabilities, the entropy and the alternatives of a
    short generation; the bf16 forward's logits differ from the fp32 one's by
    less than 0.05 (the bound of the runner's other tests)."""
    from foundry_b200 import ops
    from foundry_b200.models.llama import reference_forward

    eng = _engine(window, sinks)
    prompts = _prompts([1, 3, 70, 200, 333])
    plain = eng.generate(prompts, max_new_tokens=6)
    outs, lps = eng.generate_logprobs(prompts, max_new_tokens=6, top=5)
    assert outs == plain
    eng.capture_graphs()
    assert eng.generate_logprobs(prompts, max_new_tokens=6, top=5) == (outs, lps)
    for p, o, lp in zip(prompts, outs, lps):
        ids = torch.tensor(p + o[:-1], device="cuda")
        logits = reference_forward(eng.ecfg.model, eng.weights, ids, eng.cos_sin)[len(p) - 1:].double()
        ref = logits.log_softmax(-1)
        assert len(lp) == len(o) == 6
        for j, (token, (value, entropy, top)) in enumerate(zip(o, lp)):
            # a shift of each logit by at most d moves a log probability by at most 2 d
            assert abs(value - ref[j, token]) < 0.1
            assert top[0] == (token, value) and len(top) == 5  # greedy
            assert all(abs(v - ref[j, t]) < 0.1 for t, v in top)
            assert all(a[1] >= b[1] for a, b in zip(top, top[1:]))
            assert abs(entropy - -(ref[j].exp() * ref[j]).sum()) < 0.1 * math.log(4096)
    for img in ("attention_span", "attention_tile", "logprobs"):
        if img in ops._rt.loaded_images():
            assert ops.status(img) == 0


def test_logprobs_refusals():
    eng = _engine()
    with pytest.raises(ValueError, match="top must be"):
        eng.generate_logprobs(_prompts([3]), max_new_tokens=2, top=33)
    assert len(eng.free_pages) == eng.num_blocks


def test_a_window_over_everything_changes_nothing():
    """Greedy tokens of a window longer than every sequence, against full attention."""
    prompts = _prompts([5, 64, 300])
    full, windowed = _engine(), _engine(window=4096, sinks=3)
    a, la = full.generate_logprobs(prompts, max_new_tokens=8, top=1)
    b, lb = windowed.generate_logprobs(prompts, max_new_tokens=8, top=1)
    for x, y, lx, ly in zip(a, b, la, lb):
        for tx, ty, px, py in zip(x, y, lx, ly):
            assert abs(px[0] - py[0]) < 0.05
            if tx != ty:  # two tokens as good as one another, from where the texts differ
                break


def test_shared_prompt_windowed_and_scored_in_one_captured_step():
    """The three together as a serving step would: attention over a shared prompt,
    attention over a window of the same cache, log probabilities of what follows;
    one graph, replayed as the sequences grow."""
    from foundry_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    n, shared, n_q, n_kv, vocab = 12, 40, 32, 8, 5000
    pages = shared + 3
    table = torch.arange(n * pages, dtype=torch.int32, device="cuda").view(n, pages)
    table[:, :shared] = table[0, :shared]
    table = table.contiguous()
    kc = torch.randn(n * pages, n_kv, 64, 128, generator=g, device="cuda").to(torch.bfloat16)
    vc = torch.randn(n * pages, n_kv, 64, 128, generator=g, device="cuda").to(torch.bfloat16)
    q = torch.randn(n, n_q, 128, generator=g, device="cuda").to(torch.bfloat16)
    head = (torch.randn(vocab, n_q * 128, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    lens = torch.arange(n, dtype=torch.int32, device="cuda") + shared * 64 + 1
    plan = ops.PrefixPlan([n], [shared], n_q, n_kv, pages, share=True)
    ws, lws = ops.SpanWorkspace(plan.partials), ops.LogprobWorkspace()
    a, b = torch.empty_like(q), torch.empty_like(q)
    logits = torch.empty(n, vocab, dtype=torch.bfloat16, device="cuda")
    ids = torch.empty(n, dtype=torch.int32, device="cuda")
    lp, entropy = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")

    def step():
        ops.prefix_decode_attention(q, kc, vc, table, lens, a, plan, ws)
        ops.window_decode_attention(a, kc, vc, table, lens, b, 100, 4, ws)
        ops.linear(b.view(n, -1), head, out=logits)
        ops.argmax(logits, ids)
        ops.token_logprobs(logits, ids, lp, entropy, ws=lws)

    step()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side), ops._rt.pdl():
        step()
    for _ in range(3):
        lens += 7
        step()
        torch.cuda.synchronize()
        want = [x.clone() for x in (a, b, logits, ids, lp, entropy)]
        for x in (a, b, logits, lp, entropy):
            x.fill_(math.nan)
        ids.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((a, b, logits, ids, lp, entropy), want):
            assert torch.equal(x, y)
        ref = logits.double().log_softmax(-1)
        torch.testing.assert_close(lp.double(), ref.gather(1, ids.long()[:, None])[:, 0], atol=1e-5, rtol=1e-5)
        assert (lp.double() == ref.amax(-1).float()).float().mean() > 0.5


def test_on_another_stream():
    from foundry_b200 import ops

    x = torch.randn(64, 50_000, device="cuda").to(torch.bfloat16)
    ids = torch.zeros(64, dtype=torch.int32, device="cuda")
    ws, a, b = ops.LogprobWorkspace(), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    ops.token_logprobs(x, ids, a, None, ws=ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-3
        y = x + big[0, 0].nan_to_num(0.0, 0.0, 0.0).to(torch.bfloat16) * 0
        ops.token_logprobs(y, ids, b, None, ws=ws)
    side.synchronize()
    assert torch.equal(a, b)
