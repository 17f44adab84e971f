"""The runner's windowed attention under a mixture-of-experts model: prefill,
decode, captured decode and log probabilities against the fp32 reference. fp8
activations, which the reference does not model, move a logit by less than 0.05
(the bound of the runner's other tests of this model): a log probability by
less than twice that."""

import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(32, 4), (64, 0)])
def test_windowed_moe(window, sinks):
    from foundry_b200 import ops
    from foundry_b200.models.qwen3_moe import reference_forward, tiny_moe
    from foundry_b200.runner.engine import EngineConfig, LLMEngine

    cfg = tiny_moe(layers=2, experts=32)
    cfg.window, cfg.sinks = window, sinks
    eng = LLMEngine(EngineConfig(model=cfg, max_batch=8, max_seq_len=256, max_prefill_tokens=1024, max_prefill_seqs=8,
                                 graph_sizes=[1, 2, 4, 8], region_base=None, region_size="16GB"))
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (1, 5, 70, 130, 200)]
    outs, lps = eng.generate_logprobs(prompts, max_new_tokens=5, top=3)
    matched, moved = 0, 0.0
    for p, o, lp in zip(prompts, outs, lps):
        ids = torch.tensor(p + o[:-1], device="cuda")
        logits, full = (reference_forward(c, eng.weights, ids, eng.cos_sin)[len(p) - 1:].double()
                        for c in (cfg, dataclasses.replace(cfg, window=0)))
        ref = logits.log_softmax(-1)
        if len(p) > window + sinks:
            moved = max(moved, (ref - full.log_softmax(-1)).abs().max().item())
        for j, (token, (value, _, top)) in enumerate(zip(o, lp)):
            assert abs(value - ref[j, token]) < 0.1
            assert top[0] == (token, value) and all(abs(v - ref[j, t]) < 0.1 for t, v in top)
            best = logits[j].topk(2)
            if best.values[0] - best.values[1] > 0.1:
                assert token == int(best.indices[0])
                matched += 1
    assert matched >= 2 and moved > 0.3, (matched, moved)  # three times what the engine may be off by
    eng.capture_graphs()
    assert eng.generate_logprobs(prompts, max_new_tokens=5, top=3) == (outs, lps)
    for img in ("moe", "attention_span", "attention_tile", "logprobs"):
        assert ops.status(img) == 0, img
