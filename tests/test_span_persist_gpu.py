"""Saved and restored in fresh processes: the decode graphs of a windowed
engine, and a graph of the shared-prefix, windowed and log-probability kernels
(thread-block clusters and a programmatic edge among its nodes)."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ENGINE = r"""
import json, os, sys
sys.path.insert(0, ROOT)
import torch
from foundry_b200 import ops
from foundry_b200.models.llama import tiny
from foundry_b200.runner.engine import EngineConfig, LLMEngine
from foundry_b200.runner import persist

cfg = tiny(layers=2, vocab=4096)
cfg.window, cfg.sinks = 64, 4
g = torch.Generator().manual_seed(3)
PROMPTS = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (5, 40, 64, 200, 117)]
"""

ENGINE_SAVE = ENGINE + r"""
ecfg = EngineConfig(model=cfg, max_batch=8, max_seq_len=256, max_prefill_tokens=512, max_prefill_seqs=8,
                    graph_sizes=[1, 2, 4, 8], region_base=0x640000000000, region_size="8GB")
eng = LLMEngine(ecfg)
persist.save(eng, ARCHIVE)
out, lps = eng.generate_logprobs(PROMPTS, 12, top=3)
json.dump([out, lps], open(os.path.join(ARCHIVE, "tokens.json"), "w"))
eng.close()
print("SAVE_OK")
"""

ENGINE_LOAD = ENGINE + r"""
eng, t = persist.load(ARCHIVE)
assert eng.ecfg.model.window == 64 and eng.ecfg.model.sinks == 4
want = json.load(open(os.path.join(ARCHIVE, "tokens.json")))
for _ in range(2):
    got = json.loads(json.dumps(eng.generate_logprobs(PROMPTS, 12, top=3)))
    assert got == want, (got, want)
    eng.wait_materialized()
assert not eng.state.span_ws.tickets.any()
for img in ("attention_span", "logprobs"):
    assert ops.status(img) == 0, img
eng.close()
print("LOAD_OK")
"""

STEP = r"""
import os, sys
sys.path.insert(0, ROOT)
import torch
import foundry_b200 as fb
from foundry_b200 import ops
from foundry_b200.runner.arena import Arena

if LOADING:
    fb.load_cuda_modules_and_libraries(ARCHIVE)
torch.cuda.init()
arena = Arena(0x650000000000, "4GB", torch.device("cuda", 0))
n, shared, n_q, n_kv, vocab, pages = 40, 60, 32, 8, 40_000, 62
bf16, i32, f32 = torch.bfloat16, torch.int32, torch.float32
kc, vc = (arena.empty((shared + 2 * n, n_kv, 64, 128)) for _ in range(2))
q, a, b = (arena.empty((n, n_q, 128)) for _ in range(3))
table, lens, ids = arena.empty((n, pages), i32), arena.empty((n,), i32), arena.empty((n,), i32)
logits, lp, entropy = arena.empty((n, vocab)), arena.empty((n,), f32), arena.empty((n,), f32)
top, top_ids = arena.empty((n, 7), f32), arena.empty((n, 7), i32)
plan = ops.PrefixPlan([n], [shared], n_q, n_kv, pages, arena=arena, share=True)
assert plan.cluster > 1
ws, lws = ops.SpanWorkspace(plan.partials, arena=arena), ops.LogprobWorkspace(arena=arena)

def fill(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for x in (kc, vc, q, logits):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
    table[:, :shared] = torch.arange(shared, device="cuda", dtype=i32)
    table[:, shared:] = shared + torch.arange(2 * n, device="cuda", dtype=i32).view(n, 2)
    lens.copy_(shared * 64 + 1 + torch.randint(120, (n,), generator=g, device="cuda"))
    ids.copy_(torch.randint(vocab, (n,), generator=g, device="cuda"))

def step():
    ops.prefix_decode_attention(q, kc, vc, table, lens, a, plan, ws)
    ops.window_decode_attention(a, kc, vc, table, lens, b, 100, 4, ws)
    ops.token_logprobs(logits, ids, lp, entropy, top, top_ids, ws=lws)

OUT = (a, b, lp, entropy, top, top_ids)
"""

STEP_SAVE = "LOADING = False" + STEP + r"""
fill(1)
step()
torch.cuda.synchronize()
g = fb.CUDAGraph()
with fb.graph(g, stream=torch.cuda.Stream()), ops._rt.pdl():
    step()
os.makedirs(ARCHIVE, exist_ok=True)
g.save(os.path.join(ARCHIVE, "graph_0.json"), output_tensors=lp)
fb.pack_fatbins_to_folder(ARCHIVE)
fb.save_graph_manifest(ARCHIVE)
want = []
for seed in (2, 3):
    fill(seed)
    step()
    torch.cuda.synchronize()
    want.append([x.cpu() for x in OUT])
torch.save(want, os.path.join(ARCHIVE, "want.pt"))
print("SAVE_OK")
"""

STEP_LOAD = "LOADING = True" + STEP + r"""
g, _ = fb.CUDAGraph.load(os.path.join(ARCHIVE, "graph_0.json"))
for seed, want in zip((2, 3), torch.load(os.path.join(ARCHIVE, "want.pt"))):
    fill(seed)
    for x in OUT:
        x.zero_()
    g.replay()
    torch.cuda.synchronize()
    for x, y in zip(OUT, want):
        assert torch.equal(x.cpu(), y)
assert not ws.tickets.any() and not lws.tickets.any()
print("LOAD_OK")
"""


def _run(body, archive):
    env = dict(os.environ, PYTHONPATH=ROOT)
    code = f"ROOT={ROOT!r}; ARCHIVE={archive!r}\n" + body
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    return r.stdout


@pytest.mark.parametrize("save,load", [(ENGINE_SAVE, ENGINE_LOAD), (STEP_SAVE, STEP_LOAD)], ids=["engine", "step"])
def test_save_load(tmp_path, save, load):
    archive = str(tmp_path / "arch")
    assert "SAVE_OK" in _run(save, archive)
    assert "LOAD_OK" in _run(load, archive)
