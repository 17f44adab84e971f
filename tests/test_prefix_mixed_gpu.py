"""Shared-prefix decode of a batch in which a plan shares some groups' prompts and
reads others row by row, against every row attended to on its own. Both round p
and the output to bf16: off by 2^-8 of sum p|v| and of the output each, from
scores that are fp32 sums of 128 exact products."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, PAGE = 128, 64


@pytest.mark.parametrize("n_q,n_kv", [(32, 8), (16, 1)])
@pytest.mark.parametrize("groups", [
    [(2, 1)] * 30 + [(64, 300)] + [(1, 9)] + [(2, 1)] * 30, [(100, 300), (1, 0), (90, 40), (3, 2)],
])
def test_some_groups_shared(groups, n_q, n_kv):
    from foundry_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(len(groups))
    rows, width = sum(n for n, _ in groups), max(p for _, p in groups) + 2
    table, lens, blocks = torch.zeros(rows, width, dtype=torch.int32), [], 0
    r = 0
    for n, p in groups:
        table[r:r + n, :p] = torch.arange(blocks, blocks + p)
        blocks += p
        for _ in range(n):
            table[r, p:p + 2] = torch.arange(blocks, blocks + 2)
            blocks += 2
            lens.append(p * PAGE + (37 * r) % 120 + 1)
            r += 1
    kc, vc = (torch.randn(blocks, n_kv, PAGE, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(rows, n_q, D, generator=g, device="cuda").to(torch.bfloat16)
    plan = ops.PrefixPlan([n for n, _ in groups], [p for _, p in groups], n_q, n_kv, width)
    assert plan.items_n and 0 < (plan.row_prefix[:rows] > 0).sum() < rows  # some, not all
    ws, out = ops.SpanWorkspace(plan.partials), torch.full_like(q, 7.0)
    table, lens_t = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    ops.prefix_decode_attention(q, kc, vc, table, lens_t, out, plan, ws)
    for r in range(0, rows, 7):
        at = torch.arange(lens[r], device="cuda")
        page = table[r].long()[at // PAGE]
        k, v = (c[page, :, at % PAGE].transpose(0, 1).double() for c in (kc, vc))
        qr = q[r].view(n_kv, -1, D).double()
        p = (qr @ k.transpose(1, 2) / math.sqrt(D)).softmax(-1)
        o, a = (p @ v).reshape(n_q, D), (p @ v.abs()).reshape(n_q, D)
        worst = (qr.abs() @ k.abs().transpose(1, 2) / math.sqrt(D)).amax(-1).reshape(n_q, 1)
        tol = 2.0**-8 * (a + o.abs()) + (2 * 128 * 2.0**-23 * worst + 2.0**-20) * a
        assert ((out[r].double() - o).abs() <= tol).all(), r
    assert ops.status("attention_span") == 0 and ops.status("attention_tile") == 0 and not ws.tickets.any()
