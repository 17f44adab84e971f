"""How the attention kernels leave when a wait runs out, as far as their source
says it: no GPU is made to hang or fault for it.

A warp whose lanes leave a loop one by one would wait without a limit in the
next instruction that takes the whole warp; a block that leaves while its copies
or products are under way would have them land in another block's memory."""

import pathlib
import re

KERNELS = pathlib.Path(__file__).resolve().parent.parent / "csrc" / "kernels"


def _source(name):
    return re.sub(r"//[^\n]*", "", (KERNELS / name).read_text())


def _body(text, start):
    """The braces behind the first ``start``."""
    at = text.index("{", text.index(start))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if not depth:
            return text[at:i + 1]
    raise AssertionError("unbalanced")


def test_tile_kernel_warps_leave_together():
    text = _source("attention_tile.cu")
    helper = _body(text, "bool warp_wait(")
    assert "__all_sync(0xffffffffu, mbar_wait(" in helper
    epilogue = _body(text, "else if (EPILOGUE && warp >= 4 * QT + 4)")
    vote = "ok = __all_sync(0xffffffffu, ok);"
    assert epilogue.rindex("mbar_wait(") < epilogue.index(vote) < epilogue.index("if (!ok) break;")
    softmax = _body(text, "else if (warp < 4 * QT)")
    tiles = _body(softmax, "for (int i = 0; i < n; ++i, ++tiles)")
    # a lane's own answers decide nothing before they have been voted on: at the next tile, or behind the last
    assert tiles.index(vote) < tiles.index("if (!ok) break;") < tiles.index("mbar_wait(")
    assert tiles.count("break;") == 1 and not re.search(r"if \([^;{]*mbar_wait", tiles)
    behind = softmax[softmax.index(tiles) + len(tiles):]
    assert behind.lstrip().startswith(vote) and "mbar_wait(" not in behind
    mma = _body(text, "else if (warp == 4 * QT + 1)")
    for wait in re.finditer(r"ok = (ok && )?mbar_wait\(", mma):
        # voted on before anything else is done with it
        rest = mma[wait.start():]
        assert rest.index("__all_sync(0xffffffffu, ok)") < min(rest.find(x) % len(rest) for x in ("mma_bf16", "qk(t", "if (!ok)"))


def test_tile_kernel_waits_for_what_is_under_way():
    text = _source("attention_tile.cu")
    assert "abort" not in text  # nobody would read it
    copies = _body(text, "if (warp == 4 * QT) {")
    drain = _body(copies[copies.rindex("if (!ok)"):], "if (!ok)")
    assert "&sm.kv_full[s]" in drain and "&sm.q_full[t]" in drain
    mma = _body(text, "else if (warp == 4 * QT + 1)")
    drain = _body(mma[mma.rindex("if (!ok)"):], "if (!ok)")
    assert drain.index("commit(&sm.mma_done)") < drain.index("warp_wait(&sm.mma_done, 0")


def test_ring_drain_waits_for_every_copy_that_was_issued():
    """The parities of the drain, for a producer that stops after any number of
    copies: a wait for parity p is over when the barrier's phase is odd and p even
    or the other way round."""
    text = _source("attention_tile.cu")
    assert text.count("mbar_wait(&sm.kv_full[s], s < slot ? phase : phase ^ 1") == 1
    assert text.count("mbar_wait(&sm.q_full[t], (q_loads[t] & 1) ^ 1") == 1
    for slots in (2, 4, 5):
        for issued in range(4 * slots):
            slot, phase = issued % slots, issued // slots & 1
            for s in range(slots):
                copies = len(range(s, issued, slots))  # into this slot; all but the last have landed long since
                parity = phase if s < slot else phase ^ 1
                assert (copies & 1) != parity  # over once all have landed
                assert not copies or (copies - 1 & 1) == parity  # and not before
    for loads in range(5):
        parity = (loads & 1) ^ 1
        assert (loads & 1) != parity and (not loads or (loads - 1 & 1) == parity)


def test_span_kernel_waits_for_what_is_under_way():
    text = _source("attention_span.cu")
    copies = _body(text, "if (warp == 0)")
    empty = copies.index("ok = mbar_wait(kv ? &sm.vempty : &sm.kempty")
    # behind a wait that ran out no further copy is issued ..
    assert copies.index("if (!ok) break;") < copies.index("++loads[kv];") < copies.index("tma_load")
    assert empty < copies.index("if (!ok) break;") and "continue;\n            }" not in copies
    # .. and those that were have landed before the block leaves
    drain = _body(copies[copies.rindex("if (!ok) {"):], "if (!ok)")
    for which, at in (("k", 0), ("v", 1)):
        assert f"mbar_wait(&sm.{which}full, (loads[{at}] & 1) ^ 1" in drain
        assert f"mbar_wait(&sm.{which}empty, (loads[{at}] & 1) ^ 1" in copies
    mma = _body(text, "else if (warp == 1)")
    drain = _body(mma[mma.rindex("if (!ok) {"):], "if (!ok)")
    assert drain.index("mma_commit(&sm.mma_done)") < drain.index("mbar_wait(&sm.mma_done, 0")


def test_clusters_hold_no_tensor_memory_while_they_wait_for_each_other():
    """A CTA of a cluster that keeps its tensor memory until the others have come,
    one of which waits for tensor memory that another kernel's cluster holds in the
    same way, would wait for good."""
    body = _body(_source("attention_tile.cu"), "void tile_attention(")
    assert body.index("tmem_dealloc(") < body.index("w.finish(sm)") and "cluster_sync" not in body
