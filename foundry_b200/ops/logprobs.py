"""Log probabilities of given tokens, entropy and the most probable
alternatives (csrc/kernels/logprobs.cu), beside the greedy ``argmax``."""

from __future__ import annotations

import math

import torch

from .. import _native as native
from . import _rt

_IMG = "logprobs"
MAX_TOP = 32
CTAS_PER_SM = 3
SMEM = 75 * 1024
MIN_SHARE = 4096  # logits per CTA: below it the join of a row's pieces costs more than it saves
_KINDS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_NAMES = ("fb_logprobs_bf16", "fb_logprobs_f16", "fb_logprobs_f32")


class LogprobWorkspace:
    """Partial results of ``token_logprobs``, the same for every shape. Calls
    that may run at the same time need a workspace each; calls in stream order,
    captured graphs among them, may share one."""

    def __init__(self, arena=None, device=None):
        if arena is not None:
            empty, zeros = arena.empty, arena.zeros
        else:
            device = device or torch.device("cuda", torch.cuda.current_device())
            empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
            zeros = lambda shape, dtype: torch.zeros(shape, dtype=dtype, device=device)  # noqa: E731
        self.ctas = CTAS_PER_SM * _rt.sm_count()
        self.sums = empty((2 * self.ctas * 4,), torch.float32)
        self.keys = empty((2 * self.ctas * MAX_TOP,), torch.int64)
        self.tickets = zeros((self.ctas,), torch.int32)
        self.sums_ptr, self.keys_ptr, self.tickets_ptr = self.sums.data_ptr(), self.keys.data_ptr(), self.tickets.data_ptr()
        self.device = self.tickets.get_device()

    def clear(self) -> None:
        self.tickets.zero_()


def share_of(rows: int, vocab: int, ctas: int) -> tuple[int, int]:
    """(logits per CTA, flat distance of two rows). Up to ``ctas`` rows, each
    has a whole number of CTAs of its own; more rows are one flat sequence cut
    into equal shares. (256 rows of 128256 on 444 CTAs, k = 0 / 5 / 20: 16.7 /
    19.2 / 21.2 us so, 19.9 / 25.8 / 48.2 us in equal shares, whose CTAs end two
    rows each.)"""
    if rows <= ctas:
        parts = max(1, min(ctas // rows, vocab // MIN_SHARE))
        share = math.ceil(vocab / parts / 64) * 64
        return share, math.ceil(vocab / share) * share
    return math.ceil(rows * vocab / ctas / 64) * 64, vocab


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor | None, logprobs: torch.Tensor | None,
                   entropy: torch.Tensor | None, top_logprobs: torch.Tensor | None = None,
                   top_ids: torch.Tensor | None = None, *, ws: LogprobWorkspace) -> None:
    """For each row of ``logits`` [T, V] (bf16, fp16 or fp32, any row stride):

    ``logprobs`` [T] fp32      log softmax(row)[ids[row]]; 0 for a negative id (no token),
                               NaN (and the image's status bit) for one past the vocabulary
    ``entropy`` [T] fp32       -sum p ln p
    ``top_logprobs`` [T, k] fp32, ``top_ids`` [T, k] int32: the k <= 32 most probable
                               tokens, largest first, the lower token on ties

    Outputs that are None are left out. Masked logits may be -inf or the
    type's lowest value; a row that is -inf throughout, or holds +inf or NaN,
    gives NaN (its ``top_ids`` are the order of its logits, NaN left out and -1
    for what is missing)."""
    cur = torch.cuda.current_device()
    numbers = native.tensors().rows(logits, ids, logprobs, entropy, top_logprobs, top_ids, cur)
    if numbers is None:  # not what almost every call is
        numbers = _look(logits, ids, logprobs, entropy, top_logprobs, top_ids, cur)
    kind, t, v, k, ld, x, *outs = numbers
    if k > MAX_TOP or k > v:
        raise ValueError(f"at most {min(MAX_TOP, v)} alternatives, got {k}")
    if ws.device != cur:
        raise ValueError(f"the workspace must be on the current CUDA device {cur}")
    if not t:
        return
    share, pitch = share_of(t, v, ws.ctas)
    _rt.launch_mapped(
        _IMG, _NAMES[kind], min(ws.ctas, -(-t * pitch // share)), 1, 256, SMEM, 0, x, ld, *outs, ws.sums_ptr,
        ws.keys_ptr, ws.tickets_ptr, share, pitch, t, v, k, device=cur)


def _look(logits, ids, logprobs, entropy, top_logprobs, top_ids, cur: int) -> tuple[int, ...]:
    """(kind of logits, rows, vocabulary, alternatives, row stride, addresses) of a call, or a ValueError."""
    if logits.dim() != 2 or logits.dtype not in _KINDS or (logits.stride(1) != 1 and logits.shape[1] != 1):
        raise ValueError("logits must be bf16, fp16 or fp32 [T, V] with contiguous rows")
    t, v = logits.shape
    if not 0 < v < 1 << 30 or t >= 1 << 30:
        raise ValueError(f"{t} rows of a vocabulary of {v}")
    if (top_logprobs is None) != (top_ids is None) or (ids is None) != (logprobs is None):
        raise ValueError("top_logprobs and top_ids come together, and ids and logprobs")
    k = top_ids.shape[-1] if top_ids is not None and top_ids.dim() else 0
    if logits.get_device() != cur:
        raise ValueError(f"logits must be on the current CUDA device {cur}")
    ptrs = []
    for x, dtype, shape in ((ids, torch.int32, (t,)), (logprobs, torch.float32, (t,)), (entropy, torch.float32, (t,)),
                            (top_logprobs, torch.float32, (t, k)), (top_ids, torch.int32, (t, k))):
        if x is None:
            ptrs.append(0)
            continue
        if x.dtype is not dtype or x.shape != shape or not x.is_contiguous() or x.get_device() != cur:
            raise ValueError(f"expected contiguous {dtype} {shape} on device {cur}, got {x.dtype} {tuple(x.shape)} on {x.device}")
        ptrs.append(x.data_ptr())
    return _KINDS[logits.dtype], t, v, k, logits.stride(0), logits.data_ptr(), *ptrs
