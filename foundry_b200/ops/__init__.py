"""Hand-written sm_100a kernels of foundry_b200 and their host launchers."""

from . import _rt
from .attention import (
    DecodeWorkspace,
    decode_attention,
    decode_splits,
    prefill_attention,
    prefill_tiles,
)
from .basic import (
    add_rmsnorm_partials,
    argmax,
    copy_i32,
    decode_advance,
    embedding,
    fill_,
    init_normal_,
    rmsnorm,
    rope_cos_sin,
    rope_kv_write,
    silu_mul,
)
from .logprobs import LogprobWorkspace, token_logprobs
from .span_attention import (
    PrefixPlan,
    SpanWorkspace,
    prefix_decode_attention,
    window_decode_attention,
    window_prefill_attention,
)
from .gemm import Partial, PartialBuffer, StreamKBuffer, linear, linear_multicast, linear_swiglu, plan

status = _rt.status
clear_status = _rt.clear_status

__all__ = [
    "DecodeWorkspace", "LogprobWorkspace", "Partial", "PartialBuffer", "PrefixPlan", "SpanWorkspace", "StreamKBuffer", "add_rmsnorm_partials", "argmax", "clear_status", "copy_i32", "decode_advance",
    "decode_attention", "decode_splits", "embedding", "fill_", "init_normal_",
    "linear", "linear_multicast", "linear_swiglu", "plan", "prefill_attention", "prefill_tiles", "rmsnorm", "rope_cos_sin", "rope_kv_write",
    "prefix_decode_attention", "silu_mul", "status", "token_logprobs", "window_decode_attention",
    "window_prefill_attention",
]
