"""mxq.nn -- Schemes inside a model (mxq/nn/__init__.py:1-17).

    MXLinear(linear, scheme)     one nn.Linear computed through one Scheme (inference only)
    patch(model, rules)          a Scheme per layer name or type, first matching rule wins; (qk, pv) for a core
    is_attention                 selector for the attention projections
    attend(q, k, v, mask, scale, qk, pv)   the attention core with Q K^T and P V through two Schemes

Not in the reference, for serving in packed bytes (mxq.packed) what patch emulates:

    packed_linear(x, codes, scales, fmt, bias=, activation=, gated=, residual=)   a product and its epilogue
    route(logits, top_k)                          tokens to experts: weights and experts, differentiable
    dispatch(experts, num_experts)                the tokens' slots sorted by expert
    expert_linear(x, codes, scales, fmt, plan)    packed_linear with a weight an expert
    combine(y, weights, plan, residual=)          the experts' rows summed for each token, differentiable
    packed_cache(pages, page_size, kv_heads, head_dim, fmt)   a paged key and value cache in MX formats
    cache_write(k, v, cache, slots)               rows quantized into it
    cache_attend(q, cache, table, lengths, starts)            attention over it, prompts and single tokens
    cache_read(cache, slots, dtype)               rows of it as values
"""
from ._attention import attend
from ._cache import PackedCache, cache_attend, cache_read, cache_write, packed_cache
from ._linear import MXLinear
from ._moe import Dispatch, combine, dispatch, route
from ._packed_linear import expert_linear, packed_linear
from ._patch import is_attention, patch

__all__ = ["MXLinear", "patch", "is_attention", "attend", "packed_linear", "expert_linear", "route", "dispatch",
           "combine", "Dispatch", "PackedCache", "packed_cache", "cache_write", "cache_read", "cache_attend"]
