"""Experiments over the mxq path: the MX-Gemmini recipe (recipes), the perplexity protocol (llm_ppl), and a
mixture-of-experts layer on packed weights (moe_layer)."""
