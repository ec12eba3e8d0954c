"""The function a model calls for a decoded token's attention over a paged cache (beside retroinfer_decode_attn)."""


def paged_decode_attn(query_states, key_states, value_states, layer_idx, paged_cache):
    """query [bsz, 1, heads, dim] -> the attention's output; the token's key and value are in the cache already."""
    return paged_cache.compute(query_states.contiguous(), layer_idx)
