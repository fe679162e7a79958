"""MI355X-native MiniMax-M3 three-stage sparse attention (drop-in for ``msa_triton.triton``).

The public operators keep the reference facade (triton/__init__.py:4-29): the
implementation module is imported on first call, so importing the package does
not load the native library.

    m3_index_score(index_q, index_k, cu_seqlens, max_seqlen, *, block_size=128, scale=1.0)
    m3_topk(scores, cu_seqlens, *, block_size=128, topk_blocks=16, local_blocks=1)
    m3_sparse_attention(q, k, v, indices, cu_seqlens, max_seqlen, *, block_size=128,
                        scale=None, return_lse=False)

All three run as hand-written gfx950 HIP kernels behind the C ABI declared in
``include/msa_mi355x.h``; there is no CPU or eager fallback.

    m3_index_score_topk(index_q, index_k, cu_seqlens, max_seqlen, *, block_size=128, scale=1.0,
                        topk_blocks=16, local_blocks=1) -> (scores, indices)

is the first two stages in one call (score and selection kernels back to back);

    m3_indexer_kl(index_q, index_k, q, k, indices, cu_seqlens, max_seqlen, *, block_size=128,
                  index_scale=1.0, scale=None, return_rows=False) -> loss

is the indexer's KL training loss over the selected tokens (teacher: the detached
attention probabilities; student: the index token logits);

    m3_qk_norm_rope(q, k, q_weight, k_weight, cos_sin, cu_seqlens, *, eps=1e-6,
                    context_lens=None) -> (q_out, k_out)

norms the query and key heads and rotates them by their positions (``rope_table``), before the
stages above, with gradients;

    m3_cache_append(k, v, k_cache, v_cache, page_table, cu_seqlens, context_lens, *, index_k=None, index_cache=None,
                    k_scale=None, v_scale=None, k_weight=None, index_weight=None, cos_sin=None, eps=1e-6)

writes new keys, values and index keys into a paged cache (16-bit, or 8-bit with a scale for each page and
head), keys normed and rotated on the way;

    m3_index_score_topk_paged(index_q, index_cache, page_table, cu_seqlens, context_lens, max_seqlen, *,
                              block_size=128, scale=1.0, topk_blocks=16, local_blocks=1) -> (scores, indices)

scores new tokens against the cached index keys and selects their blocks;

    m3_sparse_attention_paged(q, k_cache, v_cache, indices, page_table, cu_seqlens, context_lens, *,
                              block_size=128, scale=None, k_scale=None, v_scale=None, return_lse=False)

is the attention of new tokens over the selected blocks of the cache;

    m3_window_attention(q, k, v, cu_seqlens, max_seqlen, *, window_size, sink_tokens=0, scale=None,
                        return_lse=False)

is causal attention with a sliding window and a few first tokens that stay visible (or without a window), for the
layers beside the block-sparse ones, with gradients;

    m3_window_attention_paged(q, k_cache, v_cache, page_table, cu_seqlens, context_lens, *, window_size, sink_tokens=0,
                              scale=None, k_scale=None, v_scale=None, return_lse=False)

is the same of new tokens over a paged cache, and

    m3_tree_attention_paged(q, k_cache, v_cache, page_table, cu_seqlens, context_lens, parents, *, window_size=None,
                            sink_tokens=0, scale=None, k_scale=None, v_scale=None, return_lse=False)

that of a tree of drafted tokens, each of which sees the cached ones and its ancestors;

    prepare_sequences(cu_seqlens, *, block_size=128) -> PackedSequences

validates ``cu_seqlens`` once and returns immutable metadata with device copies;
passed in place of ``cu_seqlens`` to any operator (and to ``build_k2q_csr``), it
removes the operators' host reads of ``cu_seqlens``, so a layer's forward and
backward run without host synchronisation and can be captured in a HIP graph.
"""

from .layout import PackedSequences


def m3_index_score(index_q, index_k, cu_seqlens, max_seqlen, *, block_size=128, scale=1.0):
    from .index_score import m3_index_score as implementation

    return implementation(index_q, index_k, cu_seqlens, max_seqlen, block_size=block_size, scale=scale)


def m3_topk(scores, cu_seqlens, *, block_size=128, topk_blocks=16, local_blocks=1):
    from .topk import m3_topk as implementation

    return implementation(
        scores, cu_seqlens, block_size=block_size, topk_blocks=topk_blocks, local_blocks=local_blocks
    )


def m3_sparse_attention(
    q, k, v, indices, cu_seqlens, max_seqlen, *, block_size=128, scale=None, return_lse=False
):
    from .sparse_attention import m3_sparse_attention as implementation

    return implementation(
        q, k, v, indices, cu_seqlens, max_seqlen,
        block_size=block_size, scale=scale, return_lse=return_lse,
    )


def m3_index_score_topk(index_q, index_k, cu_seqlens, max_seqlen, *, block_size=128, scale=1.0, topk_blocks=16,
                        local_blocks=1):
    from .index_score import m3_index_score_topk as implementation

    return implementation(index_q, index_k, cu_seqlens, max_seqlen, block_size=block_size, scale=scale,
                          topk_blocks=topk_blocks, local_blocks=local_blocks)


def m3_indexer_kl(index_q, index_k, q, k, indices, cu_seqlens, max_seqlen, *, block_size=128, index_scale=1.0,
                  scale=None, return_rows=False, teacher_lse=None):
    from .indexer_kl import m3_indexer_kl as implementation

    return implementation(index_q, index_k, q, k, indices, cu_seqlens, max_seqlen, block_size=block_size,
                          index_scale=index_scale, scale=scale, return_rows=return_rows, teacher_lse=teacher_lse)


# Where the norm and the serving operators live. Looked up on first use and bound here then: their calls are short enough
# for a wrapper (1.5 us of the 20 us of a decoding step's call) to count.
_OPERATORS = {
    "m3_qk_norm_rope": "norm_rope",
    "rope_table": "norm_rope",
    "m3_cache_append": "cache_append",
    "m3_index_score_topk_paged": "paged_score",
    "m3_sparse_attention_paged": "paged_attention",
    "m3_window_attention": "window_attention",
    "m3_window_attention_paged": "window_paged",
    "m3_tree_attention_paged": "window_paged",
}


def __getattr__(name):
    if name not in _OPERATORS:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    from importlib import import_module

    value = globals()[name] = getattr(import_module("." + _OPERATORS[name], __name__), name)
    return value


def __dir__():
    return sorted({*globals(), *_OPERATORS})


def prepare_sequences(cu_seqlens, *, block_size=128):
    from .layout import prepare_sequences as implementation

    return implementation(cu_seqlens, block_size=block_size)


__all__ = ["m3_index_score", "m3_topk", "m3_sparse_attention", "m3_index_score_topk", "m3_indexer_kl",
           "m3_qk_norm_rope", "m3_cache_append",
           "m3_index_score_topk_paged", "m3_sparse_attention_paged", "rope_table", "m3_window_attention",
           "m3_window_attention_paged", "m3_tree_attention_paged",
           "prepare_sequences", "PackedSequences"]
