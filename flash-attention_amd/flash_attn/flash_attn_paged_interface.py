"""Serving with a paged key / value cache (no counterpart in the reference): a pool of pages of a fixed number of tokens, shared by sequences that list
theirs in a page table.

    k_cache, v_cache   (pages, page size, nheads_k, headdim) fp16 or bf16, any strides with a contiguous last dimension; page size: a power of two
                       from 16 to 1024.  PagedKVCache lays a page out head by head, so that a head's keys of a page are one piece of memory.
    page_table         (batch, pages per sequence) int32: token j of sequence b is in page page_table[b, j // page_size]
    seqlens_k          (batch,) int32: tokens of each sequence that the cache holds, the new ones among them
    cu_seqlens_q       (batch + 1,) int32: where each sequence's new tokens begin in the packed (total, heads, headdim) tensors

A step of a model advances seqlens_k by the new tokens once; every layer then stores them (paged_append_func) and attends
(flash_attn_paged_func).  Nothing here waits for the GPU or reads its memory on the host: calls can be captured into a graph, whose replays
find new lengths, tables and tokens in the same tensors.  max_seqlen_k then has to hold for all of them; it bounds the work
that is cut, not the memory that is read.

What lies in page_table and seqlens_k is never trusted with an address: entries outside the pool are read as its first or last page and never written to,
lengths count as far as the table goes.  Pages that several sequences list (a common prompt) may be read by all of them and must not be appended to,
weighted or evicted from."""
import torch

from . import flash_attn_gfx950 as _backend


def _inference(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the paged cache has no backward: call it under torch.no_grad()")


def paged_append_func(q, k, v, k_cache, v_cache, page_table, cu_seqlens, seqlens_k, q_weight=None, k_weight=None, cos_half=None, sin_half=None,
                      positions=None, eps=1e-6, key_weights=None, key_positions=None):
    """Stores the new tokens' k and v (total, nheads_k, headdim) into the pages of their sequences, behind what is there: row i of sequence b goes to
    slot seqlens_k[b] - (its new tokens) + i.  In the same pass k, and q (total, nheads, headdim) if it is given, are normalised (q_weight, k_weight: see
    apply_qk_norm_rotary) and turned by their positions (cos_half, sin_half) - positions[row], or the slot.  Returns the new q, or None.
    key_weights, key_positions (pages, nheads_k, page size): set to 0 and the position for the new tokens (for paged_key_weights_func and
    paged_evict_func).  Rows behind the last sequence, and tokens for which the page table has no room, are not stored; their rows of the returned q
    hold nothing."""
    done = _backend.passes().paged_append(q, k, v, k_cache, v_cache, page_table, cu_seqlens, seqlens_k, q_weight, k_weight, cos_half, sin_half, positions, eps,
                                          key_weights, key_positions)
    if done is not None:
        return None if q is None else done
    _inference(q, k, v, q_weight, k_weight)
    return _backend.paged_append(q, k, v, k_cache, v_cache, page_table, cu_seqlens, seqlens_k, None, q_weight, k_weight, cos_half, sin_half, positions, eps,
                                 key_weights, key_positions)


def flash_attn_paged_func(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale=None, causal=True,
                          return_softmax_lse=False):
    """Attention of the new tokens q (total, nheads, headdim) over their sequences' pages; nheads is a multiple of nheads_k, and query head h attends with
    key head h // (nheads // nheads_k).  causal: a sequence's last new token sees all its keys, the one before it one less, and so on (the new tokens'
    own keys are in the cache); a token that sees no key gives zeros.  max_seqlen_q, max_seqlen_k: at least the longest of each.
    Returns out (total, nheads, headdim), or (out, softmax_lse), softmax_lse (batch, nheads, max_seqlen_q rounded up to 16) fp32, -inf for a token
    that sees no key.  Rows of out behind the last sequence hold nothing."""
    done = _backend.passes().paged_fwd(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal,
                                       return_softmax_lse)
    if done is not None:
        return done
    _inference(q, k_cache, v_cache)
    scale = q.shape[-1] ** (-0.5) if softmax_scale is None else softmax_scale
    r = _backend.paged_fwd(q, k_cache, v_cache, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal, return_softmax_lse)
    return (r[0], r[1]) if return_softmax_lse else r[0]


def paged_key_weights_func(q, softmax_lse, k_cache, key_weights, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale=None,
                           causal=True):
    """Adds to key_weights (pages, nheads_k, page size) fp32 what every key has received of the new tokens' attention: the sum of its probabilities
    over the tokens and over the query heads of its group.  q and softmax_lse: those of flash_attn_paged_func over the same cache.  In place; returns
    key_weights."""
    if _backend.passes().paged_key_weights(q, softmax_lse, k_cache, key_weights, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale,
                                           causal):
        return key_weights
    _inference(q, k_cache)
    scale = q.shape[-1] ** (-0.5) if softmax_scale is None else softmax_scale
    return _backend.paged_key_weights(q, softmax_lse, k_cache, key_weights, page_table, cu_seqlens_q, seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal)


def paged_evict_func(k_cache, v_cache, key_weights, key_positions, page_table, seqlens_k, next_positions, budget, recent, max_seqlen_k):
    """Cuts every sequence's cache to `budget` keys a head, in place, and returns the new lengths min(seqlens_k, budget).  Of a longer sequence stay
    the keys whose position is at least next_positions[b] - recent, and then those with the largest key_weights (NaN counts as -inf; ties: the lower
    slot).  Each key head chooses for itself; a kept key from behind the budget takes the place, and the weight and position, of one that goes.  Slots
    from `budget` on are left as they were.  next_positions: (batch,) int32, the position that each sequence's next token would have."""
    done = _backend.passes().paged_evict(k_cache, v_cache, key_weights, key_positions, page_table, seqlens_k, next_positions, budget, recent, max_seqlen_k)
    if done is not None:
        return done
    _inference(k_cache, v_cache)
    return _backend.paged_evict(k_cache, v_cache, key_weights, key_positions, page_table, seqlens_k, next_positions, budget, recent, max_seqlen_k)
