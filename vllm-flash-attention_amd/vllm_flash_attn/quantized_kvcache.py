"""A KV cache held in 8 bits: writing it, reading it back and attention over it.

The cache is a pair of float8_e4m3fn tensors laid out like the 16-bit cache of flash_attn_with_kvcache --
(batch_size_cache, seqlen_cache, nheads_k, headdim), or pages (num_blocks, page_block_size, nheads_k, headdim)
with a block_table -- and a pair of float8_e8m0fnu scales (first dim of the cache, blocks, nheads_k): one power
of two per KV head and block of `rows / blocks` tokens (a multiple of 16; rows = seqlen_cache or
page_block_size).  An element stands for code * scale, exactly.  e4m3 is a floating format, so a power of two
costs no precision against any other scale, and a block whose scale grows is re-encoded without a second
rounding except among the subnormals.  headdim is a multiple of 16, at most 256.

Sequence lengths are cut to the cache's capacity; a page id outside the pool is never followed (nothing is
written there, reading it gives NaN).  No gradients: a cache is not trained through.  No counterpart in the
reference, whose caches hold 16 bits (vllm_flash_attn/flash_attn_interface.py:1119-1253).
"""
from typing import Optional, Union

import torch

import vllm_flash_attn_2_cuda as flash_attn_cuda
from vllm_flash_attn.flash_attn_interface import _last_dim_contiguous


def _lengths(cache_seqlens, batch, device):
    if isinstance(cache_seqlens, int):
        return torch.full((batch,), cache_seqlens, dtype=torch.int32, device=device)
    return cache_seqlens if cache_seqlens is None else cache_seqlens.contiguous()


def _index(x):
    return None if x is None else x.contiguous()


def quantize_kvcache(k, v, k_cache, v_cache, k_scale, v_scale, cache_seqlens: Union[int, torch.Tensor],
                     cache_batch_idx: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None,
                     cu_seqlens: Optional[torch.Tensor] = None, max_seqlen: Optional[int] = None):
    """Write k / v (batch_size, seqlen_new, nheads_k, headdim) of fp16 / bf16 into the cache IN PLACE at positions
    cache_seqlens .. cache_seqlens + seqlen_new of every sequence; or ragged k / v (total, nheads_k, headdim) with
    cu_seqlens (batch_size + 1,) int32 and max_seqlen, the longest run.

    A block's scale is the least power of two that brings the largest magnitude written to it to at most 448 times the
    scale (2^-126 at least).  Tokens that join a block which holds some already can only raise its scale; what it holds
    is then re-encoded.  A block written from its first token on starts anew.  Values are rounded to nearest even, but
    from a scale of 2^8 (fp16) or 2^120 (bf16) on to at most 240 times the scale: the next code would stand for 2^16 or
    2^128, which the type does not have.  NaN and infinities become NaN and do not count for the scale.  Tokens past the capacity are dropped; rows behind
    the new tokens stay as they are.  Two sequences of one call must not write to the same block."""
    if cu_seqlens is not None and max_seqlen is None:
        raise ValueError("max_seqlen is required with cu_seqlens")
    if cu_seqlens is None and max_seqlen is not None:
        raise ValueError("max_seqlen goes with cu_seqlens")
    batch = k.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
    flash_attn_cuda.kv8_quantize(k, v, k_cache, v_cache, k_scale, v_scale, _lengths(cache_seqlens, batch, k_cache.device),
                                 _index(cache_batch_idx), _last_dim_contiguous(block_table), _index(cu_seqlens),
                                 max_seqlen or 0)


def dequantize_kvcache(k_cache, v_cache, k_scale, v_scale, cache_seqlens: torch.Tensor, max_seqlen: Optional[int] = None,
                       cu_seqlens: Optional[torch.Tensor] = None, total_seqlen: Optional[int] = None,
                       cache_batch_idx: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None,
                       dtype=torch.bfloat16):
    """The first cache_seqlens tokens of every sequence in 16 bits: k, v (batch_size, max_seqlen, nheads_k, headdim),
    or ragged (total_seqlen, nheads_k, headdim) where sequence i goes to rows cu_seqlens[i] .. cu_seqlens[i + 1]
    (what flash_attn_varlen_func takes).  Rows without a token are zeros.  Values are exact, except that fp16 cannot
    hold all that bf16 tokens can have written (they round, and overflow to infinity)."""
    if (cu_seqlens is None) == (max_seqlen is None) or (cu_seqlens is None) != (total_seqlen is None):
        raise ValueError("either max_seqlen (padded output), or cu_seqlens and total_seqlen (ragged output)")
    return tuple(flash_attn_cuda.kv8_dequantize(k_cache, v_cache, k_scale, v_scale, cache_seqlens.contiguous(),
                                                _index(cache_batch_idx), _last_dim_contiguous(block_table), _index(cu_seqlens),
                                                max_seqlen if cu_seqlens is None else total_seqlen, dtype))


def flash_attn_with_quantized_kvcache(q, k_cache, v_cache, k_scale, v_scale, k=None, v=None,
                                      cache_seqlens: Optional[Union[int, torch.Tensor]] = None,
                                      cache_batch_idx: Optional[torch.Tensor] = None,
                                      block_table: Optional[torch.Tensor] = None,
                                      cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: Optional[int] = None,
                                      softmax_scale=None, causal=False, window_size=(-1, -1), alibi_slopes=None, num_splits=0,
                                      *, out=None):
    """flash_attn_with_kvcache over an 8-bit cache: attention of q (batch_size, seqlen_q, nheads, headdim), or ragged
    (total_q, nheads, headdim) with cu_seqlens_q (batch_size + 1,) int32 and max_seqlen_q, against the first
    cache_seqlens tokens of every sequence (all of the capacity if None), aligned at the last query and the last key.

    If k / v (batch_size, seqlen_new, nheads_k, headdim) are given (dense q only) they are written first, as by
    quantize_kvcache, and attended.  The query is used as it is: rotate q and k beforehand (qk_norm_rotary_func).
    causal, window_size, alibi_slopes, num_splits, out as in flash_attn_with_kvcache, but num_splits does not cut the
    keys of a ragged batch's longer queries; softmax_scale > 0.  Returns out, shaped like q; rows of a ragged batch behind
    its last sequence stay as they are in `out`.  A row that sees no key is zero, and a key that no row of its sequence sees
    has no part in any result, whatever stands there; a NaN or an infinity in v of a key that some row sees can make the
    sequence's other rows NaN too.  An fp16 query over values past fp16's range (a cache that bf16 tokens were written to)
    sees infinities.  How the work is cut up goes by the width of block_table: one not much wider than the longest sequence
    is fastest.  No backward."""
    if (cu_seqlens_q is None) != (max_seqlen_q is None):
        raise ValueError("cu_seqlens_q and max_seqlen_q go together")
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** (-0.5)
    batch = q.shape[0] if cu_seqlens_q is None else cu_seqlens_q.numel() - 1
    out, _ = flash_attn_cuda.fwd_kv8(q, k_cache, v_cache, k_scale, v_scale, k, v, _lengths(cache_seqlens, batch, k_cache.device),
                                     _index(cache_batch_idx), _last_dim_contiguous(block_table), alibi_slopes, out,
                                     _index(cu_seqlens_q), max_seqlen_q or 0, softmax_scale, causal, window_size[0],
                                     window_size[1], num_splits)
    return out
