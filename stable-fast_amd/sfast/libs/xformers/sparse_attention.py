"""Attention over chosen key blocks beside `sfast_xformers::memory_efficient_attention` (no counterpart in the reference).

`sfast_xformers::block_means`, `::block_topk`, `::block_sparse_attention` and its `_backward` are native operators, registered by
csrc/torch/video_attention.cpp when the package is imported; hip.functional's functions of these names say what they do. A server keeps the
block means of its key cache beside the cache and passes them to `block_topk`; `sparse_attention` below makes all three calls from q, k and v.
"""
from typing import Optional

from ...hip import functional as F


def sparse_attention(query, key, value, topk: int, block_q: int = 128, block_k: int = 64, key_lengths=None, query_lengths=None,
                     scale: Optional[float] = None):
    """softmax(scale q k^T) v where every block of `block_q` queries attends to the `topk` blocks of `block_k` keys whose mean agrees best with
    the mean of the queries (summed over the heads of a group). query: [B, Sq, H, D], key / value: [B, Sk, Hk, D]; returns [B, Sq, H, D].
    The choice takes no gradient, the attention does."""
    blocks = F.block_topk(F.block_means(query, block_q, query_lengths), F.block_means(key, block_k, key_lengths), topk, block_k, key_lengths)
    return F.block_sparse_attention(query, key, value, blocks, block_q, block_k, key_lengths, query_lengths, scale)[0]
