"""Attention over chosen key blocks beside `sfast_xformers::memory_efficient_attention` (no counterpart in the reference): block means, the
choice of blocks by their products, and attention over the chosen blocks with its gradients.

A server keeps the block means of its key cache beside the cache and passes them to `block_topk`; `sparse_attention` below makes all three
calls from q, k and v.
"""
from typing import Optional

import torch

from ...hip import functional as F
from .xformers_attention import _lib

_lib.define("block_means(Tensor input, int block, Tensor? lengths=None) -> Tensor")
_lib.impl("block_means", F.block_means, "CUDA")
_lib.define("block_topk(Tensor query_means, Tensor key_means, int topk, int block_k=64, Tensor? key_lengths=None) -> Tensor")
_lib.impl("block_topk", F.block_topk, "CUDA")
_lib.define("block_sparse_attention(Tensor query, Tensor key, Tensor value, Tensor blocks, int block_q=128, int block_k=64, "
            "Tensor? key_lengths=None, Tensor? query_lengths=None, float? scale=None) -> (Tensor, Tensor)")
_lib.impl("block_sparse_attention", F.block_sparse_attention, "CUDA")
_lib.define("block_sparse_attention_backward(Tensor grad_out, Tensor? grad_lse, Tensor query, Tensor key, Tensor value, Tensor blocks, Tensor out, "
            "Tensor lse, int block_q=128, int block_k=64, Tensor? key_lengths=None, Tensor? query_lengths=None, float? scale=None) "
            "-> (Tensor, Tensor, Tensor)")
_lib.impl("block_sparse_attention_backward", F.block_sparse_attention_backward, "CUDA")


def _setup(ctx, inputs, output):
    query, key, value, blocks, ctx.block_q, ctx.block_k, key_lengths, query_lengths, ctx.scale = inputs
    ctx.save_for_backward(query, key, value, blocks, key_lengths, query_lengths, *output)
    ctx.set_materialize_grads(False)


def _backward(ctx, grad_out, grad_lse):
    query, key, value, blocks, key_lengths, query_lengths, out, lse = ctx.saved_tensors
    none = (None,) * 6
    if grad_out is None and grad_lse is None:
        return (None,) * 3 + none
    if grad_out is None:
        grad_out = torch.zeros_like(out)
    return torch.ops.sfast_xformers.block_sparse_attention_backward(grad_out, grad_lse, query, key, value, blocks, out, lse, ctx.block_q, ctx.block_k,
                                                                    key_lengths, query_lengths, ctx.scale) + none


torch.library.register_autograd("sfast_xformers::block_sparse_attention", _backward, setup_context=_setup)


def sparse_attention(query, key, value, topk: int, block_q: int = 128, block_k: int = 64, key_lengths=None, query_lengths=None,
                     scale: Optional[float] = None):
    """softmax(scale q k^T) v where every block of `block_q` queries attends to the `topk` blocks of `block_k` keys whose mean agrees best with
    the mean of the queries (summed over the heads of a group). query: [B, Sq, H, D], key / value: [B, Sk, Hk, D]; returns [B, Sq, H, D].
    The choice takes no gradient, the attention does."""
    ops = torch.ops.sfast_xformers
    blocks = ops.block_topk(ops.block_means(query.detach(), block_q, query_lengths), ops.block_means(key.detach(), block_k, key_lengths), topk,
                            block_k, key_lengths)
    return ops.block_sparse_attention(query, key, value, blocks, block_q, block_k, key_lengths, query_lengths, scale)[0]
