"""Causal attention of packed prompts on B200 (the reference leaves prompts to vLLM, src/vllm_exact/paged_attn.py:156).

A row's bits depend on its own query and the keys and values that it sees, never on the other sequences of the batch, as in
decode attention: a prompt in pieces, each over all keys so far, gives the bits of the whole.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check, launch_on, lib

__all__ = ["prompt_attention"]

_DT = {torch.bfloat16: _lib.EX_DTYPE_BF16, torch.float16: _lib.EX_DTYPE_F16}


def prompt_attention(query, key, value, cu_seqlens_q, cu_seqlens_k, scale, out=None):
    """query (tokens, H, D), key and value (keys, KV, D), all bf16 or all fp16, D = 64, 128 or 256, any token and head
    strides that are multiples of 8; sequence b has the query rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1] and the key
    rows cu_seqlens_k[b] .. cu_seqlens_k[b + 1] (int32, n + 1 entries each). Its last query is its last key's token:
    query i sees the keys j <= i + Lk - Lq, so keys may start before the queries (a continued conversation, its cached
    beginning read with kv_cache.cache_read). A query that sees no key gives zeros. Query head h reads KV head
    h // (H / KV). scale is positive. Returns out (like query; made if not given); its rows of no sequence, and those of a
    sequence whose offsets leave the arrays or run backwards, are left as they were."""
    dev = query.get_device()  # -1: not on a GPU
    if (dev < 0 or key.get_device() != dev or value.get_device() != dev or cu_seqlens_q.get_device() != dev
            or cu_seqlens_k.get_device() != dev):
        raise ValueError("prompt_attention needs CUDA tensors of one device (there is no CPU fallback)")
    if query.dtype not in _DT or key.dtype != query.dtype or value.dtype != query.dtype:
        raise TypeError("query, key and value must be all bf16 or all fp16")
    if query.dim() != 3 or key.dim() != 3 or value.shape != key.shape or key.shape[2] != query.shape[2]:
        raise ValueError("query must be (tokens, H, D), key and value (keys, KV, D)")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if out.dtype != query.dtype or out.shape != query.shape or out.get_device() != dev:
        raise ValueError("out must be like query")
    sq, sk, sv, so = query.stride(), key.stride(), value.stride(), out.stride()
    if sq[2] != 1 or sk[2] != 1 or sv[2] != 1 or so[2] != 1:
        raise ValueError("the head dimension must be contiguous")
    if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_k.dtype != torch.int32:
        raise TypeError("cu_seqlens_q and cu_seqlens_k must be int32")
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape != cu_seqlens_k.shape or cu_seqlens_q.shape[0] < 1:
        raise ValueError("cu_seqlens_q and cu_seqlens_k need n + 1 entries each")
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    T, H, D = query.shape
    with launch_on(dev) as stream:
        check("ex_prompt_attention", lib().ex_prompt_attention(
            query.data_ptr(), sq[0], sq[1], key.data_ptr(), sk[0], sk[1], value.data_ptr(), sv[0], sv[1],
            _DT[query.dtype], cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), cu_seqlens_q.shape[0] - 1, T,
            key.shape[0], H, key.shape[1], D, float(scale), out.data_ptr(), so[0], so[1], stream))
    return out
