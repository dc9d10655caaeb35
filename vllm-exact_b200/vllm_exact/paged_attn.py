"""Batch-invariant paged decode attention on B200 and the patch of vLLM's FlashAttention backend.

Mirrors the reference's src/vllm_exact/paged_attn.py:

* ``paged_decode(query, key_cache, value_cache, block_table, seq_lens, scale, out, n, max_seq_len, ...)``
  (reference paged_attn.py:97-114): same arguments, same in-place write of rows [0, n) of `out`.
* ``install()`` (reference paged_attn.py:135-163): patches ``FlashAttentionImpl.forward`` so decode tokens always go
  through ``paged_decode`` and prefill tokens through vLLM's own implementation.

Kernel parameters are module constants that never depend on the batch (reference paged_attn.py:21-28): SPLIT keys
per segment and the number of segments ceil(MAX_LEN / SPLIT) fix the floating-point reduction order of every
request, so a request's output bits are the same alone, in any batch, and under any placement of its pages.

Beside them, without a counterpart in the reference: ``paged_decode_q8``, the same over an 8-bit cache (kv_cache.py), and
``tree_attention``, up to 64 drafted tokens per request over a 16-bit or 8-bit cache under an ancestor mask. Their
segments depend on the request's own length, not on MAX_LEN, with the same invariance; their bits are not paged_decode's.
"""
from __future__ import annotations

import torch

from . import _lib, kv_cache
from ._lib import check, launch_on, lib

SPLIT = 4096       # keys per segment (fixed per deployment: it sets the reduction order)
MAX_LEN = 16384    # number of segments = ceil(MAX_LEN / SPLIT); enable() sets it to max_model_len
BLK = 64           # kept for signature compatibility; the B200 kernel's key block is fixed by the head size
WARPS = 4
STAGES = 3

_DT = {torch.float32: _lib.EX_DTYPE_F32, torch.bfloat16: _lib.EX_DTYPE_BF16, torch.float16: _lib.EX_DTYPE_F16}


def workspace_bytes(n: int, H: int, D: int, max_len: int | None = None, split: int | None = None) -> int:
    return lib().ex_paged_decode_workspace_bytes(n, H, D, MAX_LEN if max_len is None else max_len,
                                                  SPLIT if split is None else split)


def paged_decode(query, key_cache, value_cache, block_table, seq_lens, scale, out, n, max_seq_len=None, blk=None,
                 warps=None, stages=None, split=None, workspace=None, query_start_loc=None):
    """query (>=n, H, D) bf16; key_cache / value_cache (num_blocks, block_size, KV, D) bf16 views (any strides with a
    contiguous last dimension); block_table (>=n, pages) int32; seq_lens (>=n,) int32; out (>=n, H, D).
    Computes the first n requests only. `max_seq_len`, `blk`, `warps` and `stages` are accepted for signature
    compatibility with the reference; the segment count comes from MAX_LEN as in the reference.

    query_start_loc (int32, >= n + 1 entries; mixed prefill + decode steps): of the first n requests, compute only
    the leading run whose query length is 1 (the requests [0, nd) of reference paged_attn.py:153-159) and leave the
    other rows of `out` untouched. The run is found on the device, so there is no host sync."""
    if n <= 0:
        return out
    tensors = (query, key_cache, value_cache, block_table, seq_lens, out)
    if query_start_loc is not None:
        if query_start_loc.dtype != torch.int32 or query_start_loc.dim() != 1:
            raise TypeError("query_start_loc must be a 1-D int32 tensor")
        if query_start_loc.numel() < n + 1:
            raise ValueError("query_start_loc needs at least n + 1 entries")
        query_start_loc = query_start_loc.contiguous()
        tensors = tensors + (query_start_loc,)
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("paged_decode needs CUDA tensors (there is no CPU fallback)")
    if query.dtype != torch.bfloat16 or key_cache.dtype != torch.bfloat16 or value_cache.dtype != torch.bfloat16:
        raise TypeError("paged_decode expects bf16 query and KV cache")
    if key_cache.stride() != value_cache.stride():
        raise ValueError("key and value caches must share strides")
    if query.stride(2) != 1 or key_cache.stride(3) != 1 or out.stride(2) != 1 or block_table.stride(1) != 1:
        raise ValueError("the head dimension (and block table rows) must be contiguous")
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_table and seq_lens must be int32")
    seq_lens = seq_lens.contiguous()
    H, D = query.shape[1], query.shape[2]
    BS, KV = key_cache.shape[1], key_cache.shape[2]
    split = split or SPLIT
    nbytes = workspace_bytes(n, H, D, MAX_LEN, split)
    _check_workspace(workspace, query)
    if workspace is None or workspace.numel() < nbytes:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
    with torch.cuda.device(query.device):
        check("ex_paged_decode", lib().ex_paged_decode_leading(
            query.data_ptr(), query.stride(0), query.stride(1), key_cache.data_ptr(), value_cache.data_ptr(),
            key_cache.stride(0), key_cache.stride(1), key_cache.stride(2), key_cache.shape[0], block_table.data_ptr(),
            block_table.stride(0), seq_lens.data_ptr(),
            None if query_start_loc is None else query_start_loc.data_ptr(), n, H, KV, D, BS, float(scale),
            MAX_LEN, split, out.data_ptr(), out.stride(0), out.stride(1), _DT[out.dtype], workspace.data_ptr(),
            nbytes, torch.cuda.current_stream(query.device).cuda_stream))
    return out


_DT16 = {torch.bfloat16: _lib.EX_DTYPE_BF16, torch.float16: _lib.EX_DTYPE_F16}
MAX_DRAFT = 64  # drafted tokens of a request (the bits of a mask word)


def rows_workspace_bytes(tokens: int, H: int, D: int, max_len: int) -> int:
    """Bytes of workspace of paged_decode_q8 (tokens = n) and tree_attention for requests of at most max_len keys."""
    return lib().ex_paged_rows_workspace_bytes(tokens, H, D, max_len)


def _rows_operands(name, query, key_cache, value_cache, block_table, seq_lens, out, n):
    """Checks shared by paged_decode_q8 and tree_attention; the index of the device."""
    dev = query.get_device()  # -1: not on a GPU
    if (dev < 0 or key_cache.get_device() != dev or value_cache.get_device() != dev or block_table.get_device() != dev
            or seq_lens.get_device() != dev or out.get_device() != dev):
        raise ValueError(f"{name} needs CUDA tensors of one device (there is no CPU fallback)")
    if query.dtype not in _DT16 or out.dtype != query.dtype:
        raise TypeError(f"{name} expects a bf16 or fp16 query, and out of the same type")
    sq, so = query.shape, out.shape
    if len(sq) != 3 or len(so) != 3 or key_cache.dim() != 4 or sq[2] != key_cache.shape[3]:
        raise ValueError("query and out must be (tokens, H, D), caches (num_blocks, block_size, KV, D)")
    if so[1] != sq[1] or so[2] != sq[2]:
        raise ValueError("out must have a row for every row of query")
    if query.stride(2) != 1 or out.stride(2) != 1:
        raise ValueError("the head dimension must be contiguous")
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_table and seq_lens must be int32")
    if block_table.dim() != 2 or seq_lens.dim() != 1 or block_table.shape[0] < n or seq_lens.shape[0] < n:
        raise ValueError("block_table (n, pages) and seq_lens (n) need a row for every request")
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("block table rows must be contiguous")
    return dev


def _check_workspace(workspace, query):
    """A caller's workspace is written as one run of bytes: a strided or expanded view would have others' memory between."""
    if workspace is not None and (workspace.get_device() != query.get_device() or not workspace.is_contiguous()):
        raise ValueError("the workspace must be contiguous and on the query's device")


def _rows_scratch(tokens, H, D, max_len, workspace, query):
    _check_workspace(workspace, query)
    nbytes = lib().ex_paged_rows_workspace_bytes(tokens, H, D, max_len)
    if nbytes and (workspace is None or workspace.numel() * workspace.element_size() < nbytes):
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=query.device)
    return nbytes, workspace


def paged_decode_q8(query, key_cache, value_cache, key_scale, value_scale, block_table, seq_lens, scale, out, n,
                    max_seq_len=None, workspace=None):
    """paged_decode over an 8-bit cache (kv_cache.py: codes int8 or float8_e4m3fn, one float32 scale per token and KV
    head). query (>=n, H, D) bf16 or fp16, D = 64, 128 or 256, at most 16 query heads per KV head; block_size a multiple
    of 8; out (>=n, H, D) in query's type. Computes the first n requests only and returns out.

    max_seq_len: no request is longer (a bound for the workspace; default: what the block table holds). Tokens behind
    it, and tokens on pages that the cache does not have, are not seen. A request of length 0 gives zeros. workspace: as
    in paged_decode (rows_workspace_bytes; contiguous), not to be shared by calls that may run at the same time. scale: finite, not 0."""
    if n <= 0:
        return out
    if query.shape[0] < n or out.shape[0] < n:
        raise ValueError("query and out need a row for every request")
    dev = _rows_operands("paged_decode_q8", query, key_cache, value_cache, block_table, seq_lens, out, n)
    code, (nb, BS, KV, _), sc, ss = kv_cache._check_cache(key_cache, value_cache, key_scale, value_scale, dev)
    seq_lens = seq_lens.contiguous()
    _, H, D = query.shape
    width = block_table.shape[1]
    max_len = width * BS if max_seq_len is None else min(max(0, int(max_seq_len)), width * BS)
    nbytes, workspace = _rows_scratch(n, H, D, max_len, workspace, query)
    sq, so = query.stride(), out.stride()
    with launch_on(dev) as stream:
        check("ex_paged_decode_q8", lib().ex_paged_decode_q8(
            query.data_ptr(), sq[0], sq[1], _DT16[query.dtype], key_cache.data_ptr(), value_cache.data_ptr(), code, sc[0],
            sc[1], sc[2], key_scale.data_ptr(), value_scale.data_ptr(), ss[0], ss[1], nb, block_table.data_ptr(),
            block_table.stride(0), width, seq_lens.data_ptr(), n, H, KV, D, BS, float(scale), max_len, out.data_ptr(),
            so[0], so[1], workspace.data_ptr() if nbytes else None, nbytes, stream))
    return out


def tree_attention(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, scale, out, max_query_len,
                   tree_mask=None, key_scale=None, value_scale=None, max_seq_len=None, workspace=None):
    """Attention of drafted tokens over a paged cache that already holds them. query (tokens, H, D) bf16 or fp16; request
    b has the rows query_start_loc[b] .. query_start_loc[b + 1] (int32, n + 1 entries; at most max_query_len <= 64 rows,
    which are the last tokens of its seq_lens[b] cached ones). Every row sees its request's context (the tokens before
    the drafted ones); of the drafted tokens row r sees number j if bit j of tree_mask[r] (int64, one word per row of
    query) is set, its own bit included if it is to see itself. tree_mask None: a chain, each row sees the drafted tokens
    up to itself. A row that sees nothing gives zeros.

    Weights are held in the cache's 16 bits (8-bit caches: float16), where paged_decode holds them as two bf16 numbers:
    over a 16-bit cache a token's bits are not those of paged_decode, and they depend on how many tokens were drafted
    with it (requests of more than 16 rows a KV head are another kernel's). They do not depend on the other requests, nor on
    what drafted tokens hold that the row does not see. Over an 8-bit cache one drafted token is paged_decode_q8's.

    The cache is 16-bit in query's type, any strides as in paged_decode, or 8-bit with key_scale and value_scale
    (kv_cache.py); block_size a multiple of 8. A request with more rows than max_query_len is left untouched, as are rows
    of out that belong to no request. max_seq_len and workspace as in paged_decode_q8. Returns out."""
    tokens = query.shape[0]
    n = query_start_loc.shape[0] - 1
    if query_start_loc.dtype != torch.int32 or query_start_loc.dim() != 1 or n < 0:
        raise TypeError("query_start_loc must be a 1-D int32 tensor with n + 1 entries")
    if not 1 <= max_query_len <= MAX_DRAFT:
        raise ValueError(f"max_query_len must be 1 to {MAX_DRAFT}")
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.dim() != 1 or tree_mask.shape[0] < tokens:
            raise TypeError("tree_mask must be a 1-D int64 tensor with a word for every row of query")
        tree_mask = tree_mask.contiguous()
    dev = _rows_operands("tree_attention", query, key_cache, value_cache, block_table, seq_lens, out, n)
    if query_start_loc.get_device() != dev or (tree_mask is not None and tree_mask.get_device() != dev):
        raise ValueError("tree_attention needs CUDA tensors of one device (there is no CPU fallback)")
    if out.shape[0] < tokens:
        raise ValueError("out must have a row for every row of query")
    if key_cache.dtype == query.dtype:
        if value_cache.dtype != key_cache.dtype or key_scale is not None or value_scale is not None:
            raise TypeError("a 16-bit cache has query's type and no scales")
        if value_cache.shape != key_cache.shape or value_cache.stride() != key_cache.stride() or key_cache.stride(3) != 1:
            raise ValueError("key and value caches must share shape and strides, with a contiguous head dimension")
        code, ks, vs, ss = _lib.EX_CODE_NONE, None, None, (0, 0)
    else:
        if key_scale is None or value_scale is None:
            raise TypeError("the cache must be in query's type, or 8-bit with key_scale and value_scale")
        code, _, _, ss = kv_cache._check_cache(key_cache, value_cache, key_scale, value_scale, dev)
        ks, vs = key_scale.data_ptr(), value_scale.data_ptr()
    if n == 0 or tokens == 0:
        return out
    seq_lens, query_start_loc = seq_lens.contiguous(), query_start_loc.contiguous()
    _, H, D = query.shape
    nb, BS, KV, _ = key_cache.shape
    width = block_table.shape[1]
    max_len = width * BS if max_seq_len is None else min(max(0, int(max_seq_len)), width * BS)
    nbytes, workspace = _rows_scratch(tokens, H, D, max_len, workspace, query)
    sq, sc, so = query.stride(), key_cache.stride(), out.stride()
    with launch_on(dev) as stream:
        check("ex_tree_attention", lib().ex_tree_attention(
            query.data_ptr(), sq[0], sq[1], _DT16[query.dtype], key_cache.data_ptr(), value_cache.data_ptr(), code, sc[0],
            sc[1], sc[2], ks, vs, ss[0], ss[1], nb, block_table.data_ptr(), block_table.stride(0), width,
            seq_lens.data_ptr(), query_start_loc.data_ptr(), None if tree_mask is None else tree_mask.data_ptr(), n,
            tokens, max_query_len, H, KV, D, BS, float(scale), max_len, out.data_ptr(), so[0], so[1],
            workspace.data_ptr() if nbytes else None, nbytes, stream))
    return out


def kv_views(kv_cache: torch.Tensor, head_size: int):
    """(key_cache, value_cache) as (num_blocks, block_size, KV, D) views of a vLLM FlashAttention KV cache.

    vLLM 0.32 layout [num_blocks, KV, block_size, 2 * D] (reference paged_attn.py:8-9, :145) and vLLM 0.22 layout
    (2, num_blocks, block_size, KV, D) (vllm/v1/attention/backends/flash_attn.py get_kv_cache_shape) are both
    accepted; the kernel reads them through strides."""
    if kv_cache.dim() == 5 and kv_cache.shape[0] == 2:
        return kv_cache[0], kv_cache[1]
    if kv_cache.dim() == 4 and kv_cache.shape[-1] == 2 * head_size:
        return kv_cache.transpose(1, 2).split(head_size, dim=-1)
    raise ValueError(f"unrecognised KV cache layout {tuple(kv_cache.shape)}")


def mixed_step_requests(query_start_loc, block_table, seq_lens, out) -> int:
    """Number of requests handed to the kernel in a mixed step: every request query_start_loc describes, bounded by
    the rows of the block table, seq_lens and the output (shapes only: no device value is read). The kernel then
    computes the leading one-token requests among them."""
    return max(0, min(query_start_loc.shape[0] - 1, block_table.shape[0], seq_lens.shape[0], out.shape[0]))


def install():
    """Patch vLLM's FlashAttentionImpl.forward (call before creating the LLM, with VLLM_ENABLE_V1_MULTIPROCESSING=0).

    Pure decode steps (max_query_len == 1) go entirely through paged_decode (CUDA-graph safe, no host sync). Mixed
    steps run vLLM's implementation first, then overwrite the leading decode tokens (vLLM orders decodes first) with
    paged_decode, so every decode token is always computed by this kernel (reference paged_attn.py:141-160). The
    reference counts those leading decodes on the host (an .item() sync); here the kernel reads query_start_loc and
    finds them itself, so mixed steps are also free of host syncs."""
    from vllm.v1.attention.backends import flash_attn as fa
    if hasattr(fa.FlashAttentionImpl.forward, "_vllm_exact_b200_orig"):
        return fa.FlashAttentionImpl.forward._vllm_exact_b200_orig  # already installed (install is idempotent)
    orig = fa.FlashAttentionImpl.forward
    DEC = fa.AttentionType.DECODER

    def forward(self, layer, query, key, value, kv_cache, attn_metadata, output, output_scale=None,
                output_block_scale=None):
        if attn_metadata is None or self.attn_type != DEC:
            return orig(self, layer, query, key, value, kv_cache, attn_metadata, output, output_scale,
                        output_block_scale)
        D = self.head_size
        key_cache, value_cache = kv_views(kv_cache, D)
        out3 = output.view(output.shape[0], self.num_heads, D)
        if attn_metadata.max_query_len == 1:
            n = attn_metadata.num_actual_tokens
            if n > 0:  # the KV cache write happens outside forward (unified_kv_cache_update) in these vLLM versions
                paged_decode(query, key_cache, value_cache, attn_metadata.block_table, attn_metadata.seq_lens,
                             self.scale, out3, n, attn_metadata.max_seq_len)
            return output
        res = orig(self, layer, query, key, value, kv_cache, attn_metadata, output, output_scale, output_block_scale)
        qsl = attn_metadata.query_start_loc
        nreq = mixed_step_requests(qsl, attn_metadata.block_table, attn_metadata.seq_lens, out3)
        if nreq > 0:
            paged_decode(query, key_cache, value_cache, attn_metadata.block_table, attn_metadata.seq_lens,
                         self.scale, out3, nreq, attn_metadata.max_seq_len, query_start_loc=qsl)
        return res

    forward._vllm_exact_b200_orig = orig
    fa.FlashAttentionImpl.forward = forward
    return orig

