"""The 8-bit paged KV cache: quantised as it is written, read back, and (paged_attn.py) attended over.

A row of the cache is the D numbers of one token and KV head. It is held as 8-bit codes c (int8, or float8_e4m3fn) and
one float32 scale s = max|x| / Q, c = x / s rounded to nearest even, Q = 127 or 448, and stands for c * s. Against a
16-bit cache it takes half the memory and half the traffic of a decode step, plus 4 bytes of scale per row.

* ``alloc_q8_cache``   the four tensors of a cache;
* ``cache_write``      new tokens' keys and values into their slots, and on request the numbers they now stand for;
* ``cache_read``       whole sequences back as packed 16-bit rows (for prompt attention over a cached beginning).

The reference has no counterpart (its caches are bf16, src/vllm_exact/paged_attn.py:8-9). There is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check, launch_on, lib

__all__ = ["alloc_q8_cache", "cache_write", "cache_read"]

_DT = {torch.bfloat16: _lib.EX_DTYPE_BF16, torch.float16: _lib.EX_DTYPE_F16}
CODES = {torch.int8: _lib.EX_CODE_INT8, torch.float8_e4m3fn: _lib.EX_CODE_E4M3}


def alloc_q8_cache(num_blocks: int, block_size: int, KV: int, D: int, dtype=torch.float8_e4m3fn, device="cuda"):
    """(key_cache, value_cache, key_scale, value_scale) of zeros: codes (num_blocks, block_size, KV, D) of dtype int8 or
    float8_e4m3fn, scales (num_blocks, KV, block_size) float32 (a head's consecutive tokens lie side by side)."""
    if dtype not in CODES:
        raise TypeError(f"unsupported cache dtype {dtype}")
    codes = [torch.zeros(num_blocks, block_size, KV, D, dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
    scales = [torch.zeros(num_blocks, KV, block_size, dtype=torch.float32, device=device) for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def _check_cache(key_cache, value_cache, key_scale, value_scale, dev):
    """Types, shapes, strides and device of the four tensors of an 8-bit cache; its code as the library names it, its shape
    and the strides of its codes and scales."""
    kind = key_cache.dtype
    code = CODES.get(kind)
    if code is None or value_cache.dtype != kind:
        raise TypeError("an 8-bit cache holds int8 or float8_e4m3fn codes, the same for keys and values")
    if key_scale.dtype != torch.float32 or value_scale.dtype != torch.float32:
        raise TypeError("the scales of an 8-bit cache are float32")
    shape, scales = key_cache.shape, key_scale.shape
    if len(shape) != 4 or value_cache.shape != shape:
        raise ValueError("codes must be (num_blocks, block_size, KV, D), the same for keys and values")
    if len(scales) != 3 or (shape[0], shape[2], shape[1]) != scales or value_scale.shape != scales:
        raise ValueError("scales must be (num_blocks, KV, block_size)")
    st, ss = key_cache.stride(), key_scale.stride()
    if value_cache.stride() != st or value_scale.stride() != ss:
        raise ValueError("key and value caches must share strides")
    if st[3] != 1 or ss[2] != 1:
        raise ValueError("the head dimension of codes and the places of scales must be contiguous")
    if not key_cache.get_device() == value_cache.get_device() == key_scale.get_device() == value_scale.get_device() == dev:
        raise ValueError("the cache must be on the same CUDA device as the other tensors")
    return code, shape, st, ss


def _check_rows(name, a, b, KV, D):
    """Types, shapes and head dimensions of keys and values as packed rows; their type as the library names it, their number
    and strides."""
    kind, shape = a.dtype, a.shape
    dtype = _DT.get(kind)
    if dtype is None or b.dtype != kind:
        raise TypeError(f"{name} must be bf16 or fp16, the same for keys and values")
    if len(shape) != 3 or b.shape != shape or shape[1] != KV or shape[2] != D:
        raise ValueError(f"{name} must be (tokens, {KV}, {D}), the same for keys and values")
    sa, sb = a.stride(), b.stride()
    if sa[2] != 1 or sb[2] != 1:
        raise ValueError(f"the head dimension of {name} must be contiguous")
    return dtype, shape[0], sa, sb


def cache_write(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping, key_out=None, value_out=None):
    """Quantise key and value (tokens, KV, D) bf16 or fp16 (any token and head strides that are multiples of 8, for
    instance slices of one projection's output) into an 8-bit cache: token t goes to block slot_mapping[t] // block_size,
    place slot_mapping[t] % block_size. A token whose slot is negative or outside the cache is not written. The slots of
    one call must differ from each other: what a slot that is named twice holds is not defined.

    key_out, value_out (tokens, KV, D), in key's type: receive the numbers which the rows stand for, so that the prompt
    that is being cached can attend to what later steps will see. Rows with an infinity or a NaN read back as NaN."""
    dev = key.get_device()  # -1: not on a GPU
    if dev < 0 or value.get_device() != dev or slot_mapping.get_device() != dev:
        raise ValueError("cache_write needs CUDA tensors of one device (there is no CPU fallback)")
    code, (nb, BS, KV, D), sc, ss = _check_cache(key_cache, value_cache, key_scale, value_scale, dev)
    dtype, T, sk, sv = _check_rows("key and value", key, value, KV, D)
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or slot_mapping.shape[0] != T:
        raise ValueError("slot_mapping must be a 1-D int64 tensor with a slot for every token")
    if (key_out is None) != (value_out is None):
        raise ValueError("key_out and value_out are given together")
    ko, vo, sko, svo = None, None, (0, 0), (0, 0)
    if key_out is not None:
        dtype_out, T_out, sko, svo = _check_rows("key_out and value_out", key_out, value_out, KV, D)
        if dtype_out != dtype or T_out != T or key_out.get_device() != dev or value_out.get_device() != dev:
            raise ValueError("key_out and value_out must be like key")
        ko, vo = key_out.data_ptr(), value_out.data_ptr()
    slot_mapping = slot_mapping.contiguous()
    with launch_on(dev) as stream:
        check("ex_cache_write_q8", lib().ex_cache_write_q8(
            key.data_ptr(), sk[0], sk[1], value.data_ptr(), sv[0], sv[1], dtype, code, key_cache.data_ptr(),
            value_cache.data_ptr(), sc[0], sc[1], sc[2], key_scale.data_ptr(), value_scale.data_ptr(), ss[0], ss[1], nb,
            BS, slot_mapping.data_ptr(), T, KV, D, ko, sko[0], sko[1], vo, svo[0], svo[1], stream))


def cache_read(key_cache, value_cache, key_scale, value_scale, block_table, cu_seqlens, key_out, value_out):
    """Read the first cu_seqlens[b + 1] - cu_seqlens[b] tokens of every sequence b back into rows cu_seqlens[b] .. of
    key_out and value_out (rows, KV, D) bf16 or fp16; block_table (n, pages) int32, cu_seqlens (n + 1) int32. Rows of no
    sequence, behind the block table, or on a page that the cache does not have are left as they were."""
    dev = key_out.get_device()  # -1: not on a GPU
    if dev < 0 or value_out.get_device() != dev or block_table.get_device() != dev or cu_seqlens.get_device() != dev:
        raise ValueError("cache_read needs CUDA tensors of one device (there is no CPU fallback)")
    code, (nb, BS, KV, D), sc, ss = _check_cache(key_cache, value_cache, key_scale, value_scale, dev)
    dtype, rows, sk, sv = _check_rows("key_out and value_out", key_out, value_out, KV, D)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or cu_seqlens.dtype != torch.int32:
        raise TypeError("block_table (n, pages) and cu_seqlens must be int32")
    n, width = block_table.shape
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] != n + 1:
        raise ValueError("cu_seqlens needs n + 1 entries")
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError("block table rows must be contiguous")
    cu_seqlens = cu_seqlens.contiguous()
    with launch_on(dev) as stream:
        check("ex_cache_read_q8", lib().ex_cache_read_q8(
            key_cache.data_ptr(), value_cache.data_ptr(), code, sc[0], sc[1], sc[2], key_scale.data_ptr(),
            value_scale.data_ptr(), ss[0], ss[1], nb, BS, block_table.data_ptr(), block_table.stride(0), width,
            cu_seqlens.data_ptr(), n, rows, KV, D, dtype, key_out.data_ptr(),
            sk[0], sk[1], value_out.data_ptr(), sv[0], sv[1], stream))
    return key_out, value_out
