"""cscr.pos_encoding — drop-in for the reference's pybind module of the same name.

``rotary_embedding_neox(postions, query, key, head_size, cos_sin_cache)`` keeps
the reference's signature (including the ``postions`` keyword spelling of
cscr/pos_encoding.cpp:20-25), its checks and messages
(cscr/pos_encoding_kernel.cu:79-104) and its effects: returns the rotated
query as a new tensor and rotates ``key`` in place.

``rotary_embedding_neox_with_cache`` additionally writes the rotated key and
the value into the paged KV cache in the same launch (the reference's RoPE
followed by its KV write, attention.py:151-157).

``qk_norm_rotary_embedding_neox`` and ``..._with_cache`` (not in the reference)
normalise each query and key head in the same pass.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import DTYPE_CODE, torch_check
from .cache import check_quantized_caches, token_stride

_INDEX_TYPES = (torch.int32, torch.int64)


def _check_rope(postions, query, key, head_size, cos_sin_cache, out):
    torch_check(postions.is_cuda, "positions must be a CUDA tensor")
    torch_check(query.is_cuda, "query must be a CUDA tensor")
    torch_check(key.is_cuda, "key must be a CUDA tensor")
    torch_check(cos_sin_cache.is_cuda, "cos_sin_cache must be a CUDA tensor")
    torch_check(query.is_contiguous(), "query must be contiguous")
    torch_check(key.is_contiguous(), "key must be contiguous")
    torch_check(out.is_contiguous(), "out must be contiguous")
    torch_check(cos_sin_cache.is_contiguous(), "cos_sin_cache must be contiguous")
    torch_check(query.dtype == key.dtype, "query and key must share dtype")
    torch_check(query.dtype == cos_sin_cache.dtype, "query and cos_sin_cache must share dtype")
    torch_check(query.dtype == out.dtype, "query and out must share dtype")
    torch_check(query.dim() == 2, "query must be [num_tokens, num_heads * head_size]")
    torch_check(key.dim() == 2, "key must be [num_tokens, num_kv_heads * head_size]")
    torch_check(postions.dim() == 1, "positions must be [num_tokens]")
    num_tokens = postions.numel()
    torch_check(num_tokens > 0, "positions must contain at least one token")
    torch_check(query.size(0) == num_tokens, "query must have one row per token")
    torch_check(key.size(0) == num_tokens, "key must have one row per token")
    torch_check(head_size > 0, "head_size must be positive")
    torch_check(query.size(1) % head_size == 0, "query size must be divisible by head_size")
    torch_check(key.size(1) % head_size == 0, "key size must be divisible by head_size")
    rot_dim = cos_sin_cache.size(1)
    torch_check(rot_dim > 0 and rot_dim % 2 == 0, "rotary dimension must be even and positive")
    torch_check(rot_dim <= head_size, "rotary dimension must not exceed head_size")
    torch_check(postions.dtype in _INDEX_TYPES, "positions must be int32 or int64")
    torch_check(query.dtype in (torch.float16, torch.bfloat16, torch.float32),
                "dtype must be float16, bfloat16 or float32")
    dev = query.device
    torch_check(key.device == dev and postions.device == dev and cos_sin_cache.device == dev,
                "all tensors must be on the same CUDA device")
    return num_tokens, rot_dim


def rotary_embedding_neox(postions: torch.Tensor, query: torch.Tensor, key: torch.Tensor,
                          head_size: int, cos_sin_cache: torch.Tensor) -> torch.Tensor:
    """Apply GPT-NeoX style rotary embedding to query (returned) and key (in place)."""
    out = torch.empty_like(query)
    num_tokens, rot_dim = _check_rope(postions, query, key, head_size, cos_sin_cache, out)
    dev = query.device
    with _lib.device_guard(dev):
        rc = _lib.load().tlb_rotary_embedding_neox(
            out.data_ptr(), postions.data_ptr(), DTYPE_CODE[postions.dtype], query.data_ptr(),
            key.data_ptr(), num_tokens, query.size(1) // head_size, key.size(1) // head_size,
            head_size, cos_sin_cache.data_ptr(), cos_sin_cache.size(0), rot_dim,
            query.stride(0), key.stride(0), out.stride(0), DTYPE_CODE[query.dtype],
            _lib.stream_of(dev))
        _lib.check(rc)
    return out


def rotary_embedding_neox_with_cache(postions: torch.Tensor, query: torch.Tensor,
                                     key: torch.Tensor, value: torch.Tensor,
                                     key_cache: torch.Tensor, value_cache: torch.Tensor,
                                     slot_mapping: torch.Tensor | None, head_size: int,
                                     cos_sin_cache: torch.Tensor,
                                     block_tables: torch.Tensor | None = None, *,
                                     overlap_previous: bool = False) -> torch.Tensor:
    """RoPE on query/key plus the KV-cache write of the rotated key and the value.

    query [T, H * head_size], key [T, KVH * head_size] (rotated in place),
    value [T, KVH, head_size] or [T, KVH * head_size], caches
    [num_blocks, KVH, block_size, head_size]. The destination of token t is
    slot_mapping[t] (int32/int64, slot = block * block_size + offset, negative =
    no write) or, when slot_mapping is None, block_tables[t, pos // block_size]
    at offset pos % block_size as src/model_executor/layers/attention.py:96-116
    addresses it (negative block id = no write).

    overlap_previous=True launches the kernel programmatically so that it
    starts while the kernel before it on the stream finishes; until then it
    reads only positions, slots, block tables and the cos/sin table. Use it
    only when that kernel writes none of those (an attention launch or a QKV
    projection). The next launch on the stream, if it overlaps too, may then
    begin while both run: neither may write what that one reads early (for an
    attention with overlap_prologue block_tables and seq_lens).
    """
    out = torch.empty_like(query)
    num_tokens, rot_dim = _check_rope(postions, query, key, head_size, cos_sin_cache, out)
    torch_check(value.is_cuda and key_cache.is_cuda and value_cache.is_cuda,
                "value and caches must be CUDA tensors")
    torch_check(key_cache.dim() == 4 and value_cache.shape == key_cache.shape,
                "key_cache and value_cache must be [num_blocks, num_kv_heads, block_size, head_size]")
    torch_check(key_cache.is_contiguous() and value_cache.is_contiguous(),
                "key_cache and value_cache must be contiguous")
    torch_check(key_cache.dtype == query.dtype and value_cache.dtype == query.dtype
                and value.dtype == query.dtype, "value and caches must share the query dtype")
    num_kv_heads = key.size(1) // head_size
    torch_check(key_cache.size(1) == num_kv_heads and key_cache.size(3) == head_size,
                "cache heads / head_size must match key")
    v2 = value.reshape(num_tokens, -1)
    torch_check(v2.size(1) == num_kv_heads * head_size and v2.stride(1) == 1,
                "value must be [num_tokens, num_kv_heads, head_size] with unit inner stride")
    if slot_mapping is not None:
        torch_check(slot_mapping.is_cuda and slot_mapping.dim() == 1
                    and slot_mapping.numel() == num_tokens
                    and slot_mapping.dtype in _INDEX_TYPES and slot_mapping.is_contiguous(),
                    "slot_mapping must be a contiguous [num_tokens] int32/int64 CUDA tensor")
        slots_ptr, slots_code, bt_ptr, bt_cols = slot_mapping.data_ptr(), \
            DTYPE_CODE[slot_mapping.dtype], None, 0
    else:
        torch_check(block_tables is not None, "either slot_mapping or block_tables is required")
        torch_check(block_tables.is_cuda and block_tables.dim() == 2
                    and block_tables.dtype == torch.int32 and block_tables.is_contiguous()
                    and block_tables.size(0) >= num_tokens,
                    "block_tables must be a contiguous int32 CUDA tensor with a row per token")
        slots_ptr, slots_code, bt_ptr, bt_cols = None, DTYPE_CODE[torch.int64], \
            block_tables.data_ptr(), block_tables.size(1)
    dev = query.device
    with _lib.device_guard(dev):
        rc = _lib.load().tlb_rotary_embedding_neox_with_cache(
            out.data_ptr(), postions.data_ptr(), DTYPE_CODE[postions.dtype], query.data_ptr(),
            key.data_ptr(), v2.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
            slots_ptr, slots_code, bt_ptr, bt_cols, num_tokens,
            query.size(1) // head_size, num_kv_heads, head_size, cos_sin_cache.data_ptr(),
            cos_sin_cache.size(0), rot_dim, key_cache.size(0), key_cache.size(2),
            query.stride(0), key.stride(0), v2.stride(0), out.stride(0),
            DTYPE_CODE[query.dtype], 1 if overlap_previous else 0, _lib.stream_of(dev))
        _lib.check(rc)
    return out


_CACHE8_TYPES = (torch.float8_e4m3fn, torch.int8)
_FLOAT_TYPES = (torch.float16, torch.bfloat16, torch.float32)


def _check_qk_norm(positions, query, key, query_weight, key_weight, eps, head_size, cos_sin_cache):
    """The checks of ``_qk_norm_shapes`` one by one, for their messages."""
    torch_check(query.is_cuda, "query must be a CUDA tensor")
    dev, dtype = query.device, query.dtype
    torch_check(key.device == dev and positions.device == dev and cos_sin_cache.device == dev
                and query_weight.device == dev and key_weight.device == dev,
                "all tensors must be on the same CUDA device")
    torch_check(dtype in _FLOAT_TYPES, "dtype must be float16, bfloat16 or float32")
    torch_check(key.dtype == dtype and cos_sin_cache.dtype == dtype
                and query_weight.dtype == dtype and key_weight.dtype == dtype,
                "query, key, cos_sin_cache and the weights must share a dtype")
    torch_check(positions.dim() == 1 and positions.dtype in _INDEX_TYPES
                and positions.is_contiguous(),
                "positions must be a contiguous [num_tokens] int32 or int64 tensor")
    torch_check(head_size > 0, "head_size must be positive")
    for x in (query, key):
        torch_check(x.dim() == 2 and x.size(0) == positions.size(0) and x.size(1) > 0
                    and x.size(1) % head_size == 0 and x.stride(1) == 1,
                    "query and key must be [num_tokens, heads * head_size] with unit inner stride")
    torch_check(query_weight.shape == (head_size,) and key_weight.shape == (head_size,)
                and query_weight.is_contiguous() and key_weight.is_contiguous(),
                "query_weight and key_weight must be contiguous [head_size] tensors")
    torch_check(cos_sin_cache.dim() == 2 and cos_sin_cache.size(0) > 0
                and cos_sin_cache.is_contiguous(),
                "cos_sin_cache must be a contiguous [rows, rotary_dim] tensor")
    rot_dim = cos_sin_cache.size(1)
    torch_check(rot_dim > 0 and rot_dim % 2 == 0, "rotary dimension must be even and positive")
    torch_check(rot_dim <= head_size, "rotary dimension must not exceed head_size")
    torch_check(eps >= 0, "eps must not be negative")
    raise RuntimeError("qk_norm_rotary_embedding_neox: unsupported arguments")


def _qk_norm_shapes(positions, query, key, query_weight, key_weight, eps, head_size,
                    cos_sin_cache):
    """Checks shared by the two entry points below, as one expression (a call's
    host time counts in a decode step): (device index, tokens, query stride, key
    stride, query width, key width, table rows, rotary dimension)."""
    index, dtype = query.get_device(), query.dtype
    (qs, ks), (qshape, kshape, tshape) = (query.stride(), key.stride()), (
        query.shape, key.shape, cos_sin_cache.shape)
    wshape = (head_size,)
    if not (index >= 0 and len(qshape) == 2 and len(kshape) == 2 and len(tshape) == 2
            and dtype in _FLOAT_TYPES and key.dtype == dtype and cos_sin_cache.dtype == dtype
            and query_weight.dtype == dtype and key_weight.dtype == dtype and head_size > 0
            and positions.shape == qshape[:1] and positions.dtype in _INDEX_TYPES
            and kshape[0] == qshape[0] and qs[1] == 1 and ks[1] == 1 and qshape[1] > 0
            and kshape[1] > 0 and qshape[1] % head_size == 0 and kshape[1] % head_size == 0
            and query_weight.shape == wshape and key_weight.shape == wshape and tshape[0] > 0
            and 0 < tshape[1] <= head_size and tshape[1] % 2 == 0 and eps >= 0
            and positions.is_contiguous() and query_weight.is_contiguous()
            and key_weight.is_contiguous() and cos_sin_cache.is_contiguous()
            and key.get_device() == index and positions.get_device() == index
            and cos_sin_cache.get_device() == index and query_weight.get_device() == index
            and key_weight.get_device() == index):
        _check_qk_norm(positions, query, key, query_weight, key_weight, eps, head_size,
                       cos_sin_cache)
    return index, qshape[0], qs[0], ks[0], qshape[1], kshape[1], tshape[0], tshape[1]


def qk_norm_rotary_embedding_neox(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor,
                                  query_weight: torch.Tensor, key_weight: torch.Tensor,
                                  eps: float, head_size: int, cos_sin_cache: torch.Tensor
                                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each query and key head, then the NeoX rotation, in one pass.

    For each head row x: ``y = x * rsqrt(mean(x^2) + eps) * weight``, then the
    pairs (i, i + rotary_dim / 2) are rotated by their token's cos_sin_cache row;
    fp32 math, one rounding. query [T, H * head_size] and key [T, KVH *
    head_size], rows possibly strided (parts of a fused projection); weights
    [head_size]. Returns new dense (query, key); the inputs are left as they are.
    """
    if _lib.fast is not None:
        both = _lib.fast.norm(positions, query, key, None, query_weight, key_weight, eps, None,
                              None, None, head_size, cos_sin_cache, None, None, None, False)
        if both is not None:
            return both
    index, num_tokens, q_stride, k_stride, q_width, k_width, rows, rot_dim = _qk_norm_shapes(
        positions, query, key, query_weight, key_weight, eps, head_size, cos_sin_cache)
    q_out = torch.empty_like(query, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(key, memory_format=torch.contiguous_format)
    if num_tokens == 0:
        return q_out, k_out
    code = DTYPE_CODE[query.dtype]
    _lib.launch(_lib.QK_NORM_ROPE, index, q_out.data_ptr(), k_out.data_ptr(),
                positions.data_ptr(), query.data_ptr(), key.data_ptr(), 0,
                query_weight.data_ptr(), key_weight.data_ptr(), 0, 0, 0, 0, 0, 0,
                cos_sin_cache.data_ptr(), DTYPE_CODE[positions.dtype], 4, 0, num_tokens,
                q_width // head_size, k_width // head_size, head_size, rows, rot_dim, 0, 0,
                q_stride, k_stride, 0, code, code, 0, eps)
    return q_out, k_out


def qk_norm_rotary_embedding_neox_with_cache(
        positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
        query_weight: torch.Tensor, key_weight: torch.Tensor, eps: float,
        key_cache: torch.Tensor, value_cache: torch.Tensor, slot_mapping: torch.Tensor | None,
        head_size: int, cos_sin_cache: torch.Tensor, block_tables: torch.Tensor | None = None, *,
        key_scales: torch.Tensor | None = None, value_scales: torch.Tensor | None = None,
        overlap_previous: bool = False) -> torch.Tensor:
    """``qk_norm_rotary_embedding_neox`` with the KV-cache write of the key and
    the value in the same launch; returns the new query.

    The key goes to its cache row only; ``key`` and ``value`` are left as they
    are. value [T, KVH, head_size] or [T, KVH * head_size], rows possibly strided.
    The caches [num_blocks, KVH, block_size, head_size] have the query dtype, or
    are float8_e4m3fn or int8 with ``key_scales`` and ``value_scales``
    (float8_e8m0fnu): then the stored rows are those that
    ``cscr.cache.reshape_and_cache_quantized`` stores for the key as rounded to
    the query dtype. Destinations as in ``rotary_embedding_neox_with_cache``; the
    slots of one call must differ. ``overlap_previous`` is accepted and changes
    nothing: the kernel reads nothing before the one before it has ended.
    """
    if key_cache is None or value_cache is None or value is None:
        raise RuntimeError("key_cache, value_cache and value must be given "
                           "(qk_norm_rotary_embedding_neox writes no cache)")
    if _lib.fast is not None:
        out = _lib.fast.norm(positions, query, key, value, query_weight, key_weight, eps,
                             key_cache, value_cache, slot_mapping, head_size, cos_sin_cache,
                             block_tables, key_scales, value_scales, overlap_previous)
        if out is not None:
            return out
    index, num_tokens, q_stride, k_stride, q_width, k_width, rows, rot_dim = _qk_norm_shapes(
        positions, query, key, query_weight, key_weight, eps, head_size, cos_sin_cache)
    dtype, cache_dtype, cshape = query.dtype, key_cache.dtype, key_cache.shape
    kvh = k_width // head_size
    ks_ptr = vs_ptr = 0
    if cache_dtype in _CACHE8_TYPES:
        torch_check(key_scales is not None and value_scales is not None,
                    "8-bit caches need key_scales and value_scales")
        cache_index = check_quantized_caches(key_cache, value_cache, key_scales, value_scales)
        ks_ptr, vs_ptr = key_scales.data_ptr(), value_scales.data_ptr()
    else:
        torch_check(key_scales is None and value_scales is None,
                    "key_scales and value_scales belong to 8-bit caches")
        torch_check(len(cshape) == 4 and value_cache.shape == cshape,
                    "key_cache and value_cache must be [num_blocks, num_kv_heads, block_size, "
                    "head_size]")
        torch_check(cache_dtype == dtype and value_cache.dtype == dtype,
                    "the caches must have the query dtype, or be float8_e4m3fn or int8")
        torch_check(key_cache.is_contiguous() and value_cache.is_contiguous(),
                    "key_cache and value_cache must be contiguous")
        cache_index = key_cache.get_device()
        torch_check(value_cache.get_device() == cache_index,
                    "all tensors must be on the same CUDA device")
    torch_check(cache_index == index and value.get_device() == index,
                "all tensors must be on the same CUDA device")
    torch_check(cshape[1] == kvh and cshape[3] == head_size and value.dtype == dtype,
                "cache heads / head_size must match key, and value must have the query dtype")
    v_stride = token_stride(value, num_tokens, kvh, head_size, "value")
    if slot_mapping is not None:
        torch_check(slot_mapping.get_device() == index and slot_mapping.shape == (num_tokens,)
                    and slot_mapping.dtype in _INDEX_TYPES and slot_mapping.is_contiguous(),
                    "slot_mapping must be a contiguous [num_tokens] int32/int64 CUDA tensor")
        slots, slot_code, tables, width = (slot_mapping.data_ptr(),
                                           DTYPE_CODE[slot_mapping.dtype], 0, 0)
    else:
        torch_check(block_tables is not None, "either slot_mapping or block_tables is required")
        torch_check(block_tables.get_device() == index and block_tables.dim() == 2
                    and block_tables.dtype == torch.int32 and block_tables.is_contiguous()
                    and block_tables.size(0) >= num_tokens and block_tables.size(1) > 0,
                    "block_tables must be a contiguous int32 CUDA tensor with a row per token")
        slots, slot_code, tables, width = 0, 4, block_tables.data_ptr(), block_tables.size(1)
    q_out = torch.empty_like(query, memory_format=torch.contiguous_format)
    if num_tokens == 0:
        return q_out
    _lib.launch(_lib.QK_NORM_ROPE, index, q_out.data_ptr(), 0, positions.data_ptr(),
                query.data_ptr(), key.data_ptr(), value.data_ptr(), query_weight.data_ptr(),
                key_weight.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), ks_ptr,
                vs_ptr, slots, tables, cos_sin_cache.data_ptr(), DTYPE_CODE[positions.dtype],
                slot_code, width, num_tokens, q_width // head_size, kvh, head_size, rows,
                rot_dim, cshape[0], cshape[2], q_stride, k_stride, v_stride, DTYPE_CODE[dtype],
                DTYPE_CODE[cache_dtype], 1 if overlap_previous else 0, eps)
    return q_out
