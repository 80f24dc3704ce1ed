"""Layer glue of the decode step on the sm_100a ops.

``PagedAttention`` and ``PagedAttentionWithRoPE`` keep the constructors,
buffers and forward signatures of src/model_executor/layers/attention.py:7-166,
so a model built against the reference's layers runs on these unchanged.
The forward of ``PagedAttentionWithRoPE`` does the reference's three steps —
RoPE (:151-153), the KV-cache write (:155-157) and paged attention (:160-166) —
in two launches: one fused RoPE + cache-write kernel addressed through the
block tables exactly as ``_write_kv_cache`` addresses it, then the attention
kernel. Unlike the reference it does not synchronise the host (the
``valid.any()`` of :103) and converts the cos/sin table once per device and
dtype instead of on every call (:148-150).

``positions=None`` states the decode invariant the reference's worker builds
(src/worker/worker.py:144-146,154: a decode token sits at position
``context_len - 1`` and ``seq_lens`` holds the context lengths), so the
position of every token is ``seq_lens - 1``; with full-width rotary
(``rotary_dim == head_size``) the whole step then runs as ONE launch
(``cscr.attention.paged_attention_with_rope``).

``PagedAttentionWithQKNorm`` (not in the reference) is the same layer for models
that normalise each query and key head, cap their scores or limit them to a
window, over caches of the model dtype or of 8 bits.

``QuantizedLinear`` and ``QuantizedDecoderLayer`` (not in the reference) put
projections with 8-bit weights and activations (``cscr.linear``) around either
attention layer: a whole decoder layer.
"""

from __future__ import annotations

import torch
from torch import nn

from cscr import attention as _C
from cscr import cache as _Cache
from cscr import linear as _Linear
from cscr import pos_encoding as _PE

from . import metadata


class PagedAttention(nn.Module):
    def __init__(self, num_heads: int, head_size: int, scale: float):
        super().__init__()
        self.num_heads = num_heads
        self.head_size = head_size
        self.scale = scale

    def forward(self, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                block_tables: torch.Tensor, seq_lens: torch.Tensor) -> torch.Tensor:
        """query [S, H, D]; caches [NB, KVH, bs, D]; block_tables [S, maxB] int32;
        seq_lens [S] int32 -> [S, H, D]."""
        return _C.paged_attention(query=query, key_cache=key_cache, value_cache=value_cache,
                                  block_tables=block_tables, seq_lens=seq_lens, scale=self.scale)


class PagedAttentionWithRoPE(PagedAttention):
    def __init__(self, num_heads: int, head_size: int, scale: float, rotary_dim: int,
                 max_position: int = 8192, base: int = 10000):
        super().__init__(num_heads, head_size, scale)
        if rotary_dim <= 0 or rotary_dim % 2 != 0:
            raise ValueError("rotary_dim must be a positive even number")
        if rotary_dim > head_size:
            raise ValueError("rotary_dim must not exceed head_size")
        self.rotary_dim = rotary_dim
        # Same expression, same default-dtype dependence as attention.py:71-79.
        inv_freq = 1.0 / (base ** (torch.arange(0, rotary_dim, 2) / rotary_dim))
        t = torch.arange(max_position).float()
        freqs = torch.einsum("i,j -> ij", t, inv_freq.float())
        cache = torch.cat((freqs.cos(), freqs.sin()), dim=-1)
        cache = cache.to(torch.get_default_dtype())
        self.register_buffer("cos_sin_cache", cache, persistent=False)
        self._cs_cast: dict[tuple, torch.Tensor] = {}

    def _table(self, device: torch.device, dtype: torch.dtype) -> torch.Tensor:
        key = (device, dtype, self.cos_sin_cache.data_ptr(), self.cos_sin_cache._version)
        t = self._cs_cast.get(key)
        if t is None:
            self._cs_cast.clear()
            t = self.cos_sin_cache.to(device=device, dtype=dtype).contiguous()
            self._cs_cast[key] = t
        return t

    def _write_kv_cache(self, key, value, positions, key_cache, value_cache, block_tables):
        """attention.py:82-116 as one kernel (no host sync)."""
        _Cache.write_kv_cache(key, value, positions, key_cache, value_cache,
                              block_tables.to(torch.int32))

    def forward(self, positions: torch.Tensor | None, query: torch.Tensor, key: torch.Tensor,
                value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                block_tables: torch.Tensor, seq_lens: torch.Tensor) -> torch.Tensor:
        if query.dim() != 3:
            raise ValueError("query must be [num_tokens, num_heads, head_dim]")
        if key.dim() != 3:
            raise ValueError("key must be [num_tokens, num_kv_heads, head_dim]")
        if value.dim() != 3:
            raise ValueError("value must be [num_tokens, num_kv_heads, head_dim]")
        num_tokens, num_heads, head_size = query.shape
        if head_size != self.head_size:
            raise ValueError("query head_dim must match head_size")
        if num_tokens != block_tables.size(0):
            raise NotImplementedError(
                "PagedAttentionWithRoPE only supports decode: there must be one token per sequence")

        cos_sin_cache = self._table(query.device, query.dtype)
        tables = block_tables if block_tables.dtype == torch.int32 else block_tables.to(torch.int32)
        tables = tables.contiguous()
        if positions is None:
            if self.rotary_dim == head_size:
                # RoPE, cache write and attention in one launch; the key is
                # rotated in place, as rotary_embedding_neox does to it
                return _C.paged_attention_with_rope(
                    query.contiguous(), key, value, key_cache, value_cache, tables, seq_lens,
                    cos_sin_cache, self.scale)
            positions = seq_lens.to(torch.int64) - 1
        query_2d = query.reshape(num_tokens, num_heads * head_size).contiguous()
        key_2d = key.reshape(num_tokens, -1).contiguous()
        fused = key_cache.dtype == query.dtype and value.dtype == query.dtype
        if fused:
            query_2d = _PE.rotary_embedding_neox_with_cache(
                positions, query_2d, key_2d, value, key_cache, value_cache, None,
                self.head_size, cos_sin_cache, block_tables=tables)
        else:
            query_2d = _PE.rotary_embedding_neox(positions, query_2d, key_2d, self.head_size,
                                                 cos_sin_cache)
            self._write_kv_cache(key_2d, value, positions, key_cache, value_cache, tables)
        query = query_2d.view(num_tokens, num_heads, head_size)
        # The kernel just launched (RoPE + cache write) writes neither the
        # block tables nor seq_lens, so attention may overlap its prologue.
        return _C.paged_attention(query=query, key_cache=key_cache, value_cache=value_cache,
                                  block_tables=tables, seq_lens=seq_lens, scale=self.scale,
                                  overlap_prologue=fused)


class PagedAttentionWithQKNorm(PagedAttentionWithRoPE):
    """``PagedAttentionWithRoPE`` with an RMS norm of each query and key head,
    optionally capped scores (``softcap``) and a window, over 16-bit caches or
    8-bit ones with their row scales (``paged_decode.pool.
    allocate_quantized_kv_cache``).

    A decode step is two launches: norm, rotation and cache write, then
    attention. ``prompt`` serves prompt chunks; over 8-bit caches it reads the
    chunks' blocks back and runs the 16-bit prefill kernel on them.
    """

    def __init__(self, num_heads: int, head_size: int, scale: float, rotary_dim: int,
                 max_position: int = 8192, base: int = 10000, eps: float = 1e-6,
                 softcap: float = 0.0, window: int = 0):
        super().__init__(num_heads, head_size, scale, rotary_dim, max_position, base)
        self.eps, self.softcap, self.window = eps, softcap, window
        self.q_norm = nn.Parameter(torch.ones(head_size), requires_grad=False)
        self.k_norm = nn.Parameter(torch.ones(head_size), requires_grad=False)

    def _norm_rope_write(self, positions, query, key, value, key_cache, value_cache, slots, tables,
                         key_scales, value_scales):
        num_tokens, num_heads, head_size = query.shape
        if head_size != self.head_size:
            raise ValueError("query head_dim must match head_size")
        dtype = query.dtype
        out = _PE.qk_norm_rotary_embedding_neox_with_cache(
            positions, query.reshape(num_tokens, -1), key.reshape(num_tokens, -1), value,
            self.q_norm.to(dtype), self.k_norm.to(dtype), self.eps, key_cache, value_cache, slots,
            head_size, self._table(query.device, dtype), block_tables=tables,
            key_scales=key_scales, value_scales=value_scales)
        return out.view(num_tokens, num_heads, head_size)

    def forward(self, positions: torch.Tensor | None, query: torch.Tensor, key: torch.Tensor,
                value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                block_tables: torch.Tensor, seq_lens: torch.Tensor,
                key_scales: torch.Tensor | None = None,
                value_scales: torch.Tensor | None = None) -> torch.Tensor:
        """A decode step: query [S, H, D], key and value [S, KVH, D], one token per
        sequence, at ``positions`` or (None) at ``seq_lens - 1`` -> [S, H, D]."""
        if query.dim() != 3 or query.size(0) != block_tables.size(0):
            raise NotImplementedError(
                "PagedAttentionWithQKNorm.forward is a decode step: there must be one token per "
                "sequence")
        tables = block_tables.to(torch.int32).contiguous()
        if positions is None:
            positions = seq_lens.to(torch.int64) - 1
        query = self._norm_rope_write(positions, query, key, value, key_cache, value_cache, None,
                                      tables, key_scales, value_scales)
        # The kernel just launched writes neither the tables nor seq_lens, so
        # attention may overlap its prologue.
        if key_scales is not None:
            return _C.paged_attention_quantized(
                query, key_cache, value_cache, key_scales, value_scales, tables, seq_lens,
                self.scale, softcap=self.softcap, window=self.window, overlap_prologue=True)
        if self.softcap or self.window:
            return _C.paged_attention_biased(query, key_cache, value_cache, tables, seq_lens,
                                             self.scale, softcap=self.softcap, window=self.window,
                                             overlap_prologue=True)
        return _C.paged_attention(query, key_cache, value_cache, tables, seq_lens, self.scale,
                                  overlap_prologue=True)

    def prompt(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor,
               value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
               slot_mapping: torch.Tensor, block_tables: torch.Tensor, query_start: torch.Tensor,
               context_lens: torch.Tensor, max_query_len: int | None = None,
               key_scales: torch.Tensor | None = None,
               value_scales: torch.Tensor | None = None) -> torch.Tensor:
        """Prompt chunks (packed tokens [T, ...]), as ``cscr.attention.
        paged_prefill_attention`` takes them; the new rows go to ``slot_mapping``.
        Over 8-bit caches every entry of ``block_tables`` costs a block of each
        cache in the query dtype: pass no more columns than the contexts need."""
        if self.softcap or self.window:
            raise NotImplementedError("prompt chunks have plain scores: no softcap, no window")
        if query.size(0) == 0:  # a step without prompt tokens
            return torch.empty_like(query)
        query = self._norm_rope_write(positions, query, key, value, key_cache, value_cache,
                                      slot_mapping, None, key_scales, value_scales)
        tables = block_tables.to(torch.int32).contiguous()
        if key_scales is not None:
            # the chunks' blocks in the query dtype, and the table that finds them
            ids, tables = metadata.read_back_tables(tables, context_lens.contiguous(),
                                                    key_cache.size(2), key_cache.size(0))
            key_cache, value_cache = _Cache.dequantize_blocks(
                key_cache, value_cache, key_scales, value_scales, ids.view(-1), query.dtype)
        return _C.paged_prefill_attention(query, key_cache, value_cache, tables, query_start,
                                          context_lens, self.scale, max_query_len)


class QuantizedLinear(nn.Module):
    """A projection with 8-bit weights and activations (``cscr.linear.
    matmul_quantized``): [T, in_features] -> [T, out_features] of ``dtype``.

    The weight is kept as bytes, so that ``.to(dtype)`` (which sets the results' type)
    and ``state_dict`` leave it alone: ``weight_bytes`` [out_features, in_features] of float8_e4m3fn and
    ``scale_bytes`` [ceil(out / 128), ceil(in / 128)] of float8_e8m0fnu.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = False,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None):
        super().__init__()
        groups = -(-in_features // _Linear.GROUP)
        self.dtype = dtype
        self.register_buffer("weight_bytes", torch.zeros(
            (out_features, in_features), dtype=torch.uint8, device=device))
        self.register_buffer("scale_bytes", torch.full(
            (-(-out_features // _Linear.GROUP), groups), 127, dtype=torch.uint8, device=device))
        self.bias = nn.Parameter(torch.zeros(out_features, dtype=dtype, device=device),
                                 requires_grad=False) if bias else None

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None
                    ) -> QuantizedLinear:
        """The projection whose weight is ``weight`` [out, in] (float16, bfloat16 or
        float32, of finite values) in 8 bits; results and bias have its dtype."""
        m = cls(weight.size(1), weight.size(0), bias is not None, weight.dtype, weight.device)
        values, scales = _Linear.quantize_weight(weight.detach())
        m.weight_bytes, m.scale_bytes = values.view(torch.uint8), scales.view(torch.uint8)
        if bias is not None:
            m.bias = nn.Parameter(bias.detach().to(weight.dtype), requires_grad=False)
        return m

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self.dtype = fn(torch.empty(0, dtype=self.dtype)).dtype  # as the bias's
        return self

    def forward(self, x: torch.Tensor | tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
        """x: rows in float16, bfloat16 or float32 (quantised first), or 8-bit rows as
        (values, scales)."""
        values, scales = _Linear.quantize_rows(x) if isinstance(x, torch.Tensor) else x
        return _Linear.matmul_quantized(values, scales, self.weight_bytes.view(torch.float8_e4m3fn),
                                        self.scale_bytes.view(torch.float8_e8m0fnu), self.dtype,
                                        self.bias)


class QuantizedDecoderLayer(nn.Module):
    """A decoder layer with 8-bit projections around a paged attention layer.

    ``attention``: ``PagedAttentionWithRoPE`` or ``PagedAttentionWithQKNorm``.
    ``qkv`` gives each token's queries, keys and values side by side, ``gate_up`` its
    gate and up values. Each half of the layer is a norm with the residual's addition
    and an 8-bit output, the projections, and attention or the gated activation, whose
    result is quantised for the projection behind it.
    """

    def __init__(self, attention: PagedAttention, num_kv_heads: int, qkv: QuantizedLinear,
                 out: QuantizedLinear, gate_up: QuantizedLinear, down: QuantizedLinear,
                 input_norm: torch.Tensor, post_norm: torch.Tensor, eps: float = 1e-6):
        super().__init__()
        self.attention, self.num_kv_heads, self.eps = attention, num_kv_heads, eps
        self.qkv, self.out, self.gate_up, self.down = qkv, out, gate_up, down
        self.input_norm = nn.Parameter(input_norm.detach(), requires_grad=False)
        self.post_norm = nn.Parameter(post_norm.detach(), requires_grad=False)

    def _project(self, hidden, residual):
        values, scales, summed = _Linear.rms_norm_quantized(hidden, self.input_norm, self.eps,
                                                            residual)
        qkv = self.qkv((values, scales))
        d = self.attention.head_size
        q, k = self.attention.num_heads * d, self.num_kv_heads * d
        parts = [p.unflatten(1, (-1, d)) for p in qkv.split([q, k, k], 1)]
        return parts, hidden if summed is None else summed

    def _rest(self, attended, residual):
        hidden = self.out(attended.flatten(1))
        values, scales, residual = _Linear.rms_norm_quantized(hidden, self.post_norm, self.eps,
                                                              residual)
        gated = _Linear.silu_and_mul_quantized(self.gate_up((values, scales)))
        return self.down(gated), residual

    def forward(self, positions: torch.Tensor | None, hidden: torch.Tensor,
                residual: torch.Tensor | None, key_cache: torch.Tensor,
                value_cache: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                *scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """A decode step: hidden [S, width], what the layer before added to the residual
        stream ``residual`` (None in front of the first layer: hidden is the stream).
        ``scales``: key_scales and value_scales of 8-bit caches. Returns this layer's
        addition and the stream before it, the next layer's (hidden, residual); neither
        argument is modified."""
        (q, k, v), residual = self._project(hidden, residual)
        attended = self.attention(positions, q, k, v, key_cache, value_cache, block_tables,
                                  seq_lens, *scales)
        return self._rest(attended, residual)

    def prompt(self, positions: torch.Tensor, hidden: torch.Tensor,
               residual: torch.Tensor | None, key_cache: torch.Tensor,
               value_cache: torch.Tensor, slot_mapping: torch.Tensor,
               block_tables: torch.Tensor, query_start: torch.Tensor,
               context_lens: torch.Tensor, max_query_len: int | None = None,
               *scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Prompt chunks, as ``PagedAttentionWithQKNorm.prompt`` takes them."""
        if not isinstance(self.attention, PagedAttentionWithQKNorm):
            raise NotImplementedError("prompt chunks need a PagedAttentionWithQKNorm layer")
        (q, k, v), residual = self._project(hidden, residual)
        attended = self.attention.prompt(positions, q, k, v, key_cache, value_cache, slot_mapping,
                                         block_tables, query_start, context_lens, max_query_len,
                                         *scales)
        return self._rest(attended, residual)
