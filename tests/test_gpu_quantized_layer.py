"""The quantised-cache, query/key-norm and scored-attention operators together:
the layer that runs them, prompt chunks then decode steps, captured and
replayed, and block copies of 8-bit caches."""

import pytest
import torch

from cscr import _lib
from cscr import cache as C
from cscr import pos_encoding as PE
from oracle import quant_oracle as Q
from paged_decode import pool
from paged_decode.layers import PagedAttentionWithQKNorm

pytestmark = pytest.mark.gpu

KINDS = [torch.float8_e4m3fn, torch.int8, None]
H, KVH, D, BS = 16, 2, 128, 16


def short(p):
    return str(p).replace("torch.", "") if isinstance(p, torch.dtype) else None


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.device_status()
    yield
    torch.cuda.synchronize()


def layer(dtype, **kw):
    m = PagedAttentionWithQKNorm(H, D, D ** -0.5, D, max_position=4096, **kw).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    for w in (m.q_norm, m.k_norm):
        w.data = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dtype)
    return m


def caches(kind, dtype, blocks):
    if kind is None:
        return (*pool.allocate_kv_cache(1, blocks, KVH, D, BS, dtype)[0], None, None)
    return pool.allocate_quantized_kv_cache(1, blocks, KVH, D, BS, kind)[0]


def tokens(g, n, dtype):
    qkv = torch.randn(n, (H + 2 * KVH) * D, generator=g, device="cuda").to(dtype)
    q, k, v = qkv.split([H * D, KVH * D, KVH * D], 1)
    return q.view(n, H, D), k.view(n, KVH, D), v.view(n, KVH, D)


def attention_oracle(m, q, kv, tables, lens, **kw):
    return Q.attention(q, *kv, tables, lens, m.scale, **kw)


@pytest.mark.parametrize("kind", KINDS, ids=short)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=short)
@pytest.mark.parametrize("mods", [{}, dict(softcap=8.0, window=100)], ids=["plain", "modified"])
def test_decode_steps(mods, dtype, kind):
    """Four decode steps over growing contexts: every step's rows are stored as the
    separate write stores them, and its result is the oracle's over the cache."""
    g = torch.Generator(device="cuda").manual_seed(2)
    m = layer(dtype, **mods)
    lens = torch.tensor([300, 1, 16, 33, 127], dtype=torch.int32, device="cuda")
    blocks = 64
    kv = caches(kind, dtype, blocks)
    tables = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[:60].view(5, 12)
    tables = torch.cat([tables, tables[:, :0]], 1)
    lens.clamp_(max=12 * BS - 4)
    _, k0, v0 = tokens(g, blocks * BS, dtype)
    every = torch.arange(blocks * BS, device="cuda")
    if kind is None:
        C.reshape_and_cache(k0.contiguous(), v0.contiguous(), kv[0], kv[1], every)
    else:
        C.reshape_and_cache_quantized(k0, v0, *kv, every)
    for step in range(4):
        lens += 1
        q, k, v = tokens(g, 5, dtype)
        pos = lens.long() - 1
        before = [None if c is None else c.clone() for c in kv]
        out = m(None if step % 2 else pos, q, k, v, kv[0], kv[1], tables, lens, kv[2], kv[3])
        q_ref, k_ref = PE.qk_norm_rotary_embedding_neox(
            pos, q.reshape(5, -1), k.reshape(5, -1), m.q_norm, m.k_norm, m.eps, D,
            m._table(q.device, dtype))
        slots = tables[torch.arange(5, device="cuda"), pos // BS].long() * BS + pos % BS
        if kind is None:
            C.reshape_and_cache(k_ref.view(5, KVH, D), v.contiguous(), before[0], before[1], slots)
        else:
            C.reshape_and_cache_quantized(k_ref.view(5, KVH, D), v, *before, slots)
        for a, b in zip(kv, before):
            assert a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        ref = attention_oracle(m, q_ref.view(5, H, D), kv, tables, lens, **mods)
        plain16 = kind is None and not mods
        if plain16 and dtype == torch.bfloat16:
            continue  # paged_attention's own tests cover its bf16 bound
        Q.assert_within(out, ref[0], Q.attention_bound(*ref, dtype, kv[0].dtype, plain=plain16))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("kind", KINDS[:2], ids=short)
def test_prompt_chunks_then_decode(kind):
    """Two prompts in two chunks each over an 8-bit cache equal the prefill kernel
    on 16-bit caches that hold what the 8-bit rows stand for; a decode step follows."""
    from cscr import attention as A

    dtype = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    m = layer(dtype)
    kv = caches(kind, dtype, 40)
    for c in kv:
        c.view(torch.uint8).fill_(0x7F)  # unwritten rows hold NaN (e4m3)
    tables = torch.full((2, 12), -1, dtype=torch.int32, device="cuda")
    tables[:, :11] = torch.randperm(40, generator=g, device="cuda")[:22].view(2, 11)
    total = [150, 97]
    done = [0, 0]
    for part in ([100, 40], [50, 57]):
        n = sum(part)
        q, k, v = tokens(g, n, dtype)
        pos = torch.cat([torch.arange(d, d + x) for d, x in zip(done, part)]).cuda()
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(part)).cuda()
        slots = tables[seq, pos // BS].long() * BS + pos % BS
        done = [d + x for d, x in zip(done, part)]
        start = torch.tensor([0, part[0], n], dtype=torch.int32, device="cuda")
        ctx = torch.tensor(done, dtype=torch.int32, device="cuda")
        out = m.prompt(pos, q, k, v, kv[0], kv[1], slots, tables, start, ctx, max(part), kv[2],
                       kv[3])
        q_ref, _ = PE.qk_norm_rotary_embedding_neox(
            pos, q.reshape(n, -1), k.reshape(n, -1), m.q_norm, m.k_norm, m.eps, D,
            m._table(q.device, dtype))
        dense = [Q.dequantize(c, s).to(dtype) for c, s in ((kv[0], kv[2]), (kv[1], kv[3]))]
        want = A.paged_prefill_attention(q_ref.view(n, H, D), *dense, tables, start, ctx, m.scale,
                                         max(part))
        assert torch.isfinite(out).all()
        assert torch.equal(out, want)
    q, k, v = tokens(g, 2, dtype)
    lens = torch.tensor([t + 1 for t in total], dtype=torch.int32, device="cuda")
    out = m(None, q, k, v, kv[0], kv[1], tables, lens, kv[2], kv[3])
    q_ref, _ = PE.qk_norm_rotary_embedding_neox(
        lens.long() - 1, q.reshape(2, -1), k.reshape(2, -1), m.q_norm, m.k_norm, m.eps, D,
        m._table(q.device, dtype))
    ref = attention_oracle(m, q_ref.view(2, H, D), kv, tables, lens)
    Q.assert_within(out, ref[0], Q.attention_bound(*ref, dtype, kind))
    with pytest.raises(NotImplementedError, match="plain scores"):
        layer(dtype, softcap=5.0).prompt(pos, q, k, v, kv[0], kv[1], slots, tables, start, ctx)


@pytest.mark.parametrize("kind", [k for k in KINDS if k is not None], ids=short)
def test_lengths_and_tables_written_just_before_a_step(kind):
    """The attention of a step reads lengths and tables while the norm kernel before
    it runs; kernels that write them ahead of that one are complete by then. Steps
    queued without a pause, each after in-place changes of both, equal those with a
    synchronisation after every launch."""
    g = torch.Generator(device="cuda").manual_seed(9)
    m = layer(torch.bfloat16)
    n, width, blocks = 5, 12, 64
    kv = caches(kind, torch.bfloat16, blocks)
    _, k0, v0 = tokens(g, blocks * BS, torch.bfloat16)
    C.reshape_and_cache_quantized(k0, v0, *kv, torch.arange(blocks * BS, device="cuda"))
    plans = [(torch.randint(1, width * BS, (n,), generator=g, device="cuda").to(torch.int32),
              torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[:n * width]
              .view(n, width), tokens(g, n, torch.bfloat16)) for _ in range(40)]
    torch.cuda.synchronize()

    def steps(pause):
        cache = [c.clone() for c in kv]
        lens = torch.ones(n, dtype=torch.int32, device="cuda")
        tables = torch.zeros(n, width, dtype=torch.int32, device="cuda")
        pos = torch.zeros(n, dtype=torch.int64, device="cuda")
        outs = []
        for new_lens, new_tables, (q, k, v) in plans:
            pos.copy_(new_lens - 1)
            tables.copy_(new_tables)
            lens.copy_(new_lens)
            if pause:
                torch.cuda.synchronize()
            outs.append(m(pos, q, k, v, cache[0], cache[1], tables, lens, cache[2], cache[3]))
            if pause:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs

    for a, b in zip(steps(False), steps(True)):
        assert torch.equal(a, b)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("kind", KINDS, ids=short)
def test_a_captured_step_replays(kind):
    """A decode step in a graph, replayed over growing contexts, equals the eager
    step on its own caches."""
    dtype = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(4)
    m = layer(dtype, softcap=30.0)
    two = [caches(kind, dtype, 64) for _ in range(2)]
    _, k0, v0 = tokens(g, 64 * BS, dtype)
    every = torch.arange(64 * BS, device="cuda")
    for kv in two:
        if kind is None:
            C.reshape_and_cache(k0.contiguous(), v0.contiguous(), kv[0], kv[1], every)
        else:
            C.reshape_and_cache_quantized(k0, v0, *kv, every)
    tables = torch.randperm(64, generator=g, device="cuda").to(torch.int32).view(2, 32)
    lens = torch.tensor([400, 7], dtype=torch.int32, device="cuda")
    q, k, v = tokens(g, 2, dtype)
    a, b = two
    saved = [None if c is None else c.clone() for c in a]
    m(None, q, k, v, a[0], a[1], tables, lens, a[2], a[3])
    for c, s in zip(a, saved):
        if c is not None:
            c.view(torch.uint8).copy_(s.view(torch.uint8))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(None, q, k, v, a[0], a[1], tables, lens, a[2], a[3])
    for step in range(3):
        nq, nk, nv = tokens(g, 2, dtype)
        for dst, src in ((q, nq), (k, nk), (v, nv)):
            dst.copy_(src)
        lens.add_(1)
        graph.replay()
        want = m(None, nq, nk, nv, b[0], b[1], tables, lens, b[2], b[3])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for x, y in zip(a, b):
            assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_block_copies_of_quantised_caches():
    g = torch.Generator(device="cuda").manual_seed(5)
    layers = pool.allocate_quantized_kv_cache(3, 20, KVH, D, BS, torch.int8)
    _, k0, v0 = tokens(g, 20 * BS, torch.bfloat16)
    for kv in layers:
        C.reshape_and_cache_quantized(k0, v0, *kv, torch.arange(20 * BS, device="cuda"))
    C.copy_blocks([c for kv in layers for c in (kv[0], kv[2])],
                  [c for kv in layers for c in (kv[1], kv[3])], {3: [7, 9], 0: [19]})
    ids = torch.tensor([3, 7, 9, 0, 19], device="cuda")
    for kv in layers:
        for x in C.dequantize_blocks(*kv, ids, torch.float32):
            assert torch.equal(x[1], x[0]) and torch.equal(x[2], x[0]) and torch.equal(x[4], x[3])


def test_pool_sizes():
    kv = pool.allocate_quantized_kv_cache(2, 5, KVH, D, BS)
    one = sum(c.numel() for layer_ in kv for c in layer_) // 5
    assert one == pool.quantized_block_bytes(2, KVH, D, BS)
    with pytest.raises(ValueError, match="8-bit caches"):
        pool.allocate_quantized_kv_cache(1, 5, KVH, D, BS, torch.float16)
    with pytest.raises(ValueError, match="No KV cache blocks"):
        pool.allocate_quantized_kv_cache(1, 0, KVH, D, BS)


def test_calls_without_the_fast_module_are_the_same(monkeypatch):
    """Every op with its Python argument handling alone, and through cscr._fast."""
    from cscr import attention as A

    g = torch.Generator(device="cuda").manual_seed(6)
    dtype = torch.bfloat16
    m = layer(dtype)
    q, k, v = tokens(g, 40, dtype)
    pos = torch.arange(40, device="cuda")
    tables = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens = torch.tensor([40, 23], dtype=torch.int32, device="cuda")
    slots = torch.randperm(128, generator=g, device="cuda")[:40]
    table = m._table(q.device, dtype)

    def everything():
        out = []
        for kind in KINDS:
            kv = caches(kind, dtype, 8)
            for c in kv:
                if c is not None:
                    c.view(torch.uint8).fill_(0)
            out.append(PE.qk_norm_rotary_embedding_neox_with_cache(
                pos, q.view(40, -1), k.view(40, -1), v, m.q_norm, m.k_norm, 1e-6, kv[0], kv[1],
                slots, D, table, key_scales=kv[2], value_scales=kv[3]))
            if kind is not None:
                C.reshape_and_cache_quantized(v, k, *kv, slots.flip(0))
                out += C.dequantize_blocks(*kv, tables.view(-1), torch.float16)
                out.append(A.paged_attention_quantized(q[:2], *kv, tables, lens, 0.1, window=9))
            else:
                out.append(A.paged_attention_biased(q[:2], kv[0], kv[1], tables, lens, 0.1,
                                                    softcap=4.0))
            out += [c.view(torch.uint8) for c in kv if c is not None]
        out += PE.qk_norm_rotary_embedding_neox(pos, q.view(40, -1), k.view(40, -1), m.q_norm,
                                                m.k_norm, 1e-6, D, table)
        return out

    assert _lib.fast is not None
    everything()  # scratch of the stream
    quick = everything()
    monkeypatch.setattr(_lib, "fast", None)
    for a, b in zip(quick, everything(), strict=True):
        assert torch.equal(a, b)
