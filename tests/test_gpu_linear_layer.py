"""The 8-bit projection operators together and with the attention ops: the layers that
run them, prompt chunks then decode steps, captured and replayed, on several streams,
and with waits that give up."""

import threading

import pytest
import torch

from cscr import _lib
from cscr import linear as L
from oracle import linear_oracle as O
from paged_decode import pool
from paged_decode.layers import (PagedAttentionWithQKNorm, PagedAttentionWithRoPE,
                                 QuantizedDecoderLayer, QuantizedLinear)

pytestmark = pytest.mark.gpu

H, KVH, D, BS, WIDTH, INNER = 4, 2, 64, 16, 256, 640


def short(p):
    return str(p).replace("torch.", "") if isinstance(p, torch.dtype) else None


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    _lib.device_status()
    yield
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    torch.cuda.synchronize()


def layer(dtype, rope=False, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def weight(n, k):
        return (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).to(dtype)

    def vector(n):
        return (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(dtype)

    kind = PagedAttentionWithRoPE if rope else PagedAttentionWithQKNorm
    attention = kind(H, D, D ** -0.5, D, max_position=512).cuda()
    if not rope:
        attention.q_norm.data, attention.k_norm.data = vector(D), vector(D)
    return QuantizedDecoderLayer(
        attention, KVH, QuantizedLinear.from_weight(weight((H + 2 * KVH) * D, WIDTH),
                                                    vector((H + 2 * KVH) * D)),
        QuantizedLinear.from_weight(weight(WIDTH, H * D)),
        QuantizedLinear.from_weight(weight(2 * INNER, WIDTH)),
        QuantizedLinear.from_weight(weight(WIDTH, INNER)), vector(WIDTH), vector(WIDTH))


def caches(kind, dtype, blocks):
    if kind is None:
        kv = pool.allocate_kv_cache(1, blocks, KVH, D, BS, dtype)[0]
    else:
        kv = pool.allocate_quantized_kv_cache(1, blocks, KVH, D, BS, kind)[0]
    for c in kv:
        c.view(torch.uint8).zero_()
    return kv


def by_hand(m, hidden, residual, attend):
    """The layer's steps one by one, each 8-bit operator's result checked against its
    definition on the operands it got; the layer has to give the same bits."""
    def norm(x, w, res):
        q, s, h = L.rms_norm_quantized(x, w, m.eps, res)
        want, want_h = O.norm(x, w, m.eps, res)
        O.assert_rows_of(q, s, want, 2.0 ** -18)
        assert h is None or torch.equal(h, want_h)
        return q, s, x if h is None else h

    def product(lin, q, s):
        ops = (q, s, lin.weight_bytes.view(torch.float8_e4m3fn),
               lin.scale_bytes.view(torch.float8_e8m0fnu))
        got = L.matmul_quantized(*ops, lin.dtype, lin.bias)
        y, mag = O.product(*ops, lin.bias)
        bound = O.product_bound(y, mag, q.shape[1], lin.dtype)
        assert bool(((got.double() - y).abs() <= bound).all())
        return got

    q, s, residual = norm(hidden, m.input_norm, residual)
    qkv = product(m.qkv, q, s)
    parts = qkv.split([H * D, KVH * D, KVH * D], 1)
    a = attend(*(x.reshape(-1, x.shape[1] // D, D) for x in parts))
    hidden = product(m.out, *L.quantize_rows(a.reshape(-1, H * D)))
    q, s, residual = norm(hidden, m.post_norm, residual)
    gate_up = product(m.gate_up, q, s)
    q, s = L.silu_and_mul_quantized(gate_up)
    delta = (6 + 1.2 * gate_up[:, :INNER].double().abs()) * 2.0 ** -23
    O.assert_rows_of(q, s, O.silu_mul(gate_up), delta)
    return product(m.down, q, s), residual


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, None], ids=short)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=short)
def test_prompt_then_decode_steps(dtype, kind):
    g = torch.Generator(device="cuda").manual_seed(2)
    m = layer(dtype)
    kv, mine = caches(kind, dtype, 24), caches(kind, dtype, 24)
    tables = torch.randperm(24, generator=g, device="cuda").to(torch.int32).view(3, 8)
    lens = [70, 1, 33]
    starts = torch.tensor([0, 70, 71, 104], dtype=torch.int32, device="cuda")
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    row = torch.repeat_interleave(torch.arange(3), torch.tensor(lens)).cuda()
    slots = tables[row, pos // BS].long() * BS + pos % BS
    hidden = torch.randn(104, WIDTH, generator=g, device="cuda").to(dtype)
    kept = hidden.clone()
    got = m.prompt(pos, hidden, None, kv[0], kv[1], slots, tables, starts, ctx, 70, *kv[2:])
    want = by_hand(m, hidden, None, lambda q, k, v: m.attention.prompt(
        pos, q, k, v, mine[0], mine[1], slots, tables, starts, ctx, 70, *mine[2:]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(hidden, kept)
    for step in range(3):
        ctx += 1
        h = torch.randn(3, WIDTH, generator=g, device="cuda").to(dtype)
        r = torch.randn(3, WIDTH, generator=g, device="cuda").to(dtype)
        kept = r.clone()
        got = m(None, h, r, kv[0], kv[1], tables, ctx, *kv[2:])
        want = by_hand(m, h, r, lambda q, k, v: m.attention(
            None, q, k, v, mine[0], mine[1], tables, ctx, *mine[2:]))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(r, kept)
        for a, b in zip(kv, mine):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert _lib.device_status() == 0


def test_rotated_attention_and_module_conversions():
    """Around PagedAttentionWithRoPE (16-bit caches); .to(dtype) and state_dict leave
    the 8-bit weights as they are."""
    dtype = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    m = layer(dtype, rope=True)
    kv = caches(None, dtype, 8)
    tables = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    ctx = torch.tensor([1, 5, 17, 30], dtype=torch.int32, device="cuda")
    h = torch.randn(4, WIDTH, generator=g, device="cuda").to(dtype)
    want = m(None, h, None, *(c.clone() for c in kv), tables, ctx)
    mine = [c.clone() for c in kv]
    ref = by_hand(m, h, None, lambda q, k, v: m.attention(None, q, k, v, *mine, tables, ctx))
    assert torch.equal(want[0], ref[0]) and torch.equal(want[1], ref[1])
    again = layer(dtype, rope=True, seed=9).to(dtype)
    again.load_state_dict(m.state_dict())
    assert again.qkv.weight_bytes.dtype == torch.uint8
    got = again(None, h, None, *(c.clone() for c in kv), tables, ctx)
    assert torch.equal(got[0], want[0])
    half = again.to(torch.float16)
    assert half.qkv.dtype == torch.float16 and half.qkv.weight_bytes.dtype == torch.uint8
    got = half(None, h.half(), None, *(c.half() for c in kv), tables, ctx)
    assert got[0].dtype == torch.float16
    with pytest.raises(NotImplementedError, match="PagedAttentionWithQKNorm"):
        m.prompt(None, h, None, *kv, None, tables, None, ctx)


def test_steps_without_tokens():
    m = layer(torch.bfloat16)
    kv = caches(torch.float8_e4m3fn, torch.bfloat16, 2)
    none = torch.empty(0, WIDTH, dtype=torch.bfloat16, device="cuda")
    i32 = torch.zeros(0, dtype=torch.int32, device="cuda")
    out, residual = m.prompt(i32.long(), none, none, kv[0], kv[1], i32.long(), i32.view(0, 1),
                             torch.zeros(1, dtype=torch.int32, device="cuda"), i32, 0, *kv[2:])
    assert out.shape == none.shape and residual.shape == none.shape


def test_captured_steps_replayed_together():
    """Two captured decode steps of a layer over caches of their own, replayed on two
    streams at once with new inputs, equal the eager steps."""
    dtype = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(4)
    m = layer(dtype)
    tables = torch.arange(16, dtype=torch.int32, device="cuda").view(4, 4)
    ctx = torch.tensor([3, 20, 33, 60], dtype=torch.int32, device="cuda")
    graphs = []
    for i in range(2):
        kv = caches(torch.float8_e4m3fn, dtype, 16)
        h = torch.zeros(4, WIDTH, dtype=dtype, device="cuda")
        r = torch.zeros_like(h)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            m(None, h, r, kv[0], kv[1], tables, ctx, *kv[2:])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = m(None, h, r, kv[0], kv[1], tables, ctx, *kv[2:])
        graphs.append((graph, s, h, r, kv, out))
    for trial in range(3):
        want = []
        for graph, s, h, r, kv, out in graphs:
            h.copy_(torch.randn(4, WIDTH, generator=g, device="cuda"))
            r.copy_(torch.randn(4, WIDTH, generator=g, device="cuda"))
            copy = [c.clone() for c in kv]
            want.append(m(None, h, r, copy[0], copy[1], tables, ctx, *copy[2:]))
        torch.cuda.synchronize()
        for graph, s, *_ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, _, out), ref in zip(graphs, want):
            assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])
    assert _lib.device_status() == 0


def operands(g, t, k, n):
    x = L.quantize_rows(torch.randn(t, k, generator=g, device="cuda"))
    w = L.quantize_weight(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    return (*x, *w)


# a tile by one CTA; by clusters of 4 and of 2; several tiles a cluster, a CTA, a pair of
# CTAs; any alignment
WAITS = [(64, 512, 640), (64, 8192, 256), (900, 16384, 1000), (9, 8192, 20000), (1377, 64, 5528),
         (1918, 5456, 5652), (20, 100, 30)]


def test_streams_and_threads_at_once():
    """Products and rows from two threads on streams of their own, as on one."""
    g = torch.Generator(device="cuda").manual_seed(5)
    ops = [operands(g, t, k, n) for t, k, n in (*WAITS[:2], *WAITS[4:])]
    x = torch.randn(500, 1024, generator=g, device="cuda").to(torch.bfloat16)
    want = [L.matmul_quantized(*o, torch.bfloat16) for o in ops]
    rows = L.quantize_rows(x)
    torch.cuda.synchronize()
    bad = []

    def run():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = [L.matmul_quantized(*o, torch.bfloat16) for o in ops]
                q, s = L.quantize_rows(x)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)) or not torch.equal(
                        q.view(torch.uint8), rows[0].view(torch.uint8)):
                    bad.append(1)

    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and _lib.device_status() == 0


@pytest.mark.parametrize("t,k,n", WAITS)
def test_results_do_not_vary(t, k, n):
    """The same bits from every call, and for a token alone as among others."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x, xs, w, ws = operands(g, t, k, n)
    first = L.matmul_quantized(x, xs, w, ws, torch.float32)
    for _ in range(3):
        assert torch.equal(L.matmul_quantized(x, xs, w, ws, torch.float32), first)
    y, mag = O.product(x, xs, w, ws)
    bound = O.product_bound(y, mag, k, torch.float32)
    assert bool(((first.double() - y).abs() <= bound).all())


@pytest.mark.parametrize("limit", [0, 1, 4, 32, 512])
@pytest.mark.parametrize("t,k,n", WAITS)
def test_waits_that_give_up(t, k, n, limit):
    """Every input is valid and every wait ends, some before their time: the call
    returns, says so in the status word, and the next one is exact again."""
    g = torch.Generator(device="cuda").manual_seed(7)
    ops = operands(g, t, k, n)
    for dtype in (torch.bfloat16, torch.float32):
        want = L.matmul_quantized(*ops, dtype)
        torch.cuda.synchronize()
        _lib.set_wait_limit(limit)
        L.matmul_quantized(*ops, dtype)
        L.matmul_quantized(*ops, dtype)
        torch.cuda.synchronize()
        _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
        status = _lib.device_status()
        assert status & ~_lib.STATUS_WAIT_TIMEOUT == 0
        if limit == 0 and k % 16 == 0:
            assert status & _lib.STATUS_WAIT_TIMEOUT
        assert torch.equal(L.matmul_quantized(*ops, dtype), want)
        assert _lib.device_status() == 0
