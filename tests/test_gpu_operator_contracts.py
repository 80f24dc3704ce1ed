"""Calls that the documentation of the operators allows and that only a C caller,
or an unusual one, makes, on the GPU against the 64-bit oracle."""

import pytest
import torch

from cscr import _lib
from cscr import attention as A
from cscr import cache as C
from cscr import pos_encoding as PE
from cscr._lib import DTYPE_CODE
from oracle import quant_oracle as Q
from paged_decode import metadata as M
from paged_decode import pool
from paged_decode.layers import PagedAttentionWithQKNorm
from test_gpu_scored_attention import Case

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def short(p):
    return str(p).replace("torch.", "") if isinstance(p, torch.dtype) else None


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.device_status()
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,kind", [(BF16, E4M3), (F16, INT8), (BF16, BF16), (F16, F16)],
                         ids=short)
def test_outputs_off_by_an_element_through_the_c_abi(dtype, kind):
    """An `out` aligned to its elements only, for both attention entry points."""
    c = Case([70, 1, 300], 16, 2, 128, 16, dtype, kind, seed=21)
    S, H, D = c.q.shape
    buf = torch.full((S * H * D + 2,), 7.0, dtype=dtype, device="cuda")
    out = buf[1:-1].view(S, H, D)
    scales = (c.ks.data_ptr(), c.vs.data_ptr()) if c.ks is not None else (0, 0)
    _lib.launch(_lib.SCORED_ATTENTION, 0, out.data_ptr(), c.q.data_ptr(), c.k.data_ptr(),
                c.v.data_ptr(), *scales, c.tables.data_ptr(), c.lens.data_ptr(), 0, 0, 0, S, H, 2,
                D, c.k.shape[0], 16, c.tables.shape[1], H * D, 0, DTYPE_CODE[dtype],
                DTYPE_CODE[kind], 0, c.scale, 0.0)
    c.check(out)
    if kind == dtype:
        out.zero_()
        _lib.check(_lib.load().tlb_paged_attention(
            out.data_ptr(), c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.tables.data_ptr(),
            c.lens.data_ptr(), S, H, 2, D, c.k.shape[0], 16, c.tables.shape[1], c.scale,
            DTYPE_CODE[dtype], None, 0, 0, _lib.stream_of(out.device)))
        ref = Q.attention(c.q, c.k, c.v, None, None, c.tables, c.lens, c.scale)
        Q.assert_within(out, ref[0], Q.attention_bound(*ref, dtype, kind))
    assert bool((buf[0] == 7) & (buf[-1] == 7))


@pytest.mark.parametrize("before", ["rope", "attention"])
def test_early_reads_see_what_two_launches_back_wrote(before):
    """Lengths and tables written right before a launch (an attention that itself
    overlaps its predecessor, or a rotation, which must not), then an attention
    that reads them early: steps queued without a pause equal those with a
    synchronisation after every launch."""
    g = torch.Generator(device="cuda").manual_seed(22)
    h, kvh, d, bs, n, width, blocks = 16, 2, 128, 16, 24, 40, 1200
    c = Case([500] * n, h, kvh, d, bs, BF16, BF16, seed=23)
    k, v = (torch.randn(blocks, kvh, bs, d, generator=g, device="cuda").to(BF16) for _ in "kv")
    table = torch.rand(1024, d, generator=g, device="cuda").to(BF16)
    key = torch.randn(n, kvh * d, generator=g, device="cuda").to(BF16)
    value = torch.randn(n, kvh, d, generator=g, device="cuda").to(BF16)
    pos = torch.arange(n, device="cuda")
    slots = torch.full((n,), -1, device="cuda")  # nothing is written: the caches stay
    own_lens, own_tables = c.lens, c.tables[:, :-1].clamp(max=blocks - 1).contiguous()
    plans = [(torch.randint(0, width * bs, (n,), generator=g, device="cuda").to(torch.int32),
              torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[:n * width]
              .view(n, width)) for _ in range(40)]
    long = torch.randn(8192, 8192, generator=g, device="cuda")
    torch.cuda.synchronize()

    def steps(pause):
        for _ in range(0 if pause else 8):  # the steps queue up behind these
            long @ long
        lens = torch.ones(n, dtype=torch.int32, device="cuda")
        tables = torch.zeros(n, width, dtype=torch.int32, device="cuda")
        outs = []
        for new_lens, new_tables in plans:
            tables.copy_(new_tables)
            lens.copy_(new_lens)
            if pause:
                torch.cuda.synchronize()
            if before == "rope":
                PE.rotary_embedding_neox_with_cache(pos, c.q.view(n, -1), key, value, k, v,
                                                    slots, d, table)
            else:
                A.paged_attention(c.q, k, v, own_tables, own_lens, c.scale, overlap_prologue=True)
            if pause:
                torch.cuda.synchronize()
            outs.append(A.paged_attention_biased(c.q, k, v, tables, lens, c.scale, softcap=20.0,
                                                 overlap_prologue=True))
            outs.append(A.paged_attention(c.q, k, v, tables, lens, c.scale, overlap_prologue=True))
            if pause:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs

    for a, b in zip(steps(False), steps(True), strict=True):
        assert torch.equal(a, b)
    assert _lib.device_status() == 0


def test_quantised_attention_refuses_caches_without_scales():
    """Also on a stream whose scratch is there, where cscr._fast takes the calls."""
    c = Case([40, 7], 8, 2, 64, 16, F16, F16, seed=24)
    c.run()
    args = (c.tables, c.lens, c.scale)
    fast = _lib.fast.attention(c.q, c.k, c.v, None, None, *args, 0.0, None, 0, False)
    assert fast is not None and torch.equal(fast, c.run())
    for ks, vs in ((None, None), (None, c.lens)):
        with pytest.raises(RuntimeError, match="float8_e4m3fn or int8"):
            A.paged_attention_quantized(c.q, c.k, c.v, ks, vs, *args)
    assert _lib.fast.attention(c.q, c.k, c.v, None, c.lens, *args, 0.0, None, 0, False) is None
    c = Case([40, 7], 8, 2, 64, 16, F16, INT8, seed=24)
    for ks, vs in ((None, None), (c.ks, None), (None, c.vs)):
        with pytest.raises(RuntimeError, match="float8_e8m0fnu"):
            A.paged_attention_quantized(c.q, c.k, c.v, ks, vs, *args)


class NoTruth:
    def __bool__(self):
        raise ArithmeticError("neither")


def test_flags_without_a_truth_value():
    """What a flag's __bool__ raises reaches the caller, and nothing is launched."""
    c = Case([40, 7], 8, 2, 64, 16, F16, INT8, seed=25)
    want = c.run()
    with pytest.raises(ArithmeticError, match="neither"):
        c.run(overlap_prologue=NoTruth())
    with pytest.raises(RuntimeError, match="ambiguous"):
        c.run(overlap_prologue=torch.zeros(2))
    x = c.q.view(2, -1)[:, :128].contiguous()
    w, pos = torch.ones(64, dtype=F16, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    args = (w, w, 1e-6, c.k, c.v, pos, 64, x.view(4, 64))
    before = c.k.clone()
    with pytest.raises(ArithmeticError, match="neither"):
        PE.qk_norm_rotary_embedding_neox_with_cache(pos, x, x, x, *args, key_scales=c.ks,
                                                    value_scales=c.vs, overlap_previous=NoTruth())
    assert torch.equal(c.k, before) and torch.equal(c.run(), want)


@pytest.mark.parametrize("kind", [E4M3, INT8], ids=short)
def test_prompts_over_8_bit_caches_look_up_what_16_bit_ones_do(kind):
    """Stale ids past a context are not looked up; a hole and an id outside the pool
    inside one are skipped, the latter flagged: as over caches of the query dtype
    that hold the same rows."""
    h, kvh, d, bs, blocks = 8, 2, 64, 16, 30
    g = torch.Generator(device="cuda").manual_seed(26)
    m = PagedAttentionWithQKNorm(h, d, d ** -0.5, d, max_position=1024).cuda()
    kv = pool.allocate_quantized_kv_cache(1, blocks, kvh, d, bs, kind)[0]
    rows = torch.randn(2, blocks * bs, kvh, d, generator=g, device="cuda").to(BF16)
    C.reshape_and_cache_quantized(rows[0], rows[1], *kv, torch.arange(blocks * bs, device="cuda"))
    ctx = torch.tensor([100, 64, 33], dtype=torch.int32, device="cuda")
    part = [20, 64, 33]
    start = torch.tensor([0, 20, 84, 117], dtype=torch.int32, device="cuda")
    good = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)[:24].view(3, 8)
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(part)).cuda()
    pos = torch.cat([torch.arange(n - p, n) for n, p in zip(ctx.tolist(), part)]).cuda()
    slots = good[seq, pos // bs].long() * bs + pos % bs
    q = torch.randn(117, h, d, generator=g, device="cuda").to(BF16)
    k, v = torch.randn(2, 117, kvh, d, generator=g, device="cuda").to(BF16)

    def run(tables):
        out = m.prompt(pos, q, k, v, kv[0], kv[1], slots, tables, start, ctx, 64, kv[2], kv[3])
        status = _lib.device_status()
        dense = [Q.dequantize(c, s).to(BF16) for c, s in ((kv[0], kv[2]), (kv[1], kv[3]))]
        q_rot, _ = PE.qk_norm_rotary_embedding_neox(pos, q.view(117, -1), k.view(117, -1),
                                                    m.q_norm.to(BF16), m.k_norm.to(BF16), m.eps, d,
                                                    m._table(q.device, BF16))
        want = A.paged_prefill_attention(q_rot.view(117, h, d), *dense, tables, start, ctx, m.scale,
                                         64)
        assert _lib.device_status() == status
        assert torch.isfinite(out).all() and torch.equal(out, want)
        return status

    stale = good.clone()
    for c, n in enumerate(ctx.tolist()):
        stale[c, -(-n // bs):] = torch.tensor([blocks, 0, -1, 1 << 30], dtype=torch.int32,
                                              device="cuda").repeat(2)[:8 + -n // bs]
    assert run(stale) == 0
    stale[0, 2] = blocks + 3
    stale[1, 1] = -1
    assert run(stale) == 0x1


@pytest.mark.parametrize("kind", [E4M3, INT8], ids=short)
@pytest.mark.parametrize("power", [-100, 100, 126])
def test_queries_near_the_ends_of_bf16(kind, power):
    """Queries some 2^power, keys and scale that bring the scores back."""
    c = Case([100, 33], 8, 2, 64, 16, BF16, kind, seed=28)
    c.q = (c.q.clamp(-3.9, 3.9).double() * 2.0 ** power).to(BF16)
    back = 110 if power > 0 else -100
    c.ks = (c.ks.view(torch.uint8) - back).view(torch.float8_e8m0fnu)
    c.scale *= 2.0 ** (back - power)
    assert bool(torch.isfinite(c.q).all()) and int(c.ks.view(torch.uint8)[c.tables[0, 0]].min()) > 0
    c.check(c.run())
    c.check(c.run(softcap=3.0), softcap=3.0)


@pytest.mark.parametrize("kind", [E4M3, None], ids=short)
def test_norm_reads_nothing_before_the_kernel_before_it_ends(kind):
    """overlap_previous asks nothing of the caller here: positions, slots, tables,
    weights, angles and rows written right before each of a queue of calls."""
    g = torch.Generator(device="cuda").manual_seed(29)
    h, kvh, d, bs, n, blocks = 8, 2, 128, 16, 48, 64
    long = torch.randn(8192, 8192, generator=g, device="cuda")

    def new():
        slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:n]
        return (torch.randint(0, 512, (n,), generator=g, device="cuda"), slots,
                *(torch.randn(*s, generator=g, device="cuda").to(BF16)
                  for s in ((n, h * d), (n, kvh * d), (n, kvh * d), (d,), (d,), (512, d))))

    plans = [new() for _ in range(30)]

    def steps(pause):
        caches = (pool.allocate_kv_cache(1, blocks, kvh, d, bs, BF16)[0] if kind is None
                  else pool.allocate_quantized_kv_cache(1, blocks, kvh, d, bs, kind)[0])
        for c in caches:
            c.view(torch.uint8).zero_()
        scales = dict(zip(("key_scales", "value_scales"), caches[2:]))
        now = [torch.zeros_like(x) for x in plans[0]]
        outs = []
        for _ in range(0 if pause else 8):  # the steps queue up behind these
            long @ long
        for plan in plans:
            for i, x in enumerate(now):
                # each of them is once the last one written
                j = (i + len(outs)) % len(now)
                now[j].copy_(plan[j])
            if pause:
                torch.cuda.synchronize()
            pos, slots, q, k, v, wq, wk, table = now
            outs.append(PE.qk_norm_rotary_embedding_neox_with_cache(
                pos, q, k, v, wq, wk, 1e-6, *caches[:2], slots, d, table, overlap_previous=True,
                **scales))
            if pause:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return outs + [c.view(torch.uint8) for c in caches]

    for a, b in zip(steps(False), steps(True), strict=True):
        assert torch.equal(a, b)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("kind", [E4M3, INT8, BF16], ids=short)
def test_the_short_way_takes_the_ordinary_calls(kind, monkeypatch):
    """Each cscr._fast function answers an ordinary call itself, with what the op's
    Python code answers."""
    fast, h, kvh, d, bs, n = _lib.fast, 8, 2, 64, 16, 20
    c = Case([70, 33], h, kvh, d, bs, BF16, kind, seed=30)
    c.run()  # the stream's scratch
    g = torch.Generator(device="cuda").manual_seed(31)
    q, k, v = (torch.randn(n, heads * d, generator=g, device="cuda").to(BF16)
               for heads in (h, kvh, kvh))
    w, table = (torch.randn(*s, generator=g, device="cuda").to(BF16) for s in ((d,), (64, d)))
    pos, slots = torch.arange(n, device="cuda"), torch.arange(n, device="cuda").flip(0)
    ids = torch.arange(3, dtype=torch.int32, device="cuda")
    eight = kind != BF16
    new = lambda: [None if x is None else x.clone() for x in (c.k, c.v, c.ks, c.vs)]

    def calls(direct):
        out = []
        if direct:
            out.append(fast.attention(c.q, c.k, c.v, c.ks, c.vs, c.tables, c.lens, c.scale, 0.0,
                                      None, 9, False))
        else:
            out.append(c.run(window=9))
        kv = new()
        if direct:
            out.append(fast.norm(pos, q, k, v, w, w, 1e-6, kv[0], kv[1], slots, d, table, None,
                                 kv[2], kv[3], False))
            out += fast.norm(pos, q, k, None, w, w, 1e-6, None, None, None, d, table, None, None,
                             None, False)
        else:
            out.append(PE.qk_norm_rotary_embedding_neox_with_cache(
                pos, q, k, v, w, w, 1e-6, kv[0], kv[1], slots, d, table, key_scales=kv[2],
                value_scales=kv[3]))
            out += PE.qk_norm_rotary_embedding_neox(pos, q, k, w, w, 1e-6, d, table)
        if eight:
            if direct:
                assert fast.write(v, k, *kv, pos) is True
                out += fast.read(*kv, ids, F16)
            else:
                C.reshape_and_cache_quantized(v, k, *kv, pos)
                out += C.dequantize_blocks(*kv, ids, F16)
        return out + [x.view(torch.uint8) for x in kv if x is not None]

    short_way = calls(True)
    assert all(x is not None for x in short_way)
    monkeypatch.setattr(_lib, "fast", None)
    for a, b in zip(short_way, calls(False), strict=True):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("chunks,width,bs", [(1, 1, 16), (3, 7, 5), (700, 513, 16)])
def test_read_back_tables(chunks, width, bs):
    g = torch.Generator(device="cuda").manual_seed(32)
    nb = 90
    tables = torch.randint(-3, nb + 3, (chunks, width), generator=g, device="cuda").int()
    lens = torch.randint(-2, width * bs + 9, (chunks,), generator=g, device="cuda").int()
    ids, places = M.read_back_tables(tables, lens, bs, nb)
    at = torch.arange(chunks * width, device="cuda").view(chunks, width)
    seen = at % width * bs < lens[:, None]
    assert torch.equal(ids, torch.where(seen, tables, 0))
    assert torch.equal(places, torch.where(seen & (tables >= 0) & (tables < nb), at, -1).int())
    with pytest.raises(RuntimeError, match="int32"):
        M.read_back_tables(tables.long(), lens, bs, nb)
    with pytest.raises(RuntimeError, match="one row"):
        M.read_back_tables(tables, lens.new_zeros(chunks + 1), bs, nb)
    none, holes = M.read_back_tables(tables[:0], lens[:0], bs, nb)
    assert none.shape == holes.shape == (0, width)
