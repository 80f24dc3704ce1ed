"""8-bit cache rows on the GPU: the quantising write, reading blocks back and
the query/key norm with rotation and cache write, against the 64-bit oracle."""

import pytest
import torch

from cscr import _lib
from cscr import cache as C
from cscr import pos_encoding as PE
from oracle import quant_oracle as Q

pytestmark = pytest.mark.gpu

KINDS = [torch.float8_e4m3fn, torch.int8]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def short(p):
    return str(p).replace("torch.", "") if isinstance(p, torch.dtype) else None


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.device_status()
    yield
    torch.cuda.synchronize()


def pool(nb, kvh, bs, d, kind, fill=0x5A):
    """Caches and scales of known bytes: (k, v, k scales, v scales)."""
    def one(*shape, dtype):
        return torch.full(shape, fill, dtype=torch.uint8, device="cuda").view(dtype)
    if kind in Q.QMAX:
        return (one(nb, kvh, bs, d, dtype=kind), one(nb, kvh, bs, d, dtype=kind),
                one(nb, kvh, bs, dtype=torch.float8_e8m0fnu),
                one(nb, kvh, bs, dtype=torch.float8_e8m0fnu))
    return (torch.full((nb, kvh, bs, d), 7, dtype=kind, device="cuda"),
            torch.full((nb, kvh, bs, d), 7, dtype=kind, device="cuda"), None, None)


def rows(g, t, kvh, d, dtype):
    x = torch.randn(t, kvh, d, generator=g) * torch.exp(3 * torch.randn(t, kvh, 1, generator=g))
    x = x.clamp(-30000, 30000).to(dtype)
    if t > 2:
        x[1] = 0
        x[2, :, 0] = 448.0  # a maximum on the border of its scale
    return x


def same_bytes(a, b):
    if a.element_size() != 1:
        return torch.equal(a, b)
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def expected_write(before, key, value, slots, kind):
    """The caches after the write, on the host, from the oracle."""
    k, v, ks, vs = (x.cpu().clone() for x in before)
    bs = k.shape[2]
    for x, cache, scales in ((key, k, ks), (value, v, vs)):
        q, s = Q.quantize(x.cpu(), kind)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < k.shape[0] * bs:
                cache.view(torch.uint8)[slot // bs, :, slot % bs] = q.view(torch.uint8)[t]
                scales.view(torch.uint8)[slot // bs, :, slot % bs] = s.view(torch.uint8)[t]
    return k, v, ks, vs


@pytest.mark.parametrize("kind", KINDS, ids=short)
@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("tokens,kvh,d,bs", [(1, 2, 128, 16), (65, 2, 64, 8), (33, 5, 80, 16),
                                             (7, 1, 256, 32), (9, 3, 40, 5), (5, 2, 37, 16),
                                             (3, 1, 264, 16), (11, 2, 8, 16), (2, 1, 1, 1)])
def test_write_is_exact(tokens, kvh, d, bs, dtype, kind):
    g = torch.Generator().manual_seed(tokens * 131 + d)
    nb = -(-tokens // bs) + 3
    slots = torch.randperm(nb * bs, generator=g)[:tokens]
    if tokens > 4:
        slots[3] = -1
    key, value = rows(g, tokens, kvh, d, dtype), rows(g, tokens, kvh, d, dtype)
    caches = pool(nb, kvh, bs, d, kind)
    want = expected_write(caches, key, value, slots, kind)
    C.reshape_and_cache_quantized(key.cuda(), value.cuda(), *caches, slots.cuda())
    for got, ref in zip(caches, want):
        assert same_bytes(got.cpu(), ref)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("kind", KINDS, ids=short)
def test_write_of_strided_rows_odd_alignment_and_int32_slots(kind):
    """Keys and values as parts of one projection; a part that starts off a
    16-byte boundary; a broadcast value; slots past the cache are flagged."""
    g = torch.Generator().manual_seed(0)
    t, kvh, d, bs, nb = 19, 2, 128, 16, 4
    for off in (0, 1):
        qkv = (torch.randn(t, 3 * kvh * d + 8, generator=g)).to(torch.bfloat16)
        key = qkv[:, off:off + kvh * d]
        value = qkv[:1, kvh * d:2 * kvh * d].expand(t, -1)
        dev = qkv.cuda()
        slots = torch.randperm(nb * bs, generator=g)[:t].to(torch.int32)
        slots[4] = nb * bs  # outside
        caches = pool(nb, kvh, bs, d, kind)
        want = expected_write(caches, key.reshape(t, kvh, d), value.reshape(t, kvh, d), slots, kind)
        C.reshape_and_cache_quantized(dev[:, off:off + kvh * d],
                                      dev[:1, kvh * d:2 * kvh * d].expand(t, -1), *caches,
                                      slots.cuda())
        for got, ref in zip(caches, want):
            assert same_bytes(got.cpu(), ref)
        assert _lib.device_status() == 0x8


@pytest.mark.parametrize("kind", KINDS, ids=short)
@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("d", [128, 37])
def test_write_of_extreme_rows(d, dtype, kind):
    """Infinities, NaN, the type's largest and smallest values, subnormals."""
    info = torch.finfo(dtype)
    x = torch.zeros(8, 1, d)
    x[0, 0, :4] = torch.tensor([1.0, float("inf"), -float("inf"), float("nan")])
    x[1] = float("nan")
    x[2] = float("inf")
    x[3] = info.max
    x[4] = info.smallest_normal
    x[5, 0, ::2] = info.smallest_normal * info.eps * 5  # a subnormal
    x[6, 0, 0], x[6, 0, 1] = info.max, info.smallest_normal * info.eps
    x[7, 0, -1] = -info.smallest_normal * info.eps
    x = x.to(dtype)
    slots = torch.arange(8)
    caches = pool(1, 1, 8, d, kind)
    want = expected_write(caches, x, x, slots, kind)
    C.reshape_and_cache_quantized(x.cuda(), x.cuda(), *caches, slots.cuda())
    for got, ref in zip(caches, want):
        if got.dtype == torch.float8_e4m3fn:  # any NaN for a NaN, any zero for a zero
            a, b = got.cpu().float(), ref.float()
            assert torch.equal(a.isnan(), b.isnan())
            assert torch.equal(a.nan_to_num(), b.nan_to_num())
        else:
            assert same_bytes(got.cpu(), ref)


@pytest.mark.parametrize("kind", KINDS, ids=short)
@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("kvh,bs,d", [(2, 16, 128), (1, 8, 64), (3, 5, 80), (2, 16, 37)])
def test_read_back_is_exact(kvh, bs, d, dtype, kind):
    g = torch.Generator().manual_seed(d)
    nb = 9
    caches = pool(nb, kvh, bs, d, kind)
    slots = torch.arange(nb * bs, device="cuda")
    C.reshape_and_cache_quantized(rows(g, nb * bs, kvh, d, torch.float32).cuda(),
                                  rows(g, nb * bs, kvh, d, torch.float32).cuda(), *caches, slots)
    for ids in (torch.tensor([4, -1, 0, 8, 4, 9, 2], dtype=torch.int64),
                torch.tensor([7], dtype=torch.int32)):
        got = C.dequantize_blocks(*caches, ids.cuda(), dtype)
        for out, cache, scales in ((got[0], *caches[::2]), (got[1], caches[1], caches[3])):
            every = Q.dequantize(cache.cpu(), scales.cpu())
            want = torch.zeros(len(ids), kvh, bs, d, dtype=torch.float64)
            for n, b in enumerate(ids.tolist()):
                if 0 <= b < nb:
                    want[n] = every[b]
            assert torch.equal(out.cpu(), want.to(dtype))  # one rounding of an exact value
        assert _lib.device_status() == (0x1 if 9 in ids else 0)


def test_read_back_fills_the_given_tensors_and_nothing_else():
    caches = pool(3, 2, 16, 128, torch.int8)
    big = torch.full((6, 2, 16, 128), 3.0, dtype=torch.float16, device="cuda")
    out = (big[1:3], big[4:6])
    ids = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    got = C.dequantize_blocks(*caches, ids, torch.float16, out=out)
    assert got[0].data_ptr() == out[0].data_ptr()
    want = Q.dequantize(caches[0], caches[2])[ids.long()].to(torch.float16)
    assert torch.equal(out[0], want) and torch.equal(out[1], want)
    assert bool((big[0] == 3).all()) and bool((big[3] == 3).all())
    with pytest.raises(RuntimeError, match="out must be"):
        C.dequantize_blocks(*caches, ids, torch.float16, out=(big[:1], big[:2]))


def test_empty_calls():
    caches = pool(2, 2, 16, 64, torch.int8)
    before = [c.clone() for c in caches]
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    x = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    C.reshape_and_cache_quantized(x, x, *caches, none)
    k, v = C.dequantize_blocks(*caches, none, torch.float16)
    assert k.shape == (0, 2, 16, 64) and v.shape == k.shape
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    table = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(0, 128, dtype=torch.float16, device="cuda")
    a, b = PE.qk_norm_rotary_embedding_neox(none, q, q, w, w, 1e-6, 64, table)
    assert a.shape == (0, 128) and b.shape == (0, 128)
    for c, o in zip(caches, before):
        assert same_bytes(c, o)


def norm_inputs(t, h, kvh, d, rot, dtype, seed=0, max_pos=97):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(t, (h + 2 * kvh) * d, generator=g, device="cuda")
    qkv = (qkv * torch.exp(2 * torch.randn(t, 1, generator=g, device="cuda"))).to(dtype)
    q, k, v = qkv.split([h * d, kvh * d, kvh * d], 1)
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dtype) for _ in range(2))
    pos = torch.randint(0, max_pos, (t,), generator=g, device="cuda")
    ang = torch.arange(max_pos, device="cuda").double()[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, device="cuda").double() / rot)
    return q, k, v, wq, wk, pos, torch.cat((ang.cos(), ang.sin()), -1).to(dtype)


def check_normed(got, x, w, eps, pos, table, d, what):
    want, mag = Q.norm_rope(x, w, eps, pos, table, d)
    # fp32: a sum of d squares in at most log2(d) + 16 rounded steps, a root, three
    # products and one sum: under 2^-18 of the pair's magnitudes for d <= 1024
    unit = torch.finfo(got.dtype).eps / 2
    bound = want.abs() * unit * (1 + 2 ** -7) + mag * 2.0 ** -18 + torch.finfo(
        got.dtype).smallest_normal * unit * 4
    Q.assert_within(got.view(want.shape), want, bound, what)


NORM_SHAPES = [(1, 16, 2, 128, 128), (64, 14, 2, 64, 64), (37, 8, 8, 128, 64), (13, 3, 1, 80, 80),
               (5, 2, 1, 256, 256), (9, 4, 2, 40, 20), (3, 2, 2, 37, 36), (4, 1, 1, 512, 512),
               (2, 1, 1, 528, 16), (6, 5, 1, 16, 16), (700, 4, 4, 64, 32)]


@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("t,h,kvh,d,rot", NORM_SHAPES)
def test_norm_rope(t, h, kvh, d, rot, dtype):
    q, k, v, wq, wk, pos, table = norm_inputs(t, h, kvh, d, rot, dtype)
    before = q.clone(), k.clone()
    for p in (pos, pos.to(torch.int32)):
        qo, ko = PE.qk_norm_rotary_embedding_neox(p, q, k, wq, wk, 1e-5, d, table)
        check_normed(qo, q, wq, 1e-5, pos, table, d, "query")
        check_normed(ko, k, wk, 1e-5, pos, table, d, "key")
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("cache", KINDS + [None], ids=short)
@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("t,h,kvh,d,rot", NORM_SHAPES)
def test_norm_rope_with_cache_equals_its_parts(t, h, kvh, d, rot, dtype, cache):
    """The fused write stores exactly what the separate calls store, by slots and
    by block tables."""
    kind, bs = cache or dtype, 16
    q, k, v, wq, wk, pos, table = norm_inputs(t, h, kvh, d, rot, dtype, seed=1)
    q_ref, k_ref = PE.qk_norm_rotary_embedding_neox(pos, q, k, wq, wk, 1e-6, d, table)
    maxb = 97 // bs + 1
    nb = t * maxb  # every token has a table row of its own
    tables = torch.randperm(nb, device="cuda").to(torch.int32).view(t, maxb)
    if t > 3:
        tables[2] = -1
    blk = tables[torch.arange(t, device="cuda"), pos // bs].long()
    slots = torch.where(blk >= 0, blk * bs + pos % bs, -1)
    want = pool(nb, kvh, bs, d, kind)
    k3, v3 = k_ref.view(t, kvh, d), v.reshape(t, kvh, d)
    if cache:
        C.reshape_and_cache_quantized(k3, v3, *want, slots)
    else:
        C.reshape_and_cache(k3, v3, want[0], want[1], slots)
    for by_table in (False, True):
        got = pool(nb, kvh, bs, d, kind)
        q_out = PE.qk_norm_rotary_embedding_neox_with_cache(
            pos, q, k, v, wq, wk, 1e-6, got[0], got[1], None if by_table else slots, d, table,
            block_tables=tables if by_table else None, key_scales=got[2], value_scales=got[3])
        assert torch.equal(q_out, q_ref)
        for a, b in zip(got, want):
            assert a is None or same_bytes(a, b)
    assert _lib.device_status() == 0


def test_norm_rope_outside_its_tables():
    """Positions outside the table leave rows normed and unrotated and are flagged;
    so are slots and table columns outside the cache, whose rows are skipped."""
    t, h, kvh, d = 6, 2, 1, 64
    q, k, v, wq, wk, pos, table = norm_inputs(t, h, kvh, d, d, torch.bfloat16)
    pos[1], pos[2] = -1, 97
    qo, ko = PE.qk_norm_rotary_embedding_neox(pos, q, k, wq, wk, 1e-6, d, table)
    check_normed(qo, q, wq, 1e-6, pos, table, d, "query")
    check_normed(ko, k, wk, 1e-6, pos, table, d, "key")
    assert _lib.device_status() == 0x4
    got = pool(2, kvh, 16, d, torch.int8)
    fresh = [c.clone() for c in got]
    PE.qk_norm_rotary_embedding_neox_with_cache(
        pos.clamp(0, 96), q, k, v, wq, wk, 1e-6, got[0], got[1],
        torch.full((t,), 32, device="cuda"), d, table, key_scales=got[2], value_scales=got[3])
    assert _lib.device_status() == 0x8
    PE.qk_norm_rotary_embedding_neox_with_cache(
        torch.full((t,), 96, device="cuda"), q, k, v, wq, wk, 1e-6, got[0], got[1], None, d, table,
        block_tables=torch.zeros(t, 2, dtype=torch.int32, device="cuda"), key_scales=got[2],
        value_scales=got[3])
    assert _lib.device_status() == 0x8
    for a, b in zip(got, fresh):
        assert same_bytes(a, b)


def test_norm_refusals():
    q, k, v, wq, wk, pos, table = norm_inputs(4, 2, 1, 64, 64, torch.float16)
    c = pool(4, 1, 16, 64, torch.int8)
    args = (pos, q, k, v, wq, wk, 1e-6)
    with pytest.raises(RuntimeError, match="8-bit caches need"):
        PE.qk_norm_rotary_embedding_neox_with_cache(*args, c[0], c[1], pos, 64, table)
    with pytest.raises(RuntimeError, match="belong to 8-bit caches"):
        f = torch.zeros(4, 1, 16, 64, dtype=torch.float16, device="cuda")
        PE.qk_norm_rotary_embedding_neox_with_cache(*args, f, f, pos, 64, table, key_scales=c[2],
                                                    value_scales=c[3])
    with pytest.raises(RuntimeError, match="either slot_mapping or block_tables"):
        PE.qk_norm_rotary_embedding_neox_with_cache(*args, c[0], c[1], None, 64, table,
                                                    key_scales=c[2], value_scales=c[3])
    with pytest.raises(RuntimeError, match="share a dtype"):
        PE.qk_norm_rotary_embedding_neox(pos, q, k, wq.float(), wk, 1e-6, 64, table)
    with pytest.raises(RuntimeError, match="unit inner stride"):
        PE.qk_norm_rotary_embedding_neox(pos, q.t().contiguous().t(), k, wq, wk, 1e-6, 64, table)
    with pytest.raises(RuntimeError, match="heads contiguous"):
        C.reshape_and_cache_quantized(torch.zeros(4, 64, 1, device="cuda").transpose(1, 2),
                                      torch.zeros(4, 2, 64, device="cuda"), *c, pos)


def test_caches_of_one_call_can_be_large():
    """A pool whose byte offsets pass 32 bits: rows at its end are written and
    read back."""
    nb, kvh, bs, d = 1_050_000, 2, 16, 128  # 4.3 GB per cache
    k = torch.empty(nb, kvh, bs, d, dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    ks = torch.empty(nb, kvh, bs, dtype=torch.float8_e8m0fnu, device="cuda")
    vs = torch.empty_like(ks)
    g = torch.Generator().manual_seed(5)
    x, y = rows(g, 16, kvh, d, torch.bfloat16), rows(g, 16, kvh, d, torch.bfloat16)
    slots = (nb - 1) * bs + torch.randperm(16, generator=g)
    C.reshape_and_cache_quantized(x.cuda(), y.cuda(), k, v, ks, vs, slots.cuda())
    got = C.dequantize_blocks(k, v, ks, vs, torch.tensor([nb - 1], device="cuda"), torch.float32)
    for out, src in zip(got, (x, y)):
        want = Q.dequantize(*Q.quantize(src, torch.int8)).float()
        for t in range(16):
            assert torch.equal(out[0, :, int(slots[t]) % bs].cpu(), want[t])
