"""Argument checks of the quantised-cache, query/key-norm and scored-attention
operators, without a GPU: the C ABI refuses bad arguments before any CUDA call,
and the op modules refuse CPU tensors and wrong shapes or types. The 64-bit
oracle's quantiser against torch's own conversion."""

import re

import pytest
import torch

from cscr import _lib
from cscr import attention as A
from cscr import cache as C
from cscr import pos_encoding as PE
from conftest import REPO
from oracle import quant_oracle as Q

HEADER = REPO / "include" / "tinyllama_b200.h"

P = 1 << 12  # stands in for an aligned device pointer; nothing is dereferenced
OK, BAD, WORKSPACE = 0, 1, 4
F32, F16, BF16, I32, I64, E4M3, I8 = range(7)


def call(lib, entry, *fields):
    name, pack = entry
    return getattr(lib, name)(pack(*fields), None)


def test_struct_layouts_match_the_header():
    """Every struct of the header has as many fields as its packing."""
    text = HEADER.read_text()
    for name, (entry, pack) in (("quantized_write", _lib.QUANTIZED_WRITE),
                                ("dequantize", _lib.DEQUANTIZE),
                                ("qk_norm_rope", _lib.QK_NORM_ROPE),
                                ("scored_attention", _lib.SCORED_ATTENTION)):
        body = re.search(r"struct tlb_%s_args \{(.*?)\}" % name, text, re.S).group(1)
        fields = sum(len(line.split(",")) for line in body.split(";") if line.strip())
        doubles = sum(len(line.split(",")) for line in body.split(";") if "double" in line)
        assert len(pack(*[0] * (fields - doubles), *[0.0] * doubles)) == 8 * fields
        assert getattr(_lib.load(), entry)(None, None) == BAD  # no struct at all


def write(lib, key=P, slots=P, slot_dtype=I64, tokens=4, kvh=2, d=128, nb=10, bs=16, dtype=BF16,
          cache=E4M3, scales=P, kc=P):
    return call(lib, _lib.QUANTIZED_WRITE, key, P, kc, P, scales, P, slots, slot_dtype, tokens, kvh,
                d, nb, bs, kvh * d, kvh * d, dtype, cache)


def test_write_refuses_before_any_cuda_call(built_lib):
    lib = _lib.load()
    for kw, msg in ((dict(dtype=I32), "dtype must be"), (dict(cache=BF16), "cache dtype"),
                    (dict(tokens=-1), "num_tokens"), (dict(kvh=0), "positive"),
                    (dict(bs=0), "positive"), (dict(kc=0), "cache pointers"),
                    (dict(slot_dtype=F32), "slot_mapping"), (dict(scales=0), "scale pointers"),
                    (dict(key=0), "tensor pointers"), (dict(key=P + 1), "aligned")):
        assert write(lib, **kw) == BAD and msg in _lib.last_error(), kw
    assert write(lib, tokens=0) == OK  # nothing to do, nothing launched


def read(lib, out=P, ids=P, id_dtype=I32, n=4, kvh=2, d=128, nb=10, bs=16, dtype=BF16, cache=I8,
         scales=P):
    return call(lib, _lib.DEQUANTIZE, out, P, P, P, scales, P, ids, id_dtype, n, kvh, d, nb, bs,
                dtype, cache)


def test_read_refuses_before_any_cuda_call(built_lib):
    lib = _lib.load()
    for kw, msg in ((dict(dtype=I8), "dtype must be"), (dict(cache=F16), "cache dtype"),
                    (dict(n=-1), "num_tokens"), (dict(d=0), "positive"),
                    (dict(id_dtype=BF16), "block_ids"), (dict(scales=0), "scale pointers"),
                    (dict(ids=0), "tensor pointers"), (dict(out=P + 1), "aligned")):
        assert read(lib, **kw) == BAD and msg in _lib.last_error(), kw
    assert read(lib, n=0) == OK


def norm(lib, q_out=P, k_out=0, value=P, eps=1e-6, kc=P, ks=P, slots=P, tables=0, maxb=0,
         tokens=4, heads=16, kvh=2, d=128, rows=64, rot=128, nb=10, bs=16, dtype=BF16, cache=E4M3,
         flags=0, pos_dtype=I64, w=P):
    return call(lib, _lib.QK_NORM_ROPE, q_out, k_out, P, P, P, value, w, P, kc, P if kc else 0, ks,
                ks, slots, tables, P, pos_dtype, I64, maxb, tokens, heads, kvh, d, rows, rot, nb, bs,
                heads * d, kvh * d, kvh * d, dtype, cache, flags, eps)


def test_norm_refuses_before_any_cuda_call(built_lib):
    lib = _lib.load()
    for kw, msg in ((dict(dtype=E4M3), "dtype must be"), (dict(pos_dtype=F16), "positions"),
                    (dict(flags=2), "unknown flags"), (dict(heads=0), "positive"),
                    (dict(rot=63), "even"), (dict(rot=130), "must not exceed"),
                    (dict(rows=0), "at least one row"), (dict(eps=-1.0), "eps"),
                    (dict(eps=float("nan")), "eps"), (dict(cache=F16), "query dtype"),
                    (dict(ks=0), "8-bit caches need"), (dict(slots=0), "slots or block"),
                    (dict(value=0), "must not be null"), (dict(w=P + 1), "aligned"),
                    (dict(kc=0, k_out=0), "must not be null")):
        assert norm(lib, **kw) == BAD and msg in _lib.last_error(), kw
    assert norm(lib, tokens=0) == OK


def attend(lib, q=P, seqs=4, heads=16, kvh=2, d=128, nb=10, bs=16, maxb=4, stride=2048, window=0,
           cap=0.0, dtype=BF16, cache=E4M3, scales=P, flags=0, ws=0, nbytes=0):
    return call(lib, _lib.SCORED_ATTENTION, P, q, P, P, scales, scales, P, P, 0, ws, nbytes, seqs,
                heads, kvh, d, nb, bs, maxb, stride, window, dtype, cache, flags, 0.1, cap)


def test_attention_refuses_before_any_cuda_call(built_lib):
    lib = _lib.load()
    for kw, msg in ((dict(dtype=I8), "dtype must be"), (dict(cache=F16), "query dtype"),
                    (dict(flags=2), "unknown flags"), (dict(seqs=0), "at least one sequence"),
                    (dict(heads=15), "divisible"), (dict(d=2048), "1024"),
                    (dict(nb=0), "positive"), (dict(window=-1), "window"),
                    (dict(cap=-1.0), "softcap"), (dict(cap=float("inf")), "softcap"),
                    (dict(cap=1e-31), "softcap"), (dict(cap=2e30), "softcap"),
                    (dict(cap=float("nan")), "softcap"), (dict(q=0), "must not be null"),
                    (dict(scales=0), "8-bit caches need"), (dict(q=P + 1), "aligned"),
                    (dict(maxb=1 << 30, bs=16), "supported range")):
        assert attend(lib, **kw) == BAD and msg in _lib.last_error(), kw


def test_ops_refuse_cpu_tensors_and_wrong_types():
    c8 = torch.zeros(2, 2, 8, 64, dtype=torch.int8)
    sc = torch.zeros(2, 2, 8, dtype=torch.float8_e8m0fnu)
    x = torch.zeros(3, 2, 64)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="cache tensors must be CUDA tensors"):
        C.reshape_and_cache_quantized(x, x, c8, c8, sc, sc, slots)
    with pytest.raises(RuntimeError, match="cache tensors must be CUDA tensors"):
        C.dequantize_blocks(c8, c8, sc, sc, slots, torch.float16)
    tables, lens = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="query must be a CUDA tensor"):
        A.paged_attention_quantized(x, c8, c8, sc, sc, tables, lens, 0.1)
    with pytest.raises(RuntimeError, match="float8_e4m3fn or int8"):
        A.paged_attention_quantized(x, x[None], x[None], sc, sc, tables, lens, 0.1)
    with pytest.raises(RuntimeError, match="float8_e8m0fnu"):
        A.paged_attention_quantized(x, c8, c8, sc.view(torch.uint8), sc.view(torch.uint8), tables,
                                    lens, 0.1)
    with pytest.raises(RuntimeError, match="share the same dtype"):
        A.paged_attention_biased(x, c8, c8, tables, lens, 0.1)
    w = torch.ones(64)
    with pytest.raises(RuntimeError, match="query must be a CUDA tensor"):
        PE.qk_norm_rotary_embedding_neox(slots, x.view(3, -1), x.view(3, -1), w, w, 1e-6, 64,
                                         torch.zeros(4, 64))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_oracle_quantiser_agrees_with_torch(dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(257, 96, generator=g) * torch.exp(4 * torch.randn(257, 1, generator=g))).to(dtype)
    x[7] = 0
    for kind in (torch.float8_e4m3fn, torch.int8):
        q, s = Q.quantize(x, kind)
        y = x.double() / Q.scale_of(s).unsqueeze(-1)
        want = y.float().to(kind) if kind != torch.int8 else torch.round(y).to(torch.int8)
        assert torch.equal(q.view(torch.uint8), want.view(torch.uint8))
        top = y.abs().amax(-1)
        assert bool((top <= Q.QMAX[kind]).all())
        smallest = s.view(torch.uint8) == 1
        assert bool(((2 * top > Q.QMAX[kind]) | smallest).all())


def test_oracle_quantiser_on_unbounded_rows():
    x = torch.tensor([[1.0, float("inf"), -float("inf"), float("nan"), -448.0 * 4]])
    q, s = Q.quantize(x, torch.float8_e4m3fn)
    assert s.view(torch.uint8).tolist() == [129]
    assert q.float()[0, :3].tolist() == [0.25, 448.0, -448.0] and bool(q.float()[0, 3].isnan())
    q, s = Q.quantize(x, torch.int8)
    assert q[0].tolist() == [0, 127, -127, 0, -112] and s.view(torch.uint8).tolist() == [131]


def test_fast_calls_leave_everything_unusual_to_the_ops(built_lib):
    """cscr._fast answers None, and raises nothing, for what is not an ordinary
    call on the current device: other objects, other counts, CPU tensors."""
    fast = _lib.fast
    assert fast is not None
    _lib.load()
    x, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    c8 = torch.zeros(2, 2, 8, 64, dtype=torch.int8)
    sc = torch.zeros(2, 2, 8, dtype=torch.float8_e8m0fnu)
    for args in ((), (None,) * 12, ("a",) * 12, (x,) * 12,
                 (x, c8, c8, sc, sc, i.view(2, 1), i, 0.1, 0.0, None, 0, False)):
        assert fast.attention(*args) is None
    for args in ((), (1,) * 7, (x, x, c8, c8, sc, sc, i)):
        assert fast.write(*args) is None
    for args in ((), ({},) * 6, (c8, c8, sc, sc, i, torch.float16), (c8, c8, sc, sc, i, "x")):
        assert fast.read(*args) is None
    w = torch.ones(64)
    for args in ((), (None,) * 16,
                 (i, x.view(2, -1), x.view(2, -1), None, w, w, 1e-6, None, None, None, 64,
                  torch.zeros(4, 64), None, None, None, False)):
        assert fast.norm(*args) is None
