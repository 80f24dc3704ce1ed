"""Calls that the documentation of the operators allows and that only a C caller,
or an unusual one, makes: what they are served by or refused with, without a
GPU."""

import sys
import types
import weakref

import pytest
import torch

from cscr import _lib
from cscr import attention as A
from cscr import pos_encoding as PE
from paged_decode.layers import PagedAttentionWithQKNorm

P = 1 << 12  # stands in for an aligned device pointer; nothing is dereferenced
CUDA_ERROR = 3
F32, F16, BF16, I32, I64, E4M3, I8 = range(7)

# The kernel that serves a call shows in the first CUDA call, which fails where
# there is no device: the tensor-core kernels ask for it, the others are launched.
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on made-up pointers")


def scored(out=P, dtype=BF16, cache=E4M3, d=128):
    name, pack = _lib.SCORED_ATTENTION
    fields = (out, P, P, P, P, P, P, P, 0, 0, 0, 4, 16, 2, d, 10, 16, 4, 2048, 0, dtype, cache, 0,
              0.1, 0.0)
    return getattr(_lib.load(), name)(pack(*fields), None)


@no_device
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("cache", [E4M3, I8, None])
def test_scored_attention_stores_pairs_only_where_they_are_aligned(built_lib, cache, dtype):
    cache = dtype if cache is None else cache
    for out, tensor_cores in ((P, True), (P + 4, True), (P + 2, False), (P + 6, False)):
        assert scored(out, dtype, cache) == CUDA_ERROR
        assert ("device query" in _lib.last_error()) == tensor_cores, out


@no_device
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_paged_attention_stores_four_only_where_they_are_aligned(built_lib, dtype):
    lib = _lib.load()
    for out, tensor_cores in ((P, True), (P + 8, True), (P + 2, False), (P + 4, False)):
        assert lib.tlb_paged_attention(out, P, P, P, P, P, 4, 16, 2, 128, 10, 16, 4, 0.1, dtype,
                                       None, 0, 0, None) == CUDA_ERROR
        assert ("cudaGetDevice" in _lib.last_error()) == tensor_cores, out
        rc = lib.tlb_paged_attention_with_rope(out, P, P, P, P, P, P, P, P, 64, 4, 16, 2, 128, 10,
                                               16, 4, 256, 256, 0.1, dtype, None, 0, 0, None)
        assert rc == (CUDA_ERROR if tensor_cores else _lib.TLB_ERR_UNSUPPORTED), out


class AnswersAll:
    """Stands for cscr._fast on a warm stream: it has an answer to every call."""

    def __getattr__(self, name):
        return lambda *args: "answered"


def test_quantised_attention_needs_scales_on_a_warm_stream_too(monkeypatch):
    monkeypatch.setattr(_lib, "fast", AnswersAll())
    x, c8 = torch.zeros(3, 2, 64), torch.zeros(2, 2, 8, 64, dtype=torch.int8)
    tables, lens = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="float8_e4m3fn or int8"):
        A.paged_attention_quantized(x, x[None], x[None], None, None, tables, lens, 0.1)
    with pytest.raises(RuntimeError, match="float8_e8m0fnu"):
        A.paged_attention_quantized(x, c8, c8, None, None, tables, lens, 0.1)


@pytest.mark.parametrize("missing", ["value", "key_cache", "value_cache"])
def test_norm_with_cache_needs_its_caches_on_a_warm_stream_too(monkeypatch, missing):
    monkeypatch.setattr(_lib, "fast", AnswersAll())
    x, w, i = torch.zeros(3, 64), torch.ones(64), torch.zeros(3, dtype=torch.int64)
    kw = dict(value=x, key_cache=x.view(3, 1, 1, 64), value_cache=x.view(3, 1, 1, 64))
    kw[missing] = None
    with pytest.raises(RuntimeError, match="must be given"):
        PE.qk_norm_rotary_embedding_neox_with_cache(i, x, x, query_weight=w, key_weight=w, eps=1e-6,
                                                    slot_mapping=i, head_size=64, cos_sin_cache=x,
                                                    **kw)


class OnDevice(torch.Tensor):
    """A CPU tensor that passes the ops' device checks; nothing is launched on it."""

    def get_device(self):
        return 0


def test_scratch_lives_until_the_launch(monkeypatch):
    """Each call's scratch, the stream's or one of its own, is still held when the
    launch gets its address."""
    made, launched = [], []

    def workspace(query, index, nbytes, zeroed):
        ws = torch.zeros(nbytes, dtype=torch.uint8)
        made.append((weakref.ref(ws), ws.data_ptr()))
        return ws

    def launch(entry, index, *args):
        ref, address = made[-1]
        launched.append(ref() is not None and address in args)

    monkeypatch.setattr(_lib, "fast", None)
    monkeypatch.setattr(_lib, "launch", launch)
    monkeypatch.setattr(A, "_scored_workspace", workspace)
    monkeypatch.setattr(A, "_scored_workspace_bytes", lambda *key: (256, 64))

    def on(x):
        return x.as_subclass(OnDevice)

    q, c = on(torch.zeros(3, 2, 64, dtype=torch.bfloat16)), on(
        torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16))
    tables = on(torch.zeros(3, 1, dtype=torch.int32))
    lens = on(torch.ones(3, dtype=torch.int32))
    A.paged_attention_biased(q, c, c, tables, lens, 0.1)
    c8 = on(torch.zeros(2, 2, 8, 64, dtype=torch.int8))
    sc = on(torch.zeros(2, 2, 8, dtype=torch.float8_e8m0fnu))
    A.paged_attention_quantized(q, c8, c8, sc, sc, tables, lens, 0.1)
    assert launched == [True, True]


def test_a_module_of_another_torch_is_neither_used_nor_taken_as_built(built_lib, monkeypatch,
                                                                      tmp_path):
    import build as B
    import cscr

    assert _lib._load_fast() is _lib.fast and _lib.fast is not None and B._fast_up_to_date()
    for version in ("1.0.0", None):
        other = types.ModuleType("cscr._fast")
        if version is not None:
            other.torch_version = version
        monkeypatch.setitem(sys.modules, "cscr._fast", other)
        monkeypatch.setattr(cscr, "_fast", other)
        assert _lib._load_fast() is None
    module = tmp_path / "_fast.so"
    module.write_bytes(b"built against 1.0.0\0")
    monkeypatch.setattr(B, "FAST_PATH", module)
    assert not B._fast_up_to_date()


def test_a_module_that_does_not_compile_leaves_the_build_whole(built_lib, monkeypatch, tmp_path,
                                                               capsys):
    import build as B

    module = tmp_path / "_fast.so"
    module.write_bytes(b"an older one")
    source = tmp_path / "fast_calls.cpp"
    source.write_text("#error does not compile\n")
    monkeypatch.setattr(B, "FAST_PATH", module)
    monkeypatch.setattr(B, "FAST_SRC", source)
    before = B.LIB_PATH.stat().st_mtime
    assert B.build() == B.LIB_PATH and B.LIB_PATH.stat().st_mtime == before
    assert "does not compile" in capsys.readouterr().err
    assert not module.exists()


BAD = 1


def call(entry, *fields):
    name, pack = entry
    return getattr(_lib.load(), name)(pack(*fields), None)


def refused(rc):
    return rc == BAD and "aligned to the element size" in _lib.last_error()


@no_device
def test_pointers_off_their_elements_are_refused(built_lib):
    """Index arrays, tables, lengths and caches of 16-bit values: off their elements
    they are refused before any CUDA call, on them they are not."""
    for dtype, step in ((I32, 4), (I64, 8)):
        for off in (0, 1, 2, 4, 8):
            bad = off % step != 0
            at = P + off
            assert refused(call(_lib.QUANTIZED_WRITE, P, P, P, P, P, P, at, dtype, 4, 2, 128, 10,
                                16, 256, 256, BF16, E4M3)) == bad
            assert refused(call(_lib.DEQUANTIZE, P, P, P, P, P, P, at, dtype, 4, 2, 128, 10, 16,
                                BF16, I8)) == bad
            for pos, slots in ((at, P), (P, at)):
                assert refused(call(_lib.QK_NORM_ROPE, P, 0, pos, P, P, P, P, P, P, P, P, P, slots,
                                    0, P, dtype, dtype, 0, 4, 16, 2, 128, 64, 128, 10, 16, 2048,
                                    256, 256, BF16, E4M3, 0, 1e-6)) == bad
    for off in (0, 1, 2, 4):
        for kc, vc, tables in ((P + off, P, P), (P, P + off, P), (P, P, P + off)):
            rc = call(_lib.QK_NORM_ROPE, P, 0, P, P, P, P, P, P, kc, vc, 0, 0, 0, tables, P, I64, I64,
                      4, 4, 16, 2, 128, 64, 128, 10, 16, 2048, 256, 256, BF16, BF16, 0, 1e-6)
            assert refused(rc) == (off % (4 if tables != P else 2) != 0)
        for i in range(3):
            arrays = [P, P, P]
            arrays[i] += off
            rc = call(_lib.SCORED_ATTENTION, P, P, P, P, P, P, *arrays, 0, 0, 4, 16, 2, 128, 10, 16,
                      4, 2048, 0, BF16, E4M3, 0, 0.1, 0.0)
            assert refused(rc) == (off % 4 != 0)


def test_a_prompt_of_no_tokens():
    m = PagedAttentionWithQKNorm(4, 64, 0.125, 64)
    x, none = torch.zeros(0, 4, 64), torch.zeros(0, dtype=torch.int32)
    kv = torch.zeros(0, 2, 64)
    cache = torch.zeros(3, 2, 16, 64)
    out = m.prompt(none, x, kv, kv, cache, cache, none, none.view(0, 1),
                   torch.zeros(1, dtype=torch.int32), none)
    assert out.shape == x.shape and out.dtype == x.dtype


def test_read_back_tables_refuses_before_any_cuda_call(built_lib):
    lib = _lib.load()

    def tables(bt=P, lens=P, chunks=3, width=8, bs=16, nb=30, ids=P, out=P):
        return lib.tlb_read_back_tables(bt, lens, chunks, width, bs, nb, ids, out, None)

    for kw, msg in ((dict(chunks=-1), "negative"), (dict(width=-1), "negative"),
                    (dict(bs=0), "positive"), (dict(nb=0), "positive"),
                    (dict(chunks=1 << 20, width=1 << 12), "supported range"),
                    (dict(bt=0), "must not be null"), (dict(out=0), "must not be null"),
                    (dict(lens=P + 2), "aligned"), (dict(ids=P + 1), "aligned")):
        assert tables(**kw) == BAD and msg in _lib.last_error(), kw
    assert tables(chunks=0) == 0 and tables(width=0) == 0
    from paged_decode import metadata as M
    x = torch.zeros(3, 8, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device"):
        M.read_back_tables(x, x[:, 0].contiguous(), 16, 30)


def test_cscr_fast_never_holds_the_address_of_freed_scratch(monkeypatch):
    """A stream's scratch that grows or is forgotten: cscr._fast hears of it while the
    old tensor is still held (it may take another thread's call in between)."""
    held = []

    class Fast:
        @staticmethod
        def scratch(device, stream, address, nbytes):
            held.append([ref() is not None for ref in old])

    monkeypatch.setattr(_lib, "fast", Fast)
    monkeypatch.setattr(_lib, "current_device", lambda: 0)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 7)
    monkeypatch.setattr(A, "_capturing", lambda: False)
    monkeypatch.setattr(A, "_scored_workspaces", {})
    old = []
    for nbytes in (1 << 24, 1 << 25):
        ws = A._scored_workspace(torch.zeros(1), 0, nbytes, 64)
        assert A._scored_workspaces[(0, 7)] is ws
        old = [weakref.ref(ws)]
        del ws
    A.invalidate_workspaces(0)
    assert held == [[], [True], [True]]
    assert old[0]() is None and not A._scored_workspaces
