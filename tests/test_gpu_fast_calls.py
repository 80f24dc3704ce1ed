"""Allocations of cscr._fast: what watches, replaces or fills them takes part as in any
other op."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from cscr import _lib
from cscr import attention as A
from cscr import cache as C
from cscr import linear as L
from cscr import pos_encoding as PE
from paged_decode import pool
from test_gpu_scored_attention import Case

pytestmark = pytest.mark.gpu

E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    _lib.device_status()
    yield
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    torch.cuda.synchronize()


class Seen(TorchDispatchMode):
    """The shapes of tensors that are made under it."""

    def __init__(self):
        super().__init__()
        self.shapes = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if "empty" in str(func):
            self.shapes.append(tuple(out.shape))
        return out


def ordinary_calls():
    """(call, number of tensors it makes) of each op that cscr._fast answers."""
    g = torch.Generator(device="cuda").manual_seed(1)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(BF16)

    x, w, d, t = randn(6, 256), randn(256), 64, 6
    rows, weight = L.quantize_rows(x), L.quantize_weight(randn(128, 256))
    pos = torch.arange(t, device="cuda")
    q, k, v, table, head = randn(t, 4 * d), randn(t, 2 * d), randn(t, 2, d), randn(32, d), randn(d)
    kv = pool.allocate_quantized_kv_cache(1, 4, 2, d, 16, E4M3)[0]
    for c in kv:
        c.view(torch.uint8).zero_()
    c = Case([20, 33], 8, 2, 64, 16, BF16, E4M3, seed=2)
    c.run()  # its scratch is there from now on
    return {
        "rows": (lambda: L.quantize_rows(x), 2),
        "silu": (lambda: L.silu_and_mul_quantized(x), 2),
        "norm": (lambda: L.rms_norm_quantized(x, w, 1e-6, x), 3),
        "product": (lambda: (L.matmul_quantized(*rows, *weight, BF16),), 1),
        "attention": (lambda: (A.paged_attention_quantized(
            c.q, c.k, c.v, c.ks, c.vs, c.tables, c.lens, c.scale),), 1),
        "read": (lambda: C.dequantize_blocks(*kv, pos[:3], BF16), 2),
        "heads": (lambda: PE.qk_norm_rotary_embedding_neox(pos, q, k, head, head, 1e-6, d, table),
                  2),
        "heads and cache": (lambda: (PE.qk_norm_rotary_embedding_neox_with_cache(
            pos, q, k, v, head, head, 1e-6, kv[0], kv[1], pos, d, table, key_scales=kv[2],
            value_scales=kv[3]),), 1),
    }


def test_dispatch_modes_see_the_allocations():
    assert _lib.fast is not None
    for name, (call, count) in ordinary_calls().items():
        want = call()
        with Seen() as seen:
            got = call()
        shapes = [tuple(o.shape) for o in got]
        assert len(shapes) == count and sorted(seen.shapes) == sorted(shapes), name
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


def test_the_python_code_answers_the_same(monkeypatch):
    """Each of the calls with its Python argument handling alone."""
    calls = ordinary_calls()
    calls["heads and cache"][0]()  # what it writes is there for every read
    want = {name: call() for name, (call, _) in calls.items()}
    monkeypatch.setattr(_lib, "fast", None)
    for name, (call, _) in calls.items():
        for a, b in zip(call(), want[name], strict=True):
            assert a.dtype == b.dtype and a.stride() == b.stride(), name
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


def test_profilers_see_the_allocations():
    for name, (call, count) in ordinary_calls().items():
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as profile:
            call()
        assert sum(e.count for e in profile.key_averages() if e.key == "aten::empty") >= count, name


def test_deterministic_algorithms_fill_what_a_call_leaves_unwritten():
    """A product whose waits give up leaves its results as they were made: filled with NaN."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = L.quantize_rows(torch.randn(300, 512, generator=g, device="cuda"))
    w = L.quantize_weight(torch.randn(640, 512, generator=g, device="cuda"))
    L.matmul_quantized(*x, *w, BF16)
    torch.full((300, 640), 1.0, dtype=BF16, device="cuda")  # what the allocator hands out next
    torch.cuda.synchronize()
    torch.use_deterministic_algorithms(True)
    try:
        _lib.set_wait_limit(0)
        got = L.matmul_quantized(*x, *w, BF16)
        torch.cuda.synchronize()
    finally:
        torch.use_deterministic_algorithms(False)
    assert _lib.device_status() == _lib.STATUS_WAIT_TIMEOUT
    assert bool(torch.isnan(got).all())
