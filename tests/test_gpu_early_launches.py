"""Launches that begin while the kernel before them still runs, behind one that takes
far longer than the bound of a wait."""

import pytest
import torch

from cscr import _lib
from cscr import attention as A
from cscr import linear as L
from cscr import pos_encoding as PE

pytestmark = pytest.mark.gpu

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    _lib.device_status()
    yield
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def operands(g, t, k, n):
    x = L.quantize_rows(torch.randn(t, k, generator=g, device="cuda"))
    w = L.quantize_weight(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    return (*x, *w)


def long_kernel():
    """Operands of a product that takes some tenths of a second in one CTA of 256 threads
    and lets the launch behind it begin at once."""
    k = 1 << 24
    x = torch.ones(1, k, device="cuda").to(E4M3)
    one = torch.full((1, k // 128), 127, dtype=torch.uint8, device="cuda").view(E8M0)
    return x, one, x, one


# Bound of the waits in these tests: far above a wait of these calls (some us; a probe
# takes 10 ns at least), far below the long kernel's time.
FEW_PROBES = 1 << 14


@pytest.mark.parametrize("t,k,n", [(64, 2048, 2560), (64, 8192, 256), (1024, 2048, 2560),
                                   (2048, 4096, 4096)])
def test_product_behind_a_long_kernel(t, k, n):
    """A product begins while the kernel before it runs; that kernel's time does not count
    among its waits."""
    g = torch.Generator(device="cuda").manual_seed(1)
    long, ops = long_kernel(), operands(g, t, k, n)
    want = L.matmul_quantized(*ops, torch.bfloat16)
    torch.cuda.synchronize()
    _lib.set_wait_limit(FEW_PROBES)
    L.matmul_quantized(*long, torch.float32)
    got = L.matmul_quantized(*ops, torch.bfloat16)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("h,kvh,d", [(16, 2, 128), (32, 2, 64)])
def test_attention_behind_a_long_kernel(h, kvh, d):
    """A rotation that overlaps the kernel before it lets the attention behind it begin
    while that kernel still runs."""
    g = torch.Generator(device="cuda").manual_seed(2)
    seqs, bs, blocks = 8, 16, 64

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)

    query, key, value = randn(seqs, h * d), randn(seqs, kvh * d), randn(seqs, kvh, d)
    caches = [randn(blocks, kvh, bs, d) for _ in range(2)]
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda").view(seqs, -1)
    lens = torch.arange(1, 8 * bs, 8 * bs // seqs, dtype=torch.int32, device="cuda")[:seqs]
    positions, table = lens.long() - 1, randn(8 * bs, d)

    def step(overlap):
        kc, vc = (c.clone() for c in caches)
        k = key.clone()
        if overlap:
            L.matmul_quantized(*long, torch.float32)
        q = PE.rotary_embedding_neox_with_cache(positions, query, k, value, kc, vc, None, d, table,
                                                tables, overlap_previous=overlap)
        return A.paged_attention(q.view(seqs, h, d), kc, vc, tables, lens, d ** -0.5,
                                 overlap_prologue=overlap)

    long = long_kernel()
    want = step(False)
    torch.cuda.synchronize()
    _lib.set_wait_limit(FEW_PROBES)
    got = step(True)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    assert torch.equal(got, want)
