"""Launches that begin while the kernel before them still runs, behind one that takes
far longer than the bound of a wait."""

import pytest
import torch

from cscr import _lib
from cscr import linear as L

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
