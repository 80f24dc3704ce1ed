"""Each plan of the 8-bit product, over tiles of several stages and words of scales: exact on
whole numbers."""

import pytest
import torch

import product_plans as P
from cscr import _lib
from cscr import linear as L
from oracle import linear_oracle as O

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


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


@pytest.mark.parametrize("t,k,n", P.CASES)
def test_whole_numbers_are_exact(t, k, n):
    """Small whole values and scales that keep every partial sum a multiple of 1/2 below 2^23:
    each group's scale and each element shows, and results of 16 bits are rounded once."""
    g = torch.Generator(device="cuda").manual_seed(t + k + n)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda")

    x, w = whole(-2, 3, t, k).float().to(E4M3), whole(-2, 3, n, k).float().to(E4M3)
    groups = -(-k // 128)
    xs = whole(127, 131, t, groups).to(torch.uint8).view(E8M0)
    ws = whole(126, 130, -(-n // 128), groups).to(torch.uint8).view(E8M0)
    bias = whole(-50, 50, n)
    want, mag = O.product(x, xs, w, ws, bias)
    assert float(mag.max()) < 2 ** 23
    for dtype in TYPES:
        got = L.matmul_quantized(x, xs, w, ws, dtype, bias.to(dtype))
        assert torch.equal(got, want.float().to(dtype)), dtype
    assert _lib.device_status() == 0
