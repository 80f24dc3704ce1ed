"""Each plan of the 8-bit product, over tiles of several stages and words of scales: exact on
whole numbers, the same for a token alone, and with waits that give up."""

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


def operands(g, t, k, n):
    x = L.quantize_rows(torch.randn(t, k, generator=g, device="cuda"))
    w = L.quantize_weight(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    return (*x, *w)


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


@pytest.mark.parametrize("t,k,n", P.CASES)
def test_a_token_alone_and_among_others(t, k, n):
    """Within the bound of their sums, whose order goes with the sizes; the same bits from
    calls of the same sizes, wherever the token stands."""
    g = torch.Generator(device="cuda").manual_seed(t * 3 + k + n)
    x, xs, w, ws = operands(g, t, k, n)
    got = L.matmul_quantized(x, xs, w, ws, torch.float32)
    for i in (0, t // 2, t - 1):
        alone = L.matmul_quantized(x[i:i + 1], xs[i:i + 1], w, ws, torch.float32)
        y, mag = O.product(x[i:i + 1], xs[i:i + 1], w, ws)
        bound = O.product_bound(y, mag, k, torch.float32)
        assert bool(((alone.double() - y).abs() <= bound).all())
        assert bool(((got[i:i + 1].double() - y).abs() <= bound).all())
    turned = [v.view(torch.uint8).roll(1, 0).view(v.dtype) for v in (x, xs)]
    assert torch.equal(L.matmul_quantized(*turned, w, ws, torch.float32).roll(-1, 0), got)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("limit", [0, 1, 8, 64, 512])
@pytest.mark.parametrize("t,k,n", P.CASES)
def test_waits_that_give_up(t, k, n, limit):
    """Every input is valid and every wait ends, some before their time: the call returns,
    says so in the status word, and the next one is exact again."""
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
        if limit == 0:
            assert status & _lib.STATUS_WAIT_TIMEOUT
        assert torch.equal(L.matmul_quantized(*ops, dtype), want)
        assert _lib.device_status() == 0
