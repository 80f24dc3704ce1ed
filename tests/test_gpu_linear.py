"""Projections in 8 bits on the GPU: the rows' quantisers against the 64-bit oracle,
and the product of such rows with 8-bit weights."""

import pytest
import torch

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
    _lib.device_status()
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def same_bytes(a, b):
    return torch.equal(a.view(torch.uint8).cpu(), b.view(torch.uint8).cpu())


def rows(g, t, k, dtype, spread=2.0):
    x = torch.randn(t, k, generator=g) * torch.exp(spread * torch.randn(t, 1, generator=g))
    x = (x * torch.exp(torch.randn(1, k, generator=g))).clamp(-30000, 30000).to(dtype)
    if t > 2:
        x[1] = 0
        x[2, 0] = 448.0  # a maximum on the border of its scale
    return x


SHAPES = [(1, 128), (1, 1), (3, 127), (5, 129), (64, 2048), (17, 896), (2, 16384), (7, 200),
          (300, 256), (1, 37), (9, 4096), (2, 20000), (33, 640)]


@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("t,k", SHAPES)
def test_rows_are_exact(t, k, dtype):
    x = rows(torch.Generator().manual_seed(t * 131 + k), t, k, dtype).cuda()
    q, s = L.quantize_rows(x)
    want_q, want_s = O.quantize_rows(x)
    assert q.dtype == E4M3 and s.dtype == E8M0 and s.shape == (t, -(-k // 128))
    assert same_bytes(q, want_q) and same_bytes(s, want_s)


@pytest.mark.parametrize("dtype", TYPES, ids=short)
def test_rows_with_infinities_nan_and_extremes(dtype):
    """A group's scale comes from its finite values; other groups are not touched."""
    fin = torch.finfo(dtype)
    x = rows(torch.Generator().manual_seed(1), 8, 384, dtype)
    x[0, 5], x[1, 200], x[2, 383] = float("inf"), float("nan"), float("-inf")
    x[3] = float("nan")
    x[4, :128] = fin.max
    x[5, :128] = fin.smallest_normal
    x[6, :128] = fin.smallest_normal * fin.eps  # subnormal
    for v in (x.cuda(), x[:, :383].cuda()):  # whole groups, and the kernel for any width
        q, s = L.quantize_rows(v)
        want_q, want_s = O.quantize_rows(v)
        assert same_bytes(s, want_s)
        nan = torch.isnan(v)
        assert torch.equal(torch.isnan(q.float()), nan)
        keep = (~nan).cpu()
        assert torch.equal(q.float().cpu()[keep], want_q.float().cpu()[keep])


# |y' - y| <= delta |y|. The sum of squares: a lane's chain of at most 32 (80 for any
# width) additions and 10 (13) across lanes and warps, halved by the root; rsqrtf 2 ulp
# (2^-22); the quotient, eps and two products 2^-24 each: under 2^-18.
NORM_DELTA = 2.0 ** -18


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("t,k", SHAPES)
def test_norm(t, k, dtype, with_residual):
    g = torch.Generator().manual_seed(t * 7 + k)
    x = rows(g, t, k, dtype, 0.5).cuda()
    w = (1 + 0.2 * torch.randn(k, generator=g)).to(dtype).cuda()
    res = rows(g, t, k, dtype, 0.5).cuda() if with_residual else None
    before = None if res is None else res.clone()
    q, s, h = L.rms_norm_quantized(x, w, 1e-6, res)
    want, want_h = O.norm(x, w, 1e-6, res)
    if with_residual:
        assert torch.equal(h, want_h) and torch.equal(res, before)
    else:
        assert h is None
    O.assert_rows_of(q, s, want, NORM_DELTA)


@pytest.mark.parametrize("k", [256, 250, 896])
def test_norm_in_place_strided_and_unaligned(k):
    """residual_out may be the residual or x; rows may be parts of wider ones, off
    16-byte boundaries too."""
    g = torch.Generator().manual_seed(k)
    t = 11
    for off in (0, 8, 1):
        wide = rows(g, t, 2 * k + 16, torch.bfloat16, 0.5).cuda()
        x, res = wide[:, off:off + k], wide[:, off + k:off + 2 * k]
        w = (1 + 0.2 * torch.randn(k, generator=g)).to(torch.bfloat16).cuda()
        want, want_h = O.norm(x, w, 1e-5, res)
        for target in ("residual", "x"):
            mine = wide.clone()
            mx, mres = mine[:, off:off + k], mine[:, off + k:off + 2 * k]
            q, s, h = L.rms_norm_quantized(mx, w, 1e-5, mres,
                                           residual_out=mres if target == "residual" else mx)
            assert h.data_ptr() == (mres if target == "residual" else mx).data_ptr()
            assert torch.equal(h, want_h)
            O.assert_rows_of(q, s, want, NORM_DELTA)
            # nothing beside the rows of residual_out has changed
            at = off + k if target == "residual" else off
            mine[:, at:at + k] = wide[:, at:at + k]
            assert torch.equal(mine, wide)


def test_norm_of_zero_rows_and_of_infinities():
    x = torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    x[1, 3] = float("inf")
    x[2, 200] = float("nan")
    q, s, _ = L.rms_norm_quantized(x, w, 0.0)
    # 0 * rsqrt(0) is NaN, as is inf * rsqrt(inf) and all of a row with a NaN
    want, _ = O.norm(x, w, 0.0)
    assert torch.equal(torch.isnan(q.float()), torch.isnan(want))
    q, s, _ = L.rms_norm_quantized(x[:1], w, 1e-6)
    assert not q.float().any() and bool((s.view(torch.uint8) == 1).all())


@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("t,k", SHAPES)
def test_silu_and_mul(t, k, dtype):
    g = torch.Generator().manual_seed(t + 3 * k)
    x = (2 * torch.randn(t, 2 * k, generator=g)).to(dtype).cuda()
    q, s = L.silu_and_mul_quantized(x)
    # __expf is off by at most 2 + 1.173 |g| ulp (2^-23), the quotient by 2, the sum
    # and two products by half of one each
    delta = (6 + 1.2 * x[:, :k].double().abs()) * 2.0 ** -23
    O.assert_rows_of(q, s, O.silu_mul(x), delta)


def test_silu_of_far_values():
    gate = torch.tensor([-1e4, -100.0, -30.0, 0.0, 30.0, 100.0, 1e4, float("inf")])
    x = torch.cat((gate, torch.full((8,), 2.0)))[None].to(torch.float32).cuda()
    q, s = L.silu_and_mul_quantized(x)
    want_q, want_s = O.quantize_rows(torch.tensor([[-0.0, -0.0, -0.0, 0.0, 60.0, 200.0, 2e4,
                                                    float("inf")]]))
    assert same_bytes(s, want_s) and torch.equal(q.float().cpu(), want_q.float())
    x[0, 0] = float("-inf")  # -inf * 0
    assert bool(torch.isnan(L.silu_and_mul_quantized(x)[0].float()[0, 0]))


def test_strided_and_unaligned_rows():
    g = torch.Generator().manual_seed(5)
    wide = rows(g, 9, 1200, torch.float16, 0.5).cuda()
    for off in (0, 8, 3):
        x = wide[:, off:off + 512]
        q, s = L.quantize_rows(x)
        want = O.quantize_rows(x)
        assert same_bytes(q, want[0]) and same_bytes(s, want[1])
        q, s = L.silu_and_mul_quantized(x)
        delta = (6 + 1.2 * x[:, :256].double().abs()) * 2.0 ** -23
        O.assert_rows_of(q, s, O.silu_mul(x), delta)
    x = wide[:1, :256].expand(7, -1)  # one row seven times
    assert same_bytes(L.quantize_rows(x)[0], O.quantize_rows(x)[0])


@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("t,k", [(3, 8), (700, 136), (700, 2008), (2, 16376), (40, 4092),
                                 (40, 4097)])
def test_rows_that_end_in_a_short_group(t, k, dtype):
    """Rows of whole 16-byte pieces and others, parts of wider ones that hold infinities
    behind them: neither a scale nor a norm takes in what is not the row's."""
    g = torch.Generator().manual_seed(t + k)
    pad = 16 + -k % 8
    wide = torch.full((t, 2 * k + pad), float("inf"), dtype=dtype)
    wide[:, :k] = rows(g, t, k, dtype, 0.5)
    wide = wide.cuda()
    x = wide[:, :k]
    q, s = L.quantize_rows(x)
    want = O.quantize_rows(x)
    assert same_bytes(q, want[0]) and same_bytes(s, want[1])
    w = (1 + 0.2 * torch.randn(k, generator=g)).to(dtype).cuda()
    q, s, _ = L.rms_norm_quantized(x, w, 1e-6)
    O.assert_rows_of(q, s, O.norm(x, w, 1e-6, None)[0], NORM_DELTA)
    q, s, h = L.rms_norm_quantized(x, w, 1e-6, x.clone())
    want, want_h = O.norm(x, w, 1e-6, x)
    assert torch.equal(h, want_h)
    O.assert_rows_of(q, s, want, NORM_DELTA)
    wide[:, k:2 * k] = 2 * torch.randn(t, k, generator=g).to(dtype).cuda()
    x = wide[:, :2 * k]
    q, s = L.silu_and_mul_quantized(x)
    delta = (6 + 1.2 * x[:, :k].double().abs()) * 2.0 ** -23
    O.assert_rows_of(q, s, O.silu_mul(x), delta)


def test_weight_blocks():
    g = torch.Generator().manual_seed(6)
    for n, k in ((1, 1), (128, 128), (300, 200), (129, 640), (64, 1000)):
        w = (0.05 * torch.randn(n, k, generator=g)).to(torch.bfloat16)
        w[:128, :128] *= n % 2  # a block of zeros
        for dev in ("cpu", "cuda"):
            q, s = L.quantize_weight(w.to(dev))
            want_q, want_s = O.quantize_weight(w)
            assert same_bytes(q, want_q) and same_bytes(s, want_s)


def test_no_rows():
    for k in (128, 100):
        x = torch.empty(0, k, dtype=torch.bfloat16, device="cuda")
        assert L.quantize_rows(x)[0].shape == (0, k)
        assert L.silu_and_mul_quantized(torch.cat((x, x), 1))[1].shape == (0, 1)
        w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
        assert L.rms_norm_quantized(x, w, 1e-6, x)[2].shape == (0, k)
        q, s = L.quantize_rows(x)
        wq, ws = L.quantize_weight(torch.ones(5, k, device="cuda"))
        assert L.matmul_quantized(q, s, wq, ws, torch.float16).shape == (0, 5)


def test_rows_past_32_bit_offsets():
    """2^31 values and more: the last rows are those of the rows alone."""
    t, k = 68000, 32768
    x = torch.empty(t, k, dtype=torch.float16, device="cuda")
    g = torch.Generator().manual_seed(11)
    last = rows(g, 40, k, torch.float16).cuda()
    x[:-40] = 1.0
    x[-40:] = last
    want_q, want_s = O.quantize_rows(last)
    q, s = L.quantize_rows(x)
    assert same_bytes(q[-40:], want_q) and same_bytes(s[-40:], want_s)
    assert bool((q[:5].float() == 256).all())  # 1 = 256 * 2^-8, the smallest scale
    del q, s
    w = torch.ones(k, dtype=torch.float16, device="cuda")
    q, s, _ = L.rms_norm_quantized(x, w, 1e-6)
    O.assert_rows_of(q[-40:], s[-40:], O.norm(last, w, 1e-6)[0], NORM_DELTA)


# -------------------------------------------------------------------- product

def operands(g, t, k, n, spread=1.0):
    x = rows(g, t, k, torch.float32, spread).cuda()
    w = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).cuda()
    return (*O.quantize_rows(x), *O.quantize_weight(w * k ** -0.5))


def check_product(ops, dtype, bias=None, **kw):
    got = L.matmul_quantized(*ops, dtype, bias, **kw)
    y, mag = O.product(*ops, bias)
    assert got.dtype == dtype and got.shape == y.shape and got.is_contiguous()
    err, bound = (got.double() - y).abs(), O.product_bound(y, mag, ops[0].shape[1], dtype)
    assert bool((err <= bound).all()), float((err / bound).max())
    return got


PRODUCTS = [(1, 16, 1), (1, 128, 128), (1, 896, 1152), (7, 640, 100), (16, 48, 17), (64, 2048, 640),
            (65, 512, 129), (100, 144, 333), (128, 1024, 256), (200, 400, 513), (257, 2064, 384),
            (600, 896, 1152), (1000, 128, 64), (33, 8192, 128), (5, 33, 7), (70, 130, 200),
            (1, 1, 1), (228, 992, 19036), (424, 992, 13112)]


@pytest.mark.parametrize("dtype", TYPES, ids=short)
@pytest.mark.parametrize("t,k,n", PRODUCTS)
def test_product(t, k, n, dtype):
    g = torch.Generator().manual_seed(t * 31 + k + n)
    bias = torch.randn(n, generator=g).to(dtype).cuda() if n % 2 else None
    check_product(operands(g, t, k, n), dtype, bias)


@pytest.mark.parametrize("t,k,n", [(1, 2048, 256), (40, 896, 300), (300, 1152, 260), (130, 200, 129),
                                   (9, 250, 70), (520, 640, 1000), (228, 992, 19036),
                                   (424, 992, 13112)])
def test_product_of_whole_numbers_is_exact(t, k, n):
    """Small whole values and scales that keep every partial sum below 2^24: no
    rounding anywhere, so each group's scale and each element shows."""
    g = torch.Generator().manual_seed(t + k + n)
    x = torch.randint(-2, 3, (t, k), generator=g).float().to(E4M3).cuda()
    w = torch.randint(-2, 3, (n, k), generator=g).float().to(E4M3).cuda()
    groups = -(-k // 128)
    xs = torch.randint(127, 131, (t, groups), generator=g).to(torch.uint8).cuda().view(E8M0)
    ws = torch.randint(126, 130, (-(-n // 128), groups), generator=g)
    ws = ws.to(torch.uint8).cuda().view(E8M0)
    got = L.matmul_quantized(x, xs, w, ws, torch.float32)
    want, mag = O.product(x, xs, w, ws)
    assert float(mag.max()) * 2 < 2 ** 24  # the smallest step is 1/2
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=short)
def test_product_past_32_bit_offsets(dtype):
    """2^31 results and more; the last tokens' are those of the tokens alone."""
    g = torch.Generator().manual_seed(12)
    t, k, n = 68000, 128, 32000
    x, xs, w, ws = operands(g, 300, k, n)
    where = torch.arange(t, device="cuda") % 300
    x, xs = (v.view(torch.uint8)[where].view(v.dtype) for v in (x, xs))
    got = L.matmul_quantized(x, xs, w, ws, dtype)[-300:]
    y, mag = O.product(x[-300:], xs[-300:], w, ws)
    assert bool(((got.double() - y).abs() <= O.product_bound(y, mag, k, dtype)).all())


def test_product_of_rows_that_end_off_16_bytes():
    """Rows of 250 values 256 apart: what lies between them does not count."""
    g = torch.Generator().manual_seed(13)
    t, k, n = 150, 250, 300
    x, w = (torch.randint(-2, 3, (r, 256), generator=g).float() for r in (t, n))
    x[:, k:], w[:, k:] = 448, float("nan")
    x, w = (v.to(E4M3).cuda()[:, :k] for v in (x, w))
    xs = torch.randint(127, 131, (t, 2), generator=g).to(torch.uint8).cuda().view(E8M0)
    ws = torch.randint(126, 130, (3, 2), generator=g).to(torch.uint8).cuda().view(E8M0)
    for dtype in (torch.float32, torch.bfloat16):
        got = L.matmul_quantized(x, xs, w, ws, dtype)
        assert torch.equal(got, O.product(x, xs, w, ws)[0].to(torch.float32).to(dtype))


@pytest.mark.parametrize("k", [1 << 22, (1 << 22) + 256])
def test_product_of_the_widest_rows(k):
    """The tensor cores' widest rows, and wider ones; sums of ones stay below 2^24."""
    g = torch.Generator().manual_seed(14)
    x, w = (torch.randint(-1, 2, (r, k), generator=g).to(torch.int8).cuda().float().to(E4M3)
            for r in (2, 3))
    one = torch.full((3, k // 128), 127, dtype=torch.uint8, device="cuda").view(E8M0)
    got = L.matmul_quantized(x, one[:2], w, one[:1], torch.float32)
    assert torch.equal(got.double(), x.double() @ w.double().t())


def test_product_of_strided_operands():
    """Rows of wider tensors, scales among others, one scale row for all tokens."""
    g = torch.Generator().manual_seed(8)
    t, k, n = 37, 512, 200
    x, xs, w, ws = operands(g, t, k, n)
    want = L.matmul_quantized(x, xs, w, ws, torch.float32)

    def among(v, left, right):
        wide = torch.full((v.shape[0], left + v.shape[1] + right), 0x33, dtype=torch.uint8,
                          device="cuda")
        wide[:, left:left + v.shape[1]] = v.view(torch.uint8)
        return wide.view(v.dtype)[:, left:left + v.shape[1]]

    for left, right in ((0, 16), (16, 32), (3, 2)):
        got = L.matmul_quantized(among(x, left, right), among(xs, left, right),
                                 among(w, left, right), among(ws, left, right), torch.float32)
        if (left + right) % 16 == 0:
            assert torch.equal(got, want)
        check_product((among(x, left, right), among(xs, left, right), among(w, left, right),
                       among(ws, left, right)), torch.float32)
    one = xs[:1].expand(t, -1)
    check_product((x, one, w, ws), torch.bfloat16)


@pytest.mark.parametrize("k", [256, 250])
def test_product_of_nan_and_of_special_scales(k):
    """NaN values and scales reach the results of their row or block alone."""
    g = torch.Generator().manual_seed(9)
    t, n = 20, 300
    x, xs, w, ws = operands(g, t, k, n)
    x.view(torch.uint8)[3, 100] = 0x7F
    w.view(torch.uint8)[7, 130] = 0x7F
    xs.view(torch.uint8)[5, 1] = 255
    ws.view(torch.uint8)[2, 0] = 255
    xs.view(torch.uint8)[6, 0] = 0
    got = L.matmul_quantized(x, xs, w, ws, torch.float32)
    y, mag = O.product(x, xs, w, ws)
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    fine = ~torch.isnan(y)
    bound = O.product_bound(y, mag, k, torch.float32)
    assert bool(((got.double() - y).abs()[fine] <= bound[fine]).all())


@pytest.mark.parametrize("k", [256, 250])
@pytest.mark.parametrize("ex,ew", [(-60, -60), (60, 30), (-100, 100), (120, -120)])
def test_product_of_far_scales(ex, ew, k):
    g = torch.Generator().manual_seed(10)
    x, xs, w, ws = operands(g, 20, k, 150)
    xs = (xs.view(torch.uint8) * 0 + 127 + ex).view(E8M0)
    ws = (ws.view(torch.uint8) * 0 + 127 + ew).view(E8M0)
    check_product((x, xs, w, ws), torch.float32)
