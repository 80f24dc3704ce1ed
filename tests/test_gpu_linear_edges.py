"""Calls of the 8-bit projection operators at the edges of what their documentation
allows, against the 64-bit oracle."""

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
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    _lib.device_status()
    yield
    _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("k", [8, 5, 264])
@pytest.mark.parametrize("dtype", TYPES, ids=short)
def test_silu_of_far_gates_and_large_values(dtype, k):
    """Where exp(-gate) is a number of fp32, the gate's factor is none below 2^-126."""
    top = torch.finfo(dtype).max
    gate = torch.tensor([-79.5, -80.0, -84.0, -87.0, -87.5, -88.0, -88.5])  # exact in every type
    up = torch.tensor([1.0, 1e3, 1e4, -5e4, 1e20, -1e30, top, -top]).clamp(-top, top)
    x = torch.stack([v.flatten() for v in torch.meshgrid(gate, up, indexing="ij")], 1).to(dtype)
    assert torch.equal(x[::8, 0].float(), gate)
    x = x.cuda().repeat_interleave(k, 1)  # each row a value of its own
    q, s = L.silu_and_mul_quantized(x)
    delta = (6 + 1.2 * x[:, :k].double().abs()) * 2.0 ** -23
    O.assert_rows_of(q, s, O.silu_mul(x), delta)


@pytest.mark.parametrize("k", [8, 5])
def test_silu_of_gates_past_fp32(k):
    """exp(-gate) infinite: 0, and NaN times an infinite value or from an infinite gate."""
    inf = float("inf")
    gate = torch.tensor([-89.0, -120.0, -300.0, -3e38, -1e4, -inf, -inf, -90.0, inf, 3e38])
    up = torch.tensor([3e38, 3e38, 3e38, -3e38, 1.0, 0.0, 1.0, inf, 2.0, 1e-38])
    x = torch.stack((gate, up), 1).cuda().repeat_interleave(k, 1)
    q, s = L.silu_and_mul_quantized(x)
    assert not q[:5].float().any()
    assert bool(torch.isnan(q[5:8].float()).all()) and bool((q[8].float() == 448).all())
    O.assert_rows_of(q[9:], s[9:], O.silu_mul(x[9:]), 2.0 ** -20)  # a gate is not scaled up


@pytest.mark.parametrize("k", [40, 896, 1000, 1111, 1536, 2336, 3001, 3584, 5632, 13000, 20000])
@pytest.mark.parametrize("dtype", TYPES, ids=short)
def test_norm_of_values_on_a_border(dtype, k):
    """Rows of +-c have a mean square of c^2, whatever their width (sums of few bits, exact
    in any order): the normed values are the weights with x's signs, exactly, and lie on
    borders of 8 bits, which go to even."""
    g = torch.Generator(device="cuda").manual_seed(k)
    c = torch.tensor([2.0, 2.5, 3.0, 1.25, 5.0, 7.0, 0.75, 11.0, 2.75, 13.0, 3.25], device="cuda")
    x = torch.randint(0, 2, (len(c), k), generator=g, device="cuda") * 2 - 1
    w = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(torch.bfloat16).to(dtype)
    want_q, want_s = O.quantize_rows(x * w.double())
    x = (x * c[:, None]).to(dtype)
    q, s, _ = L.rms_norm_quantized(x, w, 0.0)
    assert torch.equal(s.view(torch.uint8), want_s.view(torch.uint8))
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8))


# as the other norms of random values: under 2^-18 (a chain of at most 80 additions and 13
# across lanes and warps, halved by the root, and some roundings)
NORM_DELTA = 2.0 ** -18


def norm_delta(h, w, y):
    """The same with values and results among fp32's subnormal numbers: a product of value
    and weight below 2^-126 is a multiple of 2^-149, so off by 2^-150 before the root scales
    it, and so is a result; both by as much again in the root's second part."""
    product = (h.double() * w.double()).abs()
    steps = (2.0 ** -149 / product) * (product < 2.0 ** -126) + (2.0 ** -149 / y.abs()) * (
        y.abs() < 2.0 ** -126)
    return NORM_DELTA + torch.where(y == 0, 0, steps)


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("k", [264, 1000, 1111, 4096, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=short)
def test_norm_of_far_rows(dtype, k, with_residual):
    """Rows whose squares leave fp32's range, upwards or downwards: small enough ones count
    against eps, or, without one, are normed as any other."""
    g = torch.Generator(device="cuda").manual_seed(k)
    e = torch.tensor([-132, -126, -110, -80, -70, -64, -58, -51, -49, -40, 0, 50, 58, 62, 64, 70,
                      90, 110, 124], device="cuda")
    x = torch.randn(len(e), k, generator=g, device="cuda", dtype=torch.float64).clamp(-7, 7)
    x = (x * 2.0 ** e[:, None]).to(dtype)
    w = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(dtype)
    res = x / 2 if with_residual else None
    for eps in (0.0, 1e-38, 1e-30, 1e-6, 1.0):
        q, s, h = L.rms_norm_quantized(x, w, eps, res)
        want, want_h = O.norm(x, w, eps, res)
        assert h is None or torch.equal(h, want_h)
        O.assert_rows_of(q, s, want, norm_delta(want_h, w, want))
    # a weight that takes a product of small values below 2^-126, which the root makes up for
    x = torch.full((2, k), 2.0 ** -120, device="cuda").to(dtype)
    w = torch.full((k,), 1.25 * 2.0 ** -10, device="cuda").to(dtype)
    q, s, _ = L.rms_norm_quantized(x, w, 1e-6)
    want = O.norm(x, w, 1e-6)[0]
    O.assert_rows_of(q, s, want, norm_delta(x, w, want))


def test_residual_out_over_other_rows_is_refused():
    """Written while other rows are read: an error, not a race. Rows beside them are fine."""
    k = 256
    flat = torch.randn(9 * k, device="cuda").to(torch.bfloat16)
    x, res = flat[:8 * k].view(8, k), torch.randn(8, k, device="cuda").to(torch.bfloat16)
    w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    for out in (flat[k:].view(8, k), flat[16:16 + 8 * k].view(8, k)):
        for a, b in ((x, res), (res, x)):
            with pytest.raises(RuntimeError, match="share no memory"):
                L.rms_norm_quantized(a, w, 1e-6, b, residual_out=out)
    wide = torch.randn(8, 2 * k, device="cuda").to(torch.bfloat16)
    x, out = wide[:, :k], wide[:, k:]
    want, want_h = O.norm(x, w, 1e-6, res)
    q, s, h = L.rms_norm_quantized(x, w, 1e-6, res, residual_out=out)
    assert torch.equal(out, want_h) and h.data_ptr() == out.data_ptr()
    O.assert_rows_of(q, s, want, NORM_DELTA)


@pytest.mark.parametrize("k", [256, 250])
def test_product_of_any_two_scales(k):
    """Every scale byte with every other, on the tensor cores and off: exact (sums of a few
    bits), infinite past fp32, but for sums below 2^-126, which may count as 0: each of the
    two groups', so that a result is off by less than 2^-125. Zeros are zeros at any scale."""
    for value in (1.0, -448.0, 2.0 ** -9, 0.0):
        x = torch.full((255, k), value, device="cuda").to(E4M3)
        w = torch.ones(255 * 128, k, device="cuda").to(E4M3)
        byte = torch.arange(255, dtype=torch.uint8, device="cuda")[:, None].repeat(1, 2)
        got = L.matmul_quantized(x, byte.view(E8M0), w, byte.view(E8M0), torch.float32)
        assert torch.equal(got, got[:, ::128].repeat_interleave(128, 1))
        got = got[:, ::128].double()
        e = byte[:, :1].double() + byte[:, 0].double() - 254
        want = (k * value * torch.exp2(e)).float().double()
        group = ((k - 128) * abs(value) * torch.exp2(e)).double()  # the smaller one's sum
        exact = (group >= 2.0 ** -126) | (value == 0)
        assert torch.equal(got[exact], want[exact])
        assert bool(((got - want).abs() < 2.0 ** -125)[~exact].all())


@pytest.mark.parametrize("k", [512, 500])
def test_product_of_scales_far_apart(k):
    """Groups whose scales multiply to 2^-250 and to 2^110 side by side."""
    g = torch.Generator(device="cuda").manual_seed(k)
    t, n, groups = 40, 300, 4
    x, w = (torch.randn(r, k, generator=g, device="cuda").to(E4M3) for r in (t, n))
    xs = torch.randint(2, 180, (t, groups), generator=g, device="cuda").to(torch.uint8)
    ws = torch.randint(2, 180, (3, groups), generator=g, device="cuda").to(torch.uint8)
    got = L.matmul_quantized(x, xs.view(E8M0), w, ws.view(E8M0), torch.float32)
    y, mag = O.product(x, xs.view(E8M0), w, ws.view(E8M0))
    # and each group's sum and each sum of them may be taken for 0 below 2^-126
    bound = O.product_bound(y, mag, k, torch.float32) + (2 * groups) * 2.0 ** -126
    assert bool(((got.double() - y).abs() <= bound).all())
