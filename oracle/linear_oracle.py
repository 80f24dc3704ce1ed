"""64-bit definitions of the 8-bit rows and their product, in plain torch on whatever
device the inputs are on. Test-only."""

from __future__ import annotations

import torch

from . import quant_oracle as Q

GROUP = 128
E4M3 = torch.float8_e4m3fn


def groups(x: torch.Tensor) -> torch.Tensor:
    """[T, K] -> [T, ceil(K / 128), 128], filled up with zeros."""
    t, k = x.shape
    n = -(-k // GROUP)
    out = torch.zeros(t, n * GROUP, dtype=x.dtype, device=x.device)
    out[:, :k] = x
    return out.view(t, n, GROUP)


def quantize_rows(x: torch.Tensor):
    """(values [T, K], scales [T, groups]) of rows in any float type."""
    q, s = Q.quantize(groups(x.double()), E4M3)
    return q.view(torch.uint8).flatten(1)[:, :x.shape[1]].contiguous().view(E4M3), s


def quantize_weight(w: torch.Tensor):
    n, k = w.shape
    rows = -(-n // GROUP)
    full = torch.zeros(rows * GROUP, k, dtype=torch.float64, device=w.device)
    full[:n] = w
    b = groups(full)  # [rows * 128, cols, 128]
    cols = b.shape[1]
    b = b.view(rows, GROUP, cols, GROUP).transpose(1, 2).reshape(rows, cols, GROUP * GROUP)
    q, s = Q.quantize(b, E4M3)
    q = q.view(torch.uint8).view(rows, cols, GROUP, GROUP).transpose(1, 2)
    return q.reshape(rows * GROUP, cols * GROUP)[:n, :k].contiguous().view(E4M3), s


def scale_of(s: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127), NaN for 255."""
    byte = s.view(torch.uint8).to(torch.int64)
    return torch.where(byte == 255, torch.nan, Q.power_of_two(byte - 127))


def dense_rows(q, s):
    return (groups(q.double()) * scale_of(s).unsqueeze(-1)).flatten(1)[:, :q.shape[1]]


def dense_weight(q, s):
    n, k = q.shape
    full = scale_of(s).repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    return q.double() * full


def product(x, xs, w, ws, bias=None):
    """(result, sum_k |x_k w_k| + |bias|), [T, N] in 64 bits."""
    a, b = dense_rows(x, xs), dense_weight(w, ws)
    y, mag = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag


def product_bound(y, mag, width, dtype):
    """How far a result may be off: products of two e4m3 values and powers of two are
    exact in fp32; width + 1 additions (the bias's among them) in any order, each off
    by at most 2^-23 of a partial sum (truncated or rounded), so by 2^-23 mag; then
    the result's rounding, eps / 2 of a value that is off by that much."""
    unit = torch.finfo(dtype).eps / 2
    added = mag * ((width + 1) * 2.0 ** -23)
    return added * (1 + unit) + y.abs() * unit + torch.finfo(dtype).smallest_normal * unit * 2


def norm(x, weight, eps, residual=None):
    """(the normed rows, h) in 64 bits; h rounded to x's dtype."""
    h = x.double()
    if residual is not None:
        # both are sums of few bits of a 53-bit format unless far apart, where the
        # double rounding of fp64, then fp32, then 16 bits cannot reach a tie
        h = (h + residual.double()).to(x.dtype).double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double()
    return y, h.to(x.dtype)


def silu_mul(gate_up):
    g, u = gate_up.double().chunk(2, -1)
    return g * torch.sigmoid(g) * u


def assert_rows_of(q, s, y, delta, what=""):
    """Rows (q, s) are the quantised rows of some y' with |y' - y| <= delta |y|: each
    group's scale lies between those of the smallest and largest such y', each value
    between the roundings of the smallest and largest at that scale."""
    delta = torch.as_tensor(delta, dtype=torch.float64, device=y.device).expand_as(y)
    lo, hi = y - delta * y.abs(), y + delta * y.abs()
    least = torch.minimum(lo.abs(), hi.abs())
    most = torch.maximum(lo.abs(), hi.abs())
    byte = s.view(torch.uint8)
    first = quantize_rows(least)[1].view(torch.uint8)
    last = quantize_rows(most)[1].view(torch.uint8)
    assert bool((byte >= first).all() and (byte <= last).all()), f"{what}: a scale is off"
    scale = scale_of(s).repeat_interleave(GROUP, 1)[:, :y.shape[1]]
    got = q.double()

    def rounded(v):
        v = (v / scale).clamp(-448, 448)
        step = Q.power_of_two(torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)
        return torch.round(v / step) * step

    bad = (got < rounded(lo)) | (got > rounded(hi))
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} values are off"
