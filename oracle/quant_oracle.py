"""64-bit definitions of the quantised-cache, query/key-norm and scored-attention
operators, in plain torch on whatever device the inputs are on. Test-only."""

from __future__ import annotations

import math

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def power_of_two(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64, exactly, for whole -1022 <= e <= 1023."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def scale_of(scales: torch.Tensor) -> torch.Tensor:
    return power_of_two(scales.view(torch.uint8).to(torch.int64) - 127)


def quantize(x: torch.Tensor, kind: torch.dtype):
    """Rows of x -> (8-bit values, float8_e8m0fnu scale of each row)."""
    qmax = QMAX[kind]
    x = x.double()
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    # the smallest E with top <= qmax 2^E, found by search over all of them
    every = torch.arange(-126, 128, device=x.device)
    holds = top.unsqueeze(-1) <= qmax * power_of_two(every)
    e = every[holds.to(torch.int8).argmax(-1)]
    y = (x / power_of_two(e).unsqueeze(-1)).clamp(-qmax, qmax)
    if kind == torch.int8:
        q = torch.where(torch.isnan(y), 0.0, torch.round(y)).to(torch.int8)
    else:
        # spacing of e4m3 at |y|: 2^(floor(log2 |y|) - 3), 2^-9 below 2^-6
        step = power_of_two(torch.frexp(y.abs().nan_to_num(1.0).clamp(min=2.0 ** -6))[1] - 4)
        q = (torch.round(y / step) * step).float().to(kind)  # exact by now
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def dequantize(q: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return q.double() * scale_of(scales).unsqueeze(-1)


def take(x: torch.Tensor, *index) -> torch.Tensor:
    if x.element_size() == 1:
        return x.view(torch.uint8)[index].view(x.dtype)
    return x[index]


def norm_rope(x, weight, eps, positions, table, head_size):
    """(rows [T, heads, D] normed and rotated, bound of the fp32 error's factor:
    |a| + |b| of each element's pair)."""
    T = x.shape[0]
    y = x.double().reshape(T, -1, head_size)
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    rot = table.shape[1]
    half = rot // 2
    mag = y.abs().clone()
    pair = mag[..., :half] + mag[..., half:rot]
    mag[..., :half] = pair
    mag[..., half:rot] = pair
    ok = (positions >= 0) & (positions < table.shape[0])
    cs = table.double()[torch.where(ok, positions, 0).long()][:, None, :]
    out = y.clone()
    out[..., :half] = y[..., :half] * cs[..., :half] - y[..., half:rot] * cs[..., half:]
    out[..., half:rot] = y[..., half:rot] * cs[..., :half] + y[..., :half] * cs[..., half:]
    return torch.where(ok.view(-1, 1, 1), out, y), mag


def attention(query, key_cache, value_cache, key_scales, value_scales, block_tables, seq_lens,
              scale, softcap=0.0, alibi_slopes=None, window=0):
    """(out [S, H, D], sum_j p_j |v_j| of the same shape, score error scale [S, H],
    weight floor [S, H, D]).

    The score error scale is max_j (scale * sum_d |q_d k_jd| + |bias_j|), what the
    rounding errors of a score are proportional to. The floor is
    max_j (p_j 2^Ev_j) * sum_j |v_j| 2^-Ev_j (Ev = 0 for 16-bit caches): what one
    absolute rounding of every weight is proportional to.
    """
    S, H, D = query.shape
    NB, KVH, bs, _ = key_cache.shape
    G = H // KVH
    dev = query.device
    out = torch.zeros(S, H, D, dtype=torch.float64, device=dev)
    absum, mag = torch.zeros_like(out), torch.zeros(S, H, dtype=torch.float64, device=dev)
    floor = torch.zeros_like(out)
    for i in range(S):
        L = min(max(int(seq_lens[i]), 0), block_tables.shape[1] * bs)
        first = max(0, L - window) if window else 0
        t = torch.arange(first, L, device=dev)
        blk = block_tables[i][t // bs].long()
        keep = (blk >= 0) & (blk < NB)
        t, blk = t[keep], blk[keep]
        if t.numel() == 0:
            continue
        k, v = (take(c, blk, slice(None), t % bs) for c in (key_cache, value_cache))
        if key_scales is not None:
            k = dequantize(k, take(key_scales, blk, slice(None), t % bs))
            v = dequantize(v, take(value_scales, blk, slice(None), t % bs))
        k, v = k.double(), v.double()
        q = query[i].double().view(KVH, G, D)
        s = torch.einsum("kgd,nkd->kgn", q, k) * scale
        m = torch.einsum("kgd,nkd->kgn", q.abs(), k.abs()) * abs(scale)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if alibi_slopes is not None:
            bias = alibi_slopes.double().view(KVH, G, 1) * (t - (L - 1)).double()
            s, m = s + bias, m + bias.abs()
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("kgn,nkd->kgd", p, v).reshape(H, D)
        absum[i] = torch.einsum("kgn,nkd->kgd", p, v.abs()).reshape(H, D)
        mag[i] = m.amax(-1).reshape(H)
        ev = torch.ones(t.numel(), KVH, dtype=torch.float64, device=dev)
        if value_scales is not None:
            ev = scale_of(take(value_scales, blk, slice(None), t % bs))
        top = (p * ev.t()[:, None, :]).amax(-1, keepdim=True)  # [KVH, G, 1]
        raw = (v.abs() / ev.unsqueeze(-1)).sum(0)  # [KVH, D]
        floor[i] = (top * raw[:, None, :]).reshape(H, D)
    return out, absum, mag, floor


def attention_bound(out, absum, mag, floor, dtype, cache_dtype, plain=False):
    """How far a result may be off, element by element.

    The result's rounding: eps/2 of the value. The weights: relative error
    e = e_score + e_weight + 2^-20 each, so the quotient of sums is off by at most
    2 e / (1 - e) sum p|v|. e_score: fp32 accumulation (2^-20 of mag covers
    up to 16 roundings of 2^-24 on its way). e_weight: weights are rounded to
    fp16 (2^-11) where bf16 queries meet 8-bit caches, to hi + lo pairs (2^-16)
    otherwise in 16 bits, not at all in fp32. fp16 weights (8-bit or fp16 caches)
    below fp16's normal range are off by up to half its smallest step, 2^-25, in
    a unit where the reference weight is 2^7 and the largest at least that:
    2^-32 of the largest weight for each token. `plain`: cscr's paged_attention over
    fp16 caches, whose weights are one fp16 rounding (2^-11) of values in [0, 1]
    (2^-25 of the largest below the normal range).
    """
    unit = torch.finfo(dtype).eps / 2
    eight = cache_dtype in QMAX
    if dtype == torch.float32:
        weight = 0.0
    else:
        weight = 2.0 ** -11 if plain or (eight and dtype == torch.bfloat16) else 2.0 ** -16
    e = mag.unsqueeze(-1) * 2.0 ** -20 + weight + 2.0 ** -20
    assert float(e.max()) < 0.05
    tiny = torch.finfo(dtype).smallest_normal
    fp16_weights = dtype != torch.float32 and (eight or dtype == torch.float16)
    low = floor * 2.0 ** (-25 if plain else -32) * 1.01 if fp16_weights else 0.0
    return out.abs() * unit * (1 + 2 ** -7) + 2.2 * e * absum + low + tiny * unit * 4


def assert_within(got, want, bound, what=""):
    err = (got.double() - want).abs()
    worst = (err / bound.clamp(min=1e-300)).max()
    assert bool((err <= bound).all()), f"{what}: error up to {float(worst):.3f} of the bound"
    assert not math.isnan(float(worst))
