"""The cases and plain forms by which the quantised-cache, query/key-norm and
biased-score operators are measured.

``run`` computes a case either with the framework's kernels (``own = True``:
the calls a user makes of ``cscr``) or in plain form (elementary torch
operations in 32 bits, rounded once at the end). ``exact`` gives the same
results from the definitions in 64 bits.

An 8-bit cache row (one token of one kv head) is D values of ``float8_e4m3fn``
or ``int8`` and one power-of-two scale, held as ``float8_e8m0fnu``: the
smallest 2^E with max|x| <= qmax * 2^E (qmax 448 or 127), E in [-126, 127].
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
          "float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "float8_e4m3fn": 1, "int8": 1}
QMAX = {torch.float8_e4m3fn: (448.0, 0.875, 9), torch.int8: (127.0, 127.0 / 128.0, 7)}

_ops = None


def _own_ops():
    """The framework's op modules (only when ``own``)."""
    global _ops
    if _ops is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "tinyllama.py_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from cscr import attention, cache, pos_encoding

        _ops = (attention, cache, pos_encoding)
    return _ops


# ------------------------------------------------------------------- cases

def _attention(op, name, dtype, cache, heads, block, seqs, lo, hi, lens="uniform", softcap=0.0,
               alibi=False, window=0, lens_seed=0):
    h, kvh, d = heads
    return {"op": op, "name": name, "dtype": dtype, "cache": cache, "heads": h, "kv_heads": kvh,
            "head_dim": d, "block": block, "seqs": seqs, "lo": lo, "hi": hi, "lens": lens,
            "softcap": softcap, "alibi": alibi, "window": window, "lens_seed": lens_seed}


def _write(name, dtype, cache, kv_heads, d, block, tokens, pad=0):
    return {"op": "write", "name": name, "dtype": dtype, "cache": cache, "kv_heads": kv_heads,
            "head_dim": d, "block": block, "tokens": tokens, "pad": pad}


def _read(name, dtype, cache, kv_heads, d, block, blocks):
    return {"op": "read", "name": name, "dtype": dtype, "cache": cache, "kv_heads": kv_heads,
            "head_dim": d, "block": block, "blocks": blocks}


def _norm(name, dtype, cache, heads, rot, tokens, block=16, pad=0):
    h, kvh, d = heads
    return {"op": "norm", "name": name, "dtype": dtype, "cache": cache, "heads": h,
            "kv_heads": kvh, "head_dim": d, "rot": rot, "tokens": tokens, "block": block,
            "pad": pad}


def listed():
    return [
        # a few short conversations: the call is launch and latency
        _attention("quantized", "q_small_int8", "float16", "int8", (16, 2, 128), 16, 8, 1, 512),
        # the decode step the benchmark times, its cache held in 8 bits
        _attention("quantized", "q_step_e4m3", "bfloat16", "float8_e4m3fn", (16, 2, 128), 16, 64,
                   128, 4096),
        # many long conversations on the small model's heads: the largest stream
        _attention("quantized", "q_long_e4m3", "bfloat16", "float8_e4m3fn", (14, 2, 64), 32, 256,
                   7000, 8192),
        # a capped-score model whose layer sees only the last tokens
        _attention("biased", "b_softcap_window", "bfloat16", "bfloat16", (16, 2, 128), 16, 64,
                   128, 4096, softcap=50.0, window=1024),
        # a distance-bias model with one kv head per query head, long-tailed lengths
        _attention("biased", "b_alibi", "float16", "float16", (12, 12, 64), 16, 96, 32, 16384,
                   lens="long_tail", alibi=True),
        # one decode step's new rows
        _write("w_step_e4m3", "bfloat16", "float8_e4m3fn", 2, 128, 16, 64),
        # a long prompt's rows, packed and padded to a multiple of 8
        _write("w_prompt_int8", "float16", "int8", 8, 128, 16, 16381, pad=3),
        # the shared prefix of one conversation, read for a new prompt chunk
        _read("r_prefix_int8", "float16", "int8", 2, 128, 16, 33),
        # a whole batch's cache, read back for a prompt step
        _read("r_batch_e4m3", "bfloat16", "float8_e4m3fn", 2, 128, 16, 9000),
        # a decode step's queries and keys, keys and values into a 16-bit cache
        _norm("n_step", "bfloat16", "bfloat16", (16, 2, 128), 128, 64),
        # a packed prompt step into an 8-bit cache
        _norm("n_packed_e4m3", "bfloat16", "float8_e4m3fn", (16, 2, 128), 128, 4853, pad=3),
        # a long prompt of a partly rotated model, no cache written
        _norm("n_prompt_partial", "float16", "", (32, 8, 128), 64, 16383),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantized", "quantized", "biased", "write", "read", "norm"])
    dtype = rng.choice(["float16", "bfloat16"])
    cache8 = rng.choice(["float8_e4m3fn", "int8"])
    block = rng.choice([8, 16, 32])
    if op in ("quantized", "biased"):
        heads = rng.choice([(16, 2, 128), (14, 2, 64), (12, 12, 64), (32, 8, 128), (24, 1, 128),
                            (10, 2, 64), (28, 4, 128)])
        seqs = _log_int(rng, 1, 256)
        # at most the largest listed case's cache bytes
        row = 2 * heads[1] * heads[2] * (1 if op == "quantized" else 2)
        hi = _log_int(rng, 2, max(2, min(16384, 480_000_000 // (row * seqs))))
        modified = op == "biased" or rng.random() < 0.3
        return _attention(op, "", dtype, cache8 if op == "quantized" else dtype, heads, block,
                          seqs, rng.randint(1, hi), hi, rng.choice(["uniform", "long_tail"]),
                          rng.choice([0.0, 30.0]) if modified else 0.0,
                          modified and rng.random() < 0.5,
                          _log_int(rng, 16, 8192) if modified and rng.random() < 0.5 else 0,
                          rng.randint(0, 1 << 20))
    kv_heads, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128, 256])
    if op == "write":
        return _write("", dtype, cache8, kv_heads, d, block,
                      _log_int(rng, 1, 16384 * 1024 // (kv_heads * d)), rng.randint(0, 7))
    if op == "read":
        return _read("", dtype, cache8, kv_heads, d, block,
                     _log_int(rng, 1, 36_000_000 // (kv_heads * d * block)))
    return _norm("", dtype, rng.choice(["", dtype, "float8_e4m3fn"]),
                 (kv_heads * rng.choice([1, 2, 4]), kv_heads, d), rng.choice([d, d // 2]),
                 _log_int(rng, 1, 16384 * 1024 // (kv_heads * d)) // 4 + 1, block,
                 rng.randint(0, 7))


# ------------------------------------------------------------------ inputs

def _lens(case):
    rng = np.random.default_rng(case["lens_seed"])
    lo, hi, n = case["lo"], case["hi"], case["seqs"]
    if case["lens"] == "long_tail":
        return np.clip(np.floor(lo * (1 + rng.pareto(1.2, size=n))), lo, hi).astype(np.int64)
    return rng.integers(lo, hi + 1, size=n)


def _seen(case):
    """Tokens of each sequence that its query sees."""
    lens = _lens(case)
    return np.minimum(lens, case["window"]) if case["window"] else lens


def _quantize(x, kind):
    """Rows of x (last dimension) -> (8-bit values, scale of each row), in 32 bits."""
    qmax, edge, shift = QMAX[kind]
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > edge, e - shift + 1, e - shift).clamp(-126, 127)
    scale = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    y = x / scale.float().unsqueeze(-1)
    q = torch.round(y).clamp(-qmax, qmax).to(kind) if kind == torch.int8 else y.to(kind)
    return q, scale


def _dense(q, scales):
    """The values that 8-bit rows stand for, in 32 bits."""
    return q.float() * scales.float().unsqueeze(-1)


def _take(x, i):
    """x[i] over the first dimension, for the 8-bit types too."""
    return x.view(torch.uint8)[i].view(x.dtype) if x.element_size() == 1 else x[i]


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _row_scales(g, *shape):
    """Row magnitudes as caches have them: most near 1, some far off."""
    return torch.exp(0.5 * _normal(g, *shape))


def _kv(g, blocks, case):
    """A pool of cache blocks of the case's cache type: (k, v, k scales, v scales)."""
    kvh, bs, d = case["kv_heads"], case["block"], case["head_dim"]
    kind, out, scales = DTYPES[case["cache"]], [], []
    for _ in range(2):
        x = _normal(g, blocks, kvh, bs, d) * _row_scales(g, blocks, kvh, bs, 1)
        x = x.to(DTYPES[case["dtype"]])
        if kind in QMAX:
            x, s = _quantize(x, kind)
            scales.append(s)
        out.append(x)
    return (*out, *(scales or (None, None)))


def _empty_pool(case, tokens):
    """A pool that holds `tokens` rows, and nothing yet."""
    bs, kvh, d = case["block"], case["kv_heads"], case["head_dim"]
    blocks = -(-tokens // bs) + 1
    kind = DTYPES[case["cache"]]
    if kind not in QMAX:
        k = torch.zeros(blocks, kvh, bs, d, dtype=kind, device="cuda")
        return blocks, k, torch.zeros_like(k), None, None
    caches = [torch.zeros(blocks, kvh, bs, d, dtype=torch.uint8, device="cuda").view(kind)
              for _ in range(2)]
    scales = [torch.full((blocks, kvh, bs), 127, dtype=torch.uint8,
                         device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
    return blocks, *caches, *scales


def _slots(g, case, blocks):
    """Distinct slots in shuffled blocks, the padding tokens' at -1."""
    n, bs = case["tokens"], case["block"]
    perm = torch.randperm(blocks, generator=g, device="cuda")
    i = torch.arange(n, device="cuda")
    slots = perm[i // bs] * bs + i % bs
    return torch.cat((slots, torch.full((case["pad"],), -1, dtype=torch.int64, device="cuda")))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    dtype = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] in ("quantized", "biased"):
        lens, bs = _lens(case), case["block"]
        count = -(-lens // bs)
        used = int(count.sum())
        blocks = used + 8
        st["k"], st["v"], st["ks"], st["vs"] = _kv(g, blocks, case)
        perm = torch.randperm(blocks, generator=g, device="cuda")[:used].to(torch.int32)
        width = int(count.max())
        tables = torch.zeros(case["seqs"], width, dtype=torch.int32, device="cuda")
        mask = torch.from_numpy(np.arange(width)[None, :] < count[:, None]).cuda()
        tables[mask] = perm
        st["tables"] = tables
        st["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        st["q"] = _normal(g, case["seqs"], case["heads"], case["head_dim"]).to(dtype)
        st["scale"] = case["head_dim"] ** -0.5
        h = case["heads"]
        st["slopes"] = (torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h).float()
                        if case["alibi"] else None)
        return st
    kvh, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "read":
        pool = case["blocks"] + case["blocks"] // 4 + 2
        st["k"], st["v"], st["ks"], st["vs"] = _kv(g, pool, case)
        ids = torch.randperm(pool, generator=g, device="cuda")[:case["blocks"]].to(torch.int32)
        if case["blocks"] > 2:
            ids[1] = -1  # a block that a shorter sequence of the batch does not have
        st["ids"] = ids
        return st
    total = case["tokens"] + case["pad"]
    if case["cache"]:
        blocks, st["k"], st["v"], st["ks"], st["vs"] = _empty_pool(case, case["tokens"])
        st["slots"] = _slots(g, case, blocks)
    if case["op"] == "write":
        for name in ("key", "value"):
            st[name] = (_normal(g, total, kvh, d) * _row_scales(g, total, kvh, 1)).to(dtype)
        return st
    # query, key and value are parts of one projection's rows
    h, rot = case["heads"], case["rot"]
    qkv = (_normal(g, total, (h + 2 * kvh) * d) * _row_scales(g, total, 1)).to(dtype)
    st["query"], st["key"], st["value"] = qkv.split([h * d, kvh * d, kvh * d], dim=1)
    st["wq"] = (1 + 0.2 * _normal(g, d)).to(dtype)
    st["wk"] = (1 + 0.2 * _normal(g, d)).to(dtype)
    st["eps"] = 1e-6
    rows = 8192
    st["positions"] = torch.arange(total, device="cuda") % rows
    freq = 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * freq
    st["table"] = torch.cat((angle.cos(), angle.sin()), -1).to(dtype)
    return st


# -------------------------------------------------------------- plain forms

def _plain_attention(st):
    case, q = st["case"], st["q"].float()
    s_, h, d = q.shape
    kvh, bs = case["kv_heads"], case["block"]
    at = st["tables"].long()
    k, v = _take(st["k"], at), _take(st["v"], at)  # [S, blocks, KVH, bs, D]
    if st["ks"] is not None:
        k, v = _dense(k, _take(st["ks"], at)), _dense(v, _take(st["vs"], at))
    n = at.shape[1] * bs
    k = k.float().permute(0, 2, 1, 3, 4).reshape(s_, kvh, n, d)
    v = v.float().permute(0, 2, 1, 3, 4).reshape(s_, kvh, n, d)
    q = q.view(s_, kvh, h // kvh, d)
    s = torch.matmul(q, k.transpose(-1, -2)) * st["scale"]
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    last = st["lens"].long().view(-1, 1, 1, 1) - 1
    j = torch.arange(n, device=q.device)
    if case["alibi"]:
        s = s + st["slopes"].view(1, kvh, h // kvh, 1) * (j - last).float()
    seen = j <= last
    if case["window"]:
        seen = seen & (j > last - case["window"])
    s = torch.where(seen, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = torch.where(seen, p, 0.0)
    o = torch.matmul(p, torch.where(seen.view(s_, 1, n, 1), v, 0.0))
    return (o / p.sum(-1, keepdim=True)).view(s_, h, d).to(st["q"].dtype)


def _plain_store(cache, slots, rows):
    """rows [n, KVH, D or nothing] -> cache[slot // bs, :, slot % bs]."""
    bs = cache.shape[2]
    if cache.element_size() == 1:
        cache, rows = cache.view(torch.uint8), rows.view(torch.uint8)
    cache[slots // bs, :, slots % bs] = rows


def _plain_write(st, key, value):
    n = st["case"]["tokens"]
    slots = st["slots"][:n]
    kind = st["k"].dtype
    for rows, cache, scales in ((key, st["k"], st["ks"]), (value, st["v"], st["vs"])):
        rows = rows[:n]
        if kind in QMAX:
            rows, s = _quantize(rows, kind)
            _plain_store(scales, slots, s)
        _plain_store(cache, slots, rows)


def _plain_norm(x, w, st):
    """RMS norm of each head's row, then the rotation of its first `rot` values."""
    t, d, rot = x.shape[0], st["case"]["head_dim"], st["case"]["rot"]
    y = x.float().view(t, -1, d)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"]) * w.float()
    cos, sin = st["table"].float()[st["positions"]].unsqueeze(1).chunk(2, -1)
    a, b, rest = y[..., :rot // 2], y[..., rot // 2:rot], y[..., rot:]
    y = torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)
    return y.to(x.dtype)


def _plain(st):
    case = st["case"]
    if case["op"] in ("quantized", "biased"):
        return _plain_attention(st)
    if case["op"] == "write":
        _plain_write(st, st["key"], st["value"])
        return st["k"], st["v"], st["ks"], st["vs"]
    if case["op"] == "read":
        ids = st["ids"].long()
        there = (ids >= 0).view(-1, 1, 1, 1)
        at, dtype = ids.clamp(min=0), DTYPES[case["dtype"]]
        return tuple(torch.where(there, _dense(_take(c, at), _take(s, at)), 0.0).to(dtype)
                     for c, s in ((st["k"], st["ks"]), (st["v"], st["vs"])))
    t = st["query"].shape[0]
    q = _plain_norm(st["query"], st["wq"], st)
    k = _plain_norm(st["key"], st["wk"], st)
    if not case["cache"]:
        return q.view(t, -1), k.view(t, -1)
    _plain_write(st, k, st["value"].view(t, case["kv_heads"], case["head_dim"]))
    return q.view(t, -1), st["k"], st["v"], st["ks"], st["vs"]


def _own(st):
    case = st["case"]
    attention, cache, pos_encoding = _own_ops()
    op = case["op"]
    if op == "quantized":
        return attention.paged_attention_quantized(
            st["q"], st["k"], st["v"], st["ks"], st["vs"], st["tables"], st["lens"], st["scale"],
            softcap=case["softcap"], alibi_slopes=st["slopes"], window=case["window"])
    if op == "biased":
        return attention.paged_attention_biased(
            st["q"], st["k"], st["v"], st["tables"], st["lens"], st["scale"],
            softcap=case["softcap"], alibi_slopes=st["slopes"], window=case["window"])
    if op == "write":
        cache.reshape_and_cache_quantized(st["key"], st["value"], st["k"], st["v"], st["ks"],
                                          st["vs"], st["slots"])
        return st["k"], st["v"], st["ks"], st["vs"]
    if op == "read":
        return cache.dequantize_blocks(st["k"], st["v"], st["ks"], st["vs"], st["ids"],
                                       DTYPES[case["dtype"]])
    if not case["cache"]:
        return pos_encoding.qk_norm_rotary_embedding_neox(
            st["positions"], st["query"], st["key"], st["wq"], st["wk"], st["eps"],
            case["head_dim"], st["table"])
    q = pos_encoding.qk_norm_rotary_embedding_neox_with_cache(
        st["positions"], st["query"], st["key"], st["value"], st["wq"], st["wk"], st["eps"],
        st["k"], st["v"], st["slots"], case["head_dim"], st["table"], key_scales=st["ks"],
        value_scales=st["vs"])
    return q, st["k"], st["v"], st["ks"], st["vs"]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------- work

def work(case):
    e, d, kvh = SIZES[case["dtype"]], case["head_dim"], case["kv_heads"]
    c = SIZES.get(case["cache"], 0)
    row = d * c + (1 if c == 1 else 0)  # a cache row and its scale
    if case["op"] in ("quantized", "biased"):
        seen, lens = _seen(case), _lens(case)
        tokens = int(seen.sum())
        blocks = int((-(-lens // case["block"]) - (lens - seen) // case["block"]).sum())
        h = case["heads"]
        return {"bytes": 2 * tokens * kvh * row + 2 * case["seqs"] * h * d * e + 4 * blocks
                + 4 * case["seqs"], "flops": 4 * tokens * h * d}
    if case["op"] == "read":
        n = case["blocks"] * kvh * case["block"]
        return {"bytes": 2 * n * (row + d * e) + 4 * case["blocks"], "flops": 2 * n * d}
    n = case["tokens"]
    if case["op"] == "write":
        return {"bytes": 2 * n * kvh * (d * e + row) + 8 * n, "flops": 4 * n * kvh * d}
    h, rot = case["heads"], case["rot"]
    moved = n * d * e * (2 * h + kvh) + n * (rot * e + 8)
    moved += n * (kvh * (d * e + 2 * row) + 8) if case["cache"] else n * kvh * d * e
    return {"bytes": moved, "flops": n * (h + kvh) * (4 * d + 3 * rot)}


# ------------------------------------------------------------------- exact

def _row64(x):
    return x.to(torch.float64)


def _power64(e):
    """2^e exactly, for whole e of a normal result (pow may be off by its last bit)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_attention(st):
    case = st["case"]
    h, kvh, d, bs = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    out = torch.zeros(case["seqs"], h, d, dtype=torch.float64, device="cuda")
    lens = _lens(case)
    for i, n in enumerate(lens.tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        t = torch.arange(first, n, device="cuda")
        blk, off = st["tables"][i][t // bs].long(), t % bs

        def rows(cache, scales):
            x = cache.view(torch.uint8)[blk, :, off].view(cache.dtype) \
                if cache.element_size() == 1 else cache[blk, :, off]
            x = _row64(x)
            if scales is not None:
                byte = scales.view(torch.uint8)[blk, :, off].double()
                x = x * _power64(byte - 127).unsqueeze(-1)
            return x

        k, v = rows(st["k"], st["ks"]), rows(st["v"], st["vs"])  # [n, KVH, D]
        q = _row64(st["q"][i]).view(kvh, h // kvh, d)
        s = torch.einsum("kgd,nkd->kgn", q, k) * st["scale"]
        if case["softcap"]:
            s = torch.tanh(s / case["softcap"]) * case["softcap"]
        if case["alibi"]:
            s = s - st["slopes"].double().view(kvh, -1, 1) * (n - 1 - t).double()
        out[i] = torch.einsum("kgn,nkd->kgd", torch.softmax(s, -1), v).reshape(h, d)
    return out


def _exact_quantize(x, kind):
    """From the definition: the smallest power of two, then the nearest of all values of the type."""
    qmax = QMAX[kind][0]
    x = _row64(x)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / qmax)).nan_to_num(neginf=-126.0)
    e = e.clamp(-200, 200)
    e = torch.where(_power64(e) * qmax < top, e + 1, e)
    e = torch.where(_power64(e - 1) * qmax >= top, e - 1, e).clamp(-126, 127)
    y = x / _power64(e)
    if kind == torch.int8:
        near = torch.round(y)
    else:
        # spacing of e4m3 at |y|: 2^(floor(log2|y|) - 3), 2^-9 below 2^-6
        step = _power64(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
        near = torch.round(y / step) * step
    return near, _power64(e.squeeze(-1))


def _exact_store(st, rows):
    """A pool of zeros (scales: ones) with the step's rows in their slots."""
    case = st["case"]
    n, bs = case["tokens"], case["block"]
    slots = st["slots"][:n]
    pool = torch.zeros(st["k"].shape, dtype=torch.float64, device="cuda")
    if rows.dim() == 2:
        pool = torch.ones(pool.shape[:3], dtype=torch.float64, device="cuda")
    pool[slots // bs, :, slots % bs] = rows
    return pool


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("quantized", "biased"):
        return _exact_attention(st)
    if case["op"] == "write":
        kind = st["k"].dtype
        k, ks = _exact_quantize(st["key"][:case["tokens"]], kind)
        v, vs = _exact_quantize(st["value"][:case["tokens"]], kind)
        if kind == torch.int8:  # whole numbers
            k, v = k.to(torch.int8), v.to(torch.int8)
            pools = [_exact_store(st, x.double()).to(torch.int8) for x in (k, v)]
        else:
            pools = [_exact_store(st, x) for x in (k, v)]
        return (*pools, _exact_store(st, ks), _exact_store(st, vs))
    if case["op"] == "read":
        ids = st["ids"].long()
        out = []
        for cache, scales in ((st["k"], st["ks"]), (st["v"], st["vs"])):
            x = _row64(cache)[ids.clamp(min=0)]
            byte = scales.view(torch.uint8)[ids.clamp(min=0)].long()
            x = x * _power64(byte - 127).unsqueeze(-1)
            x[ids < 0] = 0
            out.append(x)
        return tuple(out)
    t, d, rot, half = st["query"].shape[0], case["head_dim"], case["rot"], case["rot"] // 2

    def normed(x, w):
        x = _row64(x).view(t, -1, d)
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + st["eps"]) * _row64(w)
        y = x.clone()
        c = _row64(st["table"])[st["positions"]][:, None, :]
        y[..., :half] = x[..., :half] * c[..., :half] - x[..., half:rot] * c[..., half:]
        y[..., half:rot] = x[..., half:rot] * c[..., :half] + x[..., :half] * c[..., half:]
        return y

    q, k = normed(st["query"], st["wq"]), normed(st["key"], st["wk"])
    if not case["cache"]:
        return q.view(t, -1), k.view(t, -1)
    if case["cache"] in ("int8", "float8_e4m3fn"):
        # what is stored stands one rounding behind another: no value of its own in 64 bits
        return q.view(t, -1), None, None, None, None
    n = case["tokens"]
    v = _row64(st["value"][:n]).view(n, case["kv_heads"], d)
    return q.view(t, -1), _exact_store(st, k[:n]), _exact_store(st, v), None, None
