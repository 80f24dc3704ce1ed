"""The cases and plain forms by which the 8-bit projection operators are measured:
the RMS norm with the residual's addition, the gated activation and plain rows, each
with its output in 8 bits, and the product of such rows with 8-bit weights.

``run`` computes a case either with the framework's kernels (``own = True``: the
calls a user makes of ``cscr.linear``) or in plain form (elementary torch operations
in 32 bits, rounded once at the end). ``exact`` gives the same results from the
definitions in 64 bits.

8-bit rows are ``float8_e4m3fn`` [T, K] with a power-of-two scale, held as
``float8_e8m0fnu``, for each 128 values of a row (the last group of a row may be
shorter): the smallest 2^E with max|x| <= 448 * 2^E, E in [-126, 127]. 8-bit weights
are ``float8_e4m3fn`` [N, K] with such a scale for each block of 128 x 128.
"""

import math
import os
import sys

import torch

own = False

GROUP = 128
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}

_ops = None


def _own_ops():
    """The framework's op module (only when ``own``)."""
    global _ops
    if _ops is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                           "tinyllama.py_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from cscr import linear

        _ops = linear
    return _ops


# ------------------------------------------------------------------- cases

def _norm(name, dtype, tokens, width, residual=True):
    return {"op": "norm", "name": name, "dtype": dtype, "tokens": tokens, "width": width,
            "residual": residual}


def _silu(name, dtype, tokens, width):
    return {"op": "silu", "name": name, "dtype": dtype, "tokens": tokens, "width": width}


def _rows(name, dtype, tokens, width):
    return {"op": "rows", "name": name, "dtype": dtype, "tokens": tokens, "width": width}


def _product(name, dtype, tokens, width, features, bias=False):
    return {"op": "product", "name": name, "dtype": dtype, "tokens": tokens, "width": width,
            "features": features, "bias": bias}


def listed():
    return [
        # the norm before a projection in the decode step that the benchmark times
        _norm("n_step", "bfloat16", 64, 2048),
        # the first norm of a packed prompt step on the small model's width (14 heads of 64)
        _norm("n_packed", "float16", 4853, 896, residual=False),
        # a long prompt of a wide model
        _norm("n_prompt", "bfloat16", 16383, 4096),
        # a decode step's gated activation
        _silu("s_step", "bfloat16", 64, 8192),
        # a packed prompt step's
        _silu("s_packed", "float16", 4853, 5632),
        # a decode step's attention output, before the output projection
        _rows("r_step", "bfloat16", 64, 2048),
        # a long prompt's, 32 heads of 128
        _rows("r_prompt", "float16", 16381, 4096),
        # one conversation on the small model: the call is launch and latency
        _product("m_one", "float16", 1, 896, 1152, bias=True),
        # the query, key and value projection of the benchmark's decode step
        _product("m_step_qkv", "bfloat16", 64, 2048, 2560, bias=True),
        # its gate and up projections: the weights' stream
        _product("m_step_gate_up", "bfloat16", 64, 2048, 16384),
        # a packed prompt step on the small model, groups of scales not a multiple of 4
        _product("m_packed", "float16", 4853, 896, 9728),
        # a long prompt of a wide model: the tensor cores
        _product("m_prompt", "bfloat16", 16384, 4096, 8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "silu", "rows", "product", "product", "product"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "product":
        width = 16 * _log_int(rng, 4, 512)
        features = _log_int(rng, 64, 16384)
        # at most the largest listed case's operations
        most = min(16384, 500_000_000_000 // (2 * width * features))
        return _product("", dtype, _log_int(rng, 1, max(1, most)), width, features,
                        rng.random() < 0.5)
    width = _log_int(rng, 64, 16384)
    if rng.random() < 0.7:  # most widths are whole groups
        width = max(1, width // GROUP) * GROUP
    tokens = _log_int(rng, 1, max(1, min(16384, 48_000_000 // width)))
    if op == "norm":
        return _norm("", rng.choice([dtype, "bfloat16", "float32"]), tokens, width,
                     rng.random() < 0.7)
    return (_silu if op == "silu" else _rows)("", dtype, tokens, width)


# ------------------------------------------------------------------ inputs

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, tokens, width, dtype):
    """Rows as a model's layers give them: magnitudes by token, some channels far off."""
    channel = torch.exp(0.7 * _normal(g, 1, width))
    token = torch.exp(0.5 * _normal(g, tokens, 1))
    return (_normal(g, tokens, width) * channel * token).to(dtype)


def _power(e):
    """2^e as a scale, for whole e in [-126, 127]."""
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _exponent(top):
    """The smallest whole e with top <= 448 * 2^e, in [-126, 127] (32 bits)."""
    m, e = torch.frexp(top)
    return torch.where(m > 0.875, e - 8, e - 9).clamp(-126, 127)


def _groups(x):
    """[T, K] -> [T, groups, 128], the last group filled up with zeros."""
    t, k = x.shape
    n = -(-k // GROUP)
    if n * GROUP != k:
        x = torch.nn.functional.pad(x, (0, n * GROUP - k))
    return x.view(t, n, GROUP)


def _quantize(x):
    """Rows of 32-bit values -> (8-bit values, scale of each group)."""
    x, k = _groups(x), x.shape[1]
    scale = _power(_exponent(x.abs().amax(-1)))
    q = (x / scale.float().unsqueeze(-1)).to(torch.float8_e4m3fn)
    q = q.view(torch.uint8).flatten(1)[:, :k].contiguous().view(torch.float8_e4m3fn)
    return q, scale


def _quantize_weight(w):
    """32-bit weights [N, K] -> (8-bit values, scale of each block of 128 x 128)."""
    n, k = w.shape
    rows, cols = -(-n // GROUP), -(-k // GROUP)
    b = torch.nn.functional.pad(w, (0, cols * GROUP - k, 0, rows * GROUP - n))
    b = b.view(rows, GROUP, cols, GROUP)
    scale = _power(_exponent(b.abs().amax((1, 3))))
    q = (b / scale.float().view(rows, 1, cols, 1)).reshape(rows * GROUP, cols * GROUP)
    return q[:n, :k].to(torch.float8_e4m3fn).contiguous(), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 31)
    dtype, t, k = DTYPES[case["dtype"]], case["tokens"], case["width"]
    st = {"case": case, "eps": 1e-6}
    if case["op"] == "product":
        n = case["features"]
        st["x"], st["xs"] = _quantize(_activations(g, t, k, dtype).float())
        st["w"], st["ws"] = _quantize_weight(_normal(g, n, k) * (k ** -0.5))
        st["bias"] = (0.3 * _normal(g, n)).to(dtype) if case["bias"] else None
        return st
    if case["op"] == "silu":  # gate and up parts of one projection's rows
        st["x"] = (1.5 * _normal(g, t, 2 * k)
                   * torch.exp(0.3 * _normal(g, t, 1))).to(dtype)
        return st
    st["x"] = _activations(g, t, k, dtype)
    if case["op"] == "norm":
        st["weight"] = (1 + 0.2 * _normal(g, k)).to(dtype)
        st["residual"] = (2 * _activations(g, t, k, torch.float32)).to(dtype) \
            if case["residual"] else None
    return st


# -------------------------------------------------------------- plain forms

def _dense(q, scale):
    """The values that 8-bit rows stand for, in 32 bits."""
    return (_groups(q.float()) * scale.float().unsqueeze(-1)).flatten(1)[:, :q.shape[1]]


def _dense_weight(q, scale):
    n, k = q.shape
    s = scale.float().repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    return q.float() * s


def _plain(st):
    op, x = st["case"]["op"], st["x"]
    if op == "product":
        y = torch.matmul(_dense(x, st["xs"]), _dense_weight(st["w"], st["ws"]).t())
        if st["bias"] is not None:
            y = y + st["bias"].float()
        return y.to(DTYPES[st["case"]["dtype"]])
    if op == "rows":
        return _quantize(x.float())
    if op == "silu":
        gate, up = x.float().chunk(2, -1)
        return _quantize(gate / (1 + torch.exp(-gate)) * up)
    h = x if st["residual"] is None else (x.float() + st["residual"].float()).to(x.dtype)
    y = h.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"]) * st["weight"].float()
    return (*_quantize(y), None if st["residual"] is None else h)


def _own(st):
    linear, op = _own_ops(), st["case"]["op"]
    if op == "product":
        return linear.matmul_quantized(st["x"], st["xs"], st["w"], st["ws"],
                                       DTYPES[st["case"]["dtype"]], st["bias"])
    if op == "rows":
        return linear.quantize_rows(st["x"])
    if op == "silu":
        return linear.silu_and_mul_quantized(st["x"])
    return linear.rms_norm_quantized(st["x"], st["weight"], st["eps"], st["residual"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------- work

def work(case):
    e, t, k = SIZES[case["dtype"]], case["tokens"], case["width"]
    groups = -(-k // GROUP)
    row = k + groups  # an 8-bit row and its scales
    if case["op"] == "product":
        n = case["features"]
        moved = t * row + n * k + groups * -(-n // GROUP) + t * n * e
        return {"bytes": moved + (n * e if case["bias"] else 0), "flops": 2 * t * n * k}
    if case["op"] == "norm":
        both = 3 if case["residual"] else 1  # x alone, or x and the residual read, the sum written
        return {"bytes": t * (both * k * e + row) + k * e, "flops": 6 * t * k}
    if case["op"] == "silu":
        return {"bytes": t * (2 * k * e + row), "flops": 8 * t * k}
    return {"bytes": t * (k * e + row), "flops": 3 * t * k}


# ------------------------------------------------------------------- exact

def _power64(e):
    """2^e exactly, for whole e of a normal result."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_quantize(x):
    """From the definition: the smallest power of two, then the nearest value of the type."""
    t, k = x.shape
    n = -(-k // GROUP)
    y = torch.zeros(t, n * GROUP, dtype=torch.float64, device=x.device)
    y[:, :k] = x
    y = y.view(t, n, GROUP)
    top = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448.0)).nan_to_num(neginf=-126.0).clamp(-200, 200)
    e = torch.where(_power64(e) * 448.0 < top, e + 1, e)
    e = torch.where(_power64(e - 1) * 448.0 >= top, e - 1, e).clamp(-126, 127)
    y = y / _power64(e)
    # spacing of e4m3 at |y|: 2^(floor(log2|y|) - 3), 2^-9 below 2^-6
    step = _power64(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    y = (torch.round(y / step) * step).view(t, -1)[:, :k]
    return y, _power64(e.squeeze(-1))


def exact(case, seed):
    st = prepare(case, seed)
    x = st["x"].double()
    k = case["width"]
    if case["op"] == "product":
        s = _power64(st["xs"].view(torch.uint8).long() - 127)
        x = x * s.repeat_interleave(GROUP, 1)[:, :k]
        out = []
        for at in range(0, case["features"], GROUP):  # a row of weight blocks at a time
            w = st["w"][at:at + GROUP].double()
            sw = _power64(st["ws"][at // GROUP].view(torch.uint8).long() - 127)
            out.append(x @ (w * sw.repeat_interleave(GROUP)[:k]).t())
        y = torch.cat(out, 1)
        return y if st["bias"] is None else y + st["bias"].double()
    if case["op"] == "rows":
        return _exact_quantize(x)
    if case["op"] == "silu":
        return _exact_quantize(x[:, :k] * torch.sigmoid(x[:, :k]) * x[:, k:])
    h = x if st["residual"] is None else (x + st["residual"].double()).to(st["x"].dtype).double()
    y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / k + st["eps"]) * st["weight"].double()
    return (*_exact_quantize(y), None if st["residual"] is None else h)
