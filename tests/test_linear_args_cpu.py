"""Argument checks of the 8-bit projection operators, without a GPU: the C ABI refuses
bad arguments before any CUDA call, and the op module refuses CPU tensors and wrong
shapes or types. The oracle's quantisers against torch's own conversion."""

import re

import pytest
import torch

from cscr import _lib
from cscr import linear as L
from conftest import REPO
from oracle import linear_oracle as O

HEADER = REPO / "include" / "tinyllama_b200.h"

P = 1 << 12  # stands in for an aligned device pointer; nothing is dereferenced
OK, BAD = 0, 1
F32, F16, BF16, I32 = range(4)
PLAIN, SILU, NORM = range(3)


def call(lib, entry, *fields):
    name, pack = entry
    return getattr(lib, name)(pack(*fields), None)


def test_struct_layouts_match_the_header(built_lib):
    text = HEADER.read_text()
    for name, (entry, pack) in (("quantize_rows", _lib.QUANTIZE_ROWS),
                                ("matmul_quantized", _lib.MATMUL_QUANTIZED)):
        body = re.search(r"struct tlb_%s_args \{(.*?)\}" % name, text, re.S).group(1)
        fields = sum(len(line.split(",")) for line in body.split(";") if line.strip())
        doubles = sum(len(line.split(",")) for line in body.split(";") if "double" in line)
        assert len(pack(*[0] * (fields - doubles), *[0.0] * doubles)) == 8 * fields
        assert getattr(_lib.load(), entry)(None, None) == BAD  # no struct at all


def rows(lib, out=P, scales=P, h=0, x=P, res=0, w=0, op=PLAIN, n=4, width=256, dtype=BF16,
         eps=1e-6):
    return call(lib, _lib.QUANTIZE_ROWS, out, scales, h, x, res, w, op, n, width, width, width,
                width, dtype, eps)


def test_rows_refuse_before_any_cuda_call(built_lib):
    lib = _lib.load()
    for kw, msg in ((dict(op=3), "unknown op"), (dict(op=-1), "unknown op"),
                    (dict(dtype=I32), "dtype must be"), (dict(n=-1), "num_rows"),
                    (dict(width=0), "width"), (dict(width=1 << 31), "range"),
                    (dict(w=P), "belong to the norm"), (dict(op=SILU, res=P, h=P), "belong"),
                    (dict(op=NORM, w=P, eps=-1.0), "eps"),
                    (dict(op=NORM, w=P, eps=float("nan")), "eps"),
                    (dict(op=NORM), "null"), (dict(op=NORM, w=P, res=P), "null"),
                    (dict(out=0), "null"), (dict(scales=0), "null"), (dict(x=0), "null"),
                    (dict(x=P + 1), "aligned"), (dict(op=NORM, w=P + 1), "aligned"),
                    (dict(op=NORM, w=P, res=P + 1, h=P), "aligned"),
                    (dict(op=NORM, w=P, res=P, h=P + 1), "aligned")):
        assert rows(lib, **kw) == BAD and msg in _lib.last_error(), kw
    assert rows(lib, n=0) == OK  # nothing to do, nothing launched


def product(lib, out=P, x=P, xs=P, w=P, ws=P, bias=0, t=4, k=256, n=64, dtype=BF16):
    return call(lib, _lib.MATMUL_QUANTIZED, out, x, xs, w, ws, bias, t, k, n, k, 2, k, 2, n, dtype)


def test_product_refuses_before_any_cuda_call(built_lib):
    lib = _lib.load()
    for kw, msg in ((dict(dtype=I32), "out dtype"), (dict(t=-1), "negative"),
                    (dict(n=-1), "negative"), (dict(k=0), "width"), (dict(t=1 << 31), "range"),
                    (dict(out=0), "null"), (dict(x=0), "null"),
                    (dict(xs=0), "null"), (dict(w=0), "null"), (dict(ws=0), "null"),
                    (dict(out=P + 1), "aligned"), (dict(bias=P + 1), "aligned")):
        assert product(lib, **kw) == BAD and msg in _lib.last_error(), kw
    assert product(lib, t=0) == OK and product(lib, n=0) == OK


def test_ops_refuse_cpu_tensors():
    x = torch.zeros(4, 256)
    for f in (lambda: L.quantize_rows(x), lambda: L.silu_and_mul_quantized(x),
              lambda: L.rms_norm_quantized(x, torch.ones(256), 1e-6)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            f()
    q, s = L.quantize_weight(torch.zeros(128, 256))
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        L.matmul_quantized(q[:4], s.expand(4, -1), q, s, torch.float16)
    with pytest.raises(RuntimeError, match="features, width"):
        L.quantize_weight(torch.zeros(128))
    with pytest.raises(RuntimeError, match="features, width"):
        L.quantize_weight(torch.zeros(4, 4, dtype=torch.int8))


class Fake:
    """A tensor's looks on device 0, for the checks that come before any launch."""

    def __init__(self, t, index=0):
        self.t, self.index = t, index

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.index


def fakes(t=4, k=256, n=200):
    q, s = L.quantize_weight(torch.zeros(n, k))
    x = torch.zeros(t, k).to(torch.float8_e4m3fn)
    xs = torch.full((t, -(-k // 128)), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return dict(x=x, x_scales=xs, weight=q, weight_scales=s, out_dtype=torch.bfloat16, bias=None)


def test_product_refusals_name_what_is_wrong():
    good = fakes()
    for change, msg in (
            (dict(x=good["x"].float()), "float8_e4m3fn"),
            (dict(x=good["x"][:, :128]), "features, width"),
            (dict(x=good["x"].view(torch.uint8).repeat(1, 2)[:, ::2].view(torch.float8_e4m3fn)),
             "contiguously"),
            (dict(x_scales=good["x_scales"][:3]), r"x_scales must be .* \[4, 2\]"),
            (dict(x_scales=good["x_scales"].view(torch.uint8)), "x_scales"),
            (dict(x_scales=good["x_scales"].view(torch.uint8).t().contiguous().t()
                  .view(torch.float8_e8m0fnu)), "x_scales"),
            (dict(weight_scales=good["weight_scales"][:1]), r"weight_scales must be .* \[2, 2\]"),
            (dict(out_dtype=torch.int8), "out_dtype"),
            (dict(bias=torch.zeros(200)), "bias"),
            (dict(bias=torch.zeros(100, dtype=torch.bfloat16)), "bias")):
        kw = {**good, **change}
        kw = {n: Fake(v) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
        with pytest.raises(RuntimeError, match=msg):
            L.matmul_quantized(**kw)
    kw = {n: Fake(v, i) if isinstance(v, torch.Tensor) else v
          for i, (n, v) in enumerate(good.items())}
    with pytest.raises(RuntimeError, match="same CUDA device"):
        L.matmul_quantized(**kw)


def test_row_refusals_name_what_is_wrong():
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.ones(256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="gate_up must hold as many"):
        L.silu_and_mul_quantized(Fake(x[:, :255]))
    for bad, msg in ((x.long(), "float16"), (x[0], "num_tokens, width"), (x[:, :0], "num_tokens"),
                     (x.t(), "contiguously")):
        with pytest.raises(RuntimeError, match=msg):
            L.quantize_rows(Fake(bad))
    for kw, msg in ((dict(weight=w[:128]), "weight"), (dict(weight=w.float()), "weight"),
                    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                    (dict(residual=Fake(x[:2])), "residual must"),
                    (dict(residual=Fake(x.float())), "residual must"),
                    (dict(residual=Fake(x, 1)), "residual must"),
                    (dict(residual_out=Fake(x)), "belongs to residual"),
                    (dict(residual=Fake(x), residual_out=Fake(x[:1].expand(4, -1))), "overlap")):
        kw = {"weight": w, "eps": 1e-6, **kw}
        kw["weight"] = Fake(kw["weight"])
        with pytest.raises(RuntimeError, match=msg):
            L.rms_norm_quantized(Fake(x), **kw)


def test_oracle_rounds_as_torch_converts():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 300, generator=g) * torch.exp(4 * torch.randn(40, 1, generator=g))
    q, s = O.quantize_rows(x)
    back = (O.groups(x.double()) / O.scale_of(s).unsqueeze(-1)).flatten(1)[:, :300]
    assert torch.equal(back.float().to(torch.float8_e4m3fn).view(torch.uint8), q.view(torch.uint8))
    top = O.groups(x).abs().amax(-1).double()
    assert bool((top <= 448 * O.scale_of(s)).all() and (top > 224 * O.scale_of(s)).all())
    w = 0.05 * torch.randn(200, 300, generator=g)
    w[128:, :128] = 0
    for a, b in zip(L.quantize_weight(w), O.quantize_weight(w)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
