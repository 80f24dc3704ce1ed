"""Calls that the documentation of the operators allows and that only a C caller,
or an unusual one, makes, on the GPU against the 64-bit oracle."""

import pytest
import torch

from cscr import _lib
from cscr import attention as A
from cscr._lib import DTYPE_CODE
from oracle import quant_oracle as Q
from test_gpu_scored_attention import Case

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def short(p):
    return str(p).replace("torch.", "") if isinstance(p, torch.dtype) else None


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.device_status()
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,kind", [(BF16, E4M3), (F16, INT8), (BF16, BF16), (F16, F16)],
                         ids=short)
def test_outputs_off_by_an_element_through_the_c_abi(dtype, kind):
    """An `out` aligned to its elements only, for both attention entry points."""
    c = Case([70, 1, 300], 16, 2, 128, 16, dtype, kind, seed=21)
    S, H, D = c.q.shape
    buf = torch.full((S * H * D + 2,), 7.0, dtype=dtype, device="cuda")
    out = buf[1:-1].view(S, H, D)
    scales = (c.ks.data_ptr(), c.vs.data_ptr()) if c.ks is not None else (0, 0)
    _lib.launch(_lib.SCORED_ATTENTION, 0, out.data_ptr(), c.q.data_ptr(), c.k.data_ptr(),
                c.v.data_ptr(), *scales, c.tables.data_ptr(), c.lens.data_ptr(), 0, 0, 0, S, H, 2,
                D, c.k.shape[0], 16, c.tables.shape[1], H * D, 0, DTYPE_CODE[dtype],
                DTYPE_CODE[kind], 0, c.scale, 0.0)
    c.check(out)
    if kind == dtype:
        out.zero_()
        _lib.check(_lib.load().tlb_paged_attention(
            out.data_ptr(), c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.tables.data_ptr(),
            c.lens.data_ptr(), S, H, 2, D, c.k.shape[0], 16, c.tables.shape[1], c.scale,
            DTYPE_CODE[dtype], None, 0, 0, _lib.stream_of(out.device)))
        ref = Q.attention(c.q, c.k, c.v, None, None, c.tables, c.lens, c.scale)
        Q.assert_within(out, ref[0], Q.attention_bound(*ref, dtype, kind))
    assert bool((buf[0] == 7) & (buf[-1] == 7))
