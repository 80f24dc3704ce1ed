"""The 8-bit projection operators where no GPU is needed: outputs over inputs are refused,
weights are converted without a graph."""

import itertools

import pytest
import torch

from cscr import _lib
from cscr import linear as L

P = 1 << 20  # stands in for an aligned device pointer; nothing is dereferenced
BAD, BF16, NORM = 1, 2, 2
WEIGHT = 1 << 30  # far from the rows

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="calls that are taken would be "
                            "launched, on addresses that stand for none")


def norm(lib, x, residual, out, rows=4, width=8, weight=WEIGHT):
    """(pointer, stride in elements) of each; the status of the call."""
    name, pack = _lib.QUANTIZE_ROWS
    return getattr(lib, name)(pack(P << 12, P << 13, out[0], x[0], residual[0], weight, NORM, rows,
                                   width, x[1], residual[1], out[1], BF16, 1e-6), None)


def test_residual_out_over_other_rows_of_the_inputs_is_refused(built_lib):
    lib, far = _lib.load(), P << 8
    for out, why in (((P + 16, 8), "the next row"), ((P + 2, 8), "an element further"),
                     ((P, 16), "the rows' begin, other strides"), ((P - 16, 8), "the row before"),
                     ((P + 48, 8), "the last row"), ((P + 2, 12), "other strides")):
        for x, residual in (((P, 8), (far, 8)), ((far, 8), (P, 8))):
            assert norm(lib, x, residual, out) == BAD, why
            assert "share no memory" in _lib.last_error()
    assert norm(lib, (P, 8), (far, 8), (far, 8), weight=far + 32) == BAD
    assert norm(lib, (P, 0), (far, 8), (P, 8)) == BAD  # one row for all tokens
    assert norm(lib, (P, 8), (far, 8), (P << 9, 7)) == BAD and "overlap" in _lib.last_error()


@no_gpu
def test_residual_out_beside_the_inputs_is_taken(built_lib):
    """Past the checks the call asks for the device: it is refused nowhere as an argument."""
    lib, far = _lib.load(), P << 8
    for x, residual, out, rows in (
            ((P, 8), (far, 8), (P, 8), 4), ((P, 8), (far, 8), (far, 8), 4),
            ((P, 8), (P, 8), (P, 8), 4), ((P, 24), (P + 16, 24), (P + 32, 24), 4),
            ((P, 24), (P + 16, 24), (P + 16, 24), 4), ((P, 8), (far, 8), (P + 64, 8), 4),
            ((P, 8), (far, 8), (P - 64, 8), 4), ((P, 0), (far, 8), (P + 16, 8), 4),
            ((P, 8), (far, 8), (P, 16), 1), ((P, 16), (far, 8), (P + 16, 48), 2)):
        status = norm(lib, x, residual, out, rows)
        assert status not in (0, BAD), (x, residual, out, _lib.last_error())


@no_gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 5])
def test_refusals_are_those_of_rows_with_a_byte_in_common(built_lib, rows):
    """Against every row with every other, over small strides and distances."""
    lib, width, base = _lib.load(), 3, 1 << 24
    for a, b, away in itertools.product(range(0, 9), range(3, 9), range(-20, 21, 1)):
        # strides and distance in elements of two bytes
        out = [2 * away + 2 * b * r for r in range(rows)]
        ins = [2 * a * r for r in range(rows)]
        same = away == 0 and (rows == 1 or a == b)
        clash = not same and any(abs(i - o) < 2 * width for i in ins for o in out)
        got = norm(lib, (base, a), (P << 10, 8), (base + 2 * away, b), rows, width)
        assert (got == BAD) == clash, (a, b, away, _lib.last_error())


def test_product_rows_that_overlap_are_refused(built_lib):
    name, pack = _lib.MATMUL_QUANTIZED
    for stride in (0, 63, -63):
        call = pack(P, P << 1, P << 2, P << 3, P << 4, 0, 4, 256, 64, 256, 2, 256, 2, stride, BF16)
        assert getattr(_lib.load(), name)(call, None) == BAD
        assert "overlap" in _lib.last_error()


def test_weights_are_converted_without_gradients():
    """A parameter's values and scales hold no graph (with copies of its blocks in fp32)."""
    weight = torch.nn.Parameter(torch.randn(200, 300))
    values, scales = L.quantize_weight(weight)
    assert not values.requires_grad and values.grad_fn is None and not scales.requires_grad
    want = L.quantize_weight(weight.detach())
    for a, b in zip((values, scales), want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
