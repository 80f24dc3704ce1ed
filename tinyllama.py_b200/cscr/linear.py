"""cscr.linear — projections in 8 bits (not in the reference).

Activations and weights are float8_e4m3fn with power-of-two scales, the format of
the 8-bit caches: a row of activations [T, K] has one float8_e8m0fnu scale for each
128 of its values (``[T, ceil(K / 128)]``; the last group may be shorter), a weight
[N, K] one for each block of 128 x 128 (``[ceil(N / 128), ceil(K / 128)]``). A scale
is the smallest power of two 2^E with ``max|x| <= 448 * 2^E`` over the finite values
of its group (E in [-126, 127]); the values are ``x / 2^E`` rounded to nearest even,
infinities saturated, NaN kept.

* ``rms_norm_quantized``, ``silu_and_mul_quantized`` and ``quantize_rows`` make such
  rows; ``quantize_weight`` makes such weights (once, when a model is loaded).
* ``matmul_quantized`` multiplies them.

``paged_decode.layers.QuantizedLinear`` and ``QuantizedDecoderLayer`` run them
around the attention ops.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import DTYPE_CODE, torch_check

_FLOAT_TYPES = (torch.float16, torch.bfloat16, torch.float32)
GROUP = 128  # values that share a scale
_PLAIN, _SILU_AND_MUL, _RMS_NORM = 0, 1, 2


def _rows_out(x: torch.Tensor, rows: int, width: int) -> tuple[torch.Tensor, torch.Tensor]:
    return (x.new_empty((rows, width), dtype=torch.float8_e4m3fn),
            x.new_empty((rows, -(-width // GROUP)), dtype=torch.float8_e8m0fnu))


def _check_rows(x: torch.Tensor, name: str) -> int:
    """x is [T, K] with contiguous rows; returns its device index."""
    index = x.get_device()
    torch_check(index >= 0, f"{name} must be a CUDA tensor")
    torch_check(x.dtype in _FLOAT_TYPES, f"{name} must be float16, bfloat16 or float32")
    torch_check(x.dim() == 2 and x.size(1) > 0, f"{name} must be [num_tokens, width]")
    torch_check(x.stride(1) == 1 or x.size(1) == 1, f"{name} must hold each row contiguously")
    return index


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, eps: float,
                       residual: torch.Tensor | None = None, *,
                       residual_out: torch.Tensor | None = None
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """RMS norm with the residual's addition and an output in 8 bits.

    ``h = x`` or, with ``residual``, ``x + residual`` rounded to their dtype;
    ``h * rsqrt(mean(h^2) + eps) * weight`` in fp32, then quantised by groups of 128.
    x and residual [T, K] in float16, bfloat16 or float32 (one type), rows possibly
    strided; weight [K] of that type. Returns (values [T, K] float8_e4m3fn, scales
    [T, ceil(K / 128)] float8_e8m0fnu, h or None): h goes to ``residual_out``, which
    may be ``residual`` or ``x`` itself, or a tensor that shares no memory with the inputs.
    """
    if _lib.fast is not None:
        out = _lib.fast.rows(x, _RMS_NORM, weight, eps, residual, residual_out)
        if out is not None:
            return out
    index = _check_rows(x, "x")
    rows, width = x.shape
    dtype = x.dtype
    torch_check(weight.shape == (width,) and weight.dtype == dtype and weight.is_contiguous()
                and weight.get_device() == index,
                "weight must be a contiguous [width] tensor of x's dtype and device")
    torch_check(eps >= 0, "eps must not be negative")
    strides, pointers = (0, 0), (0, 0)
    torch_check(residual_out is None or residual is not None, "residual_out belongs to residual")
    for t, name in ((residual, "residual"), (residual_out, "residual_out")):
        torch_check(t is None or (t.shape == x.shape and t.dtype == dtype
                                  and t.get_device() == index
                                  and (t.stride(1) == 1 or width == 1)),
                    f"{name} must have x's shape, dtype and device, with contiguous rows")
    if residual is not None:
        if residual_out is None:
            residual_out = x.new_empty((rows, width))
        torch_check(rows < 2 or residual_out.stride(0) >= width, "residual_out's rows overlap")
        strides = residual.stride(0), residual_out.stride(0)
        pointers = residual.data_ptr(), residual_out.data_ptr()
    q, scales = _rows_out(x, rows, width)
    if rows:
        _lib.launch(_lib.QUANTIZE_ROWS, index, q.data_ptr(), scales.data_ptr(), pointers[1],
                    x.data_ptr(), pointers[0], weight.data_ptr(), _RMS_NORM, rows, width,
                    x.stride(0), *strides, DTYPE_CODE[dtype], eps)
    return q, scales, residual_out


def silu_and_mul_quantized(gate_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``gate / (1 + exp(-gate)) * up`` in 8 bits: gate_up [T, 2 K] holds each token's
    gate values, then its up values (float16, bfloat16 or float32, rows possibly
    strided). Returns (values [T, K], scales [T, ceil(K / 128)]); fp32 math, one
    rounding: gates below -88.7, whose ``exp(-gate)`` is infinite in fp32, give 0
    (NaN where up is infinite), and results below 2^-126 in magnitude may count as 0."""
    if _lib.fast is not None:
        out = _lib.fast.rows(gate_up, _SILU_AND_MUL, None, 0.0, None, None)
        if out is not None:
            return out
    index = _check_rows(gate_up, "gate_up")
    rows, both = gate_up.shape
    torch_check(both % 2 == 0, "gate_up must hold as many gate as up values")
    q, scales = _rows_out(gate_up, rows, both // 2)
    if rows:
        _lib.launch(_lib.QUANTIZE_ROWS, index, q.data_ptr(), scales.data_ptr(), 0,
                    gate_up.data_ptr(), 0, 0, _SILU_AND_MUL, rows, both // 2, gate_up.stride(0),
                    0, 0, DTYPE_CODE[gate_up.dtype], 0.0)
    return q, scales


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows of x [T, K] (float16, bfloat16 or float32, rows possibly strided) in 8
    bits: (values [T, K], scales [T, ceil(K / 128)])."""
    if _lib.fast is not None:
        out = _lib.fast.rows(x, _PLAIN, None, 0.0, None, None)
        if out is not None:
            return out
    index = _check_rows(x, "x")
    rows, width = x.shape
    q, scales = _rows_out(x, rows, width)
    if rows:
        _lib.launch(_lib.QUANTIZE_ROWS, index, q.data_ptr(), scales.data_ptr(), 0, x.data_ptr(),
                    0, 0, _PLAIN, rows, width, x.stride(0), 0, 0, DTYPE_CODE[x.dtype], 0.0)
    return q, scales


@torch.no_grad()
def quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A weight [N, K] of finite values in 8 bits, with a scale for each block of
    128 x 128: (values [N, K], scales [ceil(N / 128), ceil(K / 128)]). Plain torch, on
    the weight's device, without gradients: a model's weights are converted once."""
    torch_check(weight.dim() == 2 and weight.dtype in _FLOAT_TYPES,
                "weight must be [features, width] in float16, bfloat16 or float32")
    n, k = weight.shape
    cols = -(-k // GROUP)
    values = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=weight.device)
    scale_bytes = torch.empty((-(-n // GROUP), cols), dtype=torch.uint8, device=weight.device)
    scales = scale_bytes.view(torch.float8_e8m0fnu)
    for i in range(scales.size(0)):  # a row of blocks at a time: little memory beside the weight
        rows = weight[i * GROUP:(i + 1) * GROUP].float()
        blocks = torch.nn.functional.pad(rows, (0, cols * GROUP - k)).view(-1, cols, GROUP)
        top = blocks.abs().amax((0, 2))
        mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent; 448 = 0.875 * 2^9
        exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9)
        exponent = torch.where(top == 0, -126, exponent).clamp(-126, 127)
        scale_bytes[i] = (exponent + 127).to(torch.uint8)
        blocks = (blocks / scales[i].float().view(1, cols, 1)).view(-1, cols * GROUP)[:, :k]
        values[i * GROUP:(i + 1) * GROUP] = blocks.to(torch.float8_e4m3fn)
    return values, scales


def _check_product(x, x_scales, weight, weight_scales, out_dtype, bias):
    """The checks of ``matmul_quantized`` one by one, for their messages."""
    index = x.get_device()
    torch_check(index >= 0, "x must be a CUDA tensor")
    torch_check(x_scales.get_device() == index and weight.get_device() == index
                and weight_scales.get_device() == index
                and (bias is None or bias.get_device() == index),
                "all tensors must be on the same CUDA device")
    torch_check(x.dtype == torch.float8_e4m3fn and weight.dtype == torch.float8_e4m3fn,
                "x and weight must be float8_e4m3fn")
    torch_check(x.dim() == 2 and weight.dim() == 2 and x.size(1) == weight.size(1)
                and x.size(1) > 0,
                "x must be [num_tokens, width] and weight [features, width]")
    torch_check((x.stride(1) == 1 and weight.stride(1) == 1) or x.size(1) == 1,
                "x and weight must hold each row contiguously")
    groups = -(-x.size(1) // GROUP)
    for s, rows, name in ((x_scales, x.size(0), "x_scales"),
                          (weight_scales, -(-weight.size(0) // GROUP), "weight_scales")):
        torch_check(s.dtype == torch.float8_e8m0fnu and s.shape == (rows, groups)
                    and (groups == 1 or s.stride(1) == 1),
                    f"{name} must be a float8_e8m0fnu tensor [{rows}, {groups}] with contiguous "
                    "rows")
    torch_check(out_dtype in _FLOAT_TYPES, "out_dtype must be float16, bfloat16 or float32")
    torch_check(bias is None or (bias.dtype == out_dtype and bias.shape == weight.shape[:1]
                                 and bias.is_contiguous()),
                "bias must be a contiguous [features] tensor of out_dtype")
    raise RuntimeError("matmul_quantized: unsupported arguments")


def matmul_quantized(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor,
                     weight_scales: torch.Tensor, out_dtype: torch.dtype,
                     bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` of 8-bit rows and weights -> [T, N] of ``out_dtype``.

    x [T, K] float8_e4m3fn with x_scales [T, ceil(K / 128)], weight [N, K] with
    weight_scales [ceil(N / 128), ceil(K / 128)] (float8_e8m0fnu), bias [N] of
    ``out_dtype`` (float16, bfloat16 or float32). Sums in fp32, one rounding; their order
    goes with sizes and alignment, so a token's bits may differ between calls with other
    numbers of tokens, not between calls that are alike. Rows of any operand may be
    strided; x and weight rows on 16-byte boundaries take the tensor cores, others a
    slower kernel.

    Any scales may meet: sums past fp32 are infinite (NaN where both signs meet), those
    below 2^-126 (of a group of 128, or of all) may count as 0.
    """
    if _lib.fast is not None:
        out = _lib.fast.product(x, x_scales, weight, weight_scales, out_dtype, bias)
        if out is not None:
            return out
    index, shape, wshape = x.get_device(), x.shape, weight.shape
    sshape, wsshape = x_scales.shape, weight_scales.shape
    if not (index >= 0 and len(shape) == 2 and len(wshape) == 2 and len(sshape) == 2
            and len(wsshape) == 2 and shape[1] == wshape[1] and shape[1] > 0
            and x.dtype == torch.float8_e4m3fn and weight.dtype == torch.float8_e4m3fn
            and x_scales.dtype == torch.float8_e8m0fnu
            and weight_scales.dtype == torch.float8_e8m0fnu
            and (shape[1] == 1 or (x.stride(1) == 1 and weight.stride(1) == 1))
            and sshape[0] == shape[0] and sshape[1] == wsshape[1] == -(-shape[1] // GROUP)
            and wsshape[0] == -(-wshape[0] // GROUP)
            and (sshape[1] == 1 or (x_scales.stride(1) == 1 and weight_scales.stride(1) == 1))
            and weight.get_device() == index and x_scales.get_device() == index
            and weight_scales.get_device() == index and out_dtype in _FLOAT_TYPES
            and (bias is None or (bias.dtype == out_dtype and bias.shape == wshape[:1]
                                  and bias.is_contiguous() and bias.get_device() == index))):
        _check_product(x, x_scales, weight, weight_scales, out_dtype, bias)
    out = x.new_empty((shape[0], wshape[0]), dtype=out_dtype)
    if out.numel():
        _lib.launch(_lib.MATMUL_QUANTIZED, index, out.data_ptr(), x.data_ptr(),
                    x_scales.data_ptr(), weight.data_ptr(), weight_scales.data_ptr(),
                    0 if bias is None else bias.data_ptr(), shape[0], shape[1], wshape[0],
                    x.stride(0), x_scales.stride(0), weight.stride(0), weight_scales.stride(0),
                    wshape[0], DTYPE_CODE[out_dtype])
    return out
