"""(h) Products with weights held in 8-bit integers, with a scale for each row and channel, on the GPU (HIP kernels).

``quantize_rows(x)``: each row of a float32 or bfloat16 matrix as 8-bit integers with one float32 scale,

    scale = max |x| (1 / 127),  value = x / scale rounded to the nearest integer (ties to even)

(product, quotient and 1 / 127 in float32). ``linear_int8(x, weight, bias=None)``: ``linear`` on a weight [out, in] so rounded,

    y[m, n] = x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] + bias[n]

with the rows of x rounded on the way, or given as ``Int8Rows``. The sums are exact (32-bit integers on the matrix cores),
scales and bias are applied in float64, and each result is rounded to float32 and, where asked, from there to bfloat16. A row of
zeros has the scale 0; one that holds a value that is not finite gives NaN. For evaluation: there are no gradients, and inputs that
need them (x, scales, the bias) are refused.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch import Tensor

from fastmd_amd import _abi
from fastmd_amd._autograd import differentiated
from fastmd_amd._device import on_device_of, require_cuda, rows_view, stream

MAX_WIDTH = 131071  # 2^17 products of -128 and -128, which given values may hold, would overflow 32 bits
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


class Int8Rows(NamedTuple):
    """A matrix [rows, width] as 8-bit integers with a scale for each row: ``values * scales[:, None]``."""

    values: Tensor  # int8 [rows, width]
    scales: Tensor  # float32 [rows]

    def dense(self) -> Tensor:
        """The values that it stands for, float32."""
        return self.values.float() * self.scales[:, None]


def quantize_rows(x: Tensor) -> Int8Rows:
    """The rows of ``x`` [rows, width] (float32 or bfloat16) as ``Int8Rows``. The values' rows start on 16 bytes, so that
    ``linear_int8`` reads them in place."""
    require_cuda(x)
    if x.dim() != 2 or x.dtype not in _TYPES:
        raise ValueError(f"quantize_rows takes a float32 or bfloat16 matrix, got {x.dtype} {tuple(x.shape)}")
    if differentiated(x):
        raise ValueError("quantize_rows has no gradient: detach its input")
    rows, width = x.shape
    if width < 1:
        raise ValueError("quantize_rows takes at least one column")
    ld = -(-width // 16) * 16
    values = torch.empty((rows, ld), dtype=torch.int8, device=x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    x, x_ld = rows_view(x)
    with on_device_of(x):
        _abi.call("fmd_quantize_rows", _TYPES[x.dtype], x.data_ptr(), x_ld, rows, width, values.data_ptr(), ld,
                  scales.data_ptr(), stream())
    return Int8Rows(values[:, :width], scales)


def _in_place(values: Tensor, padded: bool) -> tuple[Tensor, int]:
    """(values, row stride in bytes) of rows on 16 bytes that can be read to the width's last 16 bytes, and, with ``padded``,
    are zero from the width on; a copy where they do not lie so."""
    rows, width = values.shape
    whole = -(-width // 16) * 16
    ld = values.stride(0) if rows > 1 else whole
    if ((values.stride(1) == 1 or width == 1) and ld % 16 == 0 and whole <= ld <= 2 ** 23 and values.data_ptr() % 16 == 0
            and (whole == width or (not padded and values.untyped_storage().nbytes()
                                    >= values.storage_offset() + (rows - 1) * ld + whole))):
        return values, ld
    out = torch.zeros((rows, whole), dtype=torch.int8, device=values.device)
    out[:, :width] = values
    return out, whole


@functools.lru_cache(maxsize=256)
def _work_size(*sizes: int) -> int:
    return _abi.load().fmd_linear_int8_work_size(*sizes)


def _check_rows(name: str, q: Int8Rows) -> None:
    if (q.values.dim() != 2 or q.values.dtype != torch.int8 or q.scales.shape != q.values.shape[:1]
            or q.scales.dtype != torch.float32):
        raise ValueError(f"{name} must be int8 [rows, width] with float32 scales [rows], got {q.values.dtype} "
                         f"{tuple(q.values.shape)} and {q.scales.dtype} {tuple(q.scales.shape)}")


def linear_int8(x: Tensor | Int8Rows, weight: Int8Rows, bias: Tensor | None = None, *, dtype: torch.dtype | None = None) -> Tensor:
    """``x weight^T + bias`` in 8 bits (see the module): ``x`` [rows, width] float32 or bfloat16, or ``Int8Rows``;
    ``weight`` [out, width] (``quantize_rows`` of it, once); ``bias`` float32 [out]; ``dtype`` of the result: x's, float32 for
    ``Int8Rows``. 8-bit values whose rows do not start on 16 bytes, or cannot be read to the width's next multiple of 16, are copied by
    every call (``quantize_rows`` lays a weight out so that they are not; of ``x``, widths that are multiples of 16 only)."""
    if not isinstance(weight, Int8Rows):
        raise ValueError("weight must be Int8Rows (quantize_rows)")
    _check_rows("weight", weight)
    rounded = isinstance(x, Int8Rows)
    if differentiated(x.scales if rounded else x, weight.scales, bias):
        raise ValueError("linear_int8 has no gradient: detach its inputs")
    if rounded:
        _check_rows("x", x)
        values, kind = x.values, torch.float32 if dtype is None else dtype
        require_cuda(values, x.scales, weight.values, weight.scales, bias)
    else:
        values, kind = x, x.dtype if dtype is None else dtype
        require_cuda(x, weight.values, weight.scales, bias)
        if x.dim() != 2 or x.dtype not in _TYPES:
            raise ValueError(f"x must be a float32 or bfloat16 matrix, or Int8Rows, got {x.dtype} {tuple(x.shape)}")
    if kind not in _TYPES:
        raise ValueError(f"the result must be float32 or bfloat16, got {kind}")
    (rows, width), out, device = values.shape, weight.values.shape[0], values.device
    if weight.values.shape[1] != width or not 1 <= width <= MAX_WIDTH:
        raise ValueError(f"x and weight must have one width, from 1 to {MAX_WIDTH}, got {width} and {weight.values.shape[1]}")
    if rows >= 2 ** 29 or out >= 2 ** 29 or rows * out >= 2 ** 36:
        raise ValueError(f"linear_int8 takes fewer than 2^29 rows and channels, and 2^36 results, got {rows} and {out}")
    if bias is not None:
        if bias.shape != (out,) or bias.dtype != torch.float32:
            raise ValueError(f"bias must be float32 [{out}], got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    y = torch.empty((rows, out), dtype=kind, device=device)
    if rows == 0 or out == 0:
        return y
    w, w_ld = _in_place(weight.values, False)
    w_scales = weight.scales.contiguous()
    size = _work_size(1 if rounded else 0, rows, width, out)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    rest = (_TYPES[kind], w.data_ptr(), w_ld, w_scales.data_ptr(), _abi.ptr(bias), rows, width, out, y.data_ptr(), _abi.ptr(work))
    with on_device_of(y):
        if rounded:
            # past the width one of the two has to be zero: rows that the call rounds itself are
            values, x_ld = _in_place(values, True)
            scales = x.scales.contiguous()
            _abi.call("fmd_linear_int8", rest[0], values.data_ptr(), x_ld, scales.data_ptr(), *rest[1:], stream())
        else:
            values, x_ld = rows_view(values)
            _abi.call("fmd_linear_int8_rows", _TYPES[x.dtype], values.data_ptr(), x_ld, *rest, stream())
    return y
