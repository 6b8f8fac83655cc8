"""(h) The gated feed-forward block on the GPU (HIP kernels), with a deterministic VJP.

``gated_feed_forward(x, w_gate, w_up, w_down, activation="silu")``:

    y = (act(x w_gate^T) * (x w_up^T)) w_down^T

on rows x [rows, width] with weights stored [out, in], as ``linear`` takes them. Both projections, the activation and the
product are one kernel: what the hidden layer holds is written once, after the product. ``activation``: "silu",
"gelu" (by erf), "relu" or None. The VJP gives the gradient of x alone (forces through a model whose weights
are fixed), of the weights, or of all.

float32 is computed on the bf16 matrix cores with every operand split into three planes (float32 accuracy; a value that is not
finite, or rounds to an infinite bfloat16, makes the results that it is a term of NaN), bfloat16 with products of bfloat16
operands. Sums are float32 in both, and so is the activation. For bfloat16 the hidden layer and, in the VJP, the
gradients of the two projections go into the next product as two bfloat16 parts (16 bits), so that each result carries the
error of one rounding, its own (an infinite value that they are multiplied by gives NaN). Gradients take no atomics: the same
call gives the same bits.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import Function

from fastmd_amd import _abi
from fastmd_amd._autograd import differentiated, first_derivatives
from fastmd_amd._device import on_device_of, require_cuda, rows_view, stream

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "relu": 3}
MAX_WIDTH = 2 ** 22 - 8
MAX_ROWS, MAX_VALUES = 2 ** 29, 2 ** 36  # within the 2^22 tiles of a launch, with every remainder
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


class FeedForwardSaved(NamedTuple):
    """What the VJP needs of the forward besides its inputs, rows of the hidden width rounded up to a multiple of 8:
    ``projections`` float32 [2, rows, .], x w_gate^T and x w_up^T, and ``hidden`` bfloat16 [planes, rows, .], what w_down
    multiplies (for float32 its three planes, for bfloat16 two). None for blocks of small weights, whose VJP forms both again."""

    projections: Tensor | None
    hidden: Tensor | None


def _refuse(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor) -> None:
    """ValueError for arguments that the block does not take (nothing for those that it does)."""
    require_cuda(x, w_gate, w_up, w_down)
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if t.dim() != 2:
            raise ValueError(f"{name} must be a matrix, got {tuple(t.shape)}")
        if t.dtype not in _TYPES or t.dtype != x.dtype:
            raise ValueError(f"x and the weights must all be float32 or bfloat16, got {x.dtype} and {t.dtype}")
    hidden, width = w_gate.shape
    if x.shape[1] != width or w_up.shape != w_gate.shape or w_down.shape[1] != hidden:
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)} and w_down "
                         f"{tuple(w_down.shape)} do not fit together")
    if not (1 <= width <= MAX_WIDTH and 1 <= hidden <= MAX_WIDTH and 1 <= w_down.shape[0] <= MAX_WIDTH):
        raise ValueError(f"the widths must be from 1 to {MAX_WIDTH}")
    rows, widest = x.shape[0], max(width, hidden, w_down.shape[0])
    if rows >= MAX_ROWS or max(rows, width, hidden, w_down.shape[0]) * widest >= MAX_VALUES:
        raise ValueError(f"the feed-forward block takes fewer than 2^29 rows, and 2^36 values of a matrix, got {rows} rows, "
                         f"widths {width}, {hidden} and {w_down.shape[0]}")


def _check(x, w_gate, w_up, w_down, activation) -> int:
    """The activation's code. The smallest calls are bound by host time: the usual case passes one condition, and what it
    excludes is named by ``_refuse``."""
    shape, dtype, device = x.shape, x.dtype, x.get_device()
    if not (len(shape) == 2 and device >= 0 and w_gate.get_device() == device and w_up.get_device() == device
            and w_down.get_device() == device and dtype in _TYPES and w_gate.dtype is dtype and w_up.dtype is dtype
            and w_down.dtype is dtype and len(w_gate.shape) == 2 and w_gate.shape == w_up.shape
            and len(w_down.shape) == 2 and w_gate.shape[1] == shape[1] and w_down.shape[1] == w_gate.shape[0]
            and 1 <= shape[1] <= MAX_WIDTH and 1 <= w_gate.shape[0] <= MAX_WIDTH
            and 1 <= w_down.shape[0] <= MAX_WIDTH and shape[0] < MAX_ROWS
            and max(shape[0], shape[1], w_down.shape[0], w_down.shape[1]) * max(shape[1], *w_down.shape) < MAX_VALUES):
        _refuse(x, w_gate, w_up, w_down)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _apart(t: Tensor, ld: int) -> bool:
    """Whether a bfloat16 matrix has to be laid out before the products read it."""
    return bool(t.shape[1] % 8 or ld % 8 or ld >= 2 ** 22 or t.data_ptr() % 16)


def _rows(t: Tensor) -> tuple[Tensor, int]:
    return (t, t.shape[1]) if t.is_contiguous() else rows_view(t)


def _operands(x, w_gate, w_up, w_down, gy=None):
    """(bits of the operands to lay out, arguments, the tensors that they point into)"""
    (x, x_ld), (w_gate, g_ld), (w_up, u_ld), (w_down, d_ld) = _rows(x), _rows(w_gate), _rows(w_up), _rows(w_down)
    if g_ld != u_ld:
        w_gate, w_up, g_ld = w_gate.contiguous(), w_up.contiguous(), w_gate.shape[1]
    lay = 15
    if x.dtype is torch.bfloat16:
        lay = ((1 if _apart(x, x_ld) else 0) | (2 if _apart(w_gate, g_ld) or _apart(w_up, g_ld) else 0)
               | (4 if _apart(w_down, d_ld) else 0))
    return lay, (x.data_ptr(), x_ld, w_gate.data_ptr(), w_up.data_ptr(), g_ld, w_down.data_ptr(), d_ld, x.shape[0],
                 x.shape[1], w_gate.shape[0], w_down.shape[0]), (x, w_gate, w_up, w_down)


@functools.lru_cache(maxsize=256)
def _saves(*sizes: int) -> bool:
    return bool(_abi.load().fmd_gated_ffn_saves(*sizes))


@functools.lru_cache(maxsize=256)
def _work_size(*sizes: int) -> int:
    return _abi.load().fmd_gated_ffn_work_size(*sizes)


@functools.lru_cache(maxsize=256)
def _work_size_vjp(*sizes: int) -> int:
    return _abi.load().fmd_gated_ffn_bwd_work_size(*sizes)


def _space(size: int, device) -> Tensor | None:
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _forward(x, w_gate, w_up, w_down, activation, save):
    act = _check(x, w_gate, w_up, w_down, activation)
    (rows, width), hidden, out, device, bf16 = x.shape, w_gate.shape[0], w_down.shape[0], x.device, _TYPES[x.dtype]
    y = torch.empty((rows, out), dtype=x.dtype, device=device)
    saved = projections = kept = None
    if save:
        if _saves(bf16, rows, width, hidden, out):
            padded = -(-hidden // 8) * 8
            projections = torch.empty((2, rows, padded), dtype=torch.float32, device=device)
            kept = torch.empty((2 if bf16 else 3, rows, padded), dtype=torch.bfloat16, device=device)
        saved = FeedForwardSaved(projections, kept)
    if rows == 0:
        return y, saved
    lay, args, keep = _operands(x, w_gate, w_up, w_down)
    work = _space(_work_size(bf16, rows, width, hidden, out, lay, 0 if kept is None else 1), device)
    with on_device_of(x):
        _abi.call("fmd_gated_ffn", bf16, act, lay, *args, y.data_ptr(), _abi.ptr(projections), _abi.ptr(kept), _abi.ptr(work),
                  stream())
    del keep
    return y, saved


def gated_feed_forward_forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *,
                               activation: str | None = "silu") -> tuple[Tensor, FeedForwardSaved]:
    """``(y, saved)`` without autograd: the output and what ``gated_feed_forward_vjp`` takes besides the inputs."""
    return _forward(x, w_gate, w_up, w_down, activation, True)


def gated_feed_forward_vjp(gy: Tensor, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, saved: FeedForwardSaved, *,
                           activation: str | None = "silu", need_x: bool = True, need_weights: bool = True):
    """``(gradient of x, of w_gate, of w_up, of w_down)`` from the gradient of the output and the forward's ``saved`` (None
    where not needed; the weights' come together)."""
    act = _check(x, w_gate, w_up, w_down, activation)
    projections, kept = saved
    (rows, width), hidden, out, device, bf16 = x.shape, w_gate.shape[0], w_down.shape[0], x.device, _TYPES[x.dtype]
    require_cuda(x, gy, projections, kept)
    if gy.shape != (rows, out) or gy.dtype != x.dtype:
        raise ValueError(f"gy must be {x.dtype} {(rows, out)}, got {gy.dtype} {tuple(gy.shape)}")
    if rows and _saves(bf16, rows, width, hidden, out):
        padded = -(-hidden // 8) * 8
        for t, shape, dtype in ((projections, (2, rows, padded), torch.float32),
                                (kept, (2 if bf16 else 3, rows, padded), torch.bfloat16)):
            if t is None or t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"saved must be the forward's: {dtype} {shape}, got "
                                 f"{None if t is None else (t.dtype, tuple(t.shape))}")
    make = torch.empty if rows else torch.zeros
    gx = make((rows, width), dtype=x.dtype, device=device) if need_x else None
    gw = [make(t.shape, dtype=x.dtype, device=device) if need_weights else None for t in (w_gate, w_up, w_down)]
    if rows == 0 or not (need_x or need_weights):
        return (gx, *gw)
    lay, args, keep = _operands(x, w_gate, w_up, w_down)
    gy, gy_ld = _rows(gy)
    if bf16 and _apart(gy, gy_ld):
        lay |= 8
    work = _space(_work_size_vjp(bf16, rows, width, hidden, out, lay, 1 if need_x else 0, 1 if need_weights else 0), device)
    with on_device_of(x):
        _abi.call("fmd_gated_ffn_bwd", bf16, act, lay, *args, gy.data_ptr(), gy_ld, _abi.ptr(projections), _abi.ptr(kept),
                  _abi.ptr(gx), *(_abi.ptr(t) for t in gw), _abi.ptr(work), stream())
    del keep
    return (gx, *gw)


class _GatedFeedForward(Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        y, saved = _forward(x, w_gate, w_up, w_down, activation, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, *saved)
        ctx.activation = activation
        return y

    @staticmethod
    def backward(ctx, gy):
        x, w_gate, w_up, w_down, *saved = ctx.saved_tensors
        grads = gated_feed_forward_vjp(gy, x, w_gate, w_up, w_down, FeedForwardSaved(*saved), activation=ctx.activation,
                                       need_x=ctx.needs_input_grad[0], need_weights=any(ctx.needs_input_grad[1:4]))
        return (*first_derivatives("gated_feed_forward", grads, gy, x, w_gate, w_up, w_down), None)


def gated_feed_forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *,
                       activation: str | None = "silu") -> Tensor:
    """The gated feed-forward block (see the module): ``x`` [rows, width], ``w_gate`` and ``w_up`` [hidden, width] (the halves of
    one packed matrix, or two), ``w_down`` [out, hidden], float32 or bfloat16, any strides and any widths (bfloat16 rows that do
    not start on 16 bytes, and widths that are no multiple of 8, are copied first). Differentiable once, in reverse mode."""
    if differentiated(x, w_gate, w_up, w_down):
        return _GatedFeedForward.apply(x, w_gate, w_up, w_down, activation)
    return _forward(x, w_gate, w_up, w_down, activation, False)[0]
