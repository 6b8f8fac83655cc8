"""(h) The norm over groups of channels, channels last, with its activation on the GPU (HIP kernels), with a deterministic VJP.

``group_norm(x, groups, weight, bias, offsets=None, eps=1e-5, activation=None)`` on x [rows, channels]:

    n = (x - mean) / sqrt(variance + eps),  y = act(n * weight + bias)

with the mean and variance of each group of ``channels / groups`` channels that lie side by side: of every row by itself
(``offsets`` None), or of all rows ``[offsets[s], offsets[s + 1])`` of segment s (the atoms of each system of a batch, the places of
each map of a batch of images [maps, height, width, channels] seen as rows). The offsets, which ascend, are read on the device only: a call
neither synchronises nor depends on lengths that the host would have to know. A row outside every segment (the unused rows of
a fixed-capacity buffer) gives zero, gets zero gradient and is not read. ``groups=1`` is the layer norm of rows.

float32 or bfloat16; statistics, sums and the activation are float32, each result rounded once. Variances are sums of
squared distances from the mean, joined over long segments by their counts: no difference of large sums. Gradients take no
atomics: the same call gives the same bits.
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
from fastmd_amd.ops.feed_forward import ACTIVATIONS

MAX_GROUP = 8192  # channels of a group
MAX_GROUPS = 65535
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


class GroupNormSaved(NamedTuple):
    """What the VJP needs of the forward: float32 [rows, groups], or [segments, groups] with offsets (undefined for an empty
    segment)."""

    mean: Tensor
    inverse: Tensor  # 1 / sqrt(variance + eps)


def _check(x: Tensor, groups: int, weight, bias, offsets, activation) -> int:
    """The activation's code, or ValueError for arguments that the kernels do not take."""
    require_cuda(x, weight, bias, offsets)
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, channels], got {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be float32 or bfloat16, got {x.dtype}")
    channels = x.shape[1]
    if not 1 <= groups <= channels or channels % groups:
        raise ValueError(f"the channels must be a multiple of the groups, got {channels} and {groups}")
    if channels // groups > MAX_GROUP or channels >= 2 ** 24:
        raise ValueError(f"a group has at most {MAX_GROUP} channels, all fewer than 2^24, got {channels // groups} and {channels}")
    if groups > MAX_GROUPS:
        raise ValueError(f"at most {MAX_GROUPS} groups, got {groups}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != (channels,) or p.dtype != x.dtype):
            raise ValueError(f"{name} must be {x.dtype} [{channels}], got {p.dtype} {tuple(p.shape)}")
    if offsets is not None and (offsets.dim() != 1 or offsets.numel() < 1 or offsets.dtype not in (torch.int32, torch.int64)):
        raise ValueError("offsets must be an integer vector [segments + 1]")
    if x.shape[0] >= 2 ** 40 or (offsets is not None and offsets.numel() > 2 ** 31 - 4):
        raise ValueError("the group norm takes fewer than 2^40 rows and 2^31 segments")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _plain(t: Tensor | None) -> Tensor | None:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _segments(offsets: Tensor | None) -> tuple[Tensor | None, int]:
    if offsets is None:
        return None, 0
    if offsets.dtype is not torch.int64 or not offsets.is_contiguous():
        offsets = offsets.to(torch.int64).contiguous()
    return offsets, offsets.shape[0] - 1


@functools.lru_cache(maxsize=256)
def _work_size(*sizes: int) -> int:
    return max(1, _abi.load().fmd_group_norm_work_size(*sizes))


@functools.lru_cache(maxsize=256)
def _work_size_vjp(*sizes: int) -> int:
    return max(1, _abi.load().fmd_group_norm_bwd_work_size(*sizes))


def _forward(x, groups, weight, bias, offsets, eps, activation, save):
    act = _check(x, groups, weight, bias, offsets, activation)
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    rows, channels = x.shape
    weight, bias = _plain(weight), _plain(bias)
    offsets, segments = _segments(offsets)
    y = torch.empty((rows, channels), dtype=x.dtype, device=x.device)
    saved = None
    if save or offsets is not None:
        stats = torch.empty((2, rows if offsets is None else segments, groups), dtype=torch.float32, device=x.device)
        saved = GroupNormSaved(stats[0], stats[1])
    if rows == 0 or (offsets is not None and segments == 0):
        return y.zero_(), saved
    x, ld = rows_view(x)
    work = None
    if offsets is not None:
        work = torch.empty(_work_size(_TYPES[x.dtype], rows, channels, groups, segments), dtype=torch.float32, device=x.device)
    with on_device_of(x):
        _abi.call("fmd_group_norm", _TYPES[x.dtype], act, x.data_ptr(), ld, _abi.ptr(weight), _abi.ptr(bias), rows, channels,
                  groups, _abi.ptr(offsets), segments, float(eps), y.data_ptr(), _abi.ptr(saved and saved.mean),
                  _abi.ptr(saved and saved.inverse), _abi.ptr(work), stream())
    return y, saved


def group_norm_forward(x: Tensor, groups: int, weight: Tensor | None = None, bias: Tensor | None = None, *,
                       offsets: Tensor | None = None, eps: float = 1e-5, activation: str | None = None
                       ) -> tuple[Tensor, GroupNormSaved]:
    """``(y, saved)`` without autograd: the output and what ``group_norm_vjp`` takes besides the inputs."""
    return _forward(x, groups, weight, bias, offsets, eps, activation, True)


def group_norm_vjp(gy: Tensor, x: Tensor, groups: int, weight: Tensor | None, bias: Tensor | None, saved: GroupNormSaved, *,
                   offsets: Tensor | None = None, activation: str | None = None, need_weights: bool = True):
    """``(gradient of x, of weight, of bias)`` from the gradient of the output and the forward's ``saved``; without
    ``need_weights`` the last two are None, and each is for a parameter that is None."""
    act = _check(x, groups, weight, bias, offsets, activation)
    mean, inverse = saved
    require_cuda(x, gy, mean, inverse)
    rows, channels = x.shape
    if gy.shape != x.shape or gy.dtype != x.dtype:
        raise ValueError(f"gy must be {x.dtype} {tuple(x.shape)}, got {gy.dtype} {tuple(gy.shape)}")
    offsets, segments = _segments(offsets)
    for t in (mean, inverse):
        if t.shape != (rows if offsets is None else segments, groups) or t.dtype != torch.float32 or not t.is_contiguous():
            raise ValueError(f"saved must be the forward's, got {t.dtype} {tuple(t.shape)}")
    weight, bias = _plain(weight), _plain(bias)
    none = rows == 0 or (offsets is not None and segments == 0)
    make = torch.zeros if none else torch.empty
    gx = make((rows, channels), dtype=x.dtype, device=x.device)
    sums = None
    if need_weights and (weight is not None or bias is not None):
        sums = make((2, channels), dtype=x.dtype, device=x.device)
    if not none:
        (x, ld), (gy, g_ld) = rows_view(x), rows_view(gy)
        bf16 = _TYPES[x.dtype]
        work = torch.empty(_work_size_vjp(bf16, rows, channels, groups, segments), dtype=torch.float32, device=x.device)
        with on_device_of(x):
            _abi.call("fmd_group_norm_bwd", bf16, act, gy.data_ptr(), g_ld, x.data_ptr(), ld, _abi.ptr(weight),
                      _abi.ptr(bias), rows, channels, groups, _abi.ptr(offsets), segments, mean.data_ptr(),
                      inverse.data_ptr(), gx.data_ptr(), None if sums is None else sums[0].data_ptr(),
                      None if sums is None else sums[1].data_ptr(), work.data_ptr(), stream())
    return (gx, None if sums is None or weight is None else sums[0], None if sums is None or bias is None else sums[1])


class _GroupNorm(Function):
    @staticmethod
    def forward(ctx, x, groups, weight, bias, offsets, eps, activation):
        y, saved = _forward(x, groups, weight, bias, offsets, eps, activation, True)
        ctx.save_for_backward(x, weight, bias, offsets, *saved)
        ctx.options = groups, activation
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight, bias, offsets, *saved = ctx.saved_tensors
        groups, activation = ctx.options
        gx, gw, gb = group_norm_vjp(gy, x, groups, weight, bias, GroupNormSaved(*saved), offsets=offsets, activation=activation,
                                    need_weights=ctx.needs_input_grad[2] or ctx.needs_input_grad[3])
        gx, gw, gb = first_derivatives("group_norm", (gx, gw, gb), gy, x, weight, bias)
        return gx, None, gw, gb, None, None, None


def group_norm(x: Tensor, groups: int, weight: Tensor | None = None, bias: Tensor | None = None, *,
               offsets: Tensor | None = None, eps: float = 1e-5, activation: str | None = None) -> Tensor:
    """The norm over groups of channels with its activation (see the module): ``x`` [rows, channels] float32 or bfloat16, any
    strides; ``weight`` and ``bias`` [channels] of its type (None: ones, zeros); ``offsets`` [segments + 1] on the device;
    ``activation`` None, "silu", "gelu" (by erf) or "relu". Differentiable once, in reverse mode."""
    if differentiated(x, weight, bias):
        return _GroupNorm.apply(x, groups, weight, bias, offsets, eps, activation)
    return _forward(x, groups, weight, bias, offsets, eps, activation, False)[0]
