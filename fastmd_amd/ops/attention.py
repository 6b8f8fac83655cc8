"""(g) Attention within segments on the GPU (HIP kernels), with a deterministic VJP.

``segment_attention(q, k, v, q_offsets, k_offsets=None, causal=False, scale=None)``:

    out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, h // group]) v[j, h // group]

over the key rows j of query i's segment. Segment s has the query rows ``[q_offsets[s], q_offsets[s + 1])`` and the
key rows ``[k_offsets[s], k_offsets[s + 1])``; the offsets, which ascend, are those of a CSR over sorted rows (the atoms of each system
of a batch, the neighbour rows of each atom, packed sequences), read on the device only: a call neither
synchronises nor depends on lengths that the host would have to know. ``group = heads / kv_heads`` query heads share a
key head. ``causal``: the last query of a segment sees all its keys, each one before it one key less. A query that sees
no key, and a row outside every segment (the unused rows of a fixed-capacity buffer), gives zero and gets zero gradient;
rows outside a query's segment are not read for it, whatever they hold, and neither an infinity nor a NaN in a key row that a
causal query does not see reaches it (nor, in the VJP, one in a query's row the keys that it does not see). One that is seen
makes the results that it is a term of NaN or infinite (a value its own column), and no others.

float32 is computed on the bf16 matrix cores with every operand split into three planes (float32 accuracy), bfloat16 with
products of bfloat16 operands. Scores, softmax statistics
and sums are float32 in both. For bfloat16, the probabilities and (in the VJP) the score gradients are operands of the
second product in two bfloat16 parts (16 bits), so that each result is as near to the exact one as its one rounding allows.
Gradients take no atomics: the same call gives the same bits.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import Function

from fastmd_amd import _abi
from fastmd_amd._autograd import differentiated, first_derivatives
from fastmd_amd._device import require_cuda, stream

MAX_DIM = 128
MAX_ROW_STRIDE = 2 ** 24  # elements; the kernels hold a lane's offset in a tile of rows in 32 bits


class AttentionSaved(NamedTuple):
    """What the VJP needs of the forward besides its output: a probability is ``exp2(score log2(e) - base) * inverse``
    (both float32 [heads, rows], 0 for a row that sees no key); ``residual`` (bfloat16 only, the output's shape) is what the
    rounding of the output dropped."""

    base: Tensor
    inverse: Tensor
    residual: Tensor | None

    @property
    def lse(self) -> Tensor:
        """Logarithm of each row's sum of exponentials [heads, rows], -inf for a row that sees no key."""
        return self.base * math.log(2.0) - torch.log(self.inverse.masked_fill(self.inverse == 0, float("inf")))


def heads_view(x: Tensor) -> tuple[Tensor, int, int]:
    """(tensor, row stride, head stride) of ``x`` [rows, heads, dim] with unit stride in dim and 16-byte aligned rows
    below MAX_ROW_STRIDE; copies only when needed (any strides otherwise: columns of a packed projection are read in
    place)."""
    rows, heads, dim = x.shape
    sr, sh, sd = x.stride()
    if rows <= 1:
        sr = heads * dim
    if heads <= 1:
        sh = dim
    if (sd != 1 or (sr | sh) % (16 // x.element_size()) or x.data_ptr() % 16 or sr >= MAX_ROW_STRIDE) and (
            rows and heads):
        x = x.clone(memory_format=torch.contiguous_format)
        sr, sh = heads * dim, dim
    return x, sr, sh


def _refuse(q: Tensor, k: Tensor, v: Tensor, q_offsets: Tensor, k_offsets: Tensor, scale) -> None:
    """ValueError for arguments that segment attention does not take (nothing for those that it does)."""
    require_cuda(q, k, v, q_offsets, k_offsets)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"q, k and v must be [rows, heads, dim], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must all be float32 or bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if k.shape != v.shape:
        raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    heads, dim, kv_heads = q.shape[1], q.shape[2], k.shape[1]
    if k.shape[2] != dim:
        raise ValueError(f"q and k must have one head width, got {dim} and {k.shape[2]}")
    if dim % 8 or not 8 <= dim <= MAX_DIM:
        raise ValueError(f"the head width must be a multiple of 8 up to {MAX_DIM}, got {dim}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"the query heads must be a multiple of the key heads, got {heads} and {kv_heads}")
    for name, off in (("q_offsets", q_offsets), ("k_offsets", k_offsets)):
        if off.dim() != 1 or off.numel() < 1 or off.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{name} must be an integer vector [segments + 1]")
    if q_offsets.numel() != k_offsets.numel():
        raise ValueError(f"q_offsets has {q_offsets.numel() - 1} segments, k_offsets {k_offsets.numel() - 1}")
    if q.shape[0] * heads // kv_heads >= 2 ** 31 or k.shape[0] >= 2 ** 31:
        raise ValueError("segment attention takes fewer than 2^31 packed query rows and key rows")
    if (max(q.shape[0] * (heads // kv_heads), k.shape[0]) // 32 + q_offsets.numel() + 1) * kv_heads >= 2 ** 31:
        raise ValueError("segment attention takes fewer than 2^31 tiles (32 rows of a key head, and one for each segment and key "
                         f"head), got {q_offsets.numel() - 1} segments of {kv_heads} key heads")
    if scale is not None and not 0.0 < float(scale) < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")


_TYPES = {torch.float32: 0, torch.bfloat16: 1}


def _prepare(q, k, v, q_offsets, k_offsets, causal, scale):
    """Checks, then the arguments that both directions share and the tensors that they point into. The smallest calls are
    bound by host time: the usual case passes one condition, and what it excludes is named by ``_refuse``."""
    shape, dtype, device = q.shape, q.dtype, q.get_device()
    if k_offsets is None:
        k_offsets = q_offsets
    if not (len(shape) == 3 and device >= 0 and k.get_device() == device and v.get_device() == device
            and q_offsets.get_device() == device and k_offsets.get_device() == device and dtype in _TYPES
            and k.dtype is dtype and v.dtype is dtype and k.shape == v.shape and len(k.shape) == 3
            and q_offsets.dtype is torch.int64 and k_offsets.dtype is torch.int64
            and q_offsets.dim() == 1 and q_offsets.shape == k_offsets.shape and scale is None):
        _refuse(q, k, v, q_offsets, k_offsets, scale)
    tq, heads, dim = shape
    tk, kv_heads, kdim = k.shape
    segments = q_offsets.shape[0] - 1
    if not (kdim == dim and 8 <= dim <= MAX_DIM and dim % 8 == 0 and heads and kv_heads and heads % kv_heads == 0
            and segments >= 0 and tq * heads < 2 ** 31 and tk < 2 ** 31
            and (tq * heads + tk * kv_heads) // 32 + (segments + 2) * kv_heads < 2 ** 31):
        _refuse(q, k, v, q_offsets, k_offsets, scale)
    (q, q_row, q_head), (k, k_row, k_head), (v, v_row, v_head) = heads_view(q), heads_view(k), heads_view(v)
    same = k_offsets is q_offsets
    if q_offsets.dtype is not torch.int64 or not q_offsets.is_contiguous():
        q_offsets = q_offsets.to(torch.int64).contiguous()
    if same:
        k_offsets = q_offsets
    elif k_offsets.dtype is not torch.int64 or not k_offsets.is_contiguous():
        k_offsets = k_offsets.to(torch.int64).contiguous()
    return ((_TYPES[dtype], q.data_ptr(), q_row, q_head, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head,
             q_offsets.data_ptr(), k_offsets.data_ptr(), tq, tk, segments, heads, kv_heads, dim, 1 if causal else 0,
             dim ** -0.5 if scale is None else float(scale)), (q, k, v, q_offsets, k_offsets))


@functools.lru_cache(maxsize=256)
def _plan(bf16: int, tq: int, tk: int, segments: int, heads: int, kv_heads: int, dim: int) -> tuple[int, int]:
    """(key splits, floats of workspace) of the forward at these sizes."""
    lib = _abi.load()
    splits = lib.fmd_segment_attention_splits(bf16, tq, tk, segments, heads, kv_heads, dim)
    return splits, lib.fmd_segment_attention_work_size(bf16, splits, tq, tk, segments, heads, kv_heads, dim)


@functools.lru_cache(maxsize=256)
def _plan_vjp(*sizes: int) -> tuple[int, int, int]:
    """(key splits of gq, query splits of gk and gv, floats of workspace) of the VJP at these sizes (as of ``_plan``)."""
    lib = _abi.load()
    q_splits, kv_splits = (lib.fmd_segment_attention_bwd_splits(*sizes, of_kv) for of_kv in (0, 1))
    return q_splits, kv_splits, lib.fmd_segment_attention_bwd_work_size(*sizes, q_splits, kv_splits)


def _forward(q, k, v, q_offsets, k_offsets, causal, scale, save):
    args, keep = _prepare(q, k, v, q_offsets, k_offsets, causal, scale)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    saved = base = inverse = residual = work = None
    if save:
        rows = torch.empty((2, q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
        saved = AttentionSaved(rows[0], rows[1], torch.empty_like(out) if args[0] else None)
        base, inverse, residual = (_abi.ptr(x) for x in saved)
    splits, size = _plan(args[0], *args[12:18])
    if size:
        work = torch.empty(size, dtype=torch.float32, device=q.device)
    _abi.call("fmd_segment_attention", *args, splits, out.data_ptr(), base, inverse, residual, _abi.ptr(work), stream())
    del keep
    return out, saved


def segment_attention_forward(q: Tensor, k: Tensor, v: Tensor, q_offsets: Tensor, k_offsets: Tensor | None = None, *,
                              causal: bool = False, scale: float | None = None) -> tuple[Tensor, AttentionSaved]:
    """``(out, saved)`` without autograd: the output and what ``segment_attention_vjp`` takes besides it."""
    return _forward(q, k, v, q_offsets, k_offsets, causal, scale, True)


def segment_attention_vjp(gout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, saved: AttentionSaved,
                          q_offsets: Tensor, k_offsets: Tensor | None = None, *, causal: bool = False,
                          scale: float | None = None, need_q: bool = True, need_kv: bool = True):
    """``(gq, gk, gv)`` from the gradient of the output and the results of ``segment_attention_forward`` (None where
    not needed; the gradients of k and v come together)."""
    args, keep = _prepare(q, k, v, q_offsets, k_offsets, causal, scale)
    base, inverse, residual = saved
    require_cuda(q, gout, out, base, inverse, residual)
    if gout.shape != q.shape or gout.dtype != q.dtype or out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError(f"gout and out must be {q.dtype} {tuple(q.shape)}, got {gout.dtype} {tuple(gout.shape)} and "
                         f"{out.dtype} {tuple(out.shape)}")
    rows = (q.shape[1], q.shape[0])
    for x in (base, inverse):
        if x.shape != rows or x.dtype != torch.float32 or not x.is_contiguous():
            raise ValueError(f"saved must be the forward's: float32 {rows} rows, got {x.dtype} {tuple(x.shape)}")
    if q.dtype == torch.bfloat16 and (residual is None or residual.shape != q.shape or residual.dtype != q.dtype
                                      or not residual.is_contiguous() or residual.data_ptr() % 16):
        raise ValueError("saved must be the forward's: the residual of a bfloat16 output")
    gout, g_row, g_head = heads_view(gout)
    if not out.is_contiguous() or out.data_ptr() % 16:
        out = out.clone(memory_format=torch.contiguous_format)
    gq = torch.empty_like(q, memory_format=torch.contiguous_format) if need_q else None
    gk = torch.empty_like(k, memory_format=torch.contiguous_format) if need_kv else None
    gv = torch.empty_like(k, memory_format=torch.contiguous_format) if need_kv else None
    q_splits, kv_splits, size = _plan_vjp(args[0], *args[12:18])
    work = torch.empty(max(4, size), dtype=torch.float32, device=q.device)
    _abi.call("fmd_segment_attention_bwd", *args, gout.data_ptr(), g_row, g_head, out.data_ptr(), base.data_ptr(),
              inverse.data_ptr(), _abi.ptr(residual), q_splits, kv_splits, work.data_ptr(), _abi.ptr(gq), _abi.ptr(gk), _abi.ptr(gv), stream())
    del keep
    return gq, gk, gv


class _SegmentAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, causal, scale):
        out, saved = _forward(q, k, v, q_offsets, k_offsets, causal, scale, True)
        ctx.save_for_backward(q, k, v, out, q_offsets, k_offsets, *saved)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    def backward(ctx, gout):
        q, k, v, out, q_offsets, k_offsets, *saved = ctx.saved_tensors
        grads = segment_attention_vjp(gout, q, k, v, out, AttentionSaved(*saved), q_offsets, k_offsets,
                                      causal=ctx.causal, scale=ctx.scale, need_q=ctx.needs_input_grad[0],
                                      need_kv=ctx.needs_input_grad[1] or ctx.needs_input_grad[2])
        return (*first_derivatives("segment_attention", grads, gout, q, k, v), None, None, None, None)


def segment_attention(q: Tensor, k: Tensor, v: Tensor, q_offsets: Tensor, k_offsets: Tensor | None = None, *,
                      causal: bool = False, scale: float | None = None) -> Tensor:
    """Attention within segments (see the module): ``q`` [rows, heads, dim], ``k`` and ``v`` [key rows, kv_heads, dim],
    float32 or bfloat16, any strides; offsets [segments + 1] on the device (``k_offsets`` None: ``q_offsets``); ``scale``
    None: ``dim ** -0.5``. One query per segment (the next token of a sequence over its cache, an atom over its neighbours) is the
    same call: a long key axis is then split over the card and joined. Differentiable once in q, k and v, in reverse mode."""
    if differentiated(q, k, v):
        return _SegmentAttention.apply(q, k, v, q_offsets, k_offsets, bool(causal), scale)
    return _forward(q, k, v, q_offsets, k_offsets, causal, scale, False)[0]
