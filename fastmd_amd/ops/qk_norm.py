"""(g) The norm of queries and keys over each head with the rotation of their positions, in one pass (HIP kernels).

``qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions)``: each head x of both becomes
``x / sqrt(mean(x^2) + eps) * weight``, and its first ``2 * cos.shape[1]`` columns turn by the angles of the token's
position: columns (i, i + half), or (2 i, 2 i + 1) when ``interleaved``,

    (a, b) -> (a cos - b sin, b cos + a sin).

``rotary(x, cos, sin, positions)`` is the rotation alone. The angles come as tables (``rotary_tables``), which a program
keeps; ``positions`` are their rows (None: token t takes row t). All arithmetic is float32, each output rounded once.
The VJP sums the weights' gradients over tokens and heads in a fixed order, without atomics.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.autograd import Function

from fastmd_amd import _abi
from fastmd_amd._autograd import differentiated, first_derivatives
from fastmd_amd._device import require_cuda, stream
from fastmd_amd.ops.attention import heads_view

MAX_DIM = 256
_TYPES = (torch.float32, torch.bfloat16)


def rotary_frequencies(width: int, *, base: float = 10000.0, factor: float = 1.0, trained_length: int | None = None,
                       low: float = 1.0, high: float = 4.0) -> Tensor:
    """The angles per position of the ``width / 2`` pairs, float64 on the host: ``base ** (-2 i / width)``.

    ``factor`` > 1 stretches them to contexts that much longer: all of them by default, and with ``trained_length`` those
    that turn fewer than ``low`` times over it, none that turns more than ``high`` times, and a linear share in between."""
    if width < 2 or width % 2:
        raise ValueError(f"the rotated width must be even and positive, got {width}")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive")
    freq = base ** (-torch.arange(0, width, 2, dtype=torch.float64) / width)
    if factor == 1.0:
        return freq
    if trained_length is None:
        return freq / factor
    if not trained_length > 0 or not low < high:
        raise ValueError("trained_length must be positive and low below high")
    turns = trained_length * freq / (2.0 * math.pi)
    keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
    return freq * keep + freq / factor * (1.0 - keep)


def rotary_tables(positions, width: int, *, device=None, amplitude: float = 1.0, **frequencies) -> tuple[Tensor, Tensor]:
    """``(cos, sin)`` float32 [positions, width / 2], formed in float64. ``positions``: a count (0, 1, ...) or a vector of
    any real positions; ``frequencies``: the arguments of ``rotary_frequencies``; ``amplitude`` scales both tables."""
    freq = rotary_frequencies(width, **frequencies)
    if not isinstance(positions, Tensor):
        positions = torch.arange(int(positions), dtype=torch.float64)
    elif device is None:
        device = positions.device
    angle = positions.to(device=device, dtype=torch.float64)[:, None] * freq.to(device)
    return (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()


def _check(q: Tensor, k: Tensor | None, q_weight, k_weight, cos: Tensor, sin: Tensor, positions) -> None:
    """ValueError for arguments that the kernels do not take. The smallest calls are bound by host time: the usual case
    (both inputs, both weights, positions) passes one condition."""
    if k is not None and q_weight is not None and k_weight is not None and positions is not None:
        shape, dtype, device = q.shape, q.dtype, q.get_device()
        if (len(shape) == 3 and len(k.shape) == 3 and device >= 0 and k.get_device() == device
                and q_weight.get_device() == device and k_weight.get_device() == device and cos.get_device() == device
                and sin.get_device() == device and positions.get_device() == device and dtype in _TYPES
                and k.dtype is dtype and q_weight.dtype is dtype and k_weight.dtype is dtype
                and cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.dim() == 2
                and cos.shape == sin.shape and positions.dtype in (torch.int32, torch.int64)):
            tokens, heads, dim = shape
            kv_tokens, kv_heads, kv_dim = k.shape
            if (kv_tokens == tokens and kv_dim == dim and heads and kv_heads and dim % 8 == 0 and 8 <= dim <= MAX_DIM
                    and q_weight.shape == k_weight.shape == (dim,) and 2 * cos.shape[1] <= dim
                    and positions.shape == (tokens,) and tokens * (heads + kv_heads) < 2 ** 31):
                return
    require_cuda(q, k, q_weight, k_weight, cos, sin, positions)
    for name, x in (("q", q), ("k", k)):
        if x is None:
            continue
        if x.dim() != 3:
            raise ValueError(f"{name} must be [tokens, heads, dim], got {tuple(x.shape)}")
        if x.dtype not in (torch.float32, torch.bfloat16) or x.dtype != q.dtype:
            raise ValueError(f"q and k must both be float32 or bfloat16, got {q.dtype} and {x.dtype}")
        if x.shape[0] != q.shape[0] or x.shape[2] != q.shape[2]:
            raise ValueError(f"q and k must share tokens and head width, got {tuple(q.shape)} and {tuple(x.shape)}")
        if x.shape[1] < 1:
            raise ValueError(f"{name} has no head")
    tokens, _, dim = q.shape
    if dim % 8 or not 8 <= dim <= MAX_DIM:
        raise ValueError(f"the head width must be a multiple of 8 up to {MAX_DIM}, got {dim}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (dim,) or w.dtype != q.dtype):
            raise ValueError(f"{name} must be {q.dtype} [{dim}], got {w.dtype} {tuple(w.shape)}")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 tables of one shape [positions, width / 2]")
    if 2 * cos.shape[1] > dim:
        raise ValueError(f"the tables turn {2 * cos.shape[1]} columns of a head of {dim}")
    if positions is None:
        if cos.shape[1] and cos.shape[0] < tokens:
            raise ValueError(f"the tables have {cos.shape[0]} rows for {tokens} tokens")
    elif positions.shape != (tokens,) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be integers [{tokens}], got {positions.dtype} {tuple(positions.shape)}")
    if tokens * (q.shape[1] + (0 if k is None else k.shape[1])) >= 2 ** 31:
        raise ValueError("the norm and rotation take fewer than 2^31 rows")


def _check_eps(eps) -> None:
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")


def _aligned(t: Tensor | None) -> Tensor | None:
    """A contiguous tensor on a 16-byte address (the same one if it is)."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _common(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm):
    q, q_row, q_head = heads_view(q)
    kv_heads = k_row = k_head = 0
    if k is not None:
        k, k_row, k_head = heads_view(k)
        kv_heads = k.shape[1]
    q_weight, k_weight, cos, sin = _aligned(q_weight), _aligned(k_weight), _aligned(cos), _aligned(sin)
    if positions is not None:
        positions = positions.contiguous()
    rot = 2 * cos.shape[1]
    args = (1 if q.dtype == torch.bfloat16 else 0, q.data_ptr(), q_row, q_head, q.shape[1], _abi.ptr(k), k_row, k_head,
            kv_heads, q.shape[0], q.shape[2], 1 if norm else 0, float(eps), _abi.ptr(q_weight), _abi.ptr(k_weight),
            cos.data_ptr(), sin.data_ptr(), cos.shape[0], rot // 2, rot, 1 if interleaved else 0, _abi.ptr(positions),
            1 if positions is not None and positions.dtype == torch.int64 else 0)
    return args, (q, k, q_weight, k_weight, cos, sin, positions)


def _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm):
    args, keep = _common(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    _abi.call("fmd_qk_norm_rotary", *args, q_out.data_ptr(), _abi.ptr(k_out), stream())
    del keep
    return q_out, k_out


def _vjp(gq, gk, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm, weights):
    for name, g, x in (("gq", gq, q), ("gk", gk, k)):
        if (g is None) != (x is None) or (x is not None and (g.shape != x.shape or g.dtype != x.dtype)):
            raise ValueError(f"{name} must have the type and shape of {name[1]}")
    require_cuda(q, gq, gk)
    args, keep = _common(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm)
    gq, gq_row, gq_head = heads_view(gq)
    gk_row = gk_head = 0
    if gk is not None:
        gk, gk_row, gk_head = heads_view(gk)
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    dim, work = q.shape[2], None
    dqw = torch.empty(dim, dtype=q.dtype, device=q.device) if weights and q_weight is not None else None
    dkw = torch.empty(dim, dtype=q.dtype, device=q.device) if weights and k_weight is not None else None
    if dqw is not None or dkw is not None:
        size = _abi.load().fmd_qk_norm_rotary_work_size(q.shape[0], q.shape[1], 0 if k is None else k.shape[1], dim)
        work = torch.empty(max(1, size), dtype=torch.float32, device=q.device)
    _abi.call("fmd_qk_norm_rotary_bwd", *args, gq.data_ptr(), gq_row, gq_head, _abi.ptr(gk), gk_row, gk_head,
              dq.data_ptr(), _abi.ptr(dk), _abi.ptr(dqw), _abi.ptr(dkw), _abi.ptr(work), stream())
    del keep
    return dq, dk, dqw, dkw


class _NormRotary(Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.set_materialize_grads(False)
        ctx.options = eps, interleaved, norm
        out = _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm)
        return out[0] if k is None else out

    @staticmethod
    def backward(ctx, gq, gk=None):
        q, k, *rest = ctx.saved_tensors
        gq = torch.zeros_like(q) if gq is None else gq
        if k is not None and gk is None:
            gk = torch.zeros_like(k)
        grads = _vjp(gq, gk, q, k, *rest, *ctx.options, ctx.needs_input_grad[2] or ctx.needs_input_grad[3])
        inputs = (gq, gk, q, k, rest[0], rest[1])
        return (*first_derivatives("qk_norm_rotary", grads, *inputs), None, None, None, None, None, None)


def _apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm):
    if differentiated(q, k, q_weight, k_weight):
        out = _NormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm)
        return (out, None) if k is None else out
    return _forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved, norm)


def qk_norm_rotary(q: Tensor, k: Tensor, q_weight: Tensor | None, k_weight: Tensor | None, cos: Tensor, sin: Tensor,
                   positions: Tensor | None = None, *, eps: float = 1e-6, interleaved: bool = False
                   ) -> tuple[Tensor, Tensor]:
    """Norm and rotation of q [tokens, heads, dim] and k [tokens, kv_heads, dim] (float32 or bfloat16, any strides: columns of
    a packed projection are read in place) in one launch; weights [dim] of their type (None: ones), shared by the
    heads. Tables without columns give the norm alone. A position outside the tables gives NaN in the turned columns.
    Differentiable once in q, k and the weights, in reverse
    mode."""
    _check(q, k, q_weight, k_weight, cos, sin, positions)
    _check_eps(eps)
    return _apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved), True)


def qk_norm_rotary_vjp(gq: Tensor, gk: Tensor, q: Tensor, k: Tensor, q_weight: Tensor | None, k_weight: Tensor | None,
                       cos: Tensor, sin: Tensor, positions: Tensor | None = None, *, eps: float = 1e-6,
                       interleaved: bool = False):
    """``(gradient of q, of k, of q_weight, of k_weight)`` from the gradients of both outputs (the last two None for
    absent weights)."""
    _check(q, k, q_weight, k_weight, cos, sin, positions)
    _check_eps(eps)
    return _vjp(gq, gk, q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved), True, True)


def rotary(x: Tensor, cos: Tensor, sin: Tensor, positions: Tensor | None = None, *, interleaved: bool = False) -> Tensor:
    """The rotation alone, of x [tokens, heads, dim]. Differentiable once in x, in reverse mode."""
    _check(x, None, None, None, cos, sin, positions)
    return _apply(x, None, None, None, cos, sin, positions, 0.0, bool(interleaved), False)[0]
