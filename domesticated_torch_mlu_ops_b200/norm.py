"""Gated RMS norm with residual sum: the norm behind the sequence mixer (with
its gate z) and the norm before a block (with the sum of the residual stream).

One pass over the rows forward and one backward (``gdn_norm.cu`` through the C
ABI); there is no CPU path.  The ops are the ``torch.library`` custom ops
``gdn_b200::norm_fwd`` and ``gdn_b200::norm_bwd``.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import _lib
from .gdn import _DT, _addr, _cuda, _first_order, _launch, _plain

Tensor = torch.Tensor
_GATE = {"silu": _lib.GDN_GATE_SILU, "swish": _lib.GDN_GATE_SILU, "sigmoid": _lib.GDN_GATE_SIGMOID}


def _row_strides(t):
    """``(tensor, heads, token stride, head stride)`` of rows over the last
    dimension: in place for up to two strided leading dimensions ([tokens, D],
    [tokens, heads, D], or more whose strides merge), else a packed copy."""
    D = t.shape[-1]
    if t.is_contiguous():
        return t, 1, D, D
    if D == 1 or t.stride(-1) == 1:
        dims = []  # (size, stride) of the leading dimensions, merged where they are one run
        for n, st in zip(t.shape[:-1], t.stride()[:-1]):
            if n == 1:
                continue
            if dims and dims[-1][1] == n * st:
                dims[-1] = (dims[-1][0] * n, st)
            else:
                dims.append((n, st))
        if len(dims) <= 2 and all(st >= 0 for _, st in dims):
            if len(dims) == 2:
                return t, dims[1][0], dims[0][1], dims[1][1]
            return t, 1, dims[0][1] if dims else D, D
    return t.contiguous(), 1, D, D


def _two_strides(x, z):
    """Row strides of x and z over one split of the rows into tokens x heads."""
    if x.is_contiguous() and (z is None or z.is_contiguous()):
        D = x.shape[-1]
        return x, z, 1, D, D, D, D
    x, hx, sxt, sxh = _row_strides(x)
    if z is None:
        return x, None, hx, sxt, sxh, 0, 0
    z, hz, szt, szh = _row_strides(z)
    if hx != hz:
        if hx == 1 and sxt * hz >= 0:  # x's rows are one run: split them as z's are
            hx, sxt, sxh = hz, sxt * hz, sxt
        elif hz == 1:
            hz, szt, szh = hx, szt * hx, szt
        else:
            x, z = x.contiguous(), z.contiguous()
            D = x.shape[-1]
            hx, sxt, sxh, szt, szh = 1, D, D, D, D
    return x, z, hx, sxt, sxh, szt, szh


def _norm_fwd_impl(x, weight, z, residual, eps, group_size, norm_before_gate, zero_centered, residual_scale,
                   activation):
    """Returns ``(y, sum)``; sum is None without a residual."""
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    total = None if residual is None else torch.empty_like(residual)
    if x.numel() == 0:
        return y, total
    D = x.shape[-1]
    x, z, heads, sxt, sxh, szt, szh = _two_strides(x, z)
    dt = _DT[x.dtype]
    packed = _lib.pack_norm(
        x.data_ptr(), _addr(z), _addr(residual), weight.data_ptr(), y.data_ptr(),
        _addr(total), 0, 0, 0, 0, 0, 0, 0, 0, x.numel() // D, heads, D, sxt, sxh, szt, szh,
        group_size, dt, dt, dt if residual is None else _DT[residual.dtype], _DT[weight.dtype], not norm_before_gate,
        zero_centered, activation, eps, residual_scale)
    _launch(_lib.load().gdn_norm_fwd, packed, dev)
    return y, total


@torch.library.custom_op("gdn_b200::norm_fwd", mutates_args=(), device_types="cuda")
def _norm_fwd_op(x: Tensor, weight: Tensor, z: Optional[Tensor], residual: Optional[Tensor], eps: float,
                 group_size: int, norm_before_gate: bool, zero_centered: bool, residual_scale: float,
                 activation: int) -> tuple[Tensor, Tensor]:
    """The sum is empty without a residual."""
    y, total = _norm_fwd_impl(x, weight, z, residual, eps, group_size, norm_before_gate, zero_centered, residual_scale,
                              activation)
    return y, x.new_empty((0,)) if total is None else total


@_norm_fwd_op.register_fake
def _(x, weight, z, residual, eps, group_size, norm_before_gate, zero_centered, residual_scale, activation):
    return x.new_empty(x.shape), x.new_empty((0,)) if residual is None else residual.new_empty(residual.shape)


@functools.lru_cache(maxsize=256)
def _bwd_workspace(rows, D, group, dtype, x_dtype):
    """Bytes of gdn_norm_bwd's workspace: they depend on the shapes alone."""
    args = _lib.NormArgs(rows=rows, heads=1, D=D, group=group, dtype=dtype, x_dtype=x_dtype, res_dtype=x_dtype)
    n = _lib.load().gdn_norm_bwd_workspace_size(ctypes.byref(args))
    if n == 0:
        _lib.check(_lib.GDN_ERR_INVALID)
    return n


def _norm_bwd_impl(dy, x, weight, z, dsum, want_dresidual, eps, group_size, norm_before_gate, zero_centered,
                   residual_scale, activation):
    """Returns ``(dx, dweight, dz, dresidual)``; the last two are None when
    there is no z or dresidual is not wanted."""
    dev = dy.device
    dx = torch.empty_like(dy)  # dy is contiguous
    dz = None if z is None else torch.empty_like(dy)
    dres = torch.empty_like(dy, dtype=x.dtype) if want_dresidual else None
    if x.numel() == 0:
        return dx, torch.zeros_like(weight), dz, dres
    dw = torch.empty_like(weight)
    D = x.shape[-1]
    x, z, heads, sxt, sxh, szt, szh = _two_strides(x, z)
    dt, xt, rows = _DT[dy.dtype], _DT[x.dtype], x.numel() // D
    nbytes = _bwd_workspace(rows, D, group_size, dt, xt)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    packed = _lib.pack_norm(
        x.data_ptr(), _addr(z), 0, weight.data_ptr(), 0, 0, dy.data_ptr(), _addr(dsum), dx.data_ptr(),
        _addr(dz), _addr(dres), dw.data_ptr(), ws.data_ptr(), nbytes,
        rows, heads, D, sxt, sxh, szt, szh, group_size, dt, xt, xt, _DT[weight.dtype], not norm_before_gate,
        zero_centered, activation, eps, residual_scale)
    _launch(_lib.load().gdn_norm_bwd, packed, dev)
    return dx, dw, dz, dres


@torch.library.custom_op("gdn_b200::norm_bwd", mutates_args=(), device_types="cuda")
def _norm_bwd_op(dy: Tensor, x: Tensor, weight: Tensor, z: Optional[Tensor], dsum: Optional[Tensor],
                 want_dresidual: bool, eps: float, group_size: int, norm_before_gate: bool, zero_centered: bool,
                 residual_scale: float, activation: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """dz and dresidual are empty when there is no z or dresidual is not wanted."""
    dx, dw, dz, dres = _norm_bwd_impl(dy, x, weight, z, dsum, want_dresidual, eps, group_size, norm_before_gate,
                                      zero_centered, residual_scale, activation)
    return dx, dw, dy.new_empty((0,)) if dz is None else dz, x.new_empty((0,)) if dres is None else dres


@_norm_bwd_op.register_fake
def _(dy, x, weight, z, dsum, want_dresidual, eps, group_size, norm_before_gate, zero_centered, residual_scale,
      activation):
    return (dy.new_empty(dy.shape), weight.new_empty(weight.shape), dy.new_empty((0,) if z is None else dy.shape),
            x.new_empty(dy.shape if want_dresidual else (0,)))


def _fwd(x, weight, z, residual, meta):
    if _plain(x, weight, z, residual):
        return _norm_fwd_impl(x, weight, z, residual, *meta)
    return torch.ops.gdn_b200.norm_fwd(x, weight, z, residual, *meta)


def _bwd(dy, x, weight, z, dsum, want_dresidual, meta):
    if _plain(dy, x, weight, z, dsum):
        return _norm_bwd_impl(dy, x, weight, z, dsum, want_dresidual, *meta)
    return torch.ops.gdn_b200.norm_bwd(dy, x, weight, z, dsum, want_dresidual, *meta)


def _check(name, x, weight, z, residual, group_size, activation):
    if x.dim() < 1:
        raise ValueError(f"{name}: x must have at least one dimension")
    if x.dtype not in _DT:
        raise ValueError(f"{name}: x dtype {x.dtype} must be float32, bfloat16 or float16")
    D = x.shape[-1]
    if tuple(weight.shape) != (D,):
        raise ValueError(f"{name}: weight {tuple(weight.shape)} must be ({D},)")
    if weight.dtype not in _DT:
        raise ValueError(f"{name}: weight dtype {weight.dtype} must be float32, bfloat16 or float16")
    if z is not None and z.shape != x.shape:
        raise ValueError(f"{name}: z {tuple(z.shape)} must match x {tuple(x.shape)}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{name}: residual {tuple(residual.shape)} must match x {tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name}: residual dtype {residual.dtype} must be {x.dtype} or float32")
    group = D if group_size is None else int(group_size)
    if group <= 0 or D % group != 0:
        raise ValueError(f"{name}: group_size={group_size} must divide {D}")
    if activation not in _GATE:
        raise ValueError(f"{name}: unsupported activation {activation!r} ('silu', 'swish' or 'sigmoid')")
    return group, _GATE[activation]


class GatedRMSNormFunction(torch.autograd.Function):
    """Autograd node of :func:`gated_rms_norm`: saves what was normed (x, or
    the sum with the residual as it was stored), z and the weight."""

    @staticmethod
    def forward(ctx, x, weight, z, residual, meta):
        y, total = _fwd(x, weight, z, residual, meta)
        ctx.save_for_backward(x if residual is None else total, weight, z)
        ctx.meta, ctx.has_residual = meta, residual is not None
        return (y, total) if residual is not None else y

    @staticmethod
    @_first_order
    def backward(ctx, dy, dsum=None):
        x, weight, z = ctx.saved_tensors
        dtype = z.dtype if z is not None else dy.dtype
        dy = dy.to(dtype).contiguous()
        dsum = None if dsum is None else dsum.contiguous()
        dx, dw, dz, dres = _bwd(dy, x, weight, z, dsum, ctx.has_residual, ctx.meta)
        return dx, dw, None if z is None else dz, dres if ctx.has_residual else None, None


def gated_rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    z: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    eps: float = 1e-6,
    group_size: int | None = None,
    norm_before_gate: bool = True,
    zero_centered: bool = False,
    residual_scale: float = 1.0,
    activation: str = "silu",
):
    """RMS norm over the last dimension, with a gate and a residual sum.

    ``r = residual + residual_scale * x`` (x without a residual);
    ``y = norm(r) * weight * act(z)``, or ``norm(r * act(z)) * weight`` with
    ``norm_before_gate=False``; ``norm(u) = u / sqrt(mean(u^2) + eps)`` over
    each ``group_size`` consecutive elements (the whole row by default).
    ``zero_centered`` multiplies by ``1 + weight``; ``activation`` of the gate
    is 'silu' or 'sigmoid'.

    x, z ``[..., D]`` of one dtype (rows of views such as ``[tokens, heads, D]``
    slices are read in place), residual ``[..., D]`` of x's dtype or float32,
    weight ``[D]`` of any float type.  Returns y in x's dtype, or
    ``(y, r)`` with r in the residual's dtype when a residual is given.  The
    norm is taken of the unrounded fp32 sum.  Differentiable once in x, weight,
    z and residual (the backward takes r as it was stored)."""
    _cuda("gated_rms_norm", x, weight, z, residual)
    group, act = _check("gated_rms_norm", x, weight, z, residual, group_size, activation)
    if z is not None and z.dtype != x.dtype:
        raise ValueError(f"gated_rms_norm: z dtype {z.dtype} must be x's {x.dtype}")
    if residual is not None:
        residual = residual.contiguous()
    weight = weight.contiguous()
    meta = (float(eps), group, bool(norm_before_gate), bool(zero_centered),
            1.0 if residual is None else float(residual_scale), act)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (z is not None and z.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return GatedRMSNormFunction.apply(x, weight, z, residual, meta)
    y, total = _fwd(x, weight, z, residual, meta)
    return y if residual is None else (y, total)


def gated_rms_norm_bwd(
    dy: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor,
    z: torch.Tensor | None = None,
    dresidual: torch.Tensor | None = None,
    eps: float = 1e-6,
    group_size: int | None = None,
    norm_before_gate: bool = True,
    zero_centered: bool = False,
    residual_scale: float = 1.0,
    activation: str = "silu",
    has_residual: bool = False,
):
    """Functional gradient of :func:`gated_rms_norm`.

    ``x`` is what was normed: the forward's x, or with ``has_residual`` its
    second output r (x's dtype or float32); ``dresidual`` is the gradient of
    that output, or None.  Returns ``(dx, dweight, dz, dresidual)``, the last
    two None where there is no z or residual."""
    _cuda("gated_rms_norm_bwd", dy, x, weight, z, dresidual)
    group, act = _check("gated_rms_norm_bwd", x, weight, z, None, group_size, activation)
    if dy.shape != x.shape or dy.dtype not in _DT:
        raise ValueError(f"gated_rms_norm_bwd: dy {tuple(dy.shape)} {dy.dtype} must match x {tuple(x.shape)}")
    if x.dtype not in (dy.dtype, torch.float32) or (z is not None and z.dtype != dy.dtype):
        raise ValueError("gated_rms_norm_bwd: x must have dy's dtype (or float32) and z dy's dtype")
    if dresidual is not None:
        if not has_residual or dresidual.shape != x.shape or dresidual.dtype != x.dtype:
            raise ValueError("gated_rms_norm_bwd: dresidual needs has_residual and must match x in shape and dtype")
        dresidual = dresidual.contiguous()
    meta = (float(eps), group, bool(norm_before_gate), bool(zero_centered),
            float(residual_scale) if has_residual else 1.0, act)
    dx, dw, dz, dres = _bwd(dy.contiguous(), x, weight.contiguous(), z, dresidual, bool(has_residual), meta)
    return dx, dw, None if z is None else dz, dres if has_residual else None
