"""Selective state space scan with one decay per head: the sibling of the
delta rule in hybrid models, for prompts (``chunk_selective_scan``) and for
single tokens on a slot-indexed cache (``selective_scan_update``).

Per head, with the step ``dt = clamp(softplus(raw + dt_bias))``::

    h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t^T        state [P, S], fp32
    y_t = (h_t C_t + D x_t) silu(z_t)

The work runs in ``libgdn_b200.so`` (``gdn_scan.cu``, ``gdn_scan_tc.cu``)
through its C ABI; there is no CPU path.  The ops are the ``torch.library``
custom ops ``gdn_b200::scan_fwd`` and ``gdn_b200::scan_update`` (which declares
the cache as mutated).
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import _lib
from .gdn import _DT, _IDT, _addr, _cuda, _err_word, _idx, _launch, _plain, _raise_err_word

Tensor = torch.Tensor
_INF = float("inf")


def _f32(t):
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


def _packed_rows(t, tail):
    """(tensor, distance between token rows) of ``t`` whose last ``tail`` (1 or
    2) dimensions are one packed row: in place when only the token rows are
    strided (views of one projection), else a packed copy."""
    shape, st = t.shape, t.stride()
    width = shape[-1] if tail == 1 else shape[-1] * shape[-2]
    # the usual views: one token dimension, or a leading one of size 1
    if st[-1] == 1 and (tail == 1 or st[-2] == shape[-1]):
        lead = len(shape) - tail
        if lead == 1 or shape[0] == 1:
            row = st[lead - 1]
            if row >= width:
                return t, row
        elif st[0] == shape[1] * st[1] and st[1] >= width:
            return t, st[1]
    return t.contiguous(), width


def _aligned_rows(t, tail):
    """:func:`_packed_rows` whose rows start on 16 bytes (what the tensor-core
    kernels read in place): other rows are copied, which costs far less than
    the recurrent kernel."""
    t, st = _packed_rows(t, tail)
    if t.data_ptr() % 16 or st * t.element_size() % 16:
        t, st = _packed_rows(t.clone(memory_format=torch.contiguous_format), tail)
    return t, st


@functools.lru_cache(maxsize=256)
def _workspace(B, T, N, H, P, G, S, dtype, force_generic):
    """Bytes of gdn_scan_fwd's workspace: they depend on the shapes alone."""
    args = _lib.ScanArgs(B=B, T=T, N=N, H=H, P=P, G=G, S=S, dtype=dtype, dt_dtype=dtype, stride_x=H * P, stride_z=H * P,
                         stride_b=G * S, stride_c=G * S, stride_dt=H, force_generic=force_generic)
    if N != B:
        args.cu_seqlens, args.cu_dtype = ctypes.c_void_p(16), _lib.GDN_I64  # packed: only whether it is there counts
    n = _lib.load().gdn_scan_workspace_size(ctypes.byref(args))
    if n == 0:
        _lib.check(_lib.GDN_ERR_INVALID)
    return n


def _scan_fwd_impl(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor],
                   dt_bias: Optional[Tensor], dt_softplus: bool, dt_min: float, dt_max: float,
                   initial_state: Optional[Tensor], output_final_state: bool, state_dtype: torch.dtype,
                   cu_seqlens: Optional[Tensor], force_generic: bool, check_errors: bool) -> tuple[Tensor, Tensor]:
    """Returns ``(y, final_state)``; final_state is empty when not requested."""
    Bt, T, H, P = x.shape
    G, S = B.shape[2], B.shape[3]
    N = Bt if cu_seqlens is None else cu_seqlens.numel() - 1
    dev = x.device
    tensor_cores = x.dtype == torch.bfloat16 and P % 64 == 0 and S in (64, 128) and not force_generic
    rows = _aligned_rows if tensor_cores else _packed_rows  # the recurrent kernel reads any rows in place
    (x, sx), (dt, sdt), (B, sb), (C, sc) = rows(x, 2), _packed_rows(dt, 1), rows(B, 2), rows(C, 2)
    z, sz = (None, 0) if z is None else rows(z, 2)
    y = torch.empty((Bt, T, H, P), dtype=x.dtype, device=dev)
    fin = torch.empty((N, H, P, S) if output_final_state else (0,), dtype=state_dtype, device=dev)
    dtype, dt_dtype = _DT[x.dtype], _DT[dt.dtype]
    nbytes = _workspace(Bt, T, N, H, P, G, S, dtype, force_generic)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    packed = _lib.pack_scan(
        x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _addr(D), _addr(z), _addr(dt_bias),
        _addr(initial_state), y.data_ptr(), fin.data_ptr() if output_final_state else 0, _addr(cu_seqlens), ws.data_ptr(),
        nbytes, Bt, T, N, sx, sdt, sb, sc, sz, H, P, G, S, dtype, dt_dtype,
        _lib.GDN_F32 if initial_state is None else _DT[initial_state.dtype], _DT[state_dtype],
        _lib.GDN_I64 if cu_seqlens is None else _IDT[cu_seqlens.dtype], dt_softplus, force_generic, dt_min, dt_max)
    lib = _lib.load()
    _launch(lib.gdn_scan_fwd, packed, dev)
    if check_errors:
        _launch(lib.gdn_chunk_check_device_error, ws.data_ptr(), dev)
    return y, fin


_scan_fwd_op = torch.library.custom_op("gdn_b200::scan_fwd", mutates_args=(), device_types="cuda")(_scan_fwd_impl)


@_scan_fwd_op.register_fake
def _(x, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_min, dt_max, initial_state, output_final_state, state_dtype,
      cu_seqlens, force_generic, check_errors):
    N = x.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1
    shape = (N, x.shape[2], x.shape[3], B.shape[3]) if output_final_state else (0,)
    return x.new_empty(x.shape), x.new_empty(shape, dtype=state_dtype)


def _scan_update_impl(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor],
                      z: Optional[Tensor], dt_bias: Optional[Tensor], dt_softplus: bool, dt_min: float, dt_max: float,
                      state: Tensor, ssm_state_indices: Optional[Tensor], check_errors: bool) -> Tensor:
    """One token per sequence; updates ``state`` in place and returns y."""
    N, H, P = x.shape
    G, S = B.shape[1], B.shape[2]
    dev = x.device
    (x, sx), (dt, sdt), (B, sb), (C, sc) = _packed_rows(x, 2), _packed_rows(dt, 1), _packed_rows(B, 2), _packed_rows(C, 2)
    z, sz = (None, 0) if z is None else _packed_rows(z, 2)
    y = torch.empty((N, H, P), dtype=x.dtype, device=dev)
    if N == 0:
        return y
    err = _err_word(dev)
    packed = _lib.pack_scan_update(
        x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _addr(D), _addr(z), _addr(dt_bias),
        state.data_ptr(), y.data_ptr(), _addr(ssm_state_indices), err.data_ptr(), N, state.shape[0],
        state.stride(0) if state.shape[0] > 1 else H * P * S, sx, sdt, sb, sc, sz, H, P, G, S, _DT[x.dtype], _DT[dt.dtype],
        _DT[state.dtype], _lib.GDN_I64 if ssm_state_indices is None else _IDT[ssm_state_indices.dtype], dt_softplus,
        dt_min, dt_max)
    _launch(_lib.load().gdn_scan_update, packed, dev)
    if check_errors:
        _raise_err_word(err)
    return y


_scan_update_op = torch.library.custom_op("gdn_b200::scan_update", mutates_args=("state",),
                                          device_types="cuda")(_scan_update_impl)


@_scan_update_op.register_fake
def _(x, dt, A, B, C, D, z, dt_bias, dt_softplus, dt_min, dt_max, state, ssm_state_indices, check_errors):
    return x.new_empty(x.shape)


def _check(name, lead, x, dt, A, B, C, D, z, dt_bias, dt_limit):
    shape, dtype = x.shape, x.dtype
    H = shape[-2]
    if dtype not in _DT:
        raise ValueError(f"{name}: x dtype {dtype} must be float32, bfloat16 or float16")
    if B.dim() != x.dim() or B.shape != C.shape or B.shape[:-2] != shape[:-2]:
        raise ValueError(f"{name}: B {tuple(B.shape)} and C {tuple(C.shape)} must be [{lead}, G, S]")
    if B.shape[-2] == 0 or H % B.shape[-2] != 0:
        raise ValueError(f"{name}: {H} heads are no multiple of {B.shape[-2]} groups")
    if B.dtype is not dtype or C.dtype is not dtype or (z is not None and z.dtype is not dtype):
        raise ValueError(f"{name}: x, B, C and z must share a dtype")
    if z is not None and z.shape != shape:
        raise ValueError(f"{name}: z {tuple(z.shape)} must match x {tuple(shape)}")
    if dt.shape != shape[:-1] or dt.dtype not in _DT:
        raise ValueError(f"{name}: dt {tuple(dt.shape)} {dt.dtype} must be {tuple(shape[:-1])} of a float type")
    for what, t in (("A", A), ("D", D), ("dt_bias", dt_bias)):
        if t is not None and (t.dim() != 1 or t.shape[0] != H):
            raise ValueError(f"{name}: {what} {tuple(t.shape)} must be ({H},), one value per head")
    lo, hi = float(dt_limit[0]), float(dt_limit[1])
    if not lo <= hi:
        raise ValueError(f"{name}: dt_limit {dt_limit} must be (least, most)")
    return lo, hi


def _no_grad(name, *ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no backward: call it under torch.no_grad() or on detached tensors")


def chunk_selective_scan(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    dt_limit: tuple[float, float] = (0.0, _INF),
    initial_state: torch.Tensor | None = None,
    output_final_state: bool = False,
    cu_seqlens: torch.LongTensor | None = None,
    *,
    state_dtype: torch.dtype = torch.float32,
    force_generic: bool = False,
    check_errors: bool = False,
):
    """Selective scan over prompts.

    x, z ``[B, T, H, P]``; dt ``[B, T, H]``; B, C ``[B, T, G, S]`` (head h uses
    group ``h // (H // G)``); A, D, dt_bias ``[H]``; initial_state
    ``[N, H, P, S]`` of any float type; with ``cu_seqlens [N + 1]`` the batch
    size is 1 and the tokens are N packed sequences (outputs of tokens outside
    them, of a padded batch, are zero).  Token rows may be strided (views of one
    projection).  ``dt_limit`` clamps the steps after softplus.
    Returns ``(y [B, T, H, P] in x's dtype, final_state [N, H, P, S] of
    state_dtype or None)``.

    bf16 with S of 64 or 128 and P a multiple of 64 runs on the tensor cores;
    other types and sizes (P, S <= 256) on an fp32 recurrence.
    ``check_errors=True`` synchronises and raises on a recorded device error.
    Serving only: inputs that require grad are refused."""
    _cuda("chunk_selective_scan", x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens)
    _no_grad("chunk_selective_scan", x, dt, A, B, C, D, z, dt_bias, initial_state)
    if x.dim() != 4:
        raise ValueError(f"chunk_selective_scan: x {tuple(x.shape)} must be [B, T, H, P]")
    lo, hi = _check("chunk_selective_scan", "B, T", x, dt, A, B, C, D, z, dt_bias, dt_limit)
    if cu_seqlens is not None and x.shape[0] != 1:
        raise ValueError("cu_seqlens requires batch size 1 (packed sequences)")
    if state_dtype not in _DT:
        raise ValueError(f"chunk_selective_scan: state_dtype {state_dtype} must be float32, bfloat16 or float16")
    cu, _ = _idx(cu_seqlens)
    if cu is not None:
        cu = cu.contiguous()
    N = x.shape[0] if cu is None else cu.shape[0] - 1
    shape = (N, x.shape[2], x.shape[3], B.shape[3])
    if initial_state is not None:
        if tuple(initial_state.shape) != shape or initial_state.dtype not in _DT:
            raise ValueError(f"initial_state must be {shape} of a float type, got {tuple(initial_state.shape)} "
                             f"{initial_state.dtype}")
        initial_state = initial_state.contiguous()
    op = (_scan_fwd_impl if _plain(x, dt, A, B, C, D, z, dt_bias, initial_state, cu) else torch.ops.gdn_b200.scan_fwd)
    y, fin = op(x, dt, _f32(A), B, C, _f32(D), z, _f32(dt_bias), bool(dt_softplus), lo, hi, initial_state,
                bool(output_final_state), state_dtype, cu, bool(force_generic), bool(check_errors))
    return y, (fin if output_final_state else None)


def selective_scan_update(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    dt_softplus: bool = False,
    dt_limit: tuple[float, float] = (0.0, _INF),
    state: torch.Tensor | None = None,
    ssm_state_indices: torch.Tensor | None = None,
    *,
    check_errors: bool = False,
):
    """One decode token per sequence, on a cache that is updated in place.

    x, z ``[N, H, P]``; dt ``[N, H]``; B, C ``[N, G, S]``; A, D, dt_bias
    ``[H]``; state ``[slots, H, P, S]`` of any float type (lines packed, the
    distance between lines free); token i works on line
    ``ssm_state_indices[i]`` (int32 / int64), or on line i without indices.  A
    negative index is padding: output zero, no line touched; one past the
    cache is treated the same and, with ``check_errors=True`` (synchronises),
    raises :class:`GdnError`.  The indices of one call must differ.  Returns
    ``(y [N, H, P], state)``."""
    if state is None:
        raise ValueError("selective_scan_update: state is required")
    _cuda("selective_scan_update", x, dt, A, B, C, D, z, dt_bias, state, ssm_state_indices)
    _no_grad("selective_scan_update", x, dt, A, B, C, D, z, dt_bias, state)
    if x.dim() != 3:
        raise ValueError(f"selective_scan_update: x {tuple(x.shape)} must be [N, H, P]")
    lo, hi = _check("selective_scan_update", "N", x, dt, A, B, C, D, z, dt_bias, dt_limit)
    N, H, P = x.shape
    S = B.shape[2]
    if state.dim() != 4 or tuple(state.shape[1:]) != (H, P, S) or state.dtype not in _DT:
        raise ValueError(f"selective_scan_update: state {tuple(state.shape)} {state.dtype} must be [slots, {H}, {P}, {S}] "
                         "of a float type")
    want = 1
    for n, st in zip(reversed(state.shape[1:]), reversed(state.stride()[1:])):
        if n != 1 and st != want:
            raise ValueError("selective_scan_update: a cache line [H, P, S] must be packed")
        want *= n
    if state.shape[0] > 1 and state.stride(0) < want:
        raise ValueError("selective_scan_update: cache lines must not overlap")
    idx = ssm_state_indices
    if idx is None:
        if state.shape[0] < N:
            raise ValueError(f"selective_scan_update: {state.shape[0]} cache lines for {N} tokens")
    else:
        if tuple(idx.shape) != (N,):
            raise ValueError(f"selective_scan_update: ssm_state_indices {tuple(idx.shape)} must be ({N},)")
        idx = _idx(idx)[0].contiguous()
    op = _scan_update_impl if _plain(x, dt, A, B, C, D, z, dt_bias, state, idx) else torch.ops.gdn_b200.scan_update
    y = op(x, dt, _f32(A), B, C, _f32(D), z, _f32(dt_bias), bool(dt_softplus), lo, hi, state, idx, bool(check_errors))
    return y, state
