"""Causal depthwise conv1d ops, drop-in for ``torch_mlu_ops.triton_ops``
(``causal_conv1d``, ``causal_conv1d_fn``) and ``triton.conv``
(``causal_conv1d_update``): the short convolution over the q/k/v channels in
front of the GDN layer of Qwen3-Next.

Same names, argument order, keyword names, defaults and return values as the
reference (``triton_ops.py:287-459``, ``triton/conv/ops.py:584-644``); the
work runs in ``libgdn_b200.so`` (``gdn_conv.cu``) through its C ABI.  There is
no CPU or Triton path.

Differences from the reference, all supersets or stricter checks:

* ``causal_conv1d_fn`` skips a sequence whose cache line is ``pad_slot_id``
  as well as ``null_block_id`` (the reference indexes line -1), and writes
  zeros for the tokens of skipped sequences (the reference leaves them
  unwritten); ``has_initial_state=None`` means no initial state and
  ``cache_indices=None`` maps sequence i to line i.
* Products are accumulated in fp32 from the inputs as given (the reference
  first casts x to the ``conv_states`` dtype and multiplies in that dtype).
* Prefix caching (``block_idx_*``, ``initial_state_idx``,
  ``num_computed_tokens``, ``block_size_to_align``) follows the reference
  kernel; ``block_size_to_align`` must be a positive multiple of 64 (the
  reference checks that only with ``validate_data``).
* An unknown ``activation`` string raises ``ValueError`` (the reference
  kernels silently apply none).
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import _lib
from .gdn import _DT, _IDT, _addr, _cuda, _first_order, _launch, _plain, _ptr, _stream


def _act(activation):
    if activation in (None, False):
        return _lib.GDN_ACT_NONE
    if activation is True or activation in ("silu", "swish"):
        return _lib.GDN_ACT_SILU
    raise ValueError(f"[CausalConv1d] unsupported activation {activation!r} (None, 'silu' or 'swish')")


def _fdt(t, name):
    if t.dtype not in _DT:
        raise ValueError(f"[CausalConv1d] {name} dtype {t.dtype} must be float32, bfloat16 or float16")
    return _DT[t.dtype]


def _fn_args(x, weight, bias, conv_states, query_start_loc, cache_indices, has_initial_state, activation,
             pad_slot_id, null_block_id, block_idx_first_scheduled_token, block_idx_last_scheduled_token,
             initial_state_idx, num_computed_tokens, block_size_to_align, out):
    """``gdn_conv1d_fn_args`` for channel-last x ``(dim, tokens)`` (and ``out``
    of the same layout, or None for the fused prefill); returns the struct and
    the converted tensors it points into (keep them alive until the launch)."""
    dim, total = x.shape
    W = weight.shape[1]
    if W < 2:
        raise ValueError("[CausalConv1d] weight.shape[-1] must be at least 2")
    if conv_states.dim() != 3 or conv_states.shape[1] != dim or conv_states.shape[2] < W - 1:
        raise ValueError(f"[CausalConv1d] conv_states {tuple(conv_states.shape)} must be (lines, {dim}, >= {W - 1})")
    if conv_states.stride(1) != 1:
        raise ValueError("[CausalConv1d] conv_states must have unit stride along dim")
    w = weight.contiguous()
    b = None if bias is None else bias.to(w.dtype).contiguous()
    qsl = (query_start_loc if query_start_loc.dtype in _IDT else query_start_loc.to(torch.int32)).contiguous()
    batch = qsl.numel() - 1
    apc = block_idx_last_scheduled_token is not None
    ci = None
    idx_dt = _lib.GDN_I32
    if cache_indices is not None:
        ci = (cache_indices if cache_indices.dtype in _IDT else cache_indices.to(torch.int32)).contiguous()
        idx_dt = _IDT[ci.dtype]
        if ci.dim() not in (1, 2) or ci.shape[0] != batch or (ci.dim() == 2 and not apc):
            raise ValueError(f"[CausalConv1d] cache_indices must be ({batch},) (or ({batch}, blocks) "
                             "with prefix caching)")
    blocks = [None] * 4
    if apc:
        if cache_indices is None:
            raise ValueError("[CausalConv1d] prefix caching needs cache_indices")
        if ci.dim() == 1:
            ci = ci[:, None]
        blocks = [t if t is None else t.to(torch.int32).contiguous()
                  for t in (block_idx_first_scheduled_token, block_idx_last_scheduled_token,
                            initial_state_idx, num_computed_tokens)]
        if any(t is None for t in blocks):
            raise ValueError("[CausalConv1d] prefix caching needs block_idx_first_scheduled_token, "
                             "block_idx_last_scheduled_token, initial_state_idx and num_computed_tokens")
    hi = None
    if has_initial_state is not None:
        hi = has_initial_state.to(torch.bool).contiguous()
        if hi.numel() != batch:
            raise ValueError(f"[CausalConv1d] has_initial_state must be ({batch},)")
    args = _lib.Conv1dFnArgs(
        x=_ptr(x), out=_ptr(out), weight=_ptr(w), bias=_ptr(b), conv_states=_ptr(conv_states),
        query_start_loc=_ptr(qsl), cache_indices=_ptr(ci), has_initial_state=_ptr(hi),
        stride_x_token=x.stride(1) if total > 1 else dim,
        stride_o_token=(out.stride(1) if total > 1 else dim) if out is not None else 0,
        stride_state_seq=conv_states.stride(0), stride_state_tok=conv_states.stride(2),
        num_cache_lines=conv_states.shape[0], batch=batch, dim=dim, total_tokens=total,
        pad_slot_id=int(pad_slot_id), null_block_id=0 if null_block_id is None else int(null_block_id),
        has_null_block=0 if null_block_id is None else 1, W=W,
        x_dtype=_fdt(x, "x"), w_dtype=_fdt(w, "weight"), state_dtype=_fdt(conv_states, "conv_states"),
        qsl_dtype=_IDT[qsl.dtype], idx_dtype=idx_dt, activation=_act(activation),
        block_idx_first=_ptr(blocks[0]), block_idx_last=_ptr(blocks[1]), initial_state_idx=_ptr(blocks[2]),
        num_computed_tokens=_ptr(blocks[3]), stride_cache_indices=ci.stride(0) if ci is not None else 0,
        block_size_to_align=int(block_size_to_align or 0), apc_dtype=_lib.GDN_I32)
    return args, (w, b, qsl, ci, hi, blocks)


@functools.lru_cache(maxsize=256)
def _bwd_workspace(B, T, N, D, W, x_dtype):
    """Bytes of gdn_causal_conv1d_bwd's workspace: they depend on the shapes alone."""
    args = _lib.Conv1dBwdArgs(B=B, T=T, N=N, D=D, stride_x_token=D, stride_dy_token=D, W=W, x_dtype=x_dtype)
    if N != B:
        args.cu_seqlens, args.cu_dtype = ctypes.c_void_p(16), _lib.GDN_I64  # packed: only whether it is there counts
    n = _lib.load().gdn_causal_conv1d_bwd_workspace_size(ctypes.byref(args))
    if n == 0:
        _lib.check(_lib.GDN_ERR_INVALID)
    return n


def _token_rows(t):
    """(tensor, distance between its B*T token rows) of ``t [B, T, D]``: in
    place when only the rows are strided (a view of one projection), else a
    packed copy."""
    B, T, D = t.shape
    if not t.is_contiguous() and t.stride(2) == 1:
        row = t.stride(1) if T > 1 else t.stride(0) if B > 1 else D
        if row >= D and (B == 1 or t.stride(0) == T * row):
            return t, row
    return t.contiguous(), D


def _conv1d_bwd_impl(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], dy: torch.Tensor,
                     initial_state: Optional[torch.Tensor], activation: int,
                     cu_seqlens: Optional[torch.Tensor]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor,
                                                                  torch.Tensor]:
    """Returns ``(dx, dweight, dbias, dinitial_state)``, the last two empty
    where there is no bias or initial state."""
    B, T, D = x.shape
    W = weight.shape[1]
    N = B if cu_seqlens is None else cu_seqlens.numel() - 1
    dev = x.device

    (x, sx), (dy, sdy) = _token_rows(x), _token_rows(dy)
    dx = torch.empty(B, T, D, dtype=x.dtype, device=dev)
    dw = torch.empty_like(weight)
    db = torch.empty(0 if bias is None else D, dtype=weight.dtype, device=dev)
    dh = torch.empty((0,) if initial_state is None else initial_state.shape,
                     dtype=x.dtype if initial_state is None else initial_state.dtype, device=dev)
    cu_dt = _lib.GDN_I64 if cu_seqlens is None else _IDT[cu_seqlens.dtype]
    xt, wt = _DT[x.dtype], _DT[weight.dtype]
    nbytes = _bwd_workspace(B, T, N, D, W, xt)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    packed = _lib.pack_conv1d_bwd(
        x.data_ptr(), weight.data_ptr(), _addr(bias), _addr(initial_state), dy.data_ptr(), dx.data_ptr(), dw.data_ptr(),
        0 if bias is None else db.data_ptr(), 0 if initial_state is None else dh.data_ptr(), _addr(cu_seqlens),
        ws.data_ptr(), nbytes, B, T, N, D, sx, sdy, W, xt, wt,
        _lib.GDN_F32 if initial_state is None else _DT[initial_state.dtype], cu_dt, activation)
    _launch(_lib.load().gdn_causal_conv1d_bwd, packed, dev)
    return dx, dw, db, dh


_conv1d_bwd_op = torch.library.custom_op("gdn_b200::causal_conv1d_bwd", mutates_args=(),
                                         device_types="cuda")(_conv1d_bwd_impl)


@_conv1d_bwd_op.register_fake
def _(x, weight, bias, dy, initial_state, activation, cu_seqlens):
    return (x.new_empty(x.shape), weight.new_empty(weight.shape),
            weight.new_empty((0,) if bias is None else bias.shape),
            x.new_empty((0,)) if initial_state is None else initial_state.new_empty(initial_state.shape))


def causal_conv1d_bwd(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None,
    dy: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    activation: str | None = None,
    cu_seqlens: torch.Tensor | None = None,
):
    """Functional gradient of :func:`causal_conv1d`: x, dy ``[B, T, D]`` (token
    rows may be strided), the other arguments as the forward took them.
    Returns ``(dx, dweight, dbias, dinitial_state)`` in the dtypes of what they
    are the gradients of, the last two None where there is no bias or initial
    state.  The residual's gradient is dy itself."""
    act = _act(activation)
    if x.dim() != 3 or dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"[CausalConv1d] dy {tuple(dy.shape)} {dy.dtype} must match x {tuple(x.shape)} {x.dtype} [B, T, D]")
    if weight.dim() != 2 or weight.shape[0] != x.shape[2]:
        raise ValueError("[CausalConv1d] x.shape[-1] must be equal to weight.shape[0].")
    if bias is not None and tuple(bias.shape) != (x.shape[2],):
        raise ValueError(f"[CausalConv1d] bias {tuple(bias.shape)} must be ({x.shape[2]},)")
    _cuda("causal_conv1d_bwd", x, weight, bias, dy, initial_state, cu_seqlens)
    _fdt(x, "x"), _fdt(weight, "weight")
    if initial_state is not None:
        _fdt(initial_state, "initial_state")
    B, T, D = x.shape
    W = weight.shape[1]
    cu = None
    N = B
    if cu_seqlens is not None:
        if B != 1:
            raise ValueError("[CausalConv1d] cu_seqlens requires batch size 1 (packed sequences)")
        cu = (cu_seqlens if cu_seqlens.dtype in _IDT else cu_seqlens.to(torch.int64)).contiguous()
        N = cu.numel() - 1
    if initial_state is not None and tuple(initial_state.shape) != (N, D, W):
        raise ValueError(f"[CausalConv1d] initial_state {tuple(initial_state.shape)} must be [N, D, W] = {(N, D, W)}")
    op = _conv1d_bwd_impl if _plain(x, weight, bias, dy, initial_state, cu) else torch.ops.gdn_b200.causal_conv1d_bwd
    w, b = weight.contiguous(), bias
    if bias is not None and bias.dtype != weight.dtype:
        # the forward's values, held in fp32: dweight and dbias come in one type, and each is rounded to its own once
        w, b = w.float(), bias.to(weight.dtype).float()
    dx, dw, db, dh = op(x, w, None if b is None else b.contiguous(), dy,
                        None if initial_state is None else initial_state.contiguous(), act, cu)
    return (dx, dw.to(weight.dtype), None if bias is None else db.to(bias.dtype), None if initial_state is None else dh)


class CausalConv1dFunction(torch.autograd.Function):
    """Autograd node of :func:`causal_conv1d`: saves its inputs and recomputes
    the pre-activations in the backward."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, initial_state, activation, cu_seqlens):
        with torch.no_grad():
            y, _ = causal_conv1d(x, weight, bias, residual, initial_state, activation=activation, cu_seqlens=cu_seqlens)
        ctx.save_for_backward(x, weight, bias, initial_state, cu_seqlens)
        ctx.activation, ctx.residual_dtype = activation, None if residual is None else residual.dtype
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight, bias, initial_state, cu = ctx.saved_tensors
        dx = dw = db = dh = None
        if any(ctx.needs_input_grad[i] for i in (0, 1, 2, 4)):  # the residual's gradient is dy
            dx, dw, db, dh = causal_conv1d_bwd(x, weight, bias, dy, initial_state, ctx.activation, cu)
        return dx, dw, db, None if ctx.residual_dtype is None else dy.to(ctx.residual_dtype), dh, None, None


def causal_conv1d(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    initial_state: torch.Tensor | None = None,
    output_final_state: bool | None = False,
    activation: str | None = None,
    backend: str | None = "triton",
    cu_seqlens: torch.Tensor | None = None,
    cu_seqlens_cpu: torch.LongTensor | None = None,
    chunk_indices: torch.LongTensor | None = None,
    cp_context=None,
    **kwargs,
):
    """y = act(conv(x) + bias) + residual over x ``[B, T, D]`` with weight
    ``[D, W]``; ``initial_state [N, D, W]`` supplies the tokens before each
    sequence (column j = token j - W).  Returns ``(y, None)``
    (``triton_ops.py:287-363``).  ``backend`` is accepted for signature
    compatibility ('triton' is the reference's only value; the work runs in
    CUDA here).  Differentiable once in x, weight, bias, residual and initial_state
    (:func:`causal_conv1d_bwd`)."""
    if cp_context is not None:
        raise ValueError("[CausalConv1d] CP Context not supported.")
    if output_final_state is True:
        raise ValueError("[CausalConv1d] output_final_state true not supported.")
    if backend != "triton":
        raise ValueError(f"[CausalConv1d] Unsupported backend: {backend}")
    if weight is None:
        raise ValueError("[CausalConv1d] weight is required")
    if x.dim() != 3:
        raise ValueError(f"[CausalConv1d] x must be [B, T, D] (got {tuple(x.shape)})")
    if x.shape[-1] != weight.shape[0]:
        raise ValueError("[CausalConv1d] x.shape[-1] must be equal to weight.shape[0].")
    _cuda("causal_conv1d", x, weight, bias, residual, initial_state, cu_seqlens)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (x, weight, bias, residual, initial_state)):
        return CausalConv1dFunction.apply(x, weight, bias, residual, initial_state, activation, cu_seqlens), None
    B, T, D = x.shape
    W = weight.shape[1]
    x = x.contiguous()
    w = weight.contiguous()
    b = None if bias is None else bias.to(w.dtype).contiguous()
    r = None if residual is None else residual.to(x.dtype).contiguous()
    if r is not None and r.shape != x.shape:
        raise ValueError(f"[CausalConv1d] residual {tuple(r.shape)} must match x {tuple(x.shape)}")
    cu, cu_dt = None, _lib.GDN_I64
    N = B
    if cu_seqlens is not None:
        cu = cu_seqlens if cu_seqlens.dtype in _IDT else cu_seqlens.to(torch.int64)
        cu_dt = _IDT[cu.dtype]
        N = cu.numel() - 1
    h0 = None if initial_state is None else initial_state.contiguous()
    if h0 is not None and tuple(h0.shape) != (N, D, W):
        raise ValueError(f"[CausalConv1d] initial_state {tuple(h0.shape)} must be [N, D, W] = {(N, D, W)}")
    y = torch.empty_like(x)
    args = _lib.Conv1dArgs(
        x=_ptr(x), weight=_ptr(w), bias=_ptr(b), residual=_ptr(r), initial_state=_ptr(h0), y=_ptr(y),
        cu_seqlens=_ptr(cu), B=B, T=T, N=N, D=D, W=W, x_dtype=_fdt(x, "x"), w_dtype=_fdt(w, "weight"),
        state_dtype=_fdt(h0, "initial_state") if h0 is not None else _lib.GDN_F32, cu_dtype=cu_dt,
        activation=_act(activation))
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().gdn_causal_conv1d_fwd(args, _stream(x.device)))
    return y, None


def causal_conv1d_fn(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None,
    conv_states: torch.Tensor,
    query_start_loc: torch.Tensor,
    cache_indices: torch.Tensor | None = None,
    has_initial_state: torch.Tensor | None = None,
    activation: str | None = "silu",
    pad_slot_id: int = -1,
    null_block_id: int = 0,
    block_idx_first_scheduled_token: torch.Tensor | None = None,
    block_idx_last_scheduled_token: torch.Tensor | None = None,
    initial_state_idx: torch.Tensor | None = None,
    num_computed_tokens: torch.Tensor | None = None,
    block_size_to_align=0,
    metadata=None,
    validate_data=False,
):
    """Continuous-batching causal conv1d (``triton_ops.py:366-459``).

    x ``(dim, total_tokens)`` channel-last (``x.stride(0) == 1``; other
    layouts are copied), weight ``(dim, W)`` with W <= 4, conv_states
    ``(lines, dim, >= W-1)`` with unit channel stride, updated in place to
    each processed sequence's last W-1 inputs.  Returns ``out`` shaped and
    strided like x."""
    if weight is not None and x.shape[0] != weight.shape[0]:
        raise ValueError("[CausalConv1d] x.shape[0] must be equal to weight.shape[0].")
    if weight is not None and weight.shape[-1] > 4:
        raise ValueError("[CausalConv1d] weight.shape[-1] must be less than or equal to 4.")
    if weight is None or x.dim() != 2:
        raise ValueError("[CausalConv1d] x must be (dim, tokens) and weight (dim, width)")
    _cuda("causal_conv1d_fn", x, weight, bias, conv_states, query_start_loc, cache_indices, has_initial_state)
    dim, total = x.shape
    if x.stride(0) != 1 and total > 1:
        x = x.t().contiguous().t()  # channel-last storage [tokens, dim]
    out = torch.empty_like(x)
    if out.stride(0) != 1 and total > 1:
        out = torch.empty(total, dim, dtype=x.dtype, device=x.device).t()
    args, _keep = _fn_args(x, weight, bias, conv_states, query_start_loc, cache_indices, has_initial_state,
                           activation, pad_slot_id, null_block_id, block_idx_first_scheduled_token,
                           block_idx_last_scheduled_token, initial_state_idx, num_computed_tokens,
                           block_size_to_align, out)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().gdn_causal_conv1d_fn(args, _stream(x.device)))
    return out


def causal_conv1d_update(
    x: torch.Tensor,
    cache: torch.Tensor,
    residual: torch.Tensor | None = None,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    activation: str | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One decode token per sequence (``triton/conv/ops.py:584-644``).

    x ``(N, D)``, ``(N, 1, D)`` or ``(1, N, D)``; cache ``[N, D, W]``
    (contiguous) holds the last W inputs and is shifted in place.  Returns
    ``(y, cache)`` with y shaped like x."""
    if x.dim() == 2:
        N, D = x.shape
        sxn = x.stride(0)
    elif x.dim() == 3 and x.shape[0] == 1:
        N, D = x.shape[1], x.shape[2]
        sxn = x.stride(1)
    elif x.dim() == 3:
        N, D = x.shape[0], x.shape[2]
        sxn = x.stride(0)
    else:
        raise ValueError(f"Unsupported input shape: {x.shape}")
    _cuda("causal_conv1d_update", x, cache, residual, weight, bias)
    if x.stride(-1) != 1 or (N > 1 and sxn < D):
        x = x.contiguous()
        sxn = D
    W = weight.shape[1] if weight is not None else (cache.shape[-1] if cache is not None else None)
    if W is None:
        raise ValueError("[CausalConv1d] weight or cache is required")
    if cache is not None:
        if tuple(cache.shape) != (N, D, W) or not cache.is_contiguous():
            raise ValueError(f"[CausalConv1d] cache must be a contiguous [N, D, W] = {(N, D, W)} tensor")
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.to(w.dtype if w is not None else bias.dtype).contiguous()
    r = None if residual is None else residual.to(x.dtype).reshape(N, D).contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    args = _lib.Conv1dUpdateArgs(
        x=_ptr(x), cache=_ptr(cache), residual=_ptr(r), weight=_ptr(w), bias=_ptr(b), y=_ptr(y),
        stride_x_n=sxn if N > 1 else D, N=N, D=D, W=W, x_dtype=_fdt(x, "x"),
        cache_dtype=_fdt(cache, "cache") if cache is not None else _lib.GDN_F32,
        w_dtype=_fdt(w if w is not None else (b if b is not None else x), "weight"), activation=_act(activation))
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().gdn_causal_conv1d_update(args, _stream(x.device)))
    return y, cache
