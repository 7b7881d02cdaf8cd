"""Linear attention with a decay per head: S <- a S + k v^T, o = scale S^T q.

The single-token and the chunked form, on the states, head layouts and dtypes
of the gated delta-rule entry points in ``api``; states may be pages of a pool
(see ``pages``).  Every call goes through the C ABI; there is no fallback.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import GDNError
from .api import _dt, _require_cuda, _same_device, check_device_status, status_word


def _launch(fn, args, dev: torch.device, what: str) -> None:
    """Calls a launcher on the tensors' device and that device's current stream."""
    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        rc = fn(ctypes.byref(args), stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(ctypes.byref(args), stream)
    if rc:
        _lib.check(rc, what)


def _check_io(q, k, v, out) -> None:
    if k.dtype != q.dtype or v.dtype != q.dtype or out.dtype != q.dtype:
        raise GDNError("q, k, v and out must share one dtype (bf16 or f16)", 4)
    if out.shape != v.shape:
        raise GDNError(f"out must have the shape of v, {tuple(v.shape)}, got {tuple(out.shape)}", 2)
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        if t.stride(-1) != 1:
            raise GDNError(f"{name}: the innermost dimension must be contiguous", 3)


def _check_states(name: str, t, page: tuple) -> int:
    """Elements between the pages of a pool [P, Hv, d_k, d_v]; raises on any other layout."""
    if t.dtype != torch.float32 or t.dim() != 4 or tuple(t.shape[1:]) != page:
        raise GDNError(f"{name} must be fp32 [P, Hv, d_k, d_v] with pages of {page}, got "
                       f"{t.dtype} {tuple(t.shape)}", 2)
    if t.stride()[1:] != (page[1] * page[2], page[2], 1):
        raise GDNError(f"{name}: each page must be contiguous", 3)
    n = page[0] * page[1] * page[2]
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), n)


def _check_index(index, rows: int, pools, name: str = "index") -> None:
    if index is None:
        for pool in pools:
            if pool is not None and pool.shape[0] != rows:
                raise GDNError(f"without index the states must have one page per sequence ({rows}), "
                               f"got {pool.shape[0]}", 2)
        return
    if index.dtype != torch.int32 or tuple(index.shape) != (rows,) or not index.is_contiguous():
        raise GDNError(f"{name} must be a contiguous int32 [{rows}] tensor", 2)


def lin_decode(q, k, v, g, state, *, scale: float = 1.0, out=None, gate: str = "log",
               state_out=None, index=None, check: bool = False) -> torch.Tensor:
    """One token of linear attention with a decay per head; ``state`` is updated
    in place (or written to ``state_out``, same pages).  Returns o [B, Hv, d_v].

    q, k [B, Hqk, d_k] bf16/f16 with d_k in {64, 128, 256}; v [B, Hv, d_v], d_v a
    multiple of 64; g [B, Hv], or [Hv] for a fixed decay per head (any float
    dtype; ``gate='log'`` means decay = exp(g)); state fp32 [B, Hv, d_k, d_v].

    With ``index`` (int32 [B] on the device) ``state`` is a pool of P pages and
    row b uses page index[b].  A negative index is an idle row: its output is
    zero and no state is touched.  An index >= P, or one that an earlier row
    holds, is treated as idle and reported (``check=True`` synchronises and
    raises).  Rows without a page leave ``state_out`` as it was.
    """
    dev = _require_cuda(q, k, v, g, state)
    if out is None:
        out = torch.empty(v.shape, dtype=q.dtype, device=dev)
    if state_out is None:
        state_out = state
    _same_device(q, out=out, state_out=state_out, index=index)
    a = _decode_args(q, k, v, g, state, state_out, out, index, scale, gate)
    a.status = status_word(dev).data_ptr()
    _launch(_lib.load().lin_decode_launch, a, dev, "lin_decode")
    if check:
        check_device_status(dev)
    return out


def _decode_args(q, k, v, g, state, state_out, out, index, scale, gate) -> _lib.LinDecodeArgs:
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[0] != q.shape[0]:
        raise GDNError("q, k must be [B, Hqk, d_k] and v [B, Hv, d_v]", 2)
    B, Hqk, dk = q.shape
    _, Hv, dv = v.shape
    _check_io(q, k, v, out)
    g_sb = 0
    if g.dim() == 2:
        g_sb = g.stride(0)
    if tuple(g.shape) not in ((B, Hv), (Hv,)):
        raise GDNError(f"g must be [B, Hv] = {(B, Hv)} or [Hv], got {tuple(g.shape)}", 2)
    if gate not in ("log", "linear"):
        raise GDNError("gate must be 'log' (decay = exp(g)) or 'linear' (decay = g)", 4)
    page = (Hv, dk, dv)
    in_sp, out_sp = _check_states("state", state, page), _check_states("state_out", state_out, page)
    if state_out.shape[0] != state.shape[0]:
        raise GDNError("state_out must have as many pages as state", 2)
    _check_index(index, B, (state,))
    return _lib.LinDecodeArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), state.data_ptr(),
        state_out.data_ptr(), out.data_ptr(), index.data_ptr() if index is not None else None,
        q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
        out.stride(0), out.stride(1), g_sb, g.stride(-1), in_sp, out_sp,
        B, Hqk, Hv, dk, dv, state.shape[0], _dt(q, "q"), _dt(g, "g"),
        _lib.GATE_LOG if gate == "log" else _lib.GATE_LINEAR, scale, None)


def lin_prefill(q, k, v, g, initial_state=None, *, scale: float = 1.0, cu_seqlens=None,
                index=None, out=None, final_state=None, workspace=None, check: bool = False):
    """Linear attention with a decay per head over T tokens, in chunks: the same
    as T calls of :func:`lin_decode` with log gates.  Returns (o, final_state).

    q, k [B, T, Hqk, d_k] bf16/f16 with d_k in {64, 128}; v [B, T, Hv, d_v], d_v
    a multiple of 64; g [B, T, Hv], or [Hv] for a fixed decay per head;
    initial_state, final_state fp32 [B, Hv, d_k, d_v] (``final_state`` may be
    the ``initial_state`` tensor: updated in place).

    ``cu_seqlens`` (int32 [N + 1] on the device) packs N sequences end to end
    into a batch of one; sequence n is rows cu_seqlens[n] .. cu_seqlens[n+1] - 1,
    possibly none, and rows outside every sequence are left as they were.

    With ``index`` (int32 on the device, one entry per sequence) the states are
    pools: sequence n starts from page index[n] of ``initial_state`` and leaves
    its state in page index[n] of ``final_state`` (required then, unless
    ``initial_state`` is to be updated in place).  A negative index starts from
    zero and keeps no state.  Indices out of range or taken by an earlier
    sequence, and offsets that are out of range or descend, are reported
    (``check=True``).  q, k, v and out may be strided views whose rows are
    contiguous and 16-byte aligned.
    """
    dev = _require_cuda(q, k, v, g)
    if out is None:
        out = torch.empty(v.shape, dtype=q.dtype, device=dev)
    if final_state is None:
        if index is not None:
            if initial_state is None:
                raise GDNError("with index, pass the pool as final_state or initial_state", 1)
            final_state = initial_state
        elif v.dim() == 4 and q.dim() == 4:
            rows = v.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
            final_state = torch.empty((rows, v.shape[2], q.shape[3], v.shape[3]),
                                      dtype=torch.float32, device=dev)
    _same_device(q, initial_state=initial_state, final_state=final_state, out=out,
                 cu_seqlens=cu_seqlens, index=index)
    a = _prefill_args(q, k, v, g, initial_state, final_state, out, cu_seqlens, index, scale)
    a.status = status_word(dev).data_ptr()
    L = _lib.load()
    need = L.lin_prefill_workspace_size(ctypes.byref(a))
    if need:
        # from the allocator on the current stream, so that calls on other streams
        # and captured graphs have workspaces of their own
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        elif workspace.device != dev or not workspace.is_contiguous():
            raise GDNError(f"workspace must be a contiguous tensor on {dev}", 2)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _launch(L.lin_prefill_launch, a, dev, "lin_prefill")
    if check:
        check_device_status(dev)
    return out, final_state


def _prefill_args(q, k, v, g, initial_state, final_state, out, cu_seqlens, index,
                  scale) -> _lib.LinPrefillArgs:
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:2] != q.shape[:2]:
        raise GDNError("q, k must be [B, T, Hqk, d_k] and v [B, T, Hv, d_v]", 2)
    B, T, Hqk, dk = q.shape
    Hv, dv = v.shape[2:]
    _check_io(q, k, v, out)
    if tuple(g.shape) == (B, T, Hv):
        g_s = g.stride()
    elif tuple(g.shape) == (Hv,):
        g_s = (0, 0, g.stride(0))
    else:
        raise GDNError(f"g must be [B, T, Hv] = {(B, T, Hv)} or [Hv], got {tuple(g.shape)}", 2)
    seqs = B
    if cu_seqlens is not None:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 \
                or not cu_seqlens.is_contiguous():
            raise GDNError("cu_seqlens must be a contiguous int32 [N + 1] tensor", 2)
        if B != 1:
            raise GDNError("packed sequences (cu_seqlens) need a batch of one", 2)
        seqs = cu_seqlens.numel() - 1
    page = (Hv, dk, dv)
    fin_sp, in_sp = _check_states("final_state", final_state, page), 0
    if initial_state is not None:
        in_sp = _check_states("initial_state", initial_state, page)
        if initial_state.shape[0] != final_state.shape[0]:
            raise GDNError("initial_state and final_state must have as many pages", 2)
    _check_index(index, seqs, (initial_state, final_state))
    return _lib.LinPrefillArgs(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
        initial_state.data_ptr() if initial_state is not None else None, final_state.data_ptr(),
        out.data_ptr(), cu_seqlens.data_ptr() if cu_seqlens is not None else None,
        index.data_ptr() if index is not None else None,
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *g_s, in_sp, fin_sp,
        seqs, T, Hqk, Hv, dk, dv, final_state.shape[0], _dt(q, "q"), _dt(g, "g"), scale,
        None, 0, None)
