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
from .api import _dt, _status_words, check_device_status, status_word


# the current stream's handle without a Stream object around it (1.2 us less per call)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") \
    else lambda dev: torch.cuda.current_stream(dev).cuda_stream
_DECODE = _lib.Packed(_lib.LinDecodeArgs, "lin_decode_launch")
_PREFILL = _lib.Packed(_lib.LinPrefillArgs, "lin_prefill_launch")
_FLOAT_MAX = torch.finfo(torch.float32).max
_UNCUT = 896  # tokens up to which no prefill is cut in time: no workspace (and 1 us less to ask for it)
_LOG, _LINEAR = _lib.GATE_LOG, _lib.GATE_LINEAR


def _on(first, *others) -> int:
    """The CUDA device that all tensors (None = absent) are on."""
    dev = first.get_device()
    if dev < 0:
        raise GDNError("tensors must be CUDA tensors (there is no CPU implementation)", 6)
    for t in others:
        if t is not None and t.get_device() != dev:
            raise GDNError(f"all tensors must be on cuda:{dev}, got {t.device}", 2)
    return dev


def _status(dev: int) -> int:
    w = _status_words.get(dev)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            # the word outlives any graph, so it cannot come from a graph's memory
            raise GDNError(f"the first call on cuda:{dev} cannot be captured: call once before", 2)
        w = status_word(dev)
    return w.data_ptr()


def _check_scale(scale) -> None:
    if not -_FLOAT_MAX <= scale <= _FLOAT_MAX:
        raise GDNError(f"scale must be a finite float, got {scale}", 2)


def _launch(packed, args: bytes, dev: int, what: str) -> None:
    """Calls a launcher on the tensors' device and that device's current stream."""
    stream = _raw_stream(dev)
    if torch.cuda.current_device() == dev:
        rc = packed.call(args, stream)
    else:
        with torch.cuda.device(dev):
            rc = packed.call(args, stream)
    if rc:
        _lib.check(rc, what)


def _check_io(q, k, v, out) -> int:
    """q's element type, which k, v and out share."""
    dt = q.dtype
    if k.dtype is not dt or v.dtype is not dt or out.dtype is not dt:
        raise GDNError("q, k, v and out must share one dtype (bf16 or f16)", 4)
    if out.shape != v.shape:
        raise GDNError(f"out must have the shape of v, {tuple(v.shape)}, got {tuple(out.shape)}", 2)
    return _dt(q, "q")


def _check_rows(**strides) -> None:
    for name, s in strides.items():
        if s[-1] != 1:
            raise GDNError(f"{name}: the innermost dimension must be contiguous", 3)


def _check_states(name: str, t, Hv: int, dk: int, dv: int) -> int:
    """Elements between the pages of a pool [P, Hv, d_k, d_v]; raises on any other layout."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not torch.float32 or len(shape) != 4 or shape[1:] != (Hv, dk, dv):
        raise GDNError(f"{name} must be fp32 [P, Hv, d_k, d_v] with pages of {(Hv, dk, dv)}, got "
                       f"{t.dtype} {tuple(shape)}", 2)
    if stride[1:] != (dk * dv, dv, 1) and not t[:1].is_contiguous():
        raise GDNError(f"{name}: each page must be contiguous", 3)
    return stride[0] if shape[0] > 1 else max(stride[0], Hv * dk * dv)


def _check_index(index, rows: int, pages: int) -> None:
    if index is None:
        if pages != rows:
            raise GDNError(f"without index the states must have one page per sequence ({rows}), "
                           f"got {pages}", 2)
    elif index.dtype is not torch.int32 or index.shape != (rows,) or not index.is_contiguous():
        raise GDNError(f"index must be a contiguous int32 [{rows}] tensor", 2)


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
    raises).  Rows without a page leave ``state_out`` as it was.  ``out`` must
    not share memory with the inputs.
    """
    dev = _on(q, k, v, g, state, state_out, out, index)
    if out is None:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    if state_out is None:
        state_out = state
    a = _decode_args(q, k, v, g, state, state_out, out, index, scale, gate, _status(dev))
    _launch(_DECODE, a, dev, "lin_decode")
    if check:
        check_device_status(dev)
    return out


def _decode_args(q, k, v, g, state, state_out, out, index, scale, gate,
                 status=0) -> bytes:
    shape, v_shape = q.shape, v.shape
    if len(shape) != 3 or k.shape != shape or len(v_shape) != 3 or v_shape[0] != shape[0]:
        raise GDNError("q, k must be [B, Hqk, d_k] and v [B, Hv, d_v]", 2)
    B, Hqk, dk = shape
    _, Hv, dv = v_shape
    io = _check_io(q, k, v, out)
    qs, ks, vs, os, gs = q.stride(), k.stride(), v.stride(), out.stride(), g.stride()
    if qs[2] != 1 or ks[2] != 1 or vs[2] != 1 or os[2] != 1:
        _check_rows(q=qs, k=ks, v=vs, out=os)
    if g.shape == (B, Hv):
        g_sb, g_sh = gs
    elif g.shape == (Hv,):
        g_sb, g_sh = 0, gs[0]
    else:
        raise GDNError(f"g must be [B, Hv] = {(B, Hv)} or [Hv], got {tuple(g.shape)}", 2)
    if gate not in ("log", "linear"):
        raise GDNError("gate must be 'log' (decay = exp(g)) or 'linear' (decay = g)", 4)
    in_sp = out_sp = _check_states("state", state, Hv, dk, dv)
    pages = state.shape[0]
    if state_out is not state:
        out_sp = _check_states("state_out", state_out, Hv, dk, dv)
        if state_out.shape[0] != pages:
            raise GDNError("state_out must have as many pages as state", 2)
    _check_index(index, B, pages)
    _check_scale(scale)
    return _DECODE.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), state.data_ptr(),
        state_out.data_ptr(), out.data_ptr(), 0 if index is None else index.data_ptr(),
        qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1], g_sb, g_sh, in_sp, out_sp,
        B, Hqk, Hv, dk, dv, pages, io, _dt(g, "g"), _LOG if gate == "log" else _LINEAR,
        scale, status)


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
    possibly none, and rows outside every sequence are left as they were (T, all
    rows, is at least 1).

    With ``index`` (int32 on the device, one entry per sequence) the states are
    pools: sequence n starts from page index[n] of ``initial_state`` and leaves
    its state in page index[n] of ``final_state`` (required then, unless
    ``initial_state`` is to be updated in place).  A negative index starts from
    zero and keeps no state.  Indices out of range or taken by an earlier
    sequence, and offsets that are out of range or descend, are reported
    (``check=True``).  q, k, v and out may be strided views whose rows are
    contiguous and 16-byte aligned; out must not share memory with them.

    Few heads and a long T: the time axis is cut, with a workspace from torch's
    allocator (or ``workspace``, at least as large).  Infinities and NaN in a row
    reach no earlier row and no other sequence; the outputs they belong to are not
    finite.  bf16: the decayed scores, and the state where the queries meet it, are
    rounded to bf16 once, the state itself takes its terms in 16 bits; under strong
    decay outputs hold up to 2^47, and a row keeps 2^-80 of the state before its chunk
    (128 tokens) where the decay would leave less, but none behind a decay of zero.  f16: scores rounded to f16 times a
    power of two of their row, the state where the queries meet it to tf32, its terms
    in 22 bits; scores and states may pass f16's range (about twice the time of bf16).
    """
    dev = _on(q, k, v, g, initial_state, final_state, out, cu_seqlens, index, workspace)
    if out is None:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    if final_state is None:
        if index is not None:
            if initial_state is None:
                raise GDNError("with index, pass the pool as final_state or initial_state", 1)
            final_state = initial_state
        elif v.dim() == 4 and q.dim() == 4 and (cu_seqlens is None or cu_seqlens.numel() > 1):
            rows = v.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
            final_state = torch.empty((rows, v.shape[2], q.shape[3], v.shape[3]),
                                      dtype=torch.float32, device=q.device)
    args = (q, k, v, g, initial_state, final_state, out, cu_seqlens, index, scale, _status(dev))
    a = _prefill_args(*args)
    need = _prefill_workspace(a, dev) if v.shape[1] > _UNCUT else 0
    if need:
        # from the allocator on the current stream, so that calls on other streams
        # and captured graphs have workspaces of their own
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif not workspace.is_contiguous():
            raise GDNError("workspace must be a contiguous tensor", 2)
        a = _prefill_args(*args, workspace.data_ptr(), workspace.numel() * workspace.element_size())
    _launch(_PREFILL, a, dev, "lin_prefill")
    if check:
        check_device_status(dev)
    return out, final_state


def _prefill_workspace(args: bytes, dev: int | None = None) -> int:
    """What the call needs on device `dev` (the current one), whose SMs decide how it is cut."""
    if dev is not None and torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _prefill_workspace(args)
    return _lib.load().lin_prefill_workspace_size(
        ctypes.cast(ctypes.c_char_p(args), ctypes.POINTER(_lib.LinPrefillArgs)))


def _prefill_args(q, k, v, g, initial_state, final_state, out, cu_seqlens, index, scale,
                  status=0, workspace=0, workspace_bytes=0) -> bytes:
    shape, v_shape = q.shape, v.shape
    if len(shape) != 4 or k.shape != shape or len(v_shape) != 4 or v_shape[:2] != shape[:2]:
        raise GDNError("q, k must be [B, T, Hqk, d_k] and v [B, T, Hv, d_v]", 2)
    B, T, Hqk, dk = shape
    _, _, Hv, dv = v_shape
    io = _check_io(q, k, v, out)
    qs, ks, vs, os, gs = q.stride(), k.stride(), v.stride(), out.stride(), g.stride()
    if qs[3] != 1 or ks[3] != 1 or vs[3] != 1 or os[3] != 1:
        _check_rows(q=qs, k=ks, v=vs, out=os)
    if g.shape == (Hv,):
        gs = (0, 0, gs[0])
    elif g.shape != (B, T, Hv):
        raise GDNError(f"g must be [B, T, Hv] = {(B, T, Hv)} or [Hv], got {tuple(g.shape)}", 2)
    seqs = B
    if cu_seqlens is not None:
        if cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 \
                or not cu_seqlens.is_contiguous():
            raise GDNError("cu_seqlens must be a contiguous int32 [N + 1] tensor", 2)
        if B != 1:
            raise GDNError("packed sequences (cu_seqlens) need a batch of one", 2)
        seqs = cu_seqlens.numel() - 1
    fin_sp, in_sp = _check_states("final_state", final_state, Hv, dk, dv), 0
    pages = final_state.shape[0]
    if initial_state is not None:
        in_sp = _check_states("initial_state", initial_state, Hv, dk, dv)
        if initial_state.shape[0] != pages:
            raise GDNError("initial_state and final_state must have as many pages", 2)
    _check_index(index, seqs, pages)
    _check_scale(scale)
    return _PREFILL.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
        0 if initial_state is None else initial_state.data_ptr(), final_state.data_ptr(),
        out.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(),
        0 if index is None else index.data_ptr(),
        *qs[:3], *ks[:3], *vs[:3], *os[:3], *gs, in_sp, fin_sp,
        seqs, T, Hqk, Hv, dk, dv, pages, io, _dt(g, "g"), scale,
        workspace, workspace_bytes, status)
