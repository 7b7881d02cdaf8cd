"""Pages of a cache of recurrent states: copy, fork, allocate, free, compact.

A pool is a tensor [P, ...] whose first axis counts pages, one page per
sequence (the states of one layer: fp32 [P, Hv, d_k, d_v]); a call takes one
pool or a list of pools of the same page count (one per layer, say; dtypes and
page sizes may differ).  ``used`` is an int32 [P] tensor, 0 where a page is
free.  Pages are handed out lowest first.  Everything is decided on the device,
so the calls can be captured in a graph; what is wrong with an index shows in
the device status (``check=True`` synchronises and raises).

After :func:`pages_compact` the live sequences' states are ``pool[:count]``,
the plain batch that ``gdn_decode`` and ``kda_decode`` take; ``lin_decode`` and
``lin_prefill`` also take pages by index.
"""
from __future__ import annotations

import ctypes
from array import array

import torch

from . import _lib
from ._lib import GDNError
from .api import check_device_status
from .lin import _launch, _on, _status


_CALLS = {name: _lib.Packed(_lib.PagesArgs, f"pages_{name}_launch")
          for name in ("copy", "fork", "free", "compact")}
_SMALL = 2048  # pages and entries up to which no call needs a workspace


def _pools(pools) -> tuple[list, array]:
    """The pools and their C descriptors (base, page stride, page bytes)."""
    pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    if len(pools) > _lib.PAGES_MAX_POOLS:
        raise GDNError(f"at most {_lib.PAGES_MAX_POOLS} pools in a call, got {len(pools)}", 2)
    flat = array("q")
    for p in pools:
        if p.dim() < 2 or p.shape[0] != pools[0].shape[0]:
            raise GDNError("pools must be [P, ...] tensors with the same number of pages", 2)
        P, size = p.shape[0], p.element_size()
        n = p.numel() // P * size if P else 0
        if not p.is_contiguous() and not p[:1].is_contiguous():
            raise GDNError("each page of a pool must be contiguous", 3)
        flat.extend((p.data_ptr(), p.stride(0) * size if P > 1 else n, n))
    return pools, flat


def _int32(name: str, t, shape=None) -> None:
    if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous() \
            or (shape is not None and t.shape != shape):
        raise GDNError(f"{name} must be a contiguous int32 [{shape[0] if shape else 'n'}] tensor", 2)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _call(name: str, like, dev: int, pages: int, *, pools=(), arr=None, used=None, used_out=None, n=0,
          src=None, dst=None, remap=None, count=None, check=False) -> None:
    if not 1 <= pages <= _lib.PAGES_MAX_PAGES:
        raise GDNError(f"a pool must have 1 to {_lib.PAGES_MAX_PAGES} pages, got {pages}", 2)
    packed = _CALLS[name]
    args = (arr.buffer_info()[0] if pools else 0, len(pools), pages, _ptr(used), _ptr(used_out), n,
            _ptr(src), _ptr(dst), _ptr(remap), _ptr(count))
    ws, need, status = 0, 0, _status(dev)
    if (pages > _SMALL or n > _SMALL) and name != "free":
        need = _lib.load().pages_workspace_size(ctypes.cast(
            ctypes.c_char_p(packed.pack(*args, 0, 0, 0)), ctypes.POINTER(_lib.PagesArgs)))
        # from the allocator on the current stream: no two calls in flight share it
        buf = torch.empty(need, dtype=torch.uint8, device=like.device)
        ws = buf.data_ptr()
    _launch(packed, packed.pack(*args, ws, need, status), dev, f"pages_{name}")
    if check:
        check_device_status(dev)


def pages_copy(pools, src, dst, *, check: bool = False) -> None:
    """Copies page src[i] to page dst[i] of every pool (int32 [n] each).

    Entries with a negative index are skipped.  So, with a device error, are
    entries whose index is out of range, whose destination another entry has
    too, or whose destination is some entry's source: what is copied does not
    depend on the order of the copies.  An entry of a page onto itself moves
    nothing and counts as neither."""
    pools, arr = _pools(pools)
    if not pools:
        raise GDNError("pages_copy needs a pool", 1)
    dev = _on(src, dst, *pools)
    _int32("src", src)
    _int32("dst", dst, tuple(src.shape))
    _call("copy", src, dev, pools[0].shape[0], pools=pools, arr=arr, n=src.numel(), src=src,
          dst=dst, check=check)


def pages_fork(pools, used, src, *, out=None, used_out=None, check: bool = False) -> torch.Tensor:
    """For each src[i] (int32 [n], the same page as often as wanted) takes the
    next free page and copies page src[i] into it, in every pool.  Returns the
    new pages, int32 [n]; ``used`` is updated in place (or into ``used_out``).

    The result is -1 where src[i] is negative and, with a device error, where
    src[i] is out of range or free, or no free page is left."""
    pools, arr = _pools(pools)
    dev = _on(used, src, out, used_out, *pools)
    _int32("src", src)
    if pools and used.numel() != pools[0].shape[0]:
        raise GDNError(f"used must be [P] = [{pools[0].shape[0]}], got {tuple(used.shape)}", 2)
    return _fork(dev, pools, arr, used, src, src.numel(), out, used_out, check)


def pages_alloc(used, n: int, *, out=None, used_out=None, check: bool = False) -> torch.Tensor:
    """Takes the n lowest free pages: int32 [n], -1 (with a device error) once
    none is left.  Their contents are left as they are."""
    dev = _on(used, out, used_out)
    if n < 0:
        raise GDNError(f"n must not be negative, got {n}", 2)
    return _fork(dev, [], None, used, None, n, out, used_out, check)


def _fork(dev, pools, arr, used, src, n, out, used_out, check):
    used_out = used if used_out is None else used_out
    if out is None:
        out = used.new_empty(n)
    _int32("used", used)
    _int32("used_out", used_out, tuple(used.shape))
    _int32("out", out, (n,))
    _call("fork", used, dev, used.numel(), pools=pools, arr=arr, used=used, used_out=used_out,
          n=n, src=src, dst=out, check=check)
    return out


def pages_free(used, index, *, used_out=None, check: bool = False) -> torch.Tensor:
    """Marks the pages index[i] (int32 [n]) free in ``used`` (or ``used_out``,
    which is returned).  Negative entries are skipped; an entry out of range, or
    of a page that is free already, is a device error."""
    dev = _on(used, index, used_out)
    used_out = used if used_out is None else used_out
    _int32("used", used)
    _int32("used_out", used_out, tuple(used.shape))
    _int32("index", index)
    _call("free", used, dev, used.numel(), used=used, used_out=used_out, n=index.numel(),
          src=index, check=check)
    return used_out


def pages_compact(pools, used, *, index=None, index_out=None, used_out=None, check: bool = False):
    """Moves the used pages that lie behind the first ``count`` places (count =
    number of used pages) into the free places among them, lowest to lowest, in
    every pool.  Returns (remap, count, index_out): remap int32 [P], where each
    page now is (-1: free); count int32 [1]; and the sequences' pages ``index``
    (int32 [n]) as they are now (None without ``index``; -1 for negative entries
    and, with a device error, for entries out of range or of free pages).
    ``used`` is updated in place (or into ``used_out``).  Pages behind the first
    ``count`` keep their bytes."""
    pools, arr = _pools(pools)
    dev = _on(used, used_out, index, index_out, *pools)
    used_out = used if used_out is None else used_out
    P, n = used.numel(), 0
    if pools and P != pools[0].shape[0]:
        raise GDNError(f"used must be [P] = [{pools[0].shape[0]}], got {tuple(used.shape)}", 2)
    _int32("used", used)
    _int32("used_out", used_out, tuple(used.shape))
    remap, count = used.new_empty(P), used.new_empty(1)
    if index is not None:
        n = index.numel()
        _int32("index", index)
        if index_out is None:
            index_out = used.new_empty(n)
        _int32("index_out", index_out, (n,))
    elif index_out is not None:
        raise GDNError("index_out needs index", 1)
    _call("compact", used, dev, P, pools=pools, arr=arr, used=used, used_out=used_out, n=n,
          src=index, dst=index_out, remap=remap, count=count, check=check)
    return remap, count, index_out
