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

import torch

from . import _lib
from ._lib import GDNError
from .api import _require_cuda, _same_device, check_device_status, status_word
from .lin import _launch


def _pools(pools) -> tuple[list, "ctypes.Array | None"]:
    pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    if len(pools) > _lib.PAGES_MAX_POOLS:
        raise GDNError(f"at most {_lib.PAGES_MAX_POOLS} pools in a call, got {len(pools)}", 2)
    arr = (_lib.PagesPool * max(1, len(pools)))()
    for i, p in enumerate(pools):
        if p.dim() < 2 or p.shape[0] != pools[0].shape[0]:
            raise GDNError("pools must be [P, ...] tensors with the same number of pages", 2)
        if not p[0].is_contiguous():
            raise GDNError("each page of a pool must be contiguous", 3)
        size, n = p.element_size(), p[0].numel()
        arr[i] = (p.data_ptr(), (p.stride(0) if p.shape[0] > 1 else n) * size, n * size)
    return pools, arr


def _int32(name: str, t, shape=None) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() \
            or (shape is not None and tuple(t.shape) != shape):
        raise GDNError(f"{name} must be a contiguous int32 [{shape[0] if shape else 'n'}] tensor", 2)


def _call(fn: str, dev, pages, *, pools=(), arr=None, used=None, used_out=None, n=0, src=None,
          dst=None, remap=None, count=None, check=False) -> None:
    if not 1 <= pages <= _lib.PAGES_MAX_PAGES:
        raise GDNError(f"a pool must have 1 to {_lib.PAGES_MAX_PAGES} pages, got {pages}", 2)
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    a = _lib.PagesArgs(arr, len(pools), pages, ptr(used), ptr(used_out), n, ptr(src), ptr(dst),
                       ptr(remap), ptr(count), None, 0, status_word(dev).data_ptr())
    L = _lib.load()
    # from the allocator on the current stream: no two calls in flight share it
    ws = torch.empty(max(16, L.pages_workspace_size(ctypes.byref(a))), dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _launch(getattr(L, fn), a, dev, fn.removesuffix("_launch"))
    if check:
        check_device_status(dev)


def pages_copy(pools, src, dst, *, check: bool = False) -> None:
    """Copies page src[i] to page dst[i] of every pool (int32 [n] each).

    Entries with a negative index are skipped.  So, with a device error, are
    entries whose index is out of range, whose destination another entry has
    too, or whose destination is some entry's source: what is copied does not
    depend on the order of the copies."""
    pools, arr = _pools(pools)
    if not pools:
        raise GDNError("pages_copy needs a pool", 1)
    dev = _require_cuda(*pools, src, dst)
    _int32("src", src)
    _int32("dst", dst, tuple(src.shape))
    _call("pages_copy_launch", dev, pools[0].shape[0], pools=pools, arr=arr, n=src.numel(), src=src,
          dst=dst, check=check)


def pages_fork(pools, used, src, *, out=None, used_out=None, check: bool = False) -> torch.Tensor:
    """For each src[i] (int32 [n], the same page as often as wanted) takes the
    next free page and copies page src[i] into it, in every pool.  Returns the
    new pages, int32 [n]; ``used`` is updated in place (or into ``used_out``).

    The result is -1 where src[i] is negative and, with a device error, where
    src[i] is out of range or free, or no free page is left."""
    pools, arr = _pools(pools)
    dev = _require_cuda(*pools, used, src)
    _int32("src", src)
    if pools and used.numel() != pools[0].shape[0]:
        raise GDNError(f"used must be [P] = [{pools[0].shape[0]}], got {tuple(used.shape)}", 2)
    return _fork(dev, pools, arr, used, src, src.numel(), out, used_out, check)


def pages_alloc(used, n: int, *, out=None, used_out=None, check: bool = False) -> torch.Tensor:
    """Takes the n lowest free pages: int32 [n], -1 (with a device error) once
    none is left.  Their contents are left as they are."""
    dev = _require_cuda(used)
    if n < 0:
        raise GDNError(f"n must not be negative, got {n}", 2)
    return _fork(dev, [], None, used, None, n, out, used_out, check)


def _fork(dev, pools, arr, used, src, n, out, used_out, check):
    used_out = used if used_out is None else used_out
    if out is None:
        out = torch.empty(n, dtype=torch.int32, device=dev)
    _same_device(used, out=out, used_out=used_out)
    _int32("used", used)
    _int32("used_out", used_out, tuple(used.shape))
    _int32("out", out, (n,))
    _call("pages_fork_launch", dev, used.numel(), pools=pools, arr=arr, used=used, used_out=used_out,
          n=n, src=src, dst=out, check=check)
    return out


def pages_free(used, index, *, used_out=None, check: bool = False) -> torch.Tensor:
    """Marks the pages index[i] (int32 [n]) free in ``used`` (or ``used_out``,
    which is returned).  Negative entries are skipped; an entry out of range, or
    of a page that is free already, is a device error."""
    dev = _require_cuda(used, index)
    used_out = used if used_out is None else used_out
    _same_device(used, used_out=used_out)
    _int32("used", used)
    _int32("used_out", used_out, tuple(used.shape))
    _int32("index", index)
    _call("pages_free_launch", dev, used.numel(), used=used, used_out=used_out, n=index.numel(),
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
    dev = _require_cuda(used, *pools)
    used_out = used if used_out is None else used_out
    P, n = used.numel(), 0
    if pools and P != pools[0].shape[0]:
        raise GDNError(f"used must be [P] = [{pools[0].shape[0]}], got {tuple(used.shape)}", 2)
    _int32("used", used)
    _int32("used_out", used_out, tuple(used.shape))
    remap = torch.empty(P, dtype=torch.int32, device=dev)
    count = torch.empty(1, dtype=torch.int32, device=dev)
    if index is not None:
        n = index.numel()
        _int32("index", index)
        if index_out is None:
            index_out = torch.empty(n, dtype=torch.int32, device=dev)
        _int32("index_out", index_out, (n,))
    elif index_out is not None:
        raise GDNError("index_out needs index", 1)
    _same_device(used, used_out=used_out, index=index, index_out=index_out)
    _call("pages_compact_launch", dev, P, pools=pools, arr=arr, used=used, used_out=used_out, n=n,
          src=index, dst=index_out, remap=remap, count=count, check=check)
    return remap, count, index_out
