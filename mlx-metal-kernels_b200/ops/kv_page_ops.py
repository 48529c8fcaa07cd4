"""Pages of a paged key/value cache: reserve, copy, fork, release and compact, for the caches of all layers at once.

The reference has static block tables only (make_identity_block_table, ops/paged_kv_ops.py:99-110); a serving loop whose
sequences come, branch and end needs to move pages around.  One block table, one ``lengths`` and one ``PagePool`` of reference
counts serve all layers.  Everything happens on the device and in stream order: no call waits, every call can be captured, and
calls on one pool must be ordered (one stream, or events between streams).

Which pages a call takes is fixed by its arguments: the lowest free ones, in the order of the call.  A call that cannot be
served - a child listed twice, a destination that is also a source, a sequence past the end of its table row, too few free
pages - changes nothing and is reported by ``_cabi.device_status()`` (event 8, or 9 for too few pages).  Negative indices are
padding, so that a captured call can serve fewer sequences than it was captured with.
"""
from __future__ import annotations

import ctypes
import operator
from dataclasses import dataclass
from typing import Any

import torch

from . import _cabi


@dataclass
class PagePool:
    """Reference counts of the pages of a pool, int32 [NUM_PAGES] on the device; 0 = free.  A page counts once for every block-table
    entry that names it."""
    ref_counts: Any
    page_size: int = 16

    @classmethod
    def empty(cls, num_pages: int, page_size: int = 16, device=None) -> "PagePool":
        if num_pages <= 0:
            raise ValueError(f"num_pages must be positive, got {num_pages}")
        return cls(torch.zeros(num_pages, dtype=torch.int32, device=device), page_size).validate()

    @classmethod
    def from_block_table(cls, block_table, num_pages: int, page_size: int = 16) -> "PagePool":
        """The pool whose pages are held as ``block_table`` says (it is read on the host)."""
        used = block_table.reshape(-1).cpu()
        used = used[used >= 0].to(torch.int64)
        if num_pages <= 0 or (used.numel() and int(used.max()) >= num_pages):
            raise ValueError(f"the block table names pages outside a pool of {num_pages}")
        return cls(torch.bincount(used, minlength=num_pages).to(torch.int32).to(block_table.device), page_size).validate()

    def validate(self) -> "PagePool":
        if self.page_size <= 0:
            raise ValueError(f"page_size must be > 0, got {self.page_size}")
        r = self.ref_counts
        if r.ndim != 1 or r.shape[0] == 0 or r.dtype != torch.int32 or not r.is_contiguous():
            raise ValueError("ref_counts must be a contiguous int32 tensor [NUM_PAGES]")
        return self

    @property
    def num_pages(self) -> int:
        return self.ref_counts.shape[0]


def _check_table(pool, block_table, lengths=None):
    pool.validate()
    if block_table.ndim != 2 or block_table.dtype != torch.int32 or not block_table.is_contiguous() or 0 in block_table.shape:
        raise ValueError("block_table must be a contiguous int32 tensor [B, MAX_BLOCKS]")
    B = block_table.shape[0]
    if lengths is not None and (tuple(lengths.shape) != (B,) or lengths.dtype != torch.int32 or not lengths.is_contiguous()):
        raise ValueError(f"lengths must be a contiguous int32 tensor [{B}]")
    return block_table.shape


def _indices(t, what: str):
    if t.ndim != 1 or t.dtype != torch.int32:
        raise ValueError(f"{what} must be an int32 tensor [n], got {t.dtype} {tuple(t.shape)}")
    return _cabi.contiguous(t)


def _layer_tensors(cache):
    """(tensors of codes or plain values, tensors of scales) of one layer."""
    if isinstance(cache, (tuple, list)):
        if len(cache) != 2:
            raise ValueError("plain caches are pairs (K_pages, V_pages)")
        return tuple(cache), ()
    if getattr(cache, "k_zeros", None) is not None or getattr(cache, "v_zeros", None) is not None:
        raise NotImplementedError("zero-point quantization is not implemented yet")
    if hasattr(cache, "k_codes"):                       # the per-layer pools of a decode stack
        return (cache.k_codes, cache.v_codes), (cache.k_scales, cache.v_scales)
    return (cache.k_pages_q, cache.v_pages_q), (cache.k_scales, cache.v_scales)


def _cache_tensors(caches, num_pages: int | None, page_size: int | None):
    """Two groups of equal tensors, (values, scales), over all layers."""
    if not isinstance(caches, (tuple, list)) or (len(caches) == 2 and all(isinstance(c, torch.Tensor) for c in caches)):
        caches = [caches]
    if len(caches) == 0:
        raise ValueError("there must be at least one cache")
    groups = ([], [])
    for cache in caches:
        for group, tensors in zip(groups, _layer_tensors(cache)):
            group.extend(tensors)
    if groups[1] and len(groups[1]) != len(groups[0]):
        raise ValueError("caches must be all quantized or all plain")
    for group, what in zip(groups, ("pages", "scales")):
        for t in group:
            if t.ndim != 4 or not t.is_contiguous() or 0 in t.shape:
                raise ValueError(f"{what} must be contiguous tensors [NUM_PAGES,PAGE_SIZE,Hkv,D], got {tuple(t.shape)}")
            if t.shape != group[0].shape or t.dtype != group[0].dtype:
                raise ValueError(f"the {what} of all layers must have one shape and dtype, got {tuple(t.shape)} {t.dtype} and "
                                 f"{tuple(group[0].shape)} {group[0].dtype}")
    want = tuple(groups[0][0].shape[:2])
    if groups[1] and tuple(groups[1][0].shape[:2]) != want:
        raise ValueError(f"pages and scales must agree in [NUM_PAGES,PAGE_SIZE], got {want} and {tuple(groups[1][0].shape[:2])}")
    if num_pages is not None and want != (num_pages, page_size):
        raise ValueError(f"caches of {want} pages and slots do not fit a pool of {(num_pages, page_size)}")
    return groups, want


def _group_args(group):
    if not group:
        return None, 0, 0
    slot = group[0][0, 0].numel() * group[0].element_size()
    return (ctypes.c_void_p * len(group))(*[t.data_ptr() for t in group]), len(group), slot


def _workspace(nbytes: int, device):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def reserve_pages(pool: PagePool, block_table, lengths, new_tokens) -> None:
    """Pages for the next tokens: sequence b gets a page for every unassigned block of the positions ``lengths[b]`` to ``lengths[b] +
    new - 1``, new being ``new_tokens`` (an int) or ``new_tokens[b]`` (int32 [B]).  ``block_table`` and the pool change in place; ``lengths`` is
    left to the caller."""
    if _cabi.host().reserve_pages(pool.ref_counts, pool.page_size, block_table, lengths, new_tokens):
        return
    B, max_blocks = _check_table(pool, block_table, lengths)
    uniform, per_row = 0, None
    if isinstance(new_tokens, torch.Tensor):
        per_row = _indices(new_tokens, "new_tokens")
        if per_row.shape[0] != B:
            raise ValueError(f"new_tokens must have shape {(B,)}, got {tuple(per_row.shape)}")
    else:
        uniform = operator.index(new_tokens)
        if not 0 <= uniform < 2 ** 31:
            raise ValueError(f"new_tokens must be in [0, 2^31), got {new_tokens}")
    device = _cabi.require_cuda(pool.ref_counts, block_table, lengths, per_row)
    lib = _cabi.load()
    with _cabi.on_device(device):
        ws = _workspace(lib.b200q_reserve_pages_workspace_bytes(B, pool.num_pages), device)
        _cabi.check(lib.b200q_reserve_pages(pool.ref_counts.data_ptr(), pool.num_pages, block_table.data_ptr(), lengths.data_ptr(),
                                            _cabi.ptr(per_row), uniform, B, max_blocks, pool.page_size, ws.data_ptr(), ws.numel(),
                                            _cabi.stream()), "b200q_reserve_pages")


def release_sequences(pool: PagePool, block_table, lengths, rows) -> None:
    """The sequences ``rows`` (int32 [n]) end: the counts of their pages fall by one, their block-table rows become -1, their lengths 0.
    A row listed twice is released once; a row that is empty stays so."""
    if _cabi.host().release_sequences(pool.ref_counts, pool.page_size, block_table, lengths, rows):
        return
    B, max_blocks = _check_table(pool, block_table, lengths)
    rows = _indices(rows, "rows")
    device = _cabi.require_cuda(pool.ref_counts, block_table, lengths, rows)
    if rows.shape[0] == 0:
        return
    with _cabi.on_device(device):
        _cabi.check(_cabi.load().b200q_release_sequences(pool.ref_counts.data_ptr(), pool.num_pages, block_table.data_ptr(),
                                                         lengths.data_ptr(), rows.data_ptr(), rows.shape[0], B, max_blocks, _cabi.stream()),
                    "b200q_release_sequences")


def copy_pages(caches, src_pages, dst_pages) -> None:
    """Page ``src_pages[i]`` to page ``dst_pages[i]`` (int32 [n]) in every tensor of ``caches``: a PagedQuantizedKVCache, a pair (K_pages,
    V_pages), or a list of them, one per layer.  Destinations must differ from one another and from all sources."""
    if _cabi.host().copy_pages(caches, src_pages, dst_pages):
        return
    src, dst = _indices(src_pages, "src_pages"), _indices(dst_pages, "dst_pages")
    if src.shape != dst.shape:
        raise ValueError(f"src_pages and dst_pages must have one shape, got {tuple(src.shape)}, {tuple(dst.shape)}")
    groups, (num_pages, page_size) = _cache_tensors(caches, None, None)
    device = _cabi.require_cuda(src, dst, *groups[0], *groups[1])
    n = src.shape[0]
    if n == 0:
        return
    lib = _cabi.load()
    with _cabi.on_device(device):
        ws = _workspace(lib.b200q_copy_pages_workspace_bytes(n, num_pages), device)
        _cabi.check(lib.b200q_copy_pages(*_group_args(groups[0]), *_group_args(groups[1]), src.data_ptr(), dst.data_ptr(), n, num_pages,
                                         page_size, ws.data_ptr(), ws.numel(), _cabi.stream()), "b200q_copy_pages")


def fork_sequences(caches, pool: PagePool, block_table, lengths, parents, children) -> None:
    """Sequence ``children[i]`` continues as ``parents[i]`` does now (int32 [n]): it shares the parent's full pages and gets the used slots of
    its last page, when that is not full, on a page of its own, in every layer of ``caches``.  A parent may have many children; a child must
    be empty (``release_sequences``), listed once, and no parent of the call.  Pages reserved behind the parent's length stay its own."""
    if _cabi.host().fork_sequences(caches, pool.ref_counts, pool.page_size, block_table, lengths, parents, children):
        return
    B, max_blocks = _check_table(pool, block_table, lengths)
    parents, children = _indices(parents, "parents"), _indices(children, "children")
    if parents.shape != children.shape:
        raise ValueError(f"parents and children must have one shape, got {tuple(parents.shape)}, {tuple(children.shape)}")
    groups, _ = _cache_tensors(caches, pool.num_pages, pool.page_size)
    device = _cabi.require_cuda(pool.ref_counts, block_table, lengths, parents, children, *groups[0], *groups[1])
    n = parents.shape[0]
    if n == 0:
        return
    lib = _cabi.load()
    with _cabi.on_device(device):
        ws = _workspace(lib.b200q_fork_sequences_workspace_bytes(n, B), device)
        _cabi.check(lib.b200q_fork_sequences(*_group_args(groups[0]), *_group_args(groups[1]), pool.ref_counts.data_ptr(), pool.num_pages,
                                             block_table.data_ptr(), lengths.data_ptr(), parents.data_ptr(), children.data_ptr(), n, B,
                                             max_blocks, pool.page_size, ws.data_ptr(), ws.numel(), _cabi.stream()),
                    "b200q_fork_sequences")


def compact_pages(caches, pool: PagePool, block_table):
    """Moves the held pages to the low end of the pool, in every layer of ``caches``, and rewrites counts and ``block_table`` (which must be the
    only one that names the pool's pages).  With L held pages the k-th held page at or above L moves to the k-th free page below L; the
    others stay.  Returns int32 [NUM_PAGES]: the new number of every held page, -1 for free ones."""
    remap = _cabi.host().compact_pages(caches, pool.ref_counts, pool.page_size, block_table)
    if remap is not None:
        return remap
    B, max_blocks = _check_table(pool, block_table)
    groups, _ = _cache_tensors(caches, pool.num_pages, pool.page_size)
    device = _cabi.require_cuda(pool.ref_counts, block_table, *groups[0], *groups[1])
    lib = _cabi.load()
    with _cabi.on_device(device):
        remap = torch.empty(pool.num_pages, dtype=torch.int32, device=device)
        ws = _workspace(lib.b200q_compact_pages_workspace_bytes(pool.num_pages), device)
        _cabi.check(lib.b200q_compact_pages(*_group_args(groups[0]), *_group_args(groups[1]), pool.ref_counts.data_ptr(), pool.num_pages,
                                            block_table.data_ptr(), B, max_blocks, pool.page_size, remap.data_ptr(), ws.data_ptr(),
                                            ws.numel(), _cabi.stream()), "b200q_compact_pages")
    return remap
