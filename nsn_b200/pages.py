"""Page operations of a paged cache whose sequences share pages (nsnkv_fork_sequences and its
companions): reference counts per page, forks that share sealed pages and copy the tail,
frees, reservations, page copies and pool compaction, in stream order with no host sync.

Conventions (include/nsnkv.h): ``page_refs`` int32 [pages] counts the block-table entries equal to
each page p > 0; a page is free when its count is 0.  Page 0 is the unassigned page: a table
entry 0 names no page.  Sequence b's entries from n_blocks[b] on are pages reserved for its
next blocks.  ``shared.SharedPagedKVCache`` keeps these arrays for a cache.
The reference has no pages: its caches grow by torch.cat per slot
(experiments/nb06/source/loop_kv_nb06_packed.py:36-50).
"""
from __future__ import annotations

import torch

from . import _lib as L
from . import primitives as w
from .kernel import workspace


def _ints(name, *tensors):
    dev = tensors[0].device
    w.require(all(t.is_cuda and t.device == dev and t.dtype == torch.int32 and (t.numel() == 0 or t.stride(-1) == 1)
                  for t in tensors), f"{name}: int32 CUDA tensors on one device")
    return dev


def _p(t):
    return t.data_ptr() if t is not None else None


def fork_sequences(block_table, n_blocks, tail_len, page_refs, k_tail, v_tail, src, dst, status=None):
    """Sequence dst[i] becomes a copy of sequence src[i]: it drops the pages it held, shares
    src's sealed pages and copies src's counters and tail rows.

    block_table [batch, max_blocks], n_blocks / tail_len [batch], page_refs [pages] and src / dst
    [count] are int32, the tails [batch, h, 64, 128] fp16 or bf16; all change in place.  The dst
    are distinct sequences and none of them is a src.
    """
    dev = _ints("fork_sequences", block_table, n_blocks, tail_len, page_refs, src, dst)
    batch = block_table.shape[0]
    w.require(block_table.ndim == 2 and n_blocks.shape == (batch,) and tail_len.shape == (batch,)
              and src.ndim == 1 and src.shape == dst.shape, "fork_sequences tables")
    w.require(k_tail.ndim == 4 and k_tail.shape == v_tail.shape and k_tail.shape[0] == batch
              and k_tail.shape[2:] == (w.BLOCK, w.DIM) and k_tail.dtype == v_tail.dtype
              and k_tail.dtype in (torch.float16, torch.bfloat16) and k_tail.is_contiguous() and v_tail.is_contiguous()
              and k_tail.device == dev and v_tail.device == dev, "fork_sequences tails [batch, h, 64, 128]")
    h = k_tail.shape[1]
    with torch.cuda.device(dev):
        rc = L.load().nsnkv_fork_sequences(
            batch, h, page_refs.numel(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            n_blocks.data_ptr(), tail_len.data_ptr(), page_refs.data_ptr(), k_tail.data_ptr(), v_tail.data_ptr(),
            h * w.BLOCK, w.BLOCK, src.numel(), src.data_ptr(), dst.data_ptr(), _p(status),
            torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, "nsnkv_fork_sequences")


def free_sequences(block_table, n_blocks, tail_len, page_refs, seqs, status=None):
    """Sequences ``seqs`` (int32 [count]) drop their pages and are empty; in place."""
    dev = _ints("free_sequences", block_table, n_blocks, tail_len, page_refs, seqs)
    batch = block_table.shape[0]
    w.require(block_table.ndim == 2 and n_blocks.shape == (batch,) and tail_len.shape == (batch,) and seqs.ndim == 1,
              "free_sequences tables")
    with torch.cuda.device(dev):
        rc = L.load().nsnkv_free_sequences(
            batch, page_refs.numel(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            n_blocks.data_ptr(), tail_len.data_ptr(), page_refs.data_ptr(), seqs.numel(), seqs.data_ptr(), _p(status),
            torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, "nsnkv_free_sequences")


def reserve_pages(block_table, n_blocks, page_refs, ahead=1, status=None):
    """Pages for every sequence's next ``ahead`` blocks where its table entries name none, in
    place: in (sequence, entry) order they take the free pages in ascending order.  ``status`` gets
    NSNKV_ST_CAPACITY when too few pages are free; the entries left over stay unassigned."""
    dev = _ints("reserve_pages", block_table, n_blocks, page_refs)
    batch = block_table.shape[0]
    w.require(block_table.ndim == 2 and n_blocks.shape == (batch,), "reserve_pages tables")
    with torch.cuda.device(dev):
        rc = L.load().nsnkv_reserve_pages(
            batch, page_refs.numel(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            n_blocks.data_ptr(), page_refs.data_ptr(), int(ahead), _p(status),
            torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, "nsnkv_reserve_pages")


def _page_arrays(arrays, dev):
    """[h, pages, ...] tensors as nsnkv_page_array descriptors: (h, pages, ctypes array)."""
    w.require(0 < len(arrays) <= 8 and all(t.ndim >= 3 and t.shape[:2] == arrays[0].shape[:2] and t.device == dev
                                           for t in arrays), "page arrays: one to eight [h, pages, ...] tensors")
    got = (L.PageArray * len(arrays))()
    for d, t in zip(got, arrays):
        size = t.element_size()
        w.require(t[0, 0].is_contiguous(), "page arrays: contiguous pages")
        d.base, d.bytes = t.data_ptr(), t[0, 0].numel() * size
        d.stride_head, d.stride_page = t.stride(0) * size, t.stride(1) * size
    return arrays[0].shape[0], arrays[0].shape[1], got


def copy_pages(arrays, src, dst, status=None):
    """Page dst[i] of every array ([h, pages, ...] tensors of a pool) becomes a copy of page
    src[i], for all heads (src, dst int32 [count]; no dst is the src of another pair)."""
    dev = _ints("copy_pages", src, dst)
    w.require(src.ndim == 1 and src.shape == dst.shape, "copy_pages src, dst")
    h, pages, arr = _page_arrays(arrays, dev)
    with torch.cuda.device(dev):
        rc = L.load().nsnkv_copy_pages(h, pages, len(arrays), arr, src.numel(), src.data_ptr(), dst.data_ptr(),
                                       _p(status), torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, "nsnkv_copy_pages")


def compact_pages(arrays, block_table, page_refs, table_out=None, refs_out=None, status=None, ws=None):
    """Bring the live pages of a pool to its front.

    With L live pages (page 0 and those with page_refs > 0), the i-th live page at or above L
    moves to the i-th free page below L, both in ascending order, in every array of the pool
    ([h, pages, ...] tensors, changed in place; freed pages keep their bytes).  Returns
    (table [batch, max_blocks], refs [pages], live int32 [1]): the block table and counts of the
    moved pages and L, in new tensors or in ``table_out`` / ``refs_out`` (which may be the inputs).
    """
    dev = _ints("compact_pages", block_table, page_refs)
    h, pages, arr = _page_arrays(arrays, dev)
    w.require(block_table.ndim == 2 and page_refs.shape == (pages,), "compact_pages tables")
    if table_out is None:
        table_out = torch.empty(block_table.shape, dtype=torch.int32, device=dev)
    if refs_out is None:
        refs_out = torch.empty_like(page_refs)
    live = torch.empty(1, dtype=torch.int32, device=dev)
    _ints("compact_pages outputs", table_out, refs_out, live)
    w.require(table_out.shape == block_table.shape and refs_out.shape == page_refs.shape, "compact_pages outputs")
    lib = L.load()
    if ws is None:
        ws = workspace(lib.nsnkv_compact_pages_workspace_bytes(pages), dev)
    with torch.cuda.device(dev):
        rc = lib.nsnkv_compact_pages(
            h, pages, len(arrays), arr, block_table.shape[0], block_table.shape[1], block_table.data_ptr(),
            block_table.stride(0), table_out.data_ptr(), table_out.stride(0), page_refs.data_ptr(),
            refs_out.data_ptr(), live.data_ptr(), ws.data_ptr(), ws.numel(), _p(status),
            torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, "nsnkv_compact_pages")
    return table_out, refs_out, live
