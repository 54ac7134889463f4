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

_I32 = torch.int32
_ARRAYS = {n: L.PageArray * n for n in range(1, 9)}


def _ints(name, dev, *tensors):
    ok = dev.type == "cuda"
    for t in tensors:
        ok = ok and t.dtype == _I32 and t.device == dev and (t.is_contiguous() or t.stride(-1) == 1)
    if not ok:
        raise w.ContractError(f"{name}: int32 CUDA tensors on one device")


def fork_sequences(block_table, n_blocks, tail_len, page_refs, k_tail, v_tail, src, dst, status=None):
    """Sequence dst[i] becomes a copy of sequence src[i]: it drops the pages it held, shares
    src's sealed pages and copies src's counters and tail rows.

    block_table [batch, max_blocks], n_blocks / tail_len [batch], page_refs [pages] and src / dst
    [count] are int32, the tails [batch, h, 64, 128] fp16 or bf16; all change in place.  The dst
    are distinct sequences and none of them is a src.
    """
    dev, (batch, max_blocks) = block_table.device, block_table.shape
    _ints("fork_sequences", dev, block_table, n_blocks, tail_len, page_refs, src, dst)
    kt = k_tail.shape
    if not (n_blocks.shape == tail_len.shape == (batch,) and src.ndim == 1 and src.shape == dst.shape
            and page_refs.ndim == 1):
        raise w.ContractError("fork_sequences tables: block_table [batch, max_blocks], counters [batch], src, dst [count]")
    if not (len(kt) == 4 and kt[0] == batch and kt[2] == w.BLOCK and kt[3] == w.DIM and v_tail.shape == kt
            and k_tail.dtype == v_tail.dtype and k_tail.dtype in (torch.float16, torch.bfloat16)
            and k_tail.is_contiguous() and v_tail.is_contiguous() and k_tail.device == dev and v_tail.device == dev):
        raise w.ContractError("fork_sequences tails: contiguous [batch, h, 64, 128] fp16 or bf16")
    index, h = dev.index, kt[1]
    rc = L.call_on(index, L.load().nsnkv_fork_sequences, batch, h, page_refs.shape[0], block_table.data_ptr(),
                   block_table.stride(0), max_blocks, n_blocks.data_ptr(), tail_len.data_ptr(), page_refs.data_ptr(),
                   k_tail.data_ptr(), v_tail.data_ptr(), h * w.BLOCK, w.BLOCK, src.shape[0], src.data_ptr(),
                   dst.data_ptr(), w.status_ptr(status, dev), L.raw_stream(index))
    if rc:
        L.check(rc, "nsnkv_fork_sequences")


def free_sequences(block_table, n_blocks, tail_len, page_refs, seqs, status=None):
    """Sequences ``seqs`` (int32 [count]) drop their pages and are empty; in place."""
    dev, (batch, max_blocks) = block_table.device, block_table.shape
    _ints("free_sequences", dev, block_table, n_blocks, tail_len, page_refs, seqs)
    if not (n_blocks.shape == tail_len.shape == (batch,) and seqs.ndim == 1 and page_refs.ndim == 1):
        raise w.ContractError("free_sequences tables: block_table [batch, max_blocks], counters [batch], seqs [count]")
    index = dev.index
    rc = L.call_on(index, L.load().nsnkv_free_sequences, batch, page_refs.shape[0], block_table.data_ptr(),
                   block_table.stride(0), max_blocks, n_blocks.data_ptr(), tail_len.data_ptr(), page_refs.data_ptr(),
                   seqs.shape[0], seqs.data_ptr(), w.status_ptr(status, dev), L.raw_stream(index))
    if rc:
        L.check(rc, "nsnkv_free_sequences")


def reserve_pages(block_table, n_blocks, page_refs, ahead=1, status=None):
    """Pages for every sequence's next ``ahead`` blocks where its table entries name none, in
    place: in (sequence, entry) order they take the free pages in ascending order.  ``status`` gets
    NSNKV_ST_CAPACITY when too few pages are free; the entries left over stay unassigned."""
    dev, (batch, max_blocks) = block_table.device, block_table.shape
    _ints("reserve_pages", dev, block_table, n_blocks, page_refs)
    if not (n_blocks.shape == (batch,) and page_refs.ndim == 1):
        raise w.ContractError("reserve_pages tables: block_table [batch, max_blocks], n_blocks [batch]")
    index = dev.index
    rc = L.call_on(index, L.load().nsnkv_reserve_pages, batch, page_refs.shape[0], block_table.data_ptr(),
                   block_table.stride(0), max_blocks, n_blocks.data_ptr(), page_refs.data_ptr(), int(ahead),
                   w.status_ptr(status, dev), L.raw_stream(index))
    if rc:
        L.check(rc, "nsnkv_reserve_pages")


def _page_arrays(arrays, dev):
    """[h, pages, ...] tensors as nsnkv_page_array descriptors: (h, pages, ctypes array)."""
    got = _ARRAYS[len(arrays)]() if 0 < len(arrays) <= 8 else None
    lead = arrays[0].shape[:2] if got is not None else None
    for i, t in enumerate(arrays):
        shape, stride, size = t.shape, t.stride(), t.element_size()
        n = 1
        for d in range(len(shape) - 1, 1, -1):  # contiguous pages
            n = n * shape[d] if stride[d] == n or shape[d] == 1 else -1
        if got is None or len(shape) < 3 or shape[:2] != lead or t.device != dev or n <= 0:
            got = None
            break
        got[i] = (t.data_ptr(), n * size, stride[0] * size, stride[1] * size)
    if got is None:
        raise w.ContractError("page arrays: one to eight [h, pages, ...] tensors of one device with contiguous pages")
    return lead[0], lead[1], got


def copy_pages(arrays, src, dst, status=None):
    """Page dst[i] of every array ([h, pages, ...] tensors of a pool) becomes a copy of page
    src[i], for all heads (src, dst int32 [count]; no dst is the src of another pair)."""
    dev = src.device
    _ints("copy_pages", dev, src, dst)
    if src.ndim != 1 or src.shape != dst.shape:
        raise w.ContractError("copy_pages src, dst: int32 [count]")
    h, pages, arr = _page_arrays(arrays, dev)
    index = dev.index
    rc = L.call_on(index, L.load().nsnkv_copy_pages, h, pages, len(arrays), arr, src.shape[0], src.data_ptr(),
                   dst.data_ptr(), w.status_ptr(status, dev), L.raw_stream(index))
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
    dev, (batch, max_blocks) = block_table.device, block_table.shape
    if table_out is None:
        table_out = block_table.new_empty((batch, max_blocks))
    if refs_out is None:
        refs_out = torch.empty_like(page_refs)
    live = page_refs.new_empty(1)
    _ints("compact_pages", dev, block_table, page_refs, table_out, refs_out)
    h, pages, arr = _page_arrays(arrays, dev)
    if not (page_refs.shape == refs_out.shape == (pages,) and table_out.shape == block_table.shape):
        raise w.ContractError("compact_pages tables: block_table and table_out [batch, max_blocks], page_refs and "
                              "refs_out [pages]")
    lib, index = L.load(), dev.index
    stream = L.raw_stream(index)
    if ws is None:
        ws = L.scratch(lib.nsnkv_compact_pages_workspace_bytes(pages), dev, stream)
    else:
        w.require_workspace(ws, dev)
    rc = L.call_on(index, lib.nsnkv_compact_pages, h, pages, len(arrays), arr, batch, max_blocks,
                   block_table.data_ptr(), block_table.stride(0), table_out.data_ptr(), table_out.stride(0),
                   page_refs.data_ptr(), refs_out.data_ptr(), live.data_ptr(), ws.data_ptr(), ws.numel(),
                   w.status_ptr(status, dev), stream)
    if rc:
        L.check(rc, "nsnkv_compact_pages")
    return table_out, refs_out, live
