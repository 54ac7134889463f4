"""Attention over a sealed prefix that many query rows share (nsnkv_prefix_attn).

A batch whose sequences start from one prompt keeps that prompt's blocks once; this operator
reads and restores each of them once per kv head for all rows, and merges the result with
what each row attended to on its own (its sequence's private blocks and tail when decoding,
its new tokens when a prompt continues after a cached one).  No counterpart in the reference,
whose caches belong to one sequence each.
"""
from __future__ import annotations

import torch

from . import _lib as L
from . import primitives as w

_TYPES = {torch.float16: L.F16, torch.bfloat16: L.BF16}
_RECORD = {bits: 2 * (w.code_bytes(bits) + 768) for bits in (3, 5)}


def _ints(t, n, dev):
    return t is None or (t.dtype == torch.int32 and t.ndim == 1 and t.shape[0] == n and t.device == dev
                         and t.is_contiguous())


def prefix_attention(q, records, page_table, n_pages=None, *, bits=3, row_offsets=None, row_index=None, max_rows=None,
                     o_part=None, lse_part=None, out=None, lse=None, status=None, ws=None):
    """Attention of q [rows, hq, 128] (fp16 or bf16) over shared sealed prefixes.

    ``records`` [h, pages, record] uint8: block records as ``paged.block_record_pools`` lays them
    out (INT3 or INT5).  ``page_table`` int32 [groups, max_pages] (or [max_pages]: one group):
    group g's prefix is its first n_pages[g] entries (``n_pages`` int32 [groups], None: all).
    ``row_offsets`` int32 [groups + 1]: group g's rows are positions row_offsets[g] ..
    row_offsets[g + 1] - 1 of ``row_index`` (int32 [rows], None: rows in order); None: one group of
    all rows.  ``max_rows``: the most rows of a group, as far as known (sizes the launch only).
    ``o_part`` [rows, hq, 128] and ``lse_part`` [rows, hq] fp32: each row's attention over its own
    tokens (normalised output and natural log-sum-exp, -inf for none), merged in.

    K and V rows are restored and rounded to q's dtype as the bridge's restore_group rounds
    them.  Returns (out [rows, hq, 128], lse [rows, hq] fp32).  ``status`` (int32 [1]): the
    NSNKV_ST_* bits of nsnkv_prefix_attn.  ``ws``: scratch of at least
    nsnkv_prefix_attn_workspace_bytes (default: one buffer per stream).  No host sync.
    """
    dt, dev, qs, rs = q.dtype, q.device, q.shape, records.shape
    rows, hq = (qs[0], qs[1]) if len(qs) == 3 else (0, 0)
    if not (hq > 0 and qs[2] == w.DIM and dt in _TYPES and q.is_contiguous() and q.is_cuda):
        raise w.ContractError("prefix attention q: contiguous [rows, hq, 128] fp16 or bf16 on CUDA")
    if not (len(rs) == 3 and rs[2] == _RECORD.get(bits) and rs[0] > 0 and hq % rs[0] == 0
            and records.dtype == torch.uint8 and records.device == dev):
        raise w.ContractError("prefix attention records: [h, pages, record] uint8 block records of INT3 or INT5 on q's "
                              "device, hq a multiple of h")
    head, page, byte = records.stride()
    if byte != 1 or (head | page) & 15:
        raise w.ContractError("prefix attention records: contiguous records, strides multiples of 16")
    table = page_table if page_table.ndim == 2 else page_table[None]
    groups, max_pages = table.shape
    if not (table.dtype == torch.int32 and table.device == dev and (max_pages <= 1 or table.stride(1) == 1)
            and _ints(n_pages, groups, dev) and _ints(row_index, rows, dev) and _ints(row_offsets, groups + 1, dev)
            and (row_offsets is not None or groups == 1)):
        raise w.ContractError("prefix attention tables: int32 on q's device: page_table [groups, max_pages], n_pages "
                              "[groups], row_offsets [groups + 1] (needed with groups), row_index [rows]")
    o_ptr = e_ptr = None
    if o_part is not None or lse_part is not None:
        if not (o_part is not None and lse_part is not None and o_part.shape == qs and lse_part.shape == qs[:2]
                and o_part.dtype == lse_part.dtype == torch.float32 and o_part.is_contiguous()
                and lse_part.is_contiguous() and o_part.device == dev and lse_part.device == dev):
            raise w.ContractError("prefix attention partial: fp32 o_part [rows, hq, 128] with lse_part [rows, hq]")
        o_ptr, e_ptr = o_part.data_ptr(), lse_part.data_ptr()
    if out is None:
        out = torch.empty_like(q)
    elif not (out.shape == qs and out.dtype == dt and out.is_contiguous() and out.device == dev):
        raise w.ContractError("prefix attention out: contiguous, of q's shape, dtype and device")
    if lse is None:
        lse = q.new_empty((rows, hq), dtype=torch.float32) if lse_part is None else torch.empty_like(lse_part)
    elif not (lse.shape == qs[:2] and lse.dtype == torch.float32 and lse.is_contiguous() and lse.device == dev):
        raise w.ContractError("prefix attention lse: contiguous fp32 [rows, hq] on q's device")
    lib, index = L.load(), dev.index
    stream = L.raw_stream(index)
    if ws is None:
        ws = L.scratch(lib.nsnkv_prefix_attn_workspace_bytes(rows, groups, hq, rs[0], max_pages), dev, stream)
    else:
        w.require_workspace(ws, dev)
    rc = L.call_on(
        index, lib.nsnkv_prefix_attn, rows, groups, int(max_rows or 0), hq, rs[0], bits, _TYPES[dt], q.data_ptr(),
        records.data_ptr(), rs[1], head, page, table.data_ptr(), table.stride(0),
        None if n_pages is None else n_pages.data_ptr(), max_pages,
        None if row_offsets is None else row_offsets.data_ptr(), None if row_index is None else row_index.data_ptr(),
        o_ptr, e_ptr, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(),
        w.status_ptr(status, dev), stream)
    if rc:
        L.check(rc, "nsnkv_prefix_attn")
    return out, lse
