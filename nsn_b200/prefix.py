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
from .kernel import workspace


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
    dt, dev = q.dtype, q.device
    rows, hq = q.shape[0], q.shape[1] if q.ndim == 3 else 0
    w.require(q.ndim == 3 and q.shape[2] == w.DIM and dt in L.DTYPE_CODE and dt is not torch.float32
              and q.is_contiguous() and q.is_cuda, "prefix attention q: contiguous [rows, hq, 128] fp16 or bf16 on CUDA")
    w.require(records.dtype == torch.uint8 and records.ndim == 3 and records.stride(2) == 1 and bits in (3, 5)
              and records.shape[2] == 2 * (w.code_bytes(bits) + 768) and hq % max(1, records.shape[0]) == 0
              and hq > 0 and not (records.stride(0) | records.stride(1)) & 15,
              "prefix attention records: [h, pages, record] uint8 block records of INT3 or INT5, hq a multiple of h")
    table = page_table if page_table.ndim == 2 else page_table[None]
    groups, max_pages = table.shape
    ints = [t for t in (table, n_pages, row_offsets, row_index) if t is not None]
    w.require(all(t.dtype == torch.int32 and t.device == dev and (t.numel() == 0 or t.stride(-1) == 1) for t in ints)
              and records.device == dev, "prefix attention tables: int32 on q's device")
    w.require((n_pages is None or n_pages.shape == (groups,)) and (row_index is None or row_index.shape == (rows,))
              and (row_offsets.shape == (groups + 1,) if row_offsets is not None else groups == 1),
              "prefix attention groups: n_pages [groups], row_offsets [groups + 1], row_index [rows]")
    w.require((o_part is None) == (lse_part is None) and
              (o_part is None or (o_part.shape == q.shape and lse_part.shape == (rows, hq)
                                  and o_part.dtype == lse_part.dtype == torch.float32 and o_part.is_contiguous()
                                  and lse_part.is_contiguous() and o_part.device == dev and lse_part.device == dev)),
              "prefix attention partial: fp32 o_part [rows, hq, 128] with lse_part [rows, hq]")
    if out is None:
        out = torch.empty_like(q)
    if lse is None:
        lse = torch.empty((rows, hq), dtype=torch.float32, device=dev)
    w.require(out.shape == q.shape and out.dtype == dt and out.is_contiguous() and lse.shape == (rows, hq)
              and lse.dtype == torch.float32 and lse.is_contiguous() and out.device == dev and lse.device == dev,
              "prefix attention outputs")
    lib, h = L.load(), records.shape[0]
    need = lib.nsnkv_prefix_attn_workspace_bytes(rows, groups, hq, h, max_pages)
    if ws is None:
        ws = workspace(need, dev)
    p = lambda t: t.data_ptr() if t is not None else None
    with torch.cuda.device(dev):
        rc = lib.nsnkv_prefix_attn(
            rows, groups, int(max_rows or 0), hq, h, bits, L.DTYPE_CODE[dt], q.data_ptr(), records.data_ptr(),
            records.shape[1], records.stride(0), records.stride(1), table.data_ptr(), table.stride(0), p(n_pages),
            max_pages, p(row_offsets), p(row_index), p(o_part), p(lse_part), out.data_ptr(), lse.data_ptr(),
            ws.data_ptr(), ws.numel(), p(status), torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, "nsnkv_prefix_attn")
    return out, lse
