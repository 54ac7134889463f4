"""Causal attention over whole prompts packed one after another (nsnkv_prompt_attn).

What the model's own attention computes over a prompt before the cache compresses it
(experiments/nb06/source/loop_kv_nb06_attention.py:33-88, the OFFICIAL arm), for a batch of
prompts of different lengths without padding and without repeating K and V for grouped heads.
"""
from __future__ import annotations

import torch

from . import _lib as L
from . import primitives as w


def prompt_attention(q, k, v, cu_seqlens, max_seqlen, *, causal=True, out=None, lse=None, status=None):
    """Attention of q [T, hq, 128] over k, v [T, h, 128] (fp16 or bf16) within each sequence
    cu_seqlens[s] .. cu_seqlens[s + 1] (int32 [seqs + 1] on the GPU, ascending from 0 to T).

    q, k and v may be views with any token and head strides that are multiples of 8 elements
    (slices of one fused projection).  ``max_seqlen``: the longest sequence, as far as known:
    it sizes the launch, not the result.  Returns (out [T, hq, 128] in the inputs' dtype,
    lse [T, hq] fp32); rows that no sequence covers are not written.  ``status`` (int32 [1]):
    NSNKV_ST_OUTPUT_NONFINITE is OR-ed in when an output is not finite.  No host sync.
    """
    dt, dev = q.dtype, q.device
    ok = (q.ndim == 3 and k.ndim == 3 and dt in L.DTYPE_CODE and dt is not torch.float32 and q.shape[2] == w.DIM
          and k.shape == v.shape and k.shape[0] == q.shape[0] and k.shape[2] == w.DIM and k.dtype == dt
          and v.dtype == dt and k.shape[1] > 0 and q.shape[1] % k.shape[1] == 0)
    w.require(ok, "prompt attention operands: q [T, hq, 128], k and v [T, h, 128], fp16 or bf16, hq a multiple of h")
    w.require(cu_seqlens.dtype == torch.int32 and cu_seqlens.ndim == 1 and cu_seqlens.numel() > 0
              and cu_seqlens.is_contiguous(), "prompt attention cu_seqlens: contiguous int32 [seqs + 1]")
    w.require(q.is_cuda and k.device == dev and v.device == dev and cu_seqlens.device == dev,
              "prompt attention operands on one CUDA device")
    (qt, qh, qc), (kt, kh, kc), (vt, vh, vc) = q.stride(), k.stride(), v.stride()
    w.require(qc == kc == vc == 1 and not (qt | qh | kt | kh | vt | vh) & 7
              and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15,
              "prompt attention strides: contiguous channels, strides multiples of 8, 16-byte aligned")
    T, hq = q.shape[0], q.shape[1]
    if out is None:
        out = torch.empty((T, hq, w.DIM), dtype=dt, device=dev)
    if lse is None:
        lse = torch.empty((T, hq), dtype=torch.float32, device=dev)
    w.require(out.shape == q.shape and out.dtype == dt and out.is_contiguous() and lse.shape == (T, hq)
              and lse.dtype == torch.float32 and lse.is_contiguous() and out.device == dev and lse.device == dev,
              "prompt attention outputs")
    with torch.cuda.device(dev):
        rc = L.load().nsnkv_prompt_attn(
            T, cu_seqlens.numel() - 1, int(max_seqlen), hq, k.shape[1], L.DTYPE_CODE[dt], int(bool(causal)),
            q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, cu_seqlens.data_ptr(), out.data_ptr(),
            lse.data_ptr(), status.data_ptr() if status is not None else None,
            torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, "nsnkv_prompt_attn")
    return out, lse
