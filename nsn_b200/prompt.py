"""Causal attention over whole prompts packed one after another (nsnkv_prompt_attn).

What the model's own attention computes over a prompt before the cache compresses it
(experiments/nb06/source/loop_kv_nb06_attention.py:33-88, the OFFICIAL arm), for a batch of
prompts of different lengths without padding and without repeating K and V for grouped heads.
"""
from __future__ import annotations

import torch

from . import _lib as L
from . import primitives as w

_TYPES = {torch.float16: L.F16, torch.bfloat16: L.BF16}


def prompt_attention(q, k, v, cu_seqlens, max_seqlen, *, causal=True, out=None, lse=None, status=None):
    """Attention of q [T, hq, 128] over k, v [T, h, 128] (fp16 or bf16) within each sequence
    cu_seqlens[s] .. cu_seqlens[s + 1] (int32 [seqs + 1] on the GPU, ascending from 0 to T).

    q, k and v may be views with any token and head strides that are multiples of 8 elements
    (slices of one fused projection).  ``max_seqlen``: the longest sequence, as far as known
    (0: not known): it sizes the launch, not the result.  Returns (out [T, hq, 128] in the inputs' dtype,
    lse [T, hq] fp32); rows that no sequence covers are not written.  ``status`` (int32 [1]):
    NSNKV_ST_OUTPUT_NONFINITE is OR-ed in when an output is not finite.  No host sync.
    """
    dt, dev = q.dtype, q.device
    qs, ks = q.shape, k.shape
    T, hq, h = (qs[0], qs[1], ks[1]) if len(qs) == 3 and len(ks) == 3 else (0, 0, 0)
    if not (h > 0 and hq % h == 0 and qs[2] == ks[2] == w.DIM and ks[0] == T and v.shape == ks and k.dtype == dt
            and v.dtype == dt and dt in _TYPES):
        raise w.ContractError("prompt attention operands: q [T, hq, 128], k and v [T, h, 128], fp16 or bf16, "
                              "hq a multiple of h")
    n = cu_seqlens.numel() - 1
    if not (cu_seqlens.dtype == torch.int32 and cu_seqlens.ndim == 1 and n >= 0 and cu_seqlens.is_contiguous()):
        raise w.ContractError("prompt attention cu_seqlens: contiguous int32 [seqs + 1]")
    if not (q.is_cuda and k.device == dev and v.device == dev and cu_seqlens.device == dev):
        raise w.ContractError("prompt attention operands on one CUDA device")
    (qt, qh, qc), (kt, kh, kc), (vt, vh, vc) = q.stride(), k.stride(), v.stride()
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not (qc == kc == vc == 1 and not (qt | qh | kt | kh | vt | vh) & 7 and not (qp | kp | vp) & 15):
        raise w.ContractError("prompt attention strides: contiguous channels, strides multiples of 8, 16-byte aligned")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(qs)
    elif not (out.shape == qs and out.dtype == dt and out.is_contiguous() and out.device == dev):
        raise w.ContractError("prompt attention out: contiguous, of q's shape, dtype and device")
    if lse is None:
        lse = q.new_empty((T, hq), dtype=torch.float32)
    elif not (lse.shape == (T, hq) and lse.dtype == torch.float32 and lse.is_contiguous() and lse.device == dev):
        raise w.ContractError("prompt attention lse: contiguous fp32 [T, hq] on q's device")
    index = dev.index
    rc = L.call_on(index, L.load().nsnkv_prompt_attn, T, n, int(max_seqlen), hq, h, _TYPES[dt], 1 if causal else 0, qp, qt,
                   qh, kp, kt, kh, vp, vt, vh, cu_seqlens.data_ptr(), out.data_ptr(), lse.data_ptr(),
                   w.status_ptr(status, dev), L.raw_stream(index))
    if rc:
        L.check(rc, "nsnkv_prompt_attn")
    return out, lse
