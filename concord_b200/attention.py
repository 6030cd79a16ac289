"""Attention over packed sequences with its gradient (concord_attention_fwd / _bwd).

The reference's trained models attend through torch's
scaled_dot_product_attention on a padded batch (notebook/src/nanogpt.py:15-101);
here a batch is its documents one after the other, with no padding between
them, read in place from the projection's output.
"""
import torch

from . import _abi, _ops

_HALVES = (torch.bfloat16, torch.float16)


def packed_attention(q, k, v, cu_seqlens, cu_seqlens_k=None, causal=True, scale=None, return_lse=False):
    """softmax(scale q k^T) v within each of several packed sequences.

    q [T, H, D], k and v [Tk, Hk, D]: bf16 or fp16, H a multiple of Hk (query
    head h reads key head h // (H // Hk)), D a multiple of 8 up to 128.  Any
    strides: views of one projection's output are read in place as long as
    rows start on 16 bytes, other layouts are copied.
    cu_seqlens [B + 1] (int32 on the device; int64 is converted): sequence b
    is rows cu_seqlens[b] .. cu_seqlens[b + 1], of any length, 0 included (the
    bounds do not fall; they are clamped to the tensors, not checked).
    cu_seqlens_k: the same for the keys, where they differ (cross attention, a
    prompt's next chunk after cached keys); default: cu_seqlens.
    causal: query i of a sequence with Lq queries and Lk keys sees the keys up
    to i + Lk - Lq.  A query that sees none gives 0 (and lse -inf).  Rows of no
    sequence give 0, and get and give no gradient.
    scale: positive, default D ** -0.5.

    Returns o [T, H, D], contiguous, and with return_lse also the fp32
    log-sum-exp [H, T] (not differentiable).  Scores, sums and lse are fp32;
    the probabilities and their gradients are rounded to the inputs' type for
    their products with v, k and q (in fp16's backward after scaling by powers
    of two, so that neither many keys nor small upstream gradients take them
    below fp16's range).  Differentiable once, without atomics: the
    same bits on every run.  A call that is differentiated keeps q, k, v, o, lse
    and what o's rounding left over (as large as o); the backward takes an fp32
    workspace for few keys with shared heads, and a small one in fp16.

    Waits inside the kernels are bounded (2 s).  If one runs out, the results
    hold NaN and every later call on the device raises until
    `attention_error(reset=True)`.
    """
    _ops.need_cuda(("q", q), ("k", k), ("v", v), ("cu_seqlens", cu_seqlens), ("cu_seqlens_k", cu_seqlens_k))
    _ops.need_type("q", q, _HALVES)
    for name, t in (("k", k), ("v", v)):
        if t.dtype != q.dtype:
            raise TypeError(f"{name} must have q's type {q.dtype}, got {t.dtype}")
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"q must be [T, H, D], k and v [Tk, Hk, D]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    H, D = q.shape[1:]
    if k.shape[2] != D or k.shape[1] < 1 or H < 1 or H % k.shape[1]:
        raise ValueError(f"q's {H} heads must be a multiple of k's, of the same size: got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"head size must be a multiple of 8 up to 128, got {D}")
    cus = []
    for name, cu in (("cu_seqlens", cu_seqlens), ("cu_seqlens_k", cu_seqlens_k)):
        if cu is None:
            cus.append(cus[0])
            continue
        _ops.need_type(name, cu, (torch.int32, torch.int64))
        if cu.dim() != 1 or cu.numel() < 2:
            raise ValueError(f"{name} must be [B + 1] with B >= 1, got shape {tuple(cu.shape)}")
        cus.append(cu.to(torch.int32).contiguous())
    if cus[0].numel() != cus[1].numel():
        raise ValueError(f"cu_seqlens and cu_seqlens_k must have one length, got {cus[0].numel()} and {cus[1].numel()}")
    if cu_seqlens_k is None and k.shape[0] != q.shape[0]:
        raise ValueError(f"k has {k.shape[0]} rows and q {q.shape[0]}: pass cu_seqlens_k")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise ValueError(f"scale must be positive, got {scale}")
    o, lse = _ops.native().attention(q, k, v, cus[0], cus[1], causal, scale)
    return (o, lse) if return_lse else o


def attention_error(reset=False):
    """Code of the first wait inside an attention kernel of the current device
    that ran out, 0 if none did.  Synchronises; `reset` clears it, after which
    calls are taken again."""
    return _abi.load().concord_attention_error(int(reset))
