"""Embedding lookup with scaling, and the table's gradient by sorted tokens
(concord_embedding_fwd / _bwd).

The reference's trained models look their tokens and positions up with torch's
nn.Embedding (notebook/src/nanogpt.py:15-101), an ordinary parameter beside
the packed layers; these kernels take its place.
"""
import torch
import torch.nn as nn

from . import _ops

_INTS = (torch.int64, torch.int32)


def embedding(ids, weight, scale=1.0, padding_idx=None, out_dtype=None):
    """weight[ids] * scale: [..., D] for ids [...] (int32 or int64) and a table [V, D].

    weight: fp32, bf16 or fp16, rows of any stride (columns that are not
    contiguous are copied).  A row whose id is outside [0, V), such as -1 for
    padding, is 0.  The result has `out_dtype` (default: weight's type).

    The gradient, of weight's type, is dense: each row the sum of its tokens'
    upstream gradients times scale, in fp32, by pieces of up to 32 tokens in
    order, rounded once: the same bits on every run.  Ids outside the table and `padding_idx` (a row that is
    looked up as any other) get none.  Differentiable once, backward only.
    """
    _ops.need_cuda(("ids", ids), ("weight", weight))
    _ops.need_type("ids", ids, _INTS)
    _ops.need_type("weight", weight, _ops.TYPES)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [V, D], got shape {tuple(weight.shape)}")
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    if out_dtype not in _ops.TYPES:
        raise TypeError(f"out_dtype must be one of {[str(t) for t in _ops.TYPES]}, got {out_dtype}")
    V = weight.shape[0]
    if padding_idx is not None and not -V <= padding_idx < V:
        raise ValueError(f"padding_idx must be a row of the table's {V}, got {padding_idx}")
    padding = -1 if padding_idx is None else padding_idx % V
    return _ops.native().embedding(ids, weight, float(scale), padding, _ops.TYPES[out_dtype])


class Embedding(nn.Embedding):
    """nn.Embedding's state on `embedding`, with `scale` (such as sqrt(dim))
    and `out_dtype` as there."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, out_dtype=None, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale, self.out_dtype = scale, out_dtype

    @classmethod
    def from_pretrained(cls, embeddings, freeze=True, padding_idx=None, scale=1.0, out_dtype=None):
        """The module around a table [V, D], which is not copied."""
        if embeddings.dim() != 2:
            raise ValueError(f"embeddings must be [V, D], got shape {tuple(embeddings.shape)}")
        module = cls(*embeddings.shape, padding_idx, scale, out_dtype, device="meta")
        module.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return module

    def forward(self, ids):
        return embedding(ids, self.weight, self.scale, self.padding_idx, self.out_dtype)
