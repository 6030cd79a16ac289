"""Layer norm with its gradient (concord_layer_norm_fwd / _bwd).

The reference's trained models normalise with torch's nn.LayerNorm around
the packed layers (notebook/src/nanogpt.py:15-101); these kernels take its
place: statistics and the sums of the weight's gradient in fp32, the output
rounded once to the type that the next layer reads.
"""
import torch
import torch.nn as nn

from . import _ops


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x: fp32, bf16 or fp16, of any shape and strides, at most 16384 wide (a
    last dimension that is not contiguous is copied).  weight and bias [D]
    (either may be None); fp32 is read as it is, other types are converted.
    The result has `out_dtype` (default: x's type); statistics, sums and the
    gradients of weight and bias are fp32.  Differentiable once, backward only.
    """
    _ops.need_cuda(("x", x), ("weight", weight), ("bias", bias))
    _ops.need_type("x", x, _ops.TYPES)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _ops.TYPES:
        raise TypeError(f"out_dtype must be one of {[str(t) for t in _ops.TYPES]}, got {out_dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    D = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (D,):
            raise ValueError(f"{name} must have shape ({D},), got {tuple(t.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if weight is not None:
        weight = weight.float().contiguous()
    if bias is not None:
        bias = bias.float().contiguous()
    return _ops.native().layer_norm(x, weight, bias, eps, _ops.TYPES[out_dtype])


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over one dimension on `layer_norm`; `out_dtype` as there
    (bf16 hands the next packed layer its input without another cast)."""

    def __init__(self, dim, eps=1e-5, elementwise_affine=True, bias=True, out_dtype=None, device=None, dtype=None):
        super().__init__(dim, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises over the last dimension only")
        self.out_dtype = out_dtype

    def forward(self, x):
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"expected a last dimension of {self.normalized_shape[0]}, got {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps, self.out_dtype)
