"""Activations kept in 8 bits for the backward pass (concord_save8, _dense8,
_gemm_dw8, concord_gated_fwd / _bwd).

With a packed layer's optimizer state inside its weight, what a training step
holds beside the weights is activations, most of them inputs of linear layers
and of the gated unit between them.  Here they are kept as 8-bit whole numbers, 32
tokens of one feature sharing a power of two (8.25 bits a value), and the
backward computes from these: a packed layer's weight gradient
(`layer(x, saved=save8(x))`, or `layer.save8 = True`) and the gated unit's.
Outputs and the gradient that goes on to earlier layers through a packed layer
do not change.
"""
import torch

from . import _abi, _ops
from . import gemm as _gemm

ACTS = {"silu": 0, "gelu": 1}


class Saved8:
    """x [..., K] in 8 bits: `data` (the bytes), `shape` and `dtype` of x."""

    def __init__(self, data, shape, dtype):
        self.data, self.shape, self.dtype = data, torch.Size(shape), dtype

    @property
    def rows(self):
        return self.shape[:-1].numel()

    @property
    def nbytes(self):
        return self.data.numel()

    def dense(self, dtype=None):
        """The values that are kept, as a tensor of x's shape and type (or `dtype`)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _ops.TYPES:
            raise TypeError(f"dtype must be one of {[str(t) for t in _ops.TYPES]}, got {dtype}")
        out = _ops.native().dense8(self.data, self.rows, self.shape[-1], _ops.TYPES[dtype])
        return out.view(self.shape)

    def __repr__(self):
        return f"Saved8({tuple(self.shape)}, {self.dtype}, {self.nbytes} bytes on {self.data.device})"


def _check_saved(saved):
    if not isinstance(saved, Saved8):
        raise TypeError(f"saved must be a Saved8 (see save8), got {type(saved).__name__}")


def save8(x):
    """x [..., K] (fp32, bf16 or fp16; columns that are not contiguous are copied) as a Saved8.

    32 tokens (rows, in order) of one feature share a power of two 2^e, the
    least with |x| <= 127 2^e, -126 at least; a value is the whole number nearest to x / 2^e, off by
    at most 2^(e - 1), which is less than the 32 values' largest magnitude / 127 (where that is above
    2^-120).  At the top of a type's range, where 64 steps are more than it holds, it ends at 63 steps: fp16's 65504 is
    kept as 64512.
    One NaN or infinity makes its 32 values NaN.  Not differentiable: the result stands for
    x in a backward pass.
    """
    _ops.need_cuda(("x", x))
    _ops.need_type("x", x, _ops.TYPES)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 1 << 20:
        raise ValueError(f"x needs a last dimension of 1 to 2^20, got shape {tuple(x.shape)}")
    return Saved8(_ops.native().save8(x), x.shape, x.dtype)


def grad_weight8(grad_y, saved):
    """dW = dY^T x, bf16 [N, K], for dY [..., N] (bf16) and the Saved8 of x [..., K]:
    the product of gemm.grad_weight with the values that `saved` keeps (exact in
    bf16), fp32 sums rounded once, the same bits on every run.  N in multiples of 8 (others read
    x back and go through torch's product)."""
    _check_saved(saved)
    _ops.need_cuda(("grad_y", grad_y), ("saved", saved.data))
    _ops.need_type("grad_y", grad_y, (torch.bfloat16,))
    if grad_y.dim() != len(saved.shape) or grad_y.shape[:-1] != saved.shape[:-1] or grad_y.shape[-1] < 1:
        raise ValueError(f"grad_y must be [..., N] beside x {tuple(saved.shape)}, got {tuple(grad_y.shape)}")
    if grad_y.shape[-1] % 8:
        return _gemm.grad_weight(grad_y.reshape(-1, grad_y.shape[-1]),
                                 saved.dense(torch.bfloat16).view(-1, saved.shape[-1]))
    return _ops.native().grad_weight8(grad_y, saved.data, saved.rows, saved.shape[-1])


def gated_unit(gate, up, act="silu", save8=False, out8=False):
    """act(gate) * up: gate and up [..., K] of one type (fp32, bf16 or fp16), act "silu" or
    "gelu" (of the error function).

    gate and up may have strides of their own (halves of one projection are
    read in place).  Arithmetic is fp32, the result (contiguous, of their type) rounded once.
    (For 16-bit types the functions are approximations, gelu's normal distribution function off by 2.9e-7, relative to it by
    1.6e-3 at -5, where gelu is 1.4e-6.)
    save8: a call that is differentiated keeps gate and up in 8 bits (see
    `save8`) in place of the tensors themselves, and their gradients are computed from these.
    out8: returns (h, Saved8 of h) in the same pass, for the packed layer that
    reads h: `layer(h, saved=h8)`.  Differentiable once, backward only.
    """
    _ops.need_cuda(("gate", gate), ("up", up))
    _ops.need_type("gate", gate, _ops.TYPES)
    if up.dtype != gate.dtype:
        raise TypeError(f"up must have gate's type {gate.dtype}, got {up.dtype}")
    if gate.dim() < 1 or up.shape != gate.shape or not 1 <= gate.shape[-1] <= 1 << 20:
        raise ValueError(f"gate and up must have one shape [..., K], got {tuple(gate.shape)} and {tuple(up.shape)}")
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}, got {act!r}")
    h, h8 = _ops.native().gated_unit(gate, up, ACTS[act], bool(save8), bool(out8))
    return (h, Saved8(h8, h.shape, h.dtype)) if out8 else h


def gemm_dw8_error(reset=False):
    """Code of the first wait inside grad_weight8's kernel that ran out on the
    current device, 0 if none did (its outputs are NaN then, and later calls raise).
    Synchronises; `reset` clears it, after which calls are taken again."""
    return _abi.load().concord_gemm_dw8_error(int(reset))
