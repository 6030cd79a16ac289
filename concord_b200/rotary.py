"""Norm of query and key heads with the position rotation in the same pass
(concord_qk_norm_rope_fwd / _bwd), between the projections and packed_attention.
"""
import torch
import torch.nn as nn

from . import _ops

_INTS = (torch.int64, torch.int32)


def rope_tables(positions, rot, base=10000.0, device="cuda"):
    """(cos, sin), fp32 [positions, rot / 2], of position * base ** (-2 i / rot):
    angles and functions in 64 bits, so that far positions lose nothing."""
    if rot < 2 or rot % 2 or positions < 1:
        raise ValueError(f"an even number of rotated columns and at least one position, got {rot} and {positions}")
    if not 0 < base < float("inf"):
        raise ValueError(f"base must be positive, got {base}")
    at = torch.arange(positions, dtype=torch.float64, device=device)
    freq = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = at[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def qk_norm_rope(q, k, cos=None, sin=None, positions=None, q_weight=None, k_weight=None, norm=True, eps=1e-6,
                 interleaved=False):
    """(q', k'): every head's root-mean-square norm, then the rotation of its
    first columns, in one pass over q and k.

    q [T, H, D], k [T, Hk, D] or None (then k' is None): one type of fp32, bf16 and
    fp16, D up to 256, any strides (columns that are not contiguous are
    copied): views of one projection's output are read in place.
    norm: x / sqrt(mean(x^2) + eps) * weight over a head's D columns, q_weight and
    k_weight [D] for all heads of q and of k (None: ones).  norm=False: rotation alone.
    cos, sin [P, R / 2] (see rope_tables; None: the norm alone): the first R columns
    turn, pair i being columns (i, i + R / 2), or (2 i, 2 i + 1) where
    `interleaved`, by the angle of the token's position.
    positions [T] (int32 or int64; default: the row's number): a position that the
    tables do not have gives NaN in the columns that turn.

    q' and k' are contiguous, of the inputs' type, rounded once; sums are fp32.  The
    gradients of the weights are fp32 sums in a fixed order: the same bits on
    every run.  Differentiable once, backward only, for q, k and the weights.
    """
    _ops.need_cuda(("q", q), ("k", k), ("cos", cos), ("sin", sin), ("positions", positions), ("q_weight", q_weight),
                   ("k_weight", k_weight))
    if q is None:
        raise TypeError("q must be a tensor, got None")
    # (a token's step waits for these checks: each shape is asked for once)
    dtype, shape = q.dtype, q.shape
    _ops.need_type("q", q, _ops.TYPES)
    if len(shape) != 3 or shape[1] < 1 or not 1 <= shape[2] <= 256:
        raise ValueError(f"q must be [T, H, D] with D up to 256, got shape {tuple(shape)}")
    T, _, D = shape
    if k is not None:
        if k.dtype != dtype:
            raise TypeError(f"k must have q's type {dtype}, got {k.dtype}")
        ks = k.shape
        if len(ks) != 3 or ks[0] != T or ks[1] < 1 or ks[2] != D:
            raise ValueError(f"k must be [T, Hk, D] beside q {tuple(shape)}, got {tuple(ks)}")
    elif k_weight is not None:
        raise ValueError("k_weight without k")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if not norm:
            raise ValueError(f"{name} belongs to the norm: pass norm=True")
        if w.shape != (D,):
            raise ValueError(f"{name} must have shape ({D},), got {tuple(w.shape)}")
        _ops.need_type(name, w, _ops.TYPES)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        _ops.need_type("cos", cos, _ops.TYPES)
        _ops.need_type("sin", sin, _ops.TYPES)
        cs = cos.shape
        if len(cs) != 2 or sin.shape != cs or cs[0] < 1 or not 1 <= cs[1] <= D // 2:
            raise ValueError(f"cos and sin must be [P, R / 2] with R up to {D}, got {tuple(cs)}, {tuple(sin.shape)}")
        if positions is not None:
            _ops.need_type("positions", positions, _INTS)
            if positions.shape != (T,):
                raise ValueError(f"positions must have shape ({T},), got {tuple(positions.shape)}")
    elif positions is not None:
        raise ValueError("positions without cos and sin")
    elif not norm:
        raise ValueError("neither norm nor rotation: nothing to do")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return _ops.native().qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, bool(norm), float(eps),
                                      bool(interleaved))


class QKNormRope(nn.Module):
    """`qk_norm_rope` with its weights (q_weight, k_weight [head_dim], ones at the start)
    and its tables for `positions` positions (not in the state dict; fp32 whatever type the module is cast to, and
    made anew where it is given memory: built on the meta device, then to_empty)."""

    base = 10000.0                  # (for modules that were pickled before they kept it)

    def __init__(self, head_dim, positions, rot=None, base=10000.0, eps=1e-6, interleaved=False, device=None):
        super().__init__()
        self.q_weight, self.k_weight = (nn.Parameter(torch.ones(head_dim, device=device)) for _ in range(2))
        cos, sin = rope_tables(positions, head_dim if rot is None else rot, base, device=self.q_weight.device)
        self.register_buffer("cos", cos, persistent=False)
        self.register_buffer("sin", sin, persistent=False)
        self.base, self.eps, self.interleaved = base, eps, interleaved

    def _apply(self, fn, recurse=True):
        # fn says where the tables go; what it makes of them (another type, to_empty's bare memory) is not theirs
        cos, sin = self.cos, self.sin
        super()._apply(fn, recurse)
        device = self.cos.device
        if cos.is_meta and device.type != "meta":
            self.cos, self.sin = rope_tables(cos.shape[0], 2 * cos.shape[1], self.base, device=device)
        else:
            self.cos, self.sin = cos.to(device), sin.to(device)
        return self

    def forward(self, q, k, positions=None):
        return qk_norm_rope(q, k, self.cos, self.sin, positions, self.q_weight, None if k is None else self.k_weight,
                            eps=self.eps, interleaved=self.interleaved)
