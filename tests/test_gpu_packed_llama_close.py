"""The decoder on packed documents beside plain operations that round where it rounds: inputs and outputs of every product in
bf16, norms, heads and the unit's output rounded to bf16 once, the residual stream in 32 bits."""
import math

import pytest
import torch
import torch.nn.functional as F

from test_gpu_packed_llama import SMALL
from test_gpu_saved8 import plain8

pytestmark = pytest.mark.gpu
DEV = "cuda"


class _Unit(torch.autograd.Function):
    """silu(g) u, rounded to bf16; gradients from what 8 bits keep of g and u."""

    @staticmethod
    def forward(ctx, g, u):
        ctx.save_for_backward(g, u)
        g, u = g.float(), u.float()
        return (g * torch.sigmoid(g) * u).bfloat16()

    @staticmethod
    def backward(ctx, dh):
        g, u = (plain8(t).float() for t in ctx.saved_tensors)
        q, d = torch.sigmoid(g), dh.float()
        return (d * u * (q + g * q * (1 - q))).bfloat16(), (d * g * q).bfloat16()


def _logits(m, idx):
    """One document."""
    T, lin = len(idx), lambda x, layer: F.linear(x, layer.weight.bfloat16())  # noqa: E731
    norm = lambda t, ln: F.layer_norm(t, (t.shape[-1],), ln.weight, None, ln.eps).bfloat16()  # noqa: E731
    x = m.emb.weight[idx] * m.emb.scale
    for b in m.blocks:
        a = norm(x, b.attn_norm)
        q, k, v = (lin(a, w).view(T, -1, b.hd) for w in (b.wq, b.wk, b.wv))
        heads = []
        for t, w in ((q, b.qk.q_weight), (k, b.qk.k_weight)):
            t = t.float()
            t = t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + b.qk.eps) * w
            lo, hi = t.chunk(2, -1)
            c, s = b.qk.cos[:T, None], b.qk.sin[:T, None]
            heads.append(torch.cat((lo * c - hi * s, lo * s + hi * c), -1).bfloat16())
        group = q.shape[1] // k.shape[1]
        q, k, v = (t.float().transpose(0, 1).repeat_interleave(n, 0) for t, n in ((heads[0], 1), (heads[1], group), (v, group)))
        score = (q @ k.transpose(1, 2) / math.sqrt(b.hd)).masked_fill(torch.ones(T, T, dtype=torch.bool, device=DEV).triu(1), -math.inf)
        x = x + lin((score.softmax(-1) @ v).transpose(0, 1).reshape(T, -1).bfloat16(), b.wo)
        f = norm(x, b.ffn_norm)
        x = x + lin(_Unit.apply(lin(f, b.w_gate), lin(f, b.w_up)), b.w_down)
    return lin(norm(x, m.norm), m.lm_head)


def _model(seed):
    import workloads
    torch.manual_seed(seed)
    m = workloads.PackedLlama(**SMALL, positions=64, device=DEV)
    for b in m.blocks:
        with torch.no_grad():
            b.qk.q_weight.uniform_(0.5, 1.5)
            b.qk.k_weight.uniform_(0.5, 1.5)
    return m


def test_logits():
    """What is left: attention's probabilities in bf16, 2^-8 in each of two blocks, and as much again for the roundings that fall
    to the other side behind it."""
    m = _model(2)
    lens = [40, 1, 64, 17]
    cu = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
    x = torch.randint(0, 300, (sum(lens),), device=DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
    with torch.no_grad():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            got = m(x, pos, cu).float()
        for i, n in enumerate(lens):
            ref = _logits(m, x[cu[i]:cu[i + 1]]).float()
            err = float((got[cu[i]:cu[i + 1]] - ref).norm() / ref.norm())
            assert err <= 4 * 2.0 ** -8


def test_gradients():
    """The same, and probabilities and their gradients in bf16 in the backward: 2^-8 for each of three roundings in each of two
    blocks, and as much again."""
    m = _model(3)
    x = torch.randint(0, 300, (64,), device=DEV)
    cu, pos = torch.tensor([0, 64], dtype=torch.int32, device=DEV), torch.arange(64, dtype=torch.int32, device=DEV)
    up = torch.randn(64, 300, device=DEV)
    params = dict(m.named_parameters())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = m(x, pos, cu)
    got = torch.autograd.grad(logits.float(), list(params.values()), up)
    ref = torch.autograd.grad(_logits(m, x).float(), list(params.values()), up)
    for name, a, b in zip(params, got, ref):
        err = float((a - b).norm() / b.norm())
        assert err <= 12 * 2.0 ** -8, name
