"""The gated unit in fp32: as exact as the functions it calls, relative to the value, where act(g) and its derivative are far
below 1 too."""
import math

import pytest
import torch

from test_gpu_saved8 import plain8

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _plain(g, u, d, act):
    """(value, bound) of h, dgate and dup.  Bounds count roundings (U each, relative) and the functions' documented errors:
    expf 2 units in the last place (4 U), erfcf 4 (8 U), division and the other operations one rounding.
    silu: e = exp(-g), q = 1 / (1 + e): off by (4 (1 - q) + 2) U q.  gelu: Phi = erfc(-g / sqrt 2) / 2, whose argument is off by
    2 U relative, which counts 2 x e^(-x^2) / (sqrt(pi) erfc x) times; g phi(g) = g c exp(-g^2 / 2), off by (g^2 / 2 + 8) U."""
    g, u, d = g.double(), u.double(), d.double()
    if act == "silu":
        q = torch.sigmoid(g)
        a, q_lim = g * q, (4 * (1 - q) + 2) * U * q
        a_lim = g.abs() * q_lim + U * a.abs()
        da = q + a * (1 - q)
        da_lim = q_lim + a.abs() * (q_lim + U) + (a_lim + U * a.abs()) * (1 - q) + U * da.abs()
    else:
        x = -g / math.sqrt(2)
        p = torch.special.erfc(x) / 2
        k = (x * torch.exp(-x.square())).abs() / (math.sqrt(math.pi) * p)
        k = torch.where(p > 0, k, 2 * x.square() + 1)
        p_lim = (2 * k + 8) * U * p
        a, phi = g * p, g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        a_lim = g.abs() * p_lim + U * a.abs()
        da = p + phi
        da_lim = p_lim + (g.square() / 2 + 8) * U * phi.abs() + U * da.abs()
    h, dg, du = a * u, d * u * da, d * a
    return ((h, a_lim * u.abs() + U * h.abs()), (dg, (d * u).abs() * da_lim + 2 * U * dg.abs()),
            (du, a_lim * d.abs() + U * du.abs()))


def _near(got, ref, lim):
    """(a second-order part of the bound: 2^-20 of it; values that fp32 holds as subnormals, or flushes: 2^-124)"""
    return bool(((got.double() - ref).abs() <= lim * (1 + 2.0 ** -20) + 2.0 ** -124).all())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("K", [4096, 4095])
def test_relative_error(K, eight, act):
    """g from -12 to 12 (and small ones of either sign), whole pieces and single elements, kept in 8 bits and as they are."""
    from concord_b200 import gated_unit
    r = torch.Generator(device=DEV).manual_seed(K)
    gate = torch.linspace(-12, 12, 64 * K, device=DEV).view(K, 64).t().contiguous()
    gate[5] *= 2.0 ** -10
    gate[6] *= 2.0 ** -40
    up, dh = (torch.randn(64, K, generator=r, device=DEV) for _ in range(2))
    gate.requires_grad_(), up.requires_grad_()
    h = gated_unit(gate, up, act, save8=eight)
    dg, du = torch.autograd.grad(h, (gate, up), dh)
    assert _near(h, *_plain(gate.detach(), up.detach(), dh, act)[0])
    kept = [plain8(t.detach()).float() if eight else t.detach() for t in (gate, up)]
    _, want_g, want_u = _plain(*kept, dh, act)
    assert _near(dg, *want_g) and _near(du, *want_u)
    with torch.no_grad():
        assert torch.equal(gated_unit(gate, up, act), h)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_borders(act):
    """What is large, infinite or no number."""
    from concord_b200 import gated_unit
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([0.0, -0.0, 1e4, -1e4, 3e38, -3e38, 1e-40, -1e-40, nan, inf], device=DEV, requires_grad=True)
    one = torch.ones(10, device=DEV)
    h = gated_unit(g, one, act)
    (dg,) = torch.autograd.grad(h, g, one)
    want = [0, 0, 1e4, 0, 3e38, 0, 0, 0]
    assert torch.allclose(h[:8].detach(), torch.tensor(want, device=DEV), rtol=1e-6, atol=1e-39)
    assert bool(h[8].isnan()) and h[9].item() == inf
    assert torch.allclose(dg[:8], torch.tensor([0.5, 0.5, 1, 0, 1, 0, 0.5, 0.5], device=DEV), rtol=1e-6, atol=0)
    assert bool(dg[8].isnan())
