"""gated_unit against its definition in 64 bits."""
import math

import pytest
import torch

from test_gpu_saved8 import plain8

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _asked():
    """Bytes that tensors asked for (a block of the allocator may be up to 1 MB larger)."""
    return torch.cuda.memory_stats()["requested_bytes.all.current"]

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def _plain(gate, up, dh, act):
    """(h, dgate, dup) and fp32's share of their errors.  sigmoid goes through 2^(-g log2 e), whose argument is off by
    |g| 2^-23 and whose value by 2^-22 and one more rounding or two: (|g| + 8) 2^-22 relative; in the derivative q + g q (1 - q) that
    many of each term.  Phi is off by 0.75e-7 + 8 units, g phi by (g^2 + 8) 2^-22 relative."""
    g, u, d = gate.double(), up.double(), dh.double()
    if act == "silu":
        q = torch.sigmoid(g)
        a, rel = g * q, (g.abs() + 8) * 4 * U
        da, a_lim, da_lim = q + a * (1 - q), rel * a.abs(), rel * (q + 2 * a.abs())
    else:
        q = torch.special.ndtr(g)
        phi = torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        a, da = g * q, q + g * phi
        p_lim = 0.75e-7 + 8 * U
        a_lim, da_lim = p_lim * g.abs() + 2 * U * a.abs(), p_lim + (g.square() + 8) * 4 * U * (g * phi).abs() + 2 * U * da.abs()
    k = 4 * U
    h, dg, du = a * u, d * u * da, d * a
    return (h, a_lim * u.abs() + k * h.abs()), (dg, (d * u).abs() * da_lim + k * dg.abs()), (du, d.abs() * a_lim + k * du.abs())


def _near(got, ref, lim, dtype):
    return bool(((got.double() - ref).abs() <= lim + HALF[dtype] * (ref.abs() + lim) + LEAST[dtype]).all())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("M,K", [(1, 1), (31, 8), (33, 129), (77, 1536), (130, 260), (64, 4098)])
def test_values_and_gradients(M, K, eight, dtype, act):
    from concord_b200 import gated_unit
    g = torch.Generator(device=DEV).manual_seed(M + K)
    randn = lambda: torch.randn(M, K, generator=g, device=DEV)  # noqa: E731
    gate, up, dh = (randn() * 2).to(dtype).requires_grad_(), randn().to(dtype).requires_grad_(), (randn() * 0.1).to(dtype)
    h = gated_unit(gate, up, act, save8=eight)
    dg, du = torch.autograd.grad(h, (gate, up), dh)
    (ref, lim), _, _ = _plain(gate.detach(), up.detach(), dh, act)
    assert h.dtype == dtype and h.is_contiguous() and _near(h, ref, lim, dtype)
    kept = [plain8(t.detach()) if eight else t.detach() for t in (gate, up)]
    _, (rg, lg), (ru, lu) = _plain(*kept, dh, act)
    assert _near(dg, rg, lg, dtype) and _near(du, ru, lu, dtype)
    with torch.no_grad():
        assert torch.equal(gated_unit(gate, up, act, save8=eight), h)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_by_differences(act):
    """Central differences of the definition in 64 bits, of step 2^-10, are off by step^2 / 6 times the third derivative, which
    is below 2 for both functions, and by 2^-42 / step from their own rounding."""
    from concord_b200 import gated_unit
    g = torch.linspace(-9, 9, 1000, device=DEV).requires_grad_()
    one = torch.ones(1000, device=DEV)
    (dg,) = torch.autograd.grad(gated_unit(g, one, act), g, one)
    f = (lambda t: t * torch.sigmoid(t)) if act == "silu" else (lambda t: t * torch.special.ndtr(t))
    x, step = g.detach().double(), 2.0 ** -10
    ref = (f(x + step) - f(x - step)) / (2 * step)
    lim = _plain(g.detach(), one, one, act)[1][1] + 2 * step ** 2 / 6 + 2.0 ** -32
    assert bool(((dg.double() - ref).abs() <= lim + U * ref.abs()).all())


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_far_values(act):
    """Large magnitudes of both signs: act is g or 0, its derivative 1 or 0, nothing overflows on the way."""
    from concord_b200 import gated_unit
    g = torch.tensor([1e4, 3e38, -1e4, -3e38, 200.0, -200.0, 0.0, -0.0], device=DEV, requires_grad=True)
    u = torch.full((8,), 0.5, device=DEV)
    h = gated_unit(g, u, act)
    (dg,) = torch.autograd.grad(h, g, torch.ones(8, device=DEV))
    assert h.tolist() == [5e3, 1.5e38, 0.0, 0.0, 100.0, 0.0, 0.0, 0.0] or \
        torch.allclose(h, torch.tensor([5e3, 1.5e38, 0, 0, 100.0, 0, 0, 0], device=DEV), rtol=1e-6, atol=0)
    assert torch.allclose(dg, torch.tensor([0.5, 0.5, 0, 0, 0.5, 0, 0.25, 0.25], device=DEV), rtol=1e-6, atol=0)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("K,gate_first", [(128, True), (5, False), (132, False), (2052, True)])
def test_halves_of_one_projection(K, gate_first, eight):
    """Views with strides of their own, odd offsets; as their copies give it, gradients into the projection's too."""
    from concord_b200 import gated_unit
    both = torch.randn(3, 30, 2 * K, device=DEV).bfloat16().requires_grad_()
    dh = torch.randn(3, 30, K, device=DEV).bfloat16()
    halves = both.chunk(2, -1) if gate_first else both.chunk(2, -1)[::-1]
    h = gated_unit(*halves, act="gelu", save8=eight)
    (got,) = torch.autograd.grad(h, both, dh)
    a, b = (t.detach().contiguous().requires_grad_() for t in halves)
    ref = gated_unit(a, b, act="gelu", save8=eight)
    grads = torch.autograd.grad(ref, (a, b), dh)
    assert torch.equal(h, ref) and torch.equal(got, torch.cat(grads if gate_first else grads[::-1], -1))


def test_strided_gradient_and_broadcast():
    from concord_b200 import gated_unit
    gate, up = (torch.randn(40, 64, device=DEV).requires_grad_() for _ in range(2))
    wide = torch.randn(40, 100, device=DEV)
    for eight in (False, True):
        a = torch.autograd.grad(gated_unit(gate, up, save8=eight), (gate, up), wide[:, 3:67])
        b = torch.autograd.grad(gated_unit(gate, up, save8=eight), (gate, up), wide[:, 3:67].contiguous())
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        c = torch.autograd.grad(gated_unit(gate, up, save8=eight).sum(), (gate, up))
        d = torch.autograd.grad(gated_unit(gate, up, save8=eight), (gate, up), torch.ones(40, 64, device=DEV))
        assert all(torch.equal(x, y) for x, y in zip(c, d))
    row = torch.randn(1, 64, device=DEV, requires_grad=True)
    (dr,) = torch.autograd.grad(gated_unit(gate, row.expand(40, 64)).sum(), row)
    (full,) = torch.autograd.grad(gated_unit(gate, up).sum(), up)
    assert dr.shape == row.shape and torch.allclose(dr[0], full.sum(0), rtol=1e-5)
    same = torch.randn(10, 64, device=DEV, requires_grad=True)                      # one tensor in both places
    (ds,) = torch.autograd.grad(gated_unit(same, same, save8=True).sum(), same)
    a, b = (same.detach().clone().requires_grad_() for _ in range(2))
    ga, gb = torch.autograd.grad(gated_unit(a, b, save8=True).sum(), (a, b))
    assert torch.equal(ds, ga + gb)


@pytest.mark.parametrize("eight", [False, True])
def test_output_in_8_bits(eight):
    """The Saved8 beside h is that of h itself, with and without a gradient to follow."""
    from concord_b200 import gated_unit, save8
    for dtype, K in ((torch.bfloat16, 96), (torch.float32, 33), (torch.float16, 50)):
        gate, up = (torch.randn(2, 45, K, device=DEV).to(dtype).requires_grad_() for _ in range(2))
        h, h8 = gated_unit(gate, up, save8=eight, out8=True)
        assert torch.equal(h8.dense(), save8(h.detach()).dense()) and h8.shape == h.shape
        a = torch.autograd.grad(h.sum(), (gate, up))
        b = torch.autograd.grad(gated_unit(gate, up, save8=eight).sum(), (gate, up))
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        with torch.no_grad():
            h, h8 = gated_unit(gate, up, out8=True)
            assert torch.equal(h8.dense(), save8(h).dense())


def test_nothing_is_kept_but_8_bits():
    from concord_b200 import gated_unit
    gate, up = (torch.randn(4096, 512, device=DEV).bfloat16().requires_grad_() for _ in range(2))
    torch.cuda.synchronize()
    before = _asked()
    h = gated_unit(gate * 1.0, up * 1.0, save8=True)
    assert _asked() - before <= h.numel() * 2 + 2 * 4096 * 512 * 66 // 64 + 4096
    h.sum().backward()


def test_empty_nan_and_refusals():
    from concord_b200 import gated_unit
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    for eight in (False, True):
        h = gated_unit(x, x, save8=eight)
        (g,) = torch.autograd.grad(h.sum(), x)
        assert h.shape == (0, 64) and g.shape == (0, 64)
    a = torch.ones(40, 8, device=DEV)
    a[35, 2] = float("nan")
    a.requires_grad_()
    h = gated_unit(a, torch.ones(40, 8, device=DEV), save8=True)
    (g,) = torch.autograd.grad(h.sum(), a)
    assert bool(h[35, 2].isnan()) and int(h.isnan().sum()) == 1
    assert bool(g[32:, 2].isnan().all()) and int(g.isnan().sum()) == 8               # its block of 32 tokens, of which 8 are there
    z = torch.zeros(4, 8, device=DEV)
    for error, match, call in (
            (TypeError, "gate must be one of", lambda: gated_unit(z.double(), z.double())),
            (TypeError, "up must have gate's type", lambda: gated_unit(z, z.half())),
            (ValueError, "one shape", lambda: gated_unit(z, z[:3])),
            (ValueError, "act must be one of", lambda: gated_unit(z, z, act="relu")),
            (RuntimeError, "CUDA tensors only", lambda: gated_unit(z, z.cpu()))):
        with pytest.raises(error, match=match):
            call()
