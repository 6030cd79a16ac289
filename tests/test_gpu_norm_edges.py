"""layer_norm's gradient on rows far off centre."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 256, 1024, 2048, 16384])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_constant_rows_have_no_deviation(D, dtype):
    """Rows of one value, whose sums are exact here (whole numbers of eighths, or of eights, below 2^24), have
    deviations of exactly 0: so has the weight's gradient, and dx = rstd (g - mean(g)) to the rounding of
    g's mean and of the result."""
    from concord_b200 import layer_norm
    g = torch.Generator(device=DEV).manual_seed(D)
    value = 1000.125 if dtype == torch.float32 and D <= 2048 else 1000.0
    x = torch.full((9, D), value, dtype=dtype, device=DEV).requires_grad_()
    w = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).requires_grad_()
    dy = torch.randn(9, D, generator=g, device=DEV)
    y = layer_norm(x, w, out_dtype=torch.float32)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert bool((y == 0).all()) and bool((dw == 0).all())
    gw = dy.double() * w.detach().double()
    ref = (gw - gw.mean(1, keepdim=True)) / 1e-5 ** 0.5
    unit = 2.0 ** -10 if dtype == torch.float16 else 0.0
    lim = unit * ref.abs() + 16 * 2.0 ** -23 * gw.abs().amax(1, keepdim=True) / 1e-5 ** 0.5
    assert bool(((dx.double() - ref).abs() <= lim).all())


def test_rows_off_centre():
    """x + 1000 for x on a grid of 2^-6 is exact, and so are the row's sums, its mean and deviations: the weight's
    gradient carries rounding relative to the deviations alone (16 units of the sum of magnitudes), none relative to
    the offset."""
    from concord_b200 import layer_norm
    g = torch.Generator(device=DEV).manual_seed(1)
    N, D = 40, 256
    x = torch.randint(-64, 65, (N, D // 2), generator=g, device=DEV).float() / 64
    x = torch.cat([x, -x], 1) + 1000.0                       # mean exactly 1000
    dy = torch.randn(N, D, generator=g, device=DEV)
    leaves = [x.requires_grad_(), torch.ones(D, device=DEV, requires_grad=True)]
    dx, dw = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    xc = x.detach().double() - 1000.0
    xh = xc / (xc.square().mean(1, keepdim=True) + 1e-5).sqrt()
    ref, mag = (dy * xh).sum(0), (dy.abs() * xh.abs()).sum(0)
    assert bool(((dw.double() - ref).abs() <= 16 * 2.0 ** -23 * mag).all())
