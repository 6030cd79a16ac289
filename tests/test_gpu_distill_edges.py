"""distill_loss where its terms are small beside the logits, and with no rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _grid(N, V, seed):
    """Logits that are multiples of 2^-6 in [-8, 8]: exact in fp32 after a shift of up to 2^14."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = torch.randint(-512, 513, (N, V), generator=g, device=DEV).float() / 64
    ids = torch.rand(N, V, generator=g, device=DEV).topk(5, 1).indices
    t = torch.randn(N, 5, generator=g, device=DEV) * 2
    y = torch.randint(0, V, (N,), generator=g, device=DEV)
    return z, ids, t, y


@pytest.mark.parametrize("V", [65, 513, 5003])
@pytest.mark.parametrize("temp", [1.0, 1.5, 2.0, 8.0])
@pytest.mark.parametrize("shift", [1024.0, -16384.0])
def test_a_shift_of_the_logits_changes_nothing(V, temp, shift):
    """Loss and gradient are functions of the differences of a row's logits, which a shift leaves as they are: the
    same bits."""
    from concord_b200 import distill_loss
    z, ids, t, y = _grid(16, V, V)
    for labels, alpha in ((y, 0.5), (y, 0.0), (None, 1.0)):
        got = []
        for leaf in (z.clone().requires_grad_(), (z + shift).requires_grad_()):
            rows = distill_loss(leaf, ids, t, labels, temp, alpha, reduction="none")
            got.append((rows.detach(), *torch.autograd.grad(rows.sum(), leaf)))
        assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("offset", [0.0, 1024.0, 16384.0])
def test_cross_entropy_of_confident_rows(offset):
    """A cross entropy of about 1e-3 is log(1 + small): the sum's roundings beside 1 (at most 32 of 2^-24: 8 pairs of
    a lane, the joins, the exponentials' own) are its whole error, wherever the logits stand."""
    from concord_b200 import distill_loss
    z, ids, t, y = _grid(64, 513, 3)
    z = z / 8
    z = (z * 64).round() / 64
    z[torch.arange(64, device=DEV), y] = 13.0
    z = z + offset
    rows = distill_loss(z, ids, t, y, 1.0, 0.0, reduction="none")
    ref = -torch.log_softmax(z.double(), 1).gather(1, y[:, None])[:, 0]
    assert 1e-4 < float(ref.min()) and float(ref.max()) < 1e-2
    assert float((rows.double() - ref).abs().max()) <= 32 * 2.0 ** -24


def test_no_rows():
    from concord_b200 import distill_loss
    z, ids, t, y = (x[:0] for x in _grid(2, 70, 0))
    z.requires_grad_()
    rows = distill_loss(z, ids, t, y, 2.0, 0.5, reduction="none")
    assert rows.shape == (0,)
    (dz,) = torch.autograd.grad(rows, z, torch.zeros(0, device=DEV))
    assert dz.shape == (0, 70)
