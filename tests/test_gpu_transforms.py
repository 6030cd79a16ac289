"""The training operators under torch's transforms: refused where the result would lack what their kernels do."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _norm():
    import concord_b200
    return concord_b200.layer_norm, [torch.randn(6, 64, device=DEV), torch.ones(64, device=DEV),
                                     torch.zeros(64, device=DEV)], (0, 1, 2)


def _attention():
    import concord_b200
    cu = torch.tensor([0, 4, 9], dtype=torch.int32, device=DEV)
    return lambda q, k, v: concord_b200.packed_attention(q, k, v, cu), [
        torch.randn(9, 2, 64, device=DEV).bfloat16() for _ in range(3)], (0, 1, 2)


def _distill():
    import concord_b200
    ids = torch.randint(0, 50, (6, 3), device=DEV)
    return lambda z, t: concord_b200.distill_loss(z, ids, t), [torch.randn(6, 50, device=DEV),
                                                               torch.randn(6, 3, device=DEV)], (0, 1)


def _distill_both():
    import concord_b200
    ids = torch.randint(0, 50, (6, 3), device=DEV)
    return lambda z, t: concord_b200.distill_loss_and_grad(z, ids, t)[1], [torch.randn(6, 50, device=DEV),
                                                                           torch.randn(6, 3, device=DEV)], (0, 1)


OPERATORS = pytest.mark.parametrize("make", [_norm, _attention, _distill, _distill_both])


@OPERATORS
def test_forward_mode_is_refused(make):
    f, args, which = make()
    for i in which:
        with fwd.dual_level():
            dual = list(args)
            dual[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*dual)
    with fwd.dual_level():
        f(*args)                          # nothing to differentiate: as ever


@OPERATORS
def test_tracing_is_refused(make):
    from torch.fx.experimental.proxy_tensor import make_fx
    f, args, _ = make()
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, tuple(args), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda *a: f(*a))(*args)
    f(*args)
