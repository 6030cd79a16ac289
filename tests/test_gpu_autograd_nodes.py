"""The training operators' autograd nodes: run again on a kept graph, refuse a
second derivative, notice inputs that were changed in place, hold only what
their inputs need."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _norm():
    from concord_b200 import layer_norm
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(40, 96, generator=g, device=DEV, requires_grad=True)
    w = torch.randn(96, generator=g, device=DEV, requires_grad=True)
    return (x, w), lambda: layer_norm(x, w)


def _attention():
    from concord_b200 import packed_attention
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(150, 2, 64, generator=g, device=DEV).bfloat16().requires_grad_() for _ in range(3))
    cu = torch.tensor([0, 100, 150], dtype=torch.int32, device=DEV)
    return (q, k, v), lambda: packed_attention(q, k, v, cu)


def _distill():
    from concord_b200 import distill_loss
    g = torch.Generator(device=DEV).manual_seed(2)
    z = torch.randn(20, 200, generator=g, device=DEV, requires_grad=True)
    ids = torch.randint(0, 200, (20, 4), generator=g, device=DEV)
    t = torch.randn(20, 4, generator=g, device=DEV)
    y = torch.randint(0, 200, (20,), generator=g, device=DEV)
    return (z,), lambda: distill_loss(z, ids, t, y, 2.0, 0.5)


OPERATORS = pytest.mark.parametrize("make", [_norm, _attention, _distill])


@OPERATORS
def test_a_kept_graph_runs_again(make):
    leaves, call = make()
    out = call()
    up = torch.ones_like(out)
    first = torch.autograd.grad(out, leaves, up, retain_graph=True)
    second = torch.autograd.grad(out, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, up)


@OPERATORS
def test_no_second_derivative(make):
    leaves, call = make()
    grads = torch.autograd.grad((call().float() ** 2).sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grads[0].float().sum().backward()


@OPERATORS
def test_changed_inputs_are_noticed(make):
    leaves, call = make()
    out = call()
    with torch.no_grad():
        leaves[0].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, torch.ones_like(out))


@OPERATORS
def test_only_what_is_wanted(make):
    leaves, call = make()
    out = call()
    want = torch.autograd.grad(out, leaves, torch.ones_like(out))
    for i, leaf in enumerate(leaves):
        (got,) = torch.autograd.grad(call(), (leaf,), torch.ones_like(out))
        assert torch.equal(got, want[i])
        for other in leaves:
            other.requires_grad_(other is leaf)
        (alone,) = torch.autograd.grad(call(), (leaf,), torch.ones_like(out))
        assert torch.equal(alone, want[i])
        for other in leaves:
            other.requires_grad_(True)
    with torch.no_grad():
        assert not call().requires_grad and torch.equal(call(), out)
