"""The decoder's operators as autograd nodes: kept graphs, second derivatives, inputs changed in place, what is wanted
alone, transforms, streams, captured graphs."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _embedding():
    from concord_b200 import embedding
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.randn(70, 64, generator=g, device=DEV, requires_grad=True)
    ids = torch.randint(-1, 70, (300,), generator=g, device=DEV)
    return [w], lambda w: embedding(ids, w, scale=2.0)


def _qk():
    from concord_b200 import qk_norm_rope, rope_tables
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k = (torch.randn(90, h, 64, generator=g, device=DEV).bfloat16().requires_grad_() for h in (4, 2))
    a, b = (torch.rand(64, generator=g, device=DEV).add_(0.5).requires_grad_() for _ in range(2))
    cos, sin = rope_tables(90, 64)

    def call(q, k, a, b):
        y, z = qk_norm_rope(q, k, cos, sin, None, a, b)
        return torch.cat((y, z), 1)
    return [q, k, a, b], call


def _gated(eight):
    from concord_b200 import gated_unit
    g = torch.Generator(device=DEV).manual_seed(2)
    gate, up = (torch.randn(50, 96, generator=g, device=DEV).requires_grad_() for _ in range(2))
    return [gate, up], lambda gate, up: gated_unit(gate, up, save8=eight)


OPERATORS = pytest.mark.parametrize("make", [_embedding, _qk, lambda: _gated(False), lambda: _gated(True)],
                                    ids=["embedding", "qk", "gated", "gated8"])


@OPERATORS
def test_a_kept_graph_runs_again(make):
    leaves, call = make()
    out = call(*leaves)
    up = torch.ones_like(out)
    first = torch.autograd.grad(out, leaves, up, retain_graph=True)
    second = torch.autograd.grad(out, leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, up)


@OPERATORS
def test_no_second_derivative(make):
    leaves, call = make()
    grads = torch.autograd.grad((call(*leaves).float() ** 2).sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grads[0].float().sum().backward()


@pytest.mark.parametrize("make", [_qk, lambda: _gated(False)], ids=["qk", "gated"])
def test_changed_inputs_are_noticed(make):
    leaves, call = make()
    out = call(*leaves)
    with torch.no_grad():
        leaves[0].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, torch.ones_like(out))


@pytest.mark.parametrize("make", [_embedding, lambda: _gated(True)], ids=["embedding", "gated8"])
def test_inputs_that_are_not_kept_may_change(make):
    """The table's values enter no gradient; of gate and up only their 8-bit form is kept."""
    leaves, call = make()
    want = torch.autograd.grad(call(*leaves), leaves, torch.ones_like(call(*leaves)))
    out = call(*leaves)
    with torch.no_grad():
        leaves[0].add_(1.0)
    got = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@OPERATORS
def test_only_what_is_wanted(make):
    leaves, call = make()
    out = call(*leaves)
    want = torch.autograd.grad(out, leaves, torch.ones_like(out))
    for i, leaf in enumerate(leaves):
        (got,) = torch.autograd.grad(call(*leaves), (leaf,), torch.ones_like(out))
        assert torch.equal(got, want[i])
        for other in leaves:
            other.requires_grad_(other is leaf)
        (alone,) = torch.autograd.grad(call(*leaves), (leaf,), torch.ones_like(out))
        assert torch.equal(alone, want[i])
        for other in leaves:
            other.requires_grad_(True)
    with torch.no_grad():
        assert not call(*leaves).requires_grad and torch.equal(call(*leaves), out)


@OPERATORS
def test_transforms_are_refused(make):
    from torch.fx.experimental.proxy_tensor import make_fx
    leaves, call = make()
    args = [t.detach() for t in leaves]
    for i in range(len(args)):
        with fwd.dual_level():
            dual = list(args)
            dual[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(*dual)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, tuple(args), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda *a: call(*a))(*args)
    call(*args)


def test_saving_and_the_weight_gradient_are_refused_in_traces():
    from torch.fx.experimental.proxy_tensor import make_fx

    from concord_b200 import grad_weight8, save8
    x = torch.randn(40, 64, device=DEV).bfloat16()
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: save8(t).dense())(x)
    s = save8(x)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: grad_weight8(t, s))(x)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            save8(fwd.make_dual(x, torch.ones_like(x)))


def _everything(ids, w, qkv, a, b, cos, sin, pos, gate, up, dy):
    """All operators on static tensors: outputs, gradients, dW from 8 bits."""
    from concord_b200 import embedding, gated_unit, grad_weight8, qk_norm_rope, save8
    y = embedding(ids, w, scale=3.0, out_dtype=torch.bfloat16)
    q, k = qk_norm_rope(qkv[:, :4], qkv[:, 4:6], cos, sin, pos, a, b)
    h, h8 = gated_unit(gate, up, save8=True, out8=True)
    grads = torch.autograd.grad((y, q, k, h), (w, qkv, a, b, gate, up),
                                (y.detach() * 0.5, q.detach() * 0.5, k.detach() * 0.5, h.detach() * 0.5))
    return [t.detach() for t in (y, q, k, h)] + list(grads) + [grad_weight8(dy, h8), grad_weight8(dy, save8(gate.detach())),
                                                               h8.dense()]


def _inputs(seed):
    from concord_b200 import rope_tables
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    T = 130
    return [torch.randint(-1, 50, (T,), generator=g, device=DEV), randn(50, 64), randn(T, 6, 64).bfloat16(), randn(64), randn(64),
            *rope_tables(T, 64), torch.randperm(T, generator=g, device=DEV).int(), randn(T, 200).bfloat16(),
            randn(T, 200).bfloat16(), randn(T, 264).bfloat16()]


def _leaves(inputs):
    return [t.clone().requires_grad_() if i in (1, 2, 3, 4, 8, 9) else t.clone() for i, t in enumerate(inputs)]


def test_captured_graphs():
    """Two graphs of forward and backward, captured one after the other, replayed in turn on new inputs, with an eager
    call between: each gives what an eager call gives."""
    eager = [[t.clone() for t in _everything(*_leaves(_inputs(s)))] for s in (1, 2, 3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            static = _leaves(_inputs(0))
            _everything(*static)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = _everything(*static)
            graphs.append((graph, static, out))
        for turn in range(3):
            for n, (graph, static, out) in enumerate(graphs):
                which = (turn + n) % 3
                with torch.no_grad():
                    for dst, src in zip(static, _inputs(which + 1)):
                        dst.copy_(src)
                graph.replay()
                _everything(*_leaves(_inputs(9)))
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(out, eager[which]))
    torch.cuda.current_stream().wait_stream(side)


def test_two_streams():
    """The same calls on two streams at once, each with its own tensors."""
    want = [[t.clone() for t in _everything(*_leaves(_inputs(s)))] for s in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = _everything(*_leaves(_inputs(i + 1)))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
