"""layer_norm and LayerNorm against a 64-bit implementation.

Tolerances: an output is rounded once to its type (half a unit in the last
place: 2^-8 of the value is a whole one for bf16, 2^-10 for fp16, 2^-23 for
fp32).  Before that, fp32 arithmetic: the mean and the deviations carry errors
of a few units of the row's largest |x|, scaled by rstd |w|; sums of n terms by
trees carry a few units of the sum of their magnitudes.  16 units are granted.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = 2.0 ** -23
ULP = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}


def reference(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    D = x.shape[-1]
    w = torch.ones(D, device=x.device).double() if w is None else w.double()
    b = torch.zeros(D, device=x.device).double() if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * rs
    g = dy * w
    dx = rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, D)  # noqa: E731
    big = x.abs().amax(-1, keepdim=True) * rs                # error scale of xh
    tol = dict(y=16 * F32 * (big * w.abs() + b.abs() + (xh * w).abs()),
               dx=16 * F32 * rs * (g.abs().amax(-1, keepdim=True) * (1 + big) ** 2),
               dw=16 * F32 * flat(dy.abs() * (xh.abs() + big)).sum(0), db=16 * F32 * flat(dy.abs()).sum(0))
    return dict(y=xh * w + b, dx=dx, dw=(flat(dy * xh)).sum(0), db=flat(dy).sum(0)), tol


def close(name, got, ref, tol):
    err = (got.double() - ref).abs()
    lim = ULP[got.dtype] * ref.abs() + tol + TINY[got.dtype]
    assert bool((err <= lim).all()), (name, float((err / lim).max()))


def inputs(shape, x_type, y_type, seed=0, offset=0.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    D = shape[-1]
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return (r(*shape) * 2 + offset).to(x_type), 1 + 0.3 * r(D), 0.2 * r(D), r(*shape).to(y_type)


def check(x, w, b, dy, eps=1e-5):
    from concord_b200 import layer_norm
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps, out_dtype=dy.dtype)
    assert y.dtype == dy.dtype and y.shape == x.shape
    wanted = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None],
                     torch.autograd.grad(y, wanted, dy)))
    ref, tol = reference(x, w, b, dy, eps)
    close("y", y.detach(), ref["y"], tol["y"])
    for name, got in grads.items():
        close(name, got, ref[name], tol[name])


# every width of a row's threads, both access forms, rows fewer and more than a wave of blocks
@pytest.mark.parametrize("N,D", [(1, 1), (3, 7), (1, 384), (77, 384), (4099, 384), (5, 512), (130, 513), (33, 1000),
                                 (700, 1280), (9, 2048), (6, 4096), (5, 5003), (3, 8192), (7, 8200), (2, 16384),
                                 (401, 16381)])
def test_shapes(N, D):
    check(*inputs((N, D), torch.bfloat16, torch.bfloat16, seed=N + D))


@pytest.mark.parametrize("x_type", list(ULP))
@pytest.mark.parametrize("y_type", list(ULP))
@pytest.mark.parametrize("D", [200, 37])
def test_types(x_type, y_type, D):
    check(*inputs((19, D), x_type, y_type, seed=D))


@pytest.mark.parametrize("has_w,has_b", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(has_w, has_b):
    x, w, b, dy = inputs((50, 96), torch.float32, torch.float32)
    check(x, w if has_w else None, b if has_b else None, dy)


def test_strides_and_leading_dims():
    x, w, b, dy = inputs((4, 6, 256), torch.bfloat16, torch.bfloat16)
    check(x[:, ::2, :128], w[:128], b[:128], dy[:, ::2, :128])        # row stride 512
    check(x[..., ::2], w[::2], b[::2], dy[..., ::2])                   # columns apart
    check(x.transpose(0, 1), w, b, dy.transpose(0, 1))
    check(x[:, :, 3:100], w[3:100], b[3:100], dy[:, :, 3:100])         # rows that start off 16 bytes
    check(x, w, b, dy[:1, :1].expand(4, 6, 256))                       # a broadcast upstream gradient


def test_constant_and_offset_rows():
    x, w, b, dy = inputs((8, 300), torch.float32, torch.float32)
    x[0] = 3.0                                                         # no spread: xh = 0
    x[1] = x[1] + 1e4                                                  # far off centre
    x[2] = 0.0
    check(x, w, b, dy)


def test_one_nan_row_stays_its_own():
    from concord_b200 import layer_norm
    x, w, b, _ = inputs((6, 520), torch.bfloat16, torch.bfloat16)
    clean = layer_norm(x, w, b)
    x2 = x.clone()
    x2[3, 7] = float("nan")
    y = layer_norm(x2, w, b)
    assert bool(y[3].isnan().all())
    keep = [0, 1, 2, 4, 5]
    assert torch.equal(y[keep], clean[keep])


def test_empty_rows():
    from concord_b200 import layer_norm
    w = torch.ones(64, device=DEV, requires_grad=True)
    b = torch.zeros(64, device=DEV, requires_grad=True)
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == (0, 64)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == (0, 64) and bool((dw == 0).all()) and bool((db == 0).all())


def test_same_bits_every_time_and_on_another_stream():
    from concord_b200 import layer_norm
    x, w, b, dy = inputs((5000, 640), torch.bfloat16, torch.bfloat16)

    def once():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = layer_norm(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
    first = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, second))


def test_gradient_against_differences():
    """Central differences of sum(y dy) along random directions, fp32: h^2 times the third derivative (under 1 for
    rows of spread 2) plus the forward's rounding over h."""
    from concord_b200 import layer_norm
    x, w, b, dy = inputs((5, 48), torch.float32, torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    h = 2.0 ** -6
    for i in range(3):
        u = torch.randn_like(leaves[i])
        u /= u.norm()
        at = lambda s: (layer_norm(*[t + s * u if k == i else t for k, t in enumerate((x, w, b))]).double()  # noqa: E731
                        * dy.double()).sum()
        diff = float((at(h) - at(-h)) / (2 * h))
        noise = 8 * F32 * float(dy.abs().sum()) * 4 / h
        assert abs(diff - float((grads[i] * u).sum())) <= float(dy.norm()) * h * h + noise


def test_module_matches_function_and_loads_state():
    from concord_b200 import LayerNorm, layer_norm
    ref = torch.nn.LayerNorm(384, device=DEV)
    torch.nn.init.normal_(ref.weight)
    m = LayerNorm(384, out_dtype=torch.bfloat16, device=DEV)
    m.load_state_dict(ref.state_dict())
    x = torch.randn(3, 5, 384, device=DEV)
    assert torch.equal(m(x), layer_norm(x, ref.weight, ref.bias, out_dtype=torch.bfloat16))
    assert m(x).dtype == torch.bfloat16


def test_weight_of_another_type_gets_its_gradient():
    from concord_b200 import layer_norm
    x, w, b, dy = inputs((9, 64), torch.bfloat16, torch.bfloat16)
    wb = w.bfloat16().requires_grad_()
    y = layer_norm(x, wb, b)
    (dw,) = torch.autograd.grad(y, wb, dy)
    assert dw.dtype == torch.bfloat16
    ref, tol = reference(x, wb.detach(), b, dy, 1e-5)
    close("dw", dw, ref["dw"], tol["dw"])


def test_captured_in_a_graph():
    from concord_b200 import layer_norm
    x, w, b, dy = inputs((64, 384), torch.float32, torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    run = lambda: torch.autograd.grad(layer_norm(*leaves, out_dtype=torch.bfloat16), leaves, dy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(eager, out))


def test_refusals():
    from concord_b200 import LayerNorm, layer_norm
    x = torch.zeros(2, 8, device=DEV)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer_norm(x.cpu())
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer_norm(x, torch.ones(8))
    with pytest.raises(TypeError, match="x must be"):
        layer_norm(x.double())
    with pytest.raises(TypeError, match="out_dtype"):
        layer_norm(x, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="weight must have shape"):
        layer_norm(x, torch.ones(7, device=DEV))
    with pytest.raises(ValueError, match="last dimension"):
        layer_norm(torch.zeros(3, 0, device=DEV))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="16384 columns"):
        layer_norm(torch.zeros(1, 16385, device=DEV))
    with pytest.raises(ValueError, match="last dimension of 8"):
        LayerNorm(8, device=DEV)(torch.zeros(2, 9, device=DEV))
