"""embedding and its gradient against plain forms in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _ids(kind, T, V, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if kind == "uniform":
        return torch.randint(-2, V + 2, (T,), generator=g, device=DEV)          # some outside the table
    if kind == "zipf":
        return ((V + 1.0) ** torch.rand(T, generator=g, device=DEV, dtype=torch.float64) - 1).long().clamp_(0, V - 1)
    if kind == "one":
        return torch.full((T,), V - 1, device=DEV)
    if kind == "none":
        return torch.full((T,), -1, device=DEV)
    return V - 1 - torch.arange(T, device=DEV) % V                              # backwards


def _ref_rows(ids, V):
    return torch.where((ids < 0) | (ids >= V), V, ids)


@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (5, 3, 7), (33, 65, 384), (300, 7, 130), (77, 1000, 64), (2049, 513, 1032)])
@pytest.mark.parametrize("wt,yt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                   (torch.float16, torch.float32), (torch.float32, torch.float32)])
def test_lookup(T, V, D, wt, yt):
    """One product in fp32 and one rounding to the result's type."""
    from concord_b200 import embedding
    ids = _ids("uniform", T, V, T)
    w = torch.randn(V, D, device=DEV).to(wt)
    y = embedding(ids, w, scale=45.25, out_dtype=yt)
    ref = torch.cat([w.double() * 45.25, torch.zeros(1, D, device=DEV, dtype=torch.float64)])[_ref_rows(ids, V)]
    assert y.shape == (T, D) and y.dtype == yt
    assert bool(((y.double() - ref).abs() <= (HALF[yt] + 2 * U) * ref.abs()).all())
    assert torch.equal(embedding(ids.int(), w, scale=45.25, out_dtype=yt), y)
    assert torch.equal(embedding(ids.view(1, T), w, scale=45.25, out_dtype=yt), y.view(1, T, D))


@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "none", "backwards"])
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (31, 5, 16), (32, 65, 384), (33, 511, 7), (64, 512, 100), (257, 513, 64),
                                   (4097, 32000, 24), (8193, 65, 96), (65536, 70000, 8), (65537, 300, 16),
                                   (70001, 262144, 8), (100000, 40, 5)])
def test_gradient_is_every_rows_sum(kind, T, V, D):
    """Whole numbers, whose sums are exact in any order: equal, each row of the table written, for sizes around the
    chunks of 32, the blocks and the 65,536 tokens of the cluster's sort, digits of one to three passes."""
    from concord_b200 import embedding
    ids = _ids(kind, T, V, T + V)
    g = torch.Generator(device=DEV).manual_seed(T)
    dy = torch.randint(-8, 9, (T, D), generator=g, device=DEV).float()
    w = torch.randn(V, D, device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(embedding(ids, w, scale=2.0), w, dy)
    ref = torch.zeros(V + 1, D, device=DEV, dtype=torch.float64).index_add_(0, _ref_rows(ids, V), dy.double())[:V] * 2
    assert dw.dtype == torch.float32 and torch.equal(dw.double(), ref)
    (again,) = torch.autograd.grad(embedding(ids.int(), w, scale=2.0), w, dy)
    assert torch.equal(again, dw)


@pytest.mark.parametrize("wt,yt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16),
                                   (torch.float16, torch.float32)])
@pytest.mark.parametrize("T,V,D", [(3000, 50, 72), (500, 2000, 65)])
def test_gradient_rounding(T, V, D, wt, yt):
    """n fp32 additions are off by at most n 2^-24 of the sum of magnitudes, scale's product by one more, then one
    rounding to the table's type (values below fp16's normal range by half of its least step)."""
    from concord_b200 import embedding
    ids = _ids("zipf", T, V, 1)
    dy = (torch.randn(T, D, device=DEV) * 0.1).to(yt)
    w = torch.randn(V, D, device=DEV).to(wt).requires_grad_()
    (dw,) = torch.autograd.grad(embedding(ids, w, scale=3.0, out_dtype=yt), w, dy)
    ref = torch.zeros(V, D, device=DEV, dtype=torch.float64).index_add_(0, ids, dy.double() * 3)
    mag = torch.zeros(V, D, device=DEV, dtype=torch.float64).index_add_(0, ids, dy.double().abs() * 3)
    n = torch.bincount(ids, minlength=V)[:, None]
    lim = (n + 1) * U * mag
    lim = lim + HALF[wt] * (ref.abs() + lim) + (2.0 ** -25 if wt == torch.float16 else 0.0)
    assert dw.dtype == wt and bool(((dw.double() - ref).abs() <= lim).all())


def test_order_repeats_bit_for_bit():
    from concord_b200 import embedding
    ids = _ids("zipf", 20000, 900, 3)
    dy = torch.randn(20000, 64, device=DEV)
    w = torch.randn(900, 64, device=DEV, requires_grad=True)
    grads = [torch.autograd.grad(embedding(ids, w), w, dy)[0] for _ in range(3)]
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


def test_strides_and_padding():
    """A table that is a part of another, upstream gradients that are a part or every row the same, padding_idx."""
    from concord_b200 import Embedding, embedding
    big = torch.randn(40, 100, device=DEV)
    w = big[:, 3:67]
    ids = torch.tensor([[0, 5, 39], [5, 5, 7]], device=DEV)
    assert torch.equal(embedding(ids, w), w[ids])
    assert torch.equal(embedding(ids, big.t()), big.t()[ids % 40])
    leaf = torch.randn(40, 64, device=DEV, requires_grad=True)
    y = embedding(ids, leaf, padding_idx=-33)                              # row 7: looked up, no gradient
    assert torch.equal(y[1, 2], leaf[7])
    (g,) = torch.autograd.grad(y.sum(), leaf)                              # (an expanded upstream gradient)
    want = torch.zeros(40, 64, device=DEV)
    want[0], want[5], want[39] = 1, 3, 1
    assert torch.equal(g, want)
    wide = torch.randn(2, 3, 80, device=DEV)
    (g,) = torch.autograd.grad(embedding(ids, leaf), leaf, wide[..., 8:72])
    assert torch.equal(g, torch.zeros(40, 64, device=DEV).index_add_(0, ids.flatten(), wide[..., 8:72].reshape(6, 64)))
    m = Embedding(40, 64, padding_idx=0, scale=8.0, out_dtype=torch.bfloat16, device=DEV)
    assert m(ids).dtype == torch.bfloat16 and bool((m(ids)[0, 0] == 0).all())
    m(ids).float().sum().backward()
    assert bool((m.weight.grad[0] == 0).all()) and bool((m.weight.grad[5] == 24).all())
    m.load_state_dict(torch.nn.Embedding(40, 64).state_dict())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset,stride", [(0, 72), (1, 72), (2, 72), (4, 72), (8, 72), (0, 68), (0, 66), (4, 68), (8, 70)])
def test_addresses(dtype, offset, stride):
    """Tables and upstream gradients whose rows begin on 2 to 32 bytes."""
    from concord_b200 import embedding
    g = torch.Generator(device=DEV).manual_seed(offset + stride)
    ids = torch.randint(-1, 30, (200,), generator=g, device=DEV)
    part = lambda rows: torch.randint(-8, 9, (rows * stride + offset,), generator=g, device=DEV).to(dtype)[offset:].view(rows, stride)[:, :56]  # noqa: E731
    w, dy = part(30), part(200)
    assert torch.equal(embedding(ids, w), torch.where(ids[:, None] < 0, 0, w[ids]))
    leaf = w.detach().clone().requires_grad_()
    (got,) = torch.autograd.grad(embedding(ids, leaf), leaf, dy)
    want = torch.zeros(31, 56, device=DEV).index_add_(0, ids % 31, dy.float())[:30]       # (whole numbers: exact)
    assert torch.equal(got, want.to(dtype))


def test_empty_and_nan():
    from concord_b200 import embedding
    w = torch.randn(10, 16, device=DEV, requires_grad=True)
    y = embedding(torch.zeros(0, 3, dtype=torch.long, device=DEV), w)
    assert y.shape == (0, 3, 16)
    (g,) = torch.autograd.grad(y.sum(), w)
    assert bool((g == 0).all())
    ids = torch.tensor([1, -1, 2, 10], device=DEV)
    dy = torch.ones(4, 16, device=DEV)
    dy[1], dy[3] = float("nan"), float("inf")                              # of tokens that count for no row
    (g,) = torch.autograd.grad(embedding(ids, w), w, dy)
    assert bool((g[1:3] == 1).all()) and float(g.sum()) == 32
    dy = torch.ones(4, 16, device=DEV)
    dy[0] = float("nan")
    (g,) = torch.autograd.grad(embedding(ids, w), w, dy)
    assert bool(g[1].isnan().all()) and bool((g[2] == 1).all()) and bool((g[3:] == 0).all())


def test_refusals():
    from concord_b200 import embedding
    w, ids = torch.zeros(5, 8, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    with pytest.raises(TypeError, match="ids must be one of"):
        embedding(ids.float(), w)
    with pytest.raises(TypeError, match="weight must be one of"):
        embedding(ids, w.double())
    with pytest.raises(TypeError, match="out_dtype"):
        embedding(ids, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match=r"weight must be \[V, D\]"):
        embedding(ids, w[0])
    with pytest.raises(ValueError, match="padding_idx"):
        embedding(ids, w, padding_idx=5)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        embedding(ids.cpu(), w)
