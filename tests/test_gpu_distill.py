"""distill_loss and distill_loss_and_grad against a 64-bit implementation.

Tolerances: a gradient is rounded once to the logits' type (at most 2^-8 of
the value for bf16, 2^-10 for fp16, 2^-23 for fp32).  Before that fp32:
exponents (z - max) / T in base 2 carry a few units of |max - min| / T, an
exponential 2 units, and where a power-of-two temperature's exponential is
squared up, T times that; 64 units of (1 + spread) per term are granted, terms
being a T softmax + a T p + (1 - a) softmax + (1 - a).  A loss is a sum of
terms of the size of lse and z / T: the same relative grant.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32 = 2.0 ** -23
ULP = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}


def reference(z, ids, t, labels, temp, alpha, ignore=-100):
    """Row losses, row gradients, which rows count, and the error scales of both (loss, gradient)."""
    z, t = z.double(), t.double() / temp
    N, V = z.shape
    ok = (ids >= 0) & (ids < V) & (t > -math.inf)
    some = ok.any(1)
    p = torch.zeros_like(t)
    p[some] = torch.softmax(t[some].masked_fill(~ok[some], -math.inf), 1)
    target = torch.zeros_like(z).scatter_add_(1, torch.where(ok, ids, 0).long(), p)
    logq = torch.log_softmax(z / temp, 1)
    part = torch.where(target > 0, target * (torch.log(target.clamp(min=1e-300)) - logq), torch.zeros_like(z))
    # entries of the same id count each with its own log p
    each = torch.where(p > 0, p * torch.log(p.clamp(min=1e-300)), torch.zeros_like(p)).sum(1)
    merged = torch.where(target > 0, target * torch.log(target.clamp(min=1e-300)), torch.zeros_like(z)).sum(1)
    loss = alpha * temp ** 2 * (part.sum(1) + each - merged)
    grad = alpha * temp * (logq.exp() * some[:, None] - target)
    mass = alpha * temp * (logq.exp() * some[:, None] + target)
    counts = some
    if labels is not None:
        counts = (labels != ignore) & (labels >= 0) & (labels < V)
        y = torch.where(counts, labels, 0).long()[:, None]
        logp = torch.log_softmax(z, 1)
        hot = torch.zeros_like(z).scatter_(1, y, 1.0)
        loss = loss - (1 - alpha) * logp.gather(1, y)[:, 0]
        grad = grad + (1 - alpha) * (logp.exp() - hot)
        mass = mass + (1 - alpha) * (logp.exp() + hot)
    zero = torch.zeros((), dtype=torch.float64, device=z.device)
    loss, grad, mass = (torch.where(counts.view(-1, *[1] * (x.dim() - 1)), x, zero) for x in (loss, grad, mass))
    fin = z.masked_fill(~z.isfinite(), 0)
    spread = 1 + (fin.amax(1) - fin.amin(1)) * max(1.0, 1 / temp) + fin.abs().amax(1) / min(temp, 1.0) + math.log(V)
    return loss, grad, counts, 64 * F32 * spread * (alpha * temp ** 2 + 1), 64 * F32 * spread[:, None] * mass * max(1, temp)


def close(got, ref, tol):
    err = (got.double() - ref).abs()
    lim = ULP[got.dtype] * ref.abs() + tol + TINY[got.dtype]
    bad = ~(err <= lim)
    assert not bool(bad.any()), (int(bad.sum()), float((err / lim)[bad].max()))


def inputs(N, V, K, dtype, labels=True, seed=0, ints=torch.int64):
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = (torch.randn(N, V, generator=g, device=DEV) * 3).to(dtype)
    ids = torch.rand(N, V, generator=g, device=DEV).topk(K, 1).indices.to(ints)
    t = torch.randn(N, K, generator=g, device=DEV) * 2
    y = torch.randint(0, V, (N,), generator=g, device=DEV).to(ints) if labels else None
    return z, ids, t, y


def check(z, ids, t, y, temp=1.0, alpha=1.0):
    from concord_b200 import distill_loss, distill_loss_and_grad
    N = z.shape[0]
    loss, grad, counts, ltol, gtol = reference(z, ids, t, y, temp, alpha)
    kw = dict(labels=y, temperature=temp, alpha=alpha)
    zl = z.detach().requires_grad_()
    rows = distill_loss(zl, ids, t, reduction="none", **kw)
    close(rows.detach(), loss, ltol)
    up = torch.linspace(0.5, 2.0, N, device=DEV)
    (g,) = torch.autograd.grad(rows, zl, up)
    close(g, grad * up.double()[:, None], gtol * 2)
    number = max(1, int(counts.sum()))
    for reduction, div in (("sum", 1), ("mean", number)):
        zl = z.detach().requires_grad_()
        one = distill_loss(zl, ids, t, reduction=reduction, **kw)
        close(one.detach(), loss.sum() / div, ltol.sum() / div)
        (g,) = torch.autograd.grad(one, zl)
        close(g, grad / div, gtol / div)
        both, fused = distill_loss_and_grad(z, ids, t, reduction=reduction, grad_scale=4.0, **kw)
        assert torch.equal(both, one.detach())
        close(fused, grad * (4.0 / div), gtol * (4.0 / div))


@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (3, 2, 2), (5, 65, 16), (700, 65, 3), (33, 1024, 64), (7, 1025, 8),
                                   (4, 4097, 5), (300, 5000, 32), (3, 32000, 100), (2, 70001, 512), (160, 8191, 1), (11, 900, 512), (9, 700, 257)])
def test_shapes(N, V, K):
    check(*inputs(N, V, K, torch.bfloat16, seed=N + V), temp=1.5, alpha=0.6)


@pytest.mark.parametrize("dtype", list(ULP))
@pytest.mark.parametrize("temp,alpha,labels", [(1.0, 1.0, False), (1.0, 0.25, True), (2.0, 0.5, True), (4.0, 0.9, True),
                                               (8.0, 0.5, True), (0.7, 0.5, True), (3.0, 1.0, False), (2.0, 0.0, True)])
def test_types_and_temperatures(dtype, temp, alpha, labels):
    check(*inputs(13, 1501, 20, dtype, labels=labels, seed=3), temp=temp, alpha=alpha)


def test_int32_ids_and_labels_give_the_same_bits():
    from concord_b200 import distill_loss_and_grad
    z, ids, t, y = inputs(20, 300, 9, torch.bfloat16)
    a = distill_loss_and_grad(z, ids, t, y, 2.0, 0.5)
    b = distill_loss_and_grad(z, ids.int(), t, y.int(), 2.0, 0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("V", [130, 6001])
def test_absent_entries_and_ignored_rows(V):
    z, ids, t, y = inputs(12, V, 8, torch.float32, seed=5)
    ids[0, 3:] = -1
    ids[1] = -1                       # no teacher entry: CE alone
    t[2, 1] = -math.inf
    t[3] = -math.inf
    ids[4, 2] = V                     # outside the vocabulary: absent
    y[5] = -100
    y[6] = V                          # outside: left out
    y[7] = -3
    z[5] = float("nan")               # a row that is left out may hold anything
    check(z.index_fill(0, torch.tensor([5], device=DEV), 0.0), ids, t, y, 2.0, 0.5)
    from concord_b200 import distill_loss, distill_loss_and_grad
    loss, dz = distill_loss_and_grad(z, ids, t, y, 2.0, 0.5)
    assert bool(loss.isfinite()) and bool(dz.isfinite().all()) and bool((dz[5] == 0).all())
    rows = distill_loss(z, ids, t, y, 2.0, 0.5, reduction="none")
    assert bool((rows[[5, 6, 7]] == 0).all())
    check(z.index_fill(0, torch.tensor([5], device=DEV), 0.0), ids, t, None, 2.0, 1.0)


def test_nothing_counts():
    from concord_b200 import distill_loss, distill_loss_and_grad
    z, ids, t, y = inputs(4, 70, 3, torch.bfloat16)
    y.fill_(-100)
    loss, dz = distill_loss_and_grad(z, ids, t, y, 1.0, 0.5)
    assert float(loss) == 0.0 and bool((dz == 0).all())
    z0 = z[:0].detach().requires_grad_()
    loss = distill_loss(z0, ids[:0], t[:0], y[:0], alpha=0.5)
    assert float(loss.detach()) == 0.0 and torch.autograd.grad(loss, z0)[0].shape == (0, 70)


def test_same_id_twice_sums():
    z, ids, t, y = inputs(6, 90, 6, torch.float32, seed=8)
    ids[:, 1] = ids[:, 0]
    ids[:, 4] = ids[:, 0]
    y[:3] = ids[:3, 0]                # the label among them
    check(z, ids, t, y, 2.0, 0.5)


def test_masked_and_extreme_logits():
    z, ids, t, y = inputs(8, 513, 4, torch.float32, seed=9)
    ids, y = ids % 256, y % 256
    z[0, 256:] = -math.inf            # a vocabulary mask
    z[1, 256:] = torch.finfo(torch.float32).min
    z[2] = z[2] + 1e4
    z[3, 7] = 300.0
    z[4, 300:] = -math.inf
    z[4, 256:300] = torch.finfo(torch.float32).min
    from concord_b200 import distill_loss_and_grad
    keep = [0, 2, 3, 5, 6, 7]
    check(z[keep], ids[keep], t[keep], y[keep], 2.0, 0.5)
    for r in (1, 4):                  # the type's lowest value weighs nothing, like -inf
        zl, zi = z[r:r + 1].clone(), z[r:r + 1].clone()      # of one alignment: the order of the sums goes by it
        zi[zi < -1e30] = -math.inf
        a = distill_loss_and_grad(zl, ids[r:r + 1], t[r:r + 1], y[r:r + 1], 2.0, 0.5)
        b = distill_loss_and_grad(zi, ids[r:r + 1], t[r:r + 1], y[r:r + 1], 2.0, 0.5)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_teacher_mass_on_a_masked_token_is_infinite():
    from concord_b200 import distill_loss
    z, ids, t, _ = inputs(2, 40, 3, torch.float32, labels=False)
    z[0, ids[0, 0]] = -math.inf
    rows = distill_loss(z, ids, t, reduction="none")
    assert float(rows[0]) == math.inf and bool(rows[1].isfinite())


@pytest.mark.parametrize("V", [64, 5003])
def test_nan_in_a_row_stays_its_own(V):
    from concord_b200 import distill_loss
    z, ids, t, y = inputs(5, V, 4, torch.bfloat16)
    clean = distill_loss(z, ids, t, y, 2.0, 0.5, reduction="none")
    z[2, V - 1] = float("nan")
    z[3] = -math.inf
    rows = distill_loss(z, ids, t, y, 2.0, 0.5, reduction="none")
    assert bool(rows[2].isnan()) and bool(rows[3].isnan())
    assert torch.equal(rows[[0, 1, 4]], clean[[0, 1, 4]])


def test_strides_and_leading_dims():
    from concord_b200 import distill_loss_and_grad
    z, ids, t, y = inputs(24, 400, 5, torch.bfloat16, seed=11)
    want = distill_loss_and_grad(z[:, 3:300].contiguous(), ids % 297, t, y % 297, 2.0, 0.5)
    got = distill_loss_and_grad(z[:, 3:300], ids % 297, t, y % 297, 2.0, 0.5)      # rows off 16 bytes
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    w3 = distill_loss_and_grad(z.view(4, 6, 400).transpose(0, 1), ids.view(4, 6, 5).transpose(0, 1),
                               t.view(4, 6, 5).transpose(0, 1), y.view(4, 6).T, 2.0, 0.5)
    flat = distill_loss_and_grad(z, ids, t, y, 2.0, 0.5)
    assert w3[1].shape == (6, 4, 400)
    assert torch.equal(w3[1].transpose(0, 1).reshape(24, 400), flat[1])
    every = z.t().contiguous().t()                                                  # columns apart: copied
    got = distill_loss_and_grad(every, ids, t, y, 2.0, 0.5)
    assert torch.equal(flat[0], got[0]) and torch.equal(flat[1], got[1])


def test_same_bits_every_time_and_on_another_stream():
    from concord_b200 import distill_loss_and_grad
    args = inputs(600, 4100, 32, torch.bfloat16, seed=12)
    first = distill_loss_and_grad(*args, 2.0, 0.5)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        second = distill_loss_and_grad(*args, 2.0, 0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, second))


def test_gradient_against_differences():
    """Central differences of the mean loss along random directions, fp32 logits: h^2 times the third derivative
    (at most alpha T^2 (1/T)^3 + 1 - alpha <= 2 for a unit direction) plus the loss's rounding over h."""
    from concord_b200 import distill_loss, distill_loss_and_grad
    z, ids, t, y = inputs(4, 67, 6, torch.float32, seed=13)
    for temp, alpha in ((2.0, 0.5), (1.3, 0.8)):
        _, dz = distill_loss_and_grad(z, ids, t, y, temp, alpha, reduction="sum")
        h = 2.0 ** -5
        for k in range(4):
            u = torch.randn_like(z)
            u /= u.norm()
            at = lambda s: distill_loss(z + s * u, ids, t, y, temp, alpha, reduction="none").double().sum()  # noqa: E731
            diff = float((at(h) - at(-h)) / (2 * h))
            noise = 64 * F32 * 40 * 4 / h
            assert abs(diff - float((dz * u).sum())) <= 2 * h * h + noise


def test_refusals():
    from concord_b200 import distill_loss, distill_loss_and_grad
    z, ids, t, y = inputs(4, 50, 3, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        distill_loss(z.cpu(), ids, t)
    with pytest.raises(TypeError, match="logits must be"):
        distill_loss(z.double(), ids, t)
    with pytest.raises(TypeError, match="top_ids must be"):
        distill_loss(z, ids.float(), t)
    with pytest.raises(ValueError, match="top_ids must be"):
        distill_loss(z, ids[:3], t[:3])
    with pytest.raises(ValueError, match="top_logits must have"):
        distill_loss(z, ids, t[:, :2])
    with pytest.raises(ValueError, match="1 to 512"):
        distill_loss(z, ids[:, :0], t[:, :0])
    with pytest.raises(ValueError, match="temperature"):
        distill_loss(z, ids, t, temperature=0.0)
    with pytest.raises(ValueError, match="alpha must be"):
        distill_loss(z, ids, t, y, alpha=1.5)
    with pytest.raises(ValueError, match="pass labels"):
        distill_loss(z, ids, t, alpha=0.5)
    with pytest.raises(ValueError, match="labels must have shape"):
        distill_loss(z, ids, t, y[:3], alpha=0.5)
    with pytest.raises(ValueError, match="reduction"):
        distill_loss(z, ids, t, reduction="avg")
    with pytest.raises(ValueError, match="reduction"):
        distill_loss_and_grad(z, ids, t, reduction="none")
