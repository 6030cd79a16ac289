"""QKNormRope's tables of cosines and sines: they belong to no state dict, so that the module itself has to have them right
wherever it is built and moved."""
import copy
import io

import pytest
import torch

META = torch.device("meta")


def _right(m, positions, rot, base=10000.0, device="cpu"):
    from concord_b200 import rope_tables
    for got, want in zip((m.cos, m.sin), rope_tables(positions, rot, base, device=device)):
        assert got.device.type == torch.device(device).type and got.dtype == torch.float32 and torch.equal(got, want)


def _on_meta(how, *a, **kw):
    from concord_b200 import QKNormRope
    if how == "argument":
        return QKNormRope(*a, device="meta", **kw)
    with META:
        return QKNormRope(*a, **kw)


@pytest.mark.parametrize("how", ["argument", "context"])
def test_built_without_memory(how):
    """Built on the meta device, given memory, then its weights: the tables are there, not what the memory held."""
    from concord_b200 import QKNormRope
    m = torch.nn.Sequential(_on_meta(how, 64, 100, rot=32, base=500.0))
    assert all(t.is_meta for t in (m[0].cos, m[0].sin, m[0].q_weight, m[0].k_weight))
    m.to_empty(device="cpu")
    _right(m[0], 100, 32, 500.0)
    full = torch.nn.Sequential(QKNormRope(64, 100, rot=32, base=500.0, device="cpu"))
    m.load_state_dict(full.state_dict())
    _right(m[0], 100, 32, 500.0)
    assert torch.equal(m[0].q_weight, torch.ones(64))


def test_built_without_memory_and_cast():
    m = torch.nn.Sequential(_on_meta("context", 64, 100)).bfloat16()
    assert m[0].cos.is_meta and m[0].cos.dtype == torch.float32 and m[0].q_weight.dtype == torch.bfloat16
    m.to_empty(device="cpu")
    _right(m[0], 100, 64)
    copied = copy.deepcopy(_on_meta("context", 64, 100))
    _right(copied.to_empty(device="cpu"), 100, 64)


def test_emptied():
    """to_empty of a module that had memory: its weights are gone, the tables are not."""
    from concord_b200 import QKNormRope
    m = QKNormRope(64, 100, rot=16, device="cpu")
    m.to_empty(device="cpu")
    _right(m, 100, 16)
    m.to_empty(device="meta")
    assert m.cos.is_meta and m.sin.is_meta and m.cos.dtype == torch.float32
    m.to_empty(device="cpu")
    _right(m, 100, 16)


def test_default_device():
    """Tables stand where the weights do."""
    from concord_b200 import QKNormRope
    with META:
        m = QKNormRope(64, 100)
        there = QKNormRope(64, 100, device="cpu")
    assert m.cos.device == m.q_weight.device and there.cos.device == there.q_weight.device == torch.device("cpu")
    _right(there, 100, 64)


def test_shared_saved_and_moved():
    from concord_b200 import QKNormRope
    m = QKNormRope(64, 100, device="cpu")
    assert m.share_memory().cos.is_shared()
    _right(m, 100, 64)
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    _right(torch.load(f, weights_only=False).double(), 100, 64)


@pytest.mark.gpu
def test_on_the_gpu():
    """A default device, and a move of tables made elsewhere: the rotation is the definition's."""
    from concord_b200 import QKNormRope
    x = torch.randn(50, 2, 64, device="cuda")
    with torch.device("cuda"):
        a = QKNormRope(64, 100)
    b = QKNormRope(64, 100, device="cpu").cuda()
    with META:
        c = QKNormRope(64, 100)
    c.to_empty(device="cuda").load_state_dict(b.state_dict())
    for m in (a, c):
        _right(m, 100, 64, device="cuda")
    _right(b.cpu(), 100, 64)
    b.cuda()
    at = torch.arange(50, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(32, device="cuda").double() / 32)
    y = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    p, q, cos, sin = y[..., :32], y[..., 32:], at.cos()[:, None], at.sin()[:, None]
    want = torch.cat((p * cos - q * sin, p * sin + q * cos), -1)
    # a table's entry is off by 2^-24, a product's and the sum's rounding, the mean's 64 terms and rsqrt's 2^-22: below 2^-18
    for m in (a, b, c):
        with torch.no_grad():
            assert bool(((m(x, x)[0].double() - want).abs() <= 2.0 ** -18 * (p.abs() + q.abs()).repeat(1, 1, 2)).all())


@pytest.mark.gpu
def test_queries_alone():
    """The module takes no keys, as the function does: k' is None, and k_weight gets no gradient."""
    from concord_b200 import QKNormRope
    m = QKNormRope(64, 100, device="cuda")
    q = torch.randn(50, 2, 64, device="cuda")
    out, none = m(q, None)
    assert none is None and torch.equal(out, m(q, q)[0])
    out.sum().backward()
    assert m.q_weight.grad is not None and m.k_weight.grad is None


def test_bases():
    """A base that is no positive number has no angles: refused, in place of tables of NaN."""
    from concord_b200 import QKNormRope, rope_tables
    for base in (0.0, -10000.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="base must be positive"):
            rope_tables(10, 8, base, device="cpu")
        with pytest.raises(ValueError, match="base must be positive"):
            QKNormRope(8, 10, base=base, device="cpu")
    assert bool(rope_tables(10, 8, 0.5, device="cpu")[0].isfinite().all())
