"""qk_norm_rope against plain forms in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}       # half of the least step


def _turn(x, c, s, rot, inter):
    """x [T, H, D] in 64 bits, c and s [T, 1, rot / 2]."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    ra, rb = a * c - b * s, a * s + b * c
    out = x.clone()
    if inter:
        out[..., 0:rot:2], out[..., 1:rot:2] = ra, rb
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = ra, rb
    return out


def _reach(x, rot, inter):
    """|a| + |b| for both of a pair: what a turned column can get from."""
    m = x.abs()
    out = m.clone()
    a, b = (m[..., 0:rot:2], m[..., 1:rot:2]) if inter else (m[..., :rot // 2], m[..., rot // 2:rot])
    if inter:
        out[..., 0:rot:2] = out[..., 1:rot:2] = a + b
    else:
        out[..., :rot // 2] = out[..., rot // 2:rot] = a + b
    return out


def _plain(x, w, dy, c, s, rot, inter, norm, eps):
    """(y, dx, dw) and what their errors go by, in 64 bits.  fp32's share: a sum of D squares is off by at most D
    units (half of it in its root), the other operations of a value by fewer than 32 together."""
    x, dy, D = x.double(), dy.double(), x.shape[-1]
    k = (D + 32) * U
    n = x
    if norm:
        r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
        n = x * r * (1.0 if w is None else w.double())
    y, y_lim = _turn(n, c, s, rot, inter), k * _reach(n, rot, inter)
    dn, dn_mag = _turn(dy, c, -s, rot, inter), _reach(dy, rot, inter)
    if not norm:
        return y, y_lim, dn, k * dn_mag, None, None
    g, g_mag = (dn, dn_mag) if w is None else (dn * w.double(), dn_mag * w.double().abs())
    dx = r * g - x * r ** 3 * (g * x).mean(-1, keepdim=True)
    dx_mag = r * g_mag + x.abs() * r ** 3 * (g_mag * x.abs()).mean(-1, keepdim=True)
    count = x.shape[0] * x.shape[1]
    dw, dw_lim = (dn * x * r).sum((0, 1)), (count + 2 * D + 32) * U * (dn_mag * x.abs() * r).sum((0, 1))
    return y, y_lim, dx, 2 * k * dx_mag, dw, dw_lim


def _case(T, H, Hk, D, rot, dtype, inter, norm, weights=True, seed=0, pos=None, packed=True):
    from concord_b200 import rope_tables
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    qkv = (randn(T, H + 2 * Hk, D) * (0.5 + 2 * torch.rand(D, generator=g, device=DEV))).to(dtype)
    q, k = qkv[:, :H], qkv[:, H:H + Hk]
    if not packed:
        q, k = q.contiguous(), k.contiguous()
    pos = torch.arange(T, device=DEV) * 7 % 50 + 1 if pos is None else pos
    cos, sin = rope_tables(int(pos.max()) + 1 if T else 60, rot) if rot else (None, None)
    qw, kw = (1 + 0.3 * randn(D), 1 + 0.3 * randn(D)) if norm and weights else (None, None)
    dq, dk = (randn(T, H, D) * 0.1).to(dtype), (randn(T, Hk, D) * 0.1).to(dtype)
    return q, k, cos, sin, pos if rot else None, qw, kw, dq, dk


def _check(args, inter, norm, eps=1e-6):
    from concord_b200 import qk_norm_rope
    q, k, cos, sin, pos, qw, kw, dq, dk = args
    dtype, rot = q.dtype, 0 if cos is None else 2 * cos.shape[1]
    leaves = [t.detach().requires_grad_() for t in (q, k, qw, kw) if t is not None]
    w = leaves[2:] if qw is not None else [None, None]
    yq, yk = qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, *w, norm=norm, eps=eps, interleaved=inter)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == yk.dtype == dtype
    T = q.shape[0]
    c, s = (t[pos.long()].double()[:, None] for t in (cos, sin)) if rot else (torch.zeros(T, 1, 0, device=DEV),) * 2
    for i, (x, wx, dy, y) in enumerate(((q, qw, dq, yq), (k, kw, dk, yk))):
        ry, ly, rx, lx, rw, lw = _plain(x, wx, dy, c, s, rot, inter, norm, eps)
        assert bool(((y.double() - ry).abs() <= HALF[dtype] * (ry.abs() + ly) + ly + LEAST[dtype]).all())
        assert bool(((grads[i].double() - rx).abs() <= HALF[dtype] * (rx.abs() + lx) + lx + LEAST[dtype]).all())
        if wx is not None:
            assert bool(((grads[2 + i].double() - rw).abs() <= lw).all())


SHAPES = [(1, 1, 1, 128, 128), (5, 16, 4, 128, 128), (37, 6, 6, 64, 64), (130, 20, 5, 80, 40), (33, 10, 2, 72, 72),
          (64, 3, 1, 96, 96), (19, 4, 4, 256, 256), (1000, 8, 2, 32, 16), (7, 5, 5, 8, 8), (21, 2, 2, 72, 36),
          (11, 3, 3, 10, 4), (9, 2, 1, 255, 254), (400, 12, 12, 64, 0), (3, 7, 7, 1, 0), (20, 32, 8, 128, 64), (40, 6, 3, 36, 36),
          (90, 4, 2, 60, 12), (33, 8, 4, 124, 124), (17, 3, 1, 132, 68), (70, 5, 5, 68, 0), (65, 3, 3, 24, 24),
          (50, 6, 2, 40, 40), (77, 12, 4, 48, 24), (300, 7, 7, 16, 16), (2100, 24, 8, 80, 80), (20011, 5, 5, 80, 40),
          (9001, 16, 4, 128, 128), (6000, 32, 32, 64, 32)]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,Hk,D,rot", SHAPES)
def test_sizes(T, H, Hk, D, rot, inter):
    _check(_case(T, H, Hk, D, rot, torch.bfloat16, inter, True), inter, True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm,weights", [(True, True), (True, False), (False, False)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,rot", [(128, 128), (80, 40), (72, 36), (60, 60), (18, 6)])
def test_types(dtype, norm, weights, inter, D, rot):
    _check(_case(70, 8, 2, D, rot, dtype, inter, norm, weights), inter, norm)


@pytest.mark.parametrize("T", [1, 2, 700, 5000, 20011])
def test_lengths(T):
    _check(_case(T, 8, 2, 64, 64, torch.bfloat16, False, True), False, True)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [2.0 ** -50, 2.0 ** 50])
def test_heads_of_any_size(scale, dtype, inter):
    """r^3 leaves fp32's range long before r x and the gradients do."""
    q, k, *rest = _case(23, 4, 2, 64, 64, dtype, inter, True)
    _check((q * scale, k * scale, *rest), inter, True, eps=0.0)


def test_far_positions():
    """Positions up to 1,000,000, whose angles fp32 products would have lost: the tables come from 64 bits, so the
    definition's own angles serve; cos and sin held in fp32 add half a unit each."""
    from concord_b200 import qk_norm_rope, rope_tables
    cos, sin = rope_tables(1_000_001, 16)
    pos = torch.tensor([0, 1, 65535, 131072, 999_999, 1_000_000], device=DEV)
    x = torch.randn(6, 2, 16, device=DEV)
    y, none = qk_norm_rope(x, None, cos, sin, pos, norm=False)
    assert none is None
    angle = pos.double()[:, None] * torch.tensor([10000.0 ** (-2 * i / 16) for i in range(8)], dtype=torch.float64, device=DEV)
    ref = _turn(x.double(), angle.cos()[:, None], angle.sin()[:, None], 16, False)
    # 1e6 radians in 64 bits are off by 2^-33: nothing here
    assert bool(((y.double() - ref).abs() <= 6 * U * _reach(x.double(), 16, False)).all())


def test_positions_of_any_type_and_the_default():
    from concord_b200 import qk_norm_rope
    q, k, cos, sin, _, qw, kw, _, _ = _case(40, 4, 2, 64, 64, torch.bfloat16, False, True, pos=torch.arange(40, device=DEV))
    a = qk_norm_rope(q, k, cos, sin, None, qw, kw)
    b = qk_norm_rope(q, k, cos, sin, torch.arange(40, device=DEV), qw, kw)
    c = qk_norm_rope(q, k, cos, sin, torch.arange(80, device=DEV, dtype=torch.int32)[:40], qw, kw)
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))


def test_positions_the_tables_do_not_have():
    """NaN in the columns that turn, the others as ever; nobody else is touched."""
    from concord_b200 import qk_norm_rope, rope_tables
    cos, sin = rope_tables(10, 16)
    for D in (32, 30):                                         # the wide path, and that of any size
        q = torch.randn(4, 3, D, device=DEV)
        y, _ = qk_norm_rope(q, None, cos, sin, torch.tensor([3, 10, -1, 9], device=DEV), norm=False)
        ok, _ = qk_norm_rope(q, None, cos, sin, torch.tensor([3, 3, 3, 9], device=DEV), norm=False)
        assert torch.equal(y[0], ok[0]) and torch.equal(y[3], ok[3])
        assert bool(y[1:3, :, :16].isnan().all()) and torch.equal(y[1:3, :, 16:], q[1:3, :, 16:])


def test_columns_that_do_not_turn_stay():
    """Infinities beside turned columns, and the other way round (inf cos and inf sin would make NaN of 0)."""
    from concord_b200 import qk_norm_rope, rope_tables
    for D in (32, 30):
        cos, sin = rope_tables(2, 16)
        q = torch.randn(2, 1, D, device=DEV)
        q[..., 16:] = float("inf")
        y, _ = qk_norm_rope(q, None, cos, sin, norm=False)
        assert bool((y[..., 16:] == float("inf")).all()) and bool(y[..., :16].isfinite().all())


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shift", [1, 2, 4, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_addresses(dtype, shift, inter):
    """q and k that begin 1 to 8 elements behind an aligned address, with token strides to match: 2 to 32 bytes."""
    T, H, D = 40, 4, 64
    args = list(_case(T, H, H, D, D, dtype, inter, True, packed=False))
    for i in (0, 1):
        room = torch.zeros(T, H * D + 8 + shift, dtype=dtype, device=DEV)
        room[:, shift:shift + H * D] = args[i].reshape(T, H * D)
        args[i] = room[:, shift:shift + H * D].view(T, H, D)
    _check(args, inter, True)


@pytest.mark.parametrize("layout", ["heads_first", "unaligned", "every_second_column", "expanded", "transposed_gradient"])
def test_layouts(layout):
    from concord_b200 import qk_norm_rope
    T, H, D = 50, 4, 64
    args = list(_case(T, H, H, D, D, torch.bfloat16, False, True, packed=False))
    q = args[0]
    if layout == "heads_first":
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "unaligned":
        q = torch.cat([q.flatten().new_zeros(1), q.flatten()])[1:].view(T, H, D)
    elif layout == "every_second_column":
        q = torch.stack([q, q], -1)[..., 0]
    elif layout == "expanded":
        q = q[:, :1].expand(T, H, D)
    else:
        args[7] = args[7].transpose(0, 1).contiguous().transpose(0, 1)
    args[0] = q
    _check(args, False, True)
    if layout == "unaligned":                                  # (another path, another order of the sums)
        return
    dense = qk_norm_rope(q.contiguous(), args[1], *args[2:7])
    assert all(torch.equal(a, b) for a, b in zip(qk_norm_rope(q, args[1], *args[2:7]), dense))


def test_one_output_alone():
    """Only q' used: k and its weight get none; the gradients of both sides otherwise."""
    from concord_b200 import qk_norm_rope
    args = _case(30, 4, 2, 64, 64, torch.float32, False, True)
    leaves = [t.detach().requires_grad_() for t in (args[0], args[1], args[5], args[6])]
    call = lambda: qk_norm_rope(leaves[0], leaves[1], *args[2:5], *leaves[2:])  # noqa: E731
    both = torch.autograd.grad(call(), leaves, (args[7], args[8]))
    q_only = torch.autograd.grad(call()[0], leaves, args[7], allow_unused=True)
    assert torch.equal(q_only[0], both[0]) and q_only[1] is None and q_only[3] is None
    # (its blocks are other ones then: another order of the fp32 sums)
    ref = _plain(args[0], args[5], args[7], *(t[args[4].long()].double()[:, None] for t in args[2:4]), 64, False, True, 1e-6)
    assert bool(((q_only[2].double() - ref[4]).abs() <= ref[5]).all())
    k_only = torch.autograd.grad(call()[1], leaves, args[8], allow_unused=True)
    assert k_only[0] is None and k_only[2] is None and torch.equal(k_only[1], both[1])
    one = torch.autograd.grad(call(), leaves[3:], (args[7], args[8]))
    assert torch.equal(one[0], both[3])


def test_zero_rows_and_no_tokens():
    from concord_b200 import qk_norm_rope, rope_tables
    cos, sin = rope_tables(5, 64)
    w = torch.ones(64, device=DEV, requires_grad=True)
    q = torch.zeros(5, 2, 64, device=DEV, requires_grad=True)
    y, _ = qk_norm_rope(q, None, cos, sin, None, w, eps=1e-6)
    dq, dw = torch.autograd.grad(y, (q, w), torch.ones_like(y))
    assert bool((y == 0).all()) and bool(dq.isfinite().all()) and bool((dw == 0).all())
    q = torch.zeros(0, 2, 64, device=DEV, requires_grad=True)
    k = torch.zeros(0, 1, 64, device=DEV, requires_grad=True)
    y, z = qk_norm_rope(q, k, cos, sin, None, w, w)
    assert y.shape == (0, 2, 64) and z.shape == (0, 1, 64)
    dw, = torch.autograd.grad((y, z), (w,), (torch.ones_like(y), torch.ones_like(z)))
    assert bool((dw == 0).all())


def test_module():
    from concord_b200 import QKNormRope, qk_norm_rope
    m = QKNormRope(64, 100, rot=32, device=DEV)
    assert sorted(m.state_dict()) == ["k_weight", "q_weight"]
    q, k = torch.randn(9, 4, 64, device=DEV), torch.randn(9, 2, 64, device=DEV)
    a, b = m(q, k), qk_norm_rope(q, k, m.cos, m.sin, None, m.q_weight, m.k_weight)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and m.cos.shape == (100, 16)
    (a[0].sum() + a[1].sum()).backward()
    assert m.q_weight.grad is not None and m.k_weight.grad is not None


def test_refusals():
    from concord_b200 import qk_norm_rope, rope_tables
    q, k = torch.zeros(4, 2, 64, device=DEV), torch.zeros(4, 2, 64, device=DEV)
    cos, sin = rope_tables(4, 64)
    w = torch.ones(64, device=DEV)
    for error, match, call in (
            (TypeError, "q must be one of", lambda: qk_norm_rope(q.double(), None)),
            (TypeError, "k must have q's type", lambda: qk_norm_rope(q, k.half())),
            (ValueError, "q must be", lambda: qk_norm_rope(q[0], None)),
            (ValueError, "q must be", lambda: qk_norm_rope(torch.zeros(4, 1, 257, device=DEV), None)),
            (ValueError, "k must be", lambda: qk_norm_rope(q, k[:3])),
            (ValueError, "belongs to the norm", lambda: qk_norm_rope(q, k, cos, sin, None, w, norm=False)),
            (ValueError, "k_weight without k", lambda: qk_norm_rope(q, None, cos, sin, None, w, w)),
            (ValueError, "q_weight must have shape", lambda: qk_norm_rope(q, k, cos, sin, None, w[:32])),
            (ValueError, "come together", lambda: qk_norm_rope(q, k, cos)),
            (ValueError, "cos and sin must be", lambda: qk_norm_rope(q, k, *rope_tables(4, 66))),
            (ValueError, "positions must have shape", lambda: qk_norm_rope(q, k, cos, sin, torch.zeros(3, dtype=torch.long, device=DEV))),
            (TypeError, "positions must be one of", lambda: qk_norm_rope(q, k, cos, sin, torch.zeros(4, device=DEV))),
            (ValueError, "positions without", lambda: qk_norm_rope(q, k, positions=torch.zeros(4, dtype=torch.long, device=DEV))),
            (ValueError, "nothing to do", lambda: qk_norm_rope(q, k, norm=False)),
            (ValueError, "eps", lambda: qk_norm_rope(q, k, eps=-1.0)),
            (ValueError, "even number", lambda: rope_tables(4, 5)),
            (RuntimeError, "CUDA tensors only", lambda: qk_norm_rope(q.cpu(), None))):
        with pytest.raises(error, match=match):
            call()
