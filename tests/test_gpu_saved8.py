"""Activations kept in 8 bits: the format, the weight gradient from it, the packed layer that uses both."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _asked():
    """Bytes that tensors asked for (a block of the allocator may be up to 1 MB larger)."""
    return torch.cuda.memory_stats()["requested_bytes.all.current"]

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def plain8(x):
    """What 8 bits keep of x [M, K], in 64 bits, by the definition: the least e with |x| <= 127 2^e."""
    M, K = x.shape
    pad = torch.zeros(-(-M // 32) * 32, K, dtype=torch.float64, device=x.device)
    pad[:M] = x.double()
    b = pad.view(-1, 32, K)
    most = b.abs().amax(1, keepdim=True)
    e = torch.full_like(most, -126.0)
    for _ in range(400):
        more = most > 127 * torch.exp2(e)
        if not bool(more.any()):
            break
        e = e + more.double()
    step = torch.exp2(e)
    return (b / step).round().mul(step).view(-1, K)[:M]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,K", [(1, 1), (31, 7), (32, 16), (33, 129), (64, 128), (65, 260), (100, 384), (257, 1000)])
def test_values(M, K, dtype):
    """Exactly the definition's values, in every type that holds them, read back from any odd size."""
    from concord_b200 import save8
    g = torch.Generator(device=DEV).manual_seed(M * K)
    x = torch.randn(M, K, generator=g, device=DEV) * torch.exp2(torch.randint(-12, 6, (K,), generator=g, device=DEV).float())
    x[torch.rand(M, K, generator=g, device=DEV) < 0.3] = 0.0
    x = x.to(dtype)
    s = save8(x)
    want = plain8(x)
    assert s.shape == x.shape and s.dtype == dtype and s.dense().dtype == dtype
    assert torch.equal(s.dense(torch.float32).double(), want) and torch.equal(s.dense(torch.bfloat16).double(), want)
    pad = (K + 15) // 16 * 16
    assert s.nbytes == -(-M // 64) * 66 * pad
    # half a step off at most, less than the block's largest / 127
    b = torch.zeros(-(-M // 32) * 32, K, dtype=torch.float64, device=DEV)
    b[:M] = x.double()
    most = b.view(-1, 32, K).abs().amax(1, keepdim=True).expand(-1, 32, K).reshape(-1, K)[:M]
    assert bool(((want - x.double()).abs() <= most / 127).all())


def test_layout():
    """The bytes stand where the header says: tiles of 64 tokens x 128 features, codes [4][features][16], bytes [2][features]."""
    from concord_b200 import save8
    M, K = 150, 300
    x = torch.randn(M, K, device=DEV)
    data, want = save8(x).data.cpu(), plain8(x).cpu()
    at, pad = 0, 304
    for t in range(3):
        for k0 in range(0, pad, 128):
            w = min(128, pad - k0)
            codes = data[at:at + 64 * w].view(torch.int8).view(4, w, 16).permute(0, 2, 1).reshape(64, w)
            scale = data[at + 64 * w:at + 66 * w].view(2, w)
            at += 66 * w
            value = codes.double() * torch.exp2(scale.double() - 127).repeat_interleave(32, 0)
            for r in range(64):
                for c in (0, w // 2, w - 1):
                    row, col = 64 * t + r, k0 + c
                    inside = row < M and col < K
                    assert value[r, c] == (want[row, col] if inside else 0), (row, col)
    assert at == data.numel()


def test_extremes():
    """The least and largest values of each type, ties, steps' borders, and what is not a number."""
    from concord_b200 import save8
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        info = torch.finfo(dtype)
        top = torch.full((32, 8), info.max, dtype=dtype, device=DEV)
        kept = save8(top).dense()
        assert bool(kept.isfinite().all()) and bool((kept.double() >= info.max * 62.9 / 64).all())
        tiny = torch.full((32, 8), info.smallest_normal * info.eps, dtype=dtype, device=DEV)       # the least subnormal
        kept = save8(tiny).dense(torch.float32)
        if dtype == torch.float16:
            assert torch.equal(kept.double(), plain8(tiny))
        else:                            # steps are 2^-126 at least
            assert bool((kept == 0).all())
    x = torch.zeros(32, 6, device=DEV)
    x[:, 0] = 127.0                      # step 1
    x[0, 1], x[1, 1], x[2, 1], x[3, 1] = 127.0, 0.5, 1.5, -2.5         # ties to even
    x[0, 2] = 127.0000076                # just above: step 2
    x[0, 3], x[1, 3] = float("inf"), 1.0
    x[0, 4] = float("nan")
    x[0, 5] = 1e-42
    d = save8(x).dense()
    assert bool((d[:, 0] == 127).all()) and d[:4, 1].tolist() == [127.0, 0.0, 2.0, -2.0] and float(d[0, 2]) == 128.0
    assert bool(d[:, 3:5].isnan().all()) and bool((d[:, 5] == 0).all())
    assert save8(torch.full((5, 3), float("nan"), device=DEV, dtype=torch.bfloat16)).dense().isnan().all()


def test_shapes_and_strides():
    from concord_b200 import save8
    x = torch.randn(3, 50, 96, device=DEV).bfloat16()
    assert torch.equal(save8(x).dense(), save8(x.view(150, 96)).dense().view(3, 50, 96))
    part = x[..., 5:40]
    assert torch.equal(save8(part).dense(), save8(part.contiguous()).dense())
    turned = x[0].t()
    assert torch.equal(save8(turned).dense(), save8(turned.contiguous()).dense())
    row = torch.randn(64, device=DEV)
    assert save8(row).dense().shape == (64,) and save8(row.expand(40, 64)).dense().shape == (40, 64)
    empty = save8(x[:0])
    assert empty.dense().shape == (0, 50, 96) and empty.nbytes == 0


DW = [(1, 8, 1), (33, 8, 16), (64, 256, 256), (65, 264, 130), (100, 1536, 384), (129, 72, 129), (1000, 512, 300),
      (4096, 2048, 520), (16381, 1536, 384), (700, 128, 5000), (64 * 37 + 5, 2560, 2568)]


@pytest.mark.parametrize("M,N,K", DW)
def test_weight_gradient_of_whole_numbers(M, N, K):
    """Whole numbers whose products' sums stay below 2^24 are exact in fp32: the result is the sum, rounded once to
    bf16; partial tiles, features and tokens, tiles cut along the tokens."""
    from concord_b200 import gemm_dw8_error, grad_weight8, save8
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    x = torch.randint(-30, 31, (M, K), generator=g, device=DEV).bfloat16()
    dy = torch.randint(-4, 5, (M, N), generator=g, device=DEV).bfloat16()
    s = save8(x)
    assert torch.equal(s.dense(), x)
    got = grad_weight8(dy, s)
    ref = (dy.double().t() @ x.double()).float().bfloat16()
    assert got.shape == (N, K) and torch.equal(got, ref) and gemm_dw8_error() == 0
    assert torch.equal(grad_weight8(dy, s), got)


@pytest.mark.parametrize("M,N,K", [(77, 64, 100), (3000, 512, 640), (16384, 384, 384)])
def test_weight_gradient_rounding(M, N, K):
    """fp32 sums of M exact products, whose additions may cut what lies below their last bit: M 2^-23 of the sum of
    magnitudes, and the result's rounding."""
    from concord_b200 import grad_weight8, save8
    x, dy = torch.randn(M, K, device=DEV), (torch.randn(M, N, device=DEV) * 0.01).bfloat16()
    s = save8(x)
    v = s.dense(torch.float32).double()
    ref, mag = dy.double().t() @ v, dy.double().abs().t() @ v.abs()
    lim = M * 2 * U * mag
    assert bool(((grad_weight8(dy, s).double() - ref).abs() <= lim + 2.0 ** -8 * (ref.abs() + lim)).all())


def test_weight_gradient_operands():
    """A gradient that is a part of another, leading dimensions, an unaligned one, N that is no multiple of 8, no rows."""
    from concord_b200 import grad_weight8, save8
    x = torch.randint(-9, 10, (2, 60, 48), device=DEV).bfloat16()
    dy = torch.randint(-4, 5, (2, 60, 80), device=DEV).bfloat16()
    ref = lambda d: (d.reshape(120, -1).double().t() @ x.view(120, 48).double()).bfloat16()  # noqa: E731
    s = save8(x)
    assert torch.equal(grad_weight8(dy, s), ref(dy))
    for part in (dy[..., 8:72], dy[..., 3:67], dy[..., :61], dy[..., :1]):
        assert torch.equal(grad_weight8(part, s), ref(part))
    assert torch.equal(grad_weight8(torch.ones(2, 60, 1, device=DEV).bfloat16().expand(2, 60, 16), s),
                       x.double().sum((0, 1)).bfloat16().expand(16, 48))
    none = grad_weight8(dy[:, :0], save8(x[:, :0]))
    assert none.shape == (80, 48) and bool((none == 0).all())


def test_not_a_number_reaches_its_feature_alone():
    from concord_b200 import grad_weight8, save8
    x, dy = torch.ones(70, 200, device=DEV), torch.ones(70, 16, device=DEV).bfloat16()
    x[40, 3], x[5, 150] = float("nan"), float("inf")
    got = grad_weight8(dy, save8(x))
    bad = torch.zeros(200, dtype=torch.bool, device=DEV)
    bad[3] = bad[150] = True
    assert bool(got[:, bad].isnan().all()) and bool((got[:, ~bad] == 70).all())


def _layer(seed=0, K=256, N=128, bias=False):
    from concord_b200 import ConcordLinearPackedB
    from concord_b200.checkpoint import set_step_salt
    torch.manual_seed(seed)
    set_step_salt(torch.device(DEV, torch.cuda.current_device()), seed)
    lay = ConcordLinearPackedB(K, N, bias=bias, device=DEV, lr=1e-2)
    lay.load_weights(torch.randn(N, K, device=DEV) * 0.05)
    return lay


@pytest.mark.parametrize("how", ["argument", "attribute"])
@pytest.mark.parametrize("K,N", [(256, 128), (104, 40), (64, 20)])
def test_packed_layer(how, K, N):
    """Forward and the input's gradient as without; the step is the one that dW from the kept values makes."""
    from concord_b200 import grad_weight8, save8
    torch.manual_seed(7)
    x, dy = torch.randn(2, 50, K, device=DEV).bfloat16(), torch.randn(2, 50, N, device=DEV).bfloat16()
    plain = _layer(K=K, N=N)
    a = x.clone().requires_grad_()
    ya = plain(a)
    ya.backward(dy)
    eight = _layer(K=K, N=N)
    b = x.clone().requires_grad_()
    if how == "attribute":
        eight.save8 = True
        yb = eight(b)
    else:
        yb = eight(b, saved=save8(b.detach()))
    yb.backward(dy)
    assert torch.equal(ya, yb) and torch.equal(a.grad, b.grad)
    given = _layer(K=K, N=N)
    given(x)
    given.optimizer_step(grad_weight8(dy, save8(x)))
    assert torch.equal(eight.packed_w, given.packed_w) and torch.equal(eight.v_row, given.v_row)
    assert not torch.equal(eight.packed_w, plain.packed_w)


def test_packed_layer_of_whole_numbers():
    """Inputs that 8 bits keep exactly and sums that fp32 holds: the same step as without."""
    torch.manual_seed(8)
    x, dy = (torch.randint(-n, n + 1, (300, k), device=DEV).bfloat16() for n, k in ((30, 256), (4, 128)))
    plain = _layer()
    plain(x.clone().requires_grad_()).backward(dy)
    eight = _layer()
    eight.save8 = True
    eight(x.clone().requires_grad_()).backward(dy)
    assert torch.equal(eight.packed_w, plain.packed_w) and torch.equal(eight._bf16_weight_buf, plain._bf16_weight_buf)


def test_packed_layer_with_gradient_noise():
    """The noise's statistics come from the kept values: whole numbers, the same as without."""
    from concord_b200 import packed_b
    torch.manual_seed(9)
    x, dy = (torch.randint(-n, n + 1, (200, k), device=DEV).bfloat16() for n, k in ((30, 256), (4, 128)))
    packed_b.set_sigmag_noise(True)
    try:
        words = []
        for eight in (False, True):
            lay = _layer()
            lay.save8 = eight
            y = lay(x.clone().requires_grad_())
            torch.manual_seed(10)
            y.backward(dy)
            words.append(lay.packed_w.clone())
        assert torch.equal(words[0], words[1])
    finally:
        packed_b.set_sigmag_noise(False)


def test_packed_layer_keeps_8_bits():
    """What a forward holds until its backward: the codes, not x."""
    from concord_b200 import save8
    lay = _layer(K=1024, N=1024)
    lay.save8 = True
    x = torch.randn(4096, 1024, device=DEV).bfloat16().requires_grad_()
    lay(x * 1.0).sum().backward()                           # (buffers and workspaces made)
    torch.cuda.synchronize()
    before = _asked()
    y = lay(x * 1.0)
    held = _asked() - before - y.numel() * 2
    assert held <= save8(x.detach()).nbytes + 4096
    with torch.no_grad():
        assert not lay(x).requires_grad
    y.sum().backward()


def test_packed_layer_bias_fp32_input_and_refusals():
    from concord_b200 import save8
    lay = _layer(bias=True)
    x = torch.randn(30, 256, device=DEV, requires_grad=True)
    y = lay(x, saved=save8(x.detach()))
    assert y.dtype == torch.float32
    y.sum().backward()
    assert torch.equal(lay.bias.grad, torch.full_like(lay.bias.grad, 30)) and x.grad.shape == x.shape
    with pytest.raises(TypeError, match="saved must be a Saved8"):
        lay(x, saved=x)
    other = save8(x.detach())
    other.data = other.data.cpu()
    with pytest.raises(RuntimeError, match="saved is on cpu"):
        lay(x, saved=other)
    with pytest.raises(ValueError, match="saved is of shape"):
        lay(x, saved=save8(x[:3].detach()))


def test_refusals():
    from concord_b200 import Saved8, grad_weight8, save8
    x = torch.zeros(4, 8, device=DEV)
    s = save8(x)
    for error, match, call in (
            (TypeError, "x must be one of", lambda: save8(x.double())),
            (ValueError, "last dimension", lambda: save8(torch.zeros((), device=DEV))),
            (RuntimeError, "CUDA tensors only", lambda: save8(x.cpu())),
            (TypeError, "must be a Saved8", lambda: grad_weight8(x.bfloat16(), x)),
            (TypeError, "grad_y must be one of", lambda: grad_weight8(x, s)),
            (ValueError, "grad_y must be", lambda: grad_weight8(x[:3].bfloat16(), s)),
            (TypeError, "dtype must be one of", lambda: s.dense(torch.float64)),
            (RuntimeError, "saved must hold", lambda: Saved8(s.data, (65, 8), torch.float32).dense()),
            (RuntimeError, "saved must hold", lambda: Saved8(s.data[1:], (4, 8), torch.float32).dense()),
            (RuntimeError, "saved must hold", lambda: Saved8(s.data.float(), (4, 8), torch.float32).dense()),
            (RuntimeError, "saved must hold", lambda: grad_weight8(torch.zeros(65, 8, device=DEV).bfloat16(),
                                                                   Saved8(s.data, (65, 8), torch.float32)))):
        with pytest.raises(error, match=match):
            call()


def _conv(C=16, O=24, k=3, stride=1):
    from concord_b200 import ConcordConv2dPackedB
    from concord_b200.checkpoint import set_step_salt
    torch.manual_seed(0)
    set_step_salt(torch.device(DEV, torch.cuda.current_device()), 0)
    lay = ConcordConv2dPackedB(C, O, k, stride=stride, padding=k // 2, bias=False, device=DEV, lr=1e-2)
    lay.load_weights(torch.randn(O, C * k * k, device=DEV) * 0.1)
    return lay


@pytest.mark.parametrize("k", [1, 3])
def test_convolution(k):
    """Channels-last inputs in 8 bits, pixels as tokens: forward and the input's gradient as without; the step is the one
    of the kept values' dW, and that of x itself where x is kept exactly."""
    from concord_b200 import gemm, save8
    torch.manual_seed(3)
    for whole in (False, True):
        x = torch.randint(-30, 31, (2, 16, 9, 7), device=DEV) if whole else torch.randn(2, 16, 9, 7, device=DEV)
        x = x.bfloat16().contiguous(memory_format=torch.channels_last)
        dy = torch.randint(-4, 5, (2, 24, 9, 7), device=DEV).bfloat16().contiguous(memory_format=torch.channels_last)
        plain, eight = _conv(k=k), _conv(k=k)
        _conv(k=k)                                           # (the salt at its start)
        a = x.clone(memory_format=torch.preserve_format).requires_grad_()
        ya = plain(a)
        ya.backward(dy)
        eight.save8 = True
        _conv(k=k)
        b = x.clone(memory_format=torch.preserve_format).requires_grad_()
        yb = eight(b)
        yb.backward(dy)
        assert torch.equal(ya, yb) and torch.equal(a.grad, b.grad)
        if whole:
            assert torch.equal(plain.packed_w, eight.packed_w)
            continue
        given = _conv(k=k)
        given(x)
        kept = save8(x.permute(0, 2, 3, 1)).dense().permute(0, 3, 1, 2)
        w = gemm.filter_krsc(given._bf16_weight_buf, 16, k, k)
        given.optimizer_step(gemm.conv2d_backward_nhwc(kept, w, dy, k, k, 1, k // 2)[1])
        assert torch.equal(eight.packed_w, given.packed_w) and not torch.equal(eight.packed_w, plain.packed_w)


def test_other_convolutions_keep_their_input():
    """A stride that the implicit kernels do not run: the switch changes nothing."""
    x = torch.randn(2, 16, 8, 8, device=DEV).bfloat16().contiguous(memory_format=torch.channels_last)
    words = []
    for eight in (False, True):
        lay = _conv(stride=2)
        lay.save8 = eight
        y = lay(x.clone(memory_format=torch.preserve_format).requires_grad_())
        y.backward(torch.ones_like(y))
        words.append(lay.packed_w.clone())
    assert torch.equal(words[0], words[1])


def test_a_whole_model_of_layers():
    """concordify(save8=True): linear layers and convolutions; the ordinary ones beside them train as ever."""
    from concord_b200.convert import concordify
    torch.manual_seed(4)
    m = torch.nn.Sequential(torch.nn.Conv2d(8, 16, 3, padding=1), torch.nn.SiLU(), torch.nn.Flatten(), torch.nn.Linear(16 * 36, 40),
                            torch.nn.LayerNorm(40), torch.nn.Linear(40, 8)).to(DEV)
    layers = concordify(m, lr=1e-3, convs=True, save8=True)
    assert len(layers) == 3 and all(lay.save8 for lay in layers)
    x = torch.randn(5, 8, 6, 6, device=DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = m(x)
    before = [lay.packed_w.clone() for lay in layers]
    out.float().square().sum().backward()
    assert all(not torch.equal(a, lay.packed_w) for a, lay in zip(before, layers)) and bool(x.grad.isfinite().all())
