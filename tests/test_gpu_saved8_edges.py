"""Activations in 8 bits at their edges: waits that run out, the border of a type's range, the shares of the weight gradient."""
import pytest
import torch

DEV = "cuda"


@pytest.mark.gpu
def test_a_wait_that_ran_out_is_reported():
    """A rehearsal: a wait that nothing ends sets the error 2 s later, without a synchronisation of the caller's; then
    grad_weight8 and a packed layer's backward refuse, and the layer keeps its words, until the error is cleared."""
    import concord_b200
    from concord_b200 import ConcordLinearPackedB, _abi, grad_weight8, save8
    lib = _abi.load()
    torch.manual_seed(0)
    x, dy = (torch.randint(-9, 10, (200, n), device=DEV).bfloat16() for n in (96, 64))
    s = save8(x)
    want = grad_weight8(dy, s)
    lay = ConcordLinearPackedB(96, 64, bias=False, device=DEV, lr=1e-2)
    lay.load_weights(torch.randn(64, 96, device=DEV) * 0.05)
    lay.save8 = True
    y = lay(x.clone().requires_grad_())
    words = lay.packed_w.clone()
    word = lib.concord_gemm_dw8_error_word()
    assert word[0] == 0 and concord_b200.gemm_dw8_error() == 0
    try:
        assert lib.concord_gemm_dw8_wait_check(torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert word[0] == 99 and concord_b200.gemm_dw8_error() == 99
        with pytest.raises(RuntimeError, match="a wait inside an earlier weight gradient's kernel ran out .code 99."):
            grad_weight8(dy, s)
        with pytest.raises(RuntimeError, match="ran out"):
            y.backward(dy)
        assert torch.equal(lay.packed_w, words)
        assert lib.concord_gemm_dw8_wait_check(None) == -8
        assert concord_b200.attention_error() == 0           # (its word is its own)
    finally:
        assert concord_b200.gemm_dw8_error(reset=True) == 99
    assert word[0] == 0 and concord_b200.gemm_dw8_error() == 0
    assert torch.equal(grad_weight8(dy, s), want)
    word[0] = 5                          # another program's handler, or a kernel, wrote the host's word alone
    try:
        with pytest.raises(RuntimeError, match="code 5"):
            grad_weight8(dy, s)
    finally:
        assert concord_b200.gemm_dw8_error(reset=True) == 5
    assert torch.equal(grad_weight8(dy, s), want)


@pytest.mark.gpu
def test_copies_of_a_pair_land():
    """The rehearsal's CTAs stop after 3 and 3 stages, 7 and 3, 3 and 8: what each has sent lands, or the code is 98."""
    import concord_b200
    from concord_b200 import _abi
    lib = _abi.load()
    torch.zeros(1, device=DEV)
    try:
        assert lib.concord_gemm_dw8_wait_check(torch.cuda.current_stream().cuda_stream) == 0
    finally:
        assert concord_b200.gemm_dw8_error(reset=True) == 99


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_top_and_bottom_of_the_range(dtype):
    """Exactly the documented values: above 127 steps of the last block that is whole, codes end at 63 (less than one step
    off); steps are 2^-126 at least."""
    from concord_b200 import save8
    top = 9 if dtype == torch.float16 else 121
    info = torch.finfo(dtype)
    border = torch.tensor(127.0 * 2.0 ** top, dtype=dtype, device=DEV)           # (exact in each type)
    assert float(border) == 127 * 2.0 ** top
    above = torch.nextafter(border, torch.tensor(float("inf"), device=DEV, dtype=dtype))
    x = torch.zeros(64, 4, dtype=dtype, device=DEV)
    x[:32, 0], x[:32, 1], x[:32, 2] = border, above, -info.max
    x[1:32] *= torch.linspace(0.01, 1, 31, device=DEV)[:, None].to(dtype)
    x[32:, 3] = info.max
    kept = save8(x).dense().double()
    step = torch.tensor([2.0 ** top] + 3 * [2.0 ** (top + 1)], dtype=torch.float64, device=DEV)
    ends = torch.tensor([127.0, 63.0, 63.0, 63.0], dtype=torch.float64, device=DEV)
    want = (x.double() / step).round().clamp(-ends, ends) * step
    assert torch.equal(kept, want)
    off = (kept - x.double()).abs()
    assert bool((off[:, 1:] < step[1:]).all()) and bool((off[:, 0] <= step[0] / 2).all())
    if dtype == torch.float16:
        assert float(kept[0, 2]) == -64512 and float(off[0, 2]) == 992
        return
    small = torch.tensor([126.0, 2.5, 0.75, 0.5, 2.0 ** -7, 0.0], device=DEV).repeat(32, 1) * 2.0 ** -126     # a step is 2^-126
    got = save8(small.to(dtype)).dense(torch.float32)[0] * 2.0 ** 126
    assert got.tolist() == [126.0, 2.0, 1.0, 0.0, 0.0, 0.0]


def test_error_word_without_a_device():
    """No device: no word, and nothing that crashes."""
    from concord_b200 import _abi, build
    build.build()
    lib = _abi.load()
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    assert lib.concord_gemm_dw8_error(0) == -1 and not lib.concord_gemm_dw8_error_word()
    assert lib.concord_gemm_dw8_wait_check(None) < 0
