"""packed_attention at the ends of its types' ranges, in layouts of one row or one head, and after a wait that ran
out.  Tolerances as in test_gpu_attention.py, with half of fp16's smallest number as the absolute part where results
are that small."""
import math

import pytest
import torch

from test_gpu_attention import DEV, U, check, cum, inputs, reference, run

pytestmark = pytest.mark.gpu


def close(name, got, ref, mag, u, least):
    err, lim = (got.double() - ref).abs(), u * (ref.abs() + mag) + least
    assert bool((err <= lim).all()), (name, float((err / lim).max()))


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("D", [64, 128])
def test_nan_reaches_all_that_depends_on_it(dtype, D):
    """Without a mask every query sees a key that is NaN, and every gradient hangs on their scores; a value that is
    NaN reaches what delta enters (dq, dk) but not dv."""
    q, k, v, do = inputs(200, 1, 1, D, dtype, seed=21)
    cu = cum([200])
    want = run(q, k, v, do, cu, causal=False)
    bad = k.clone()
    bad[50] = math.nan
    got = run(q, bad, v, do, cu, causal=False)
    assert all(bool(got[n].isnan().all()) for n in got)
    bad = v.clone()
    bad[50, 0, 0] = math.nan
    got = run(q, k, bad, do, cu, causal=False)
    assert bool(got["dq"].isnan().all()) and bool(got["dk"].isnan().all())
    assert torch.equal(got["dv"], want["dv"]) and torch.equal(got["lse"], want["lse"])


@pytest.mark.parametrize("dtype", list(U))
def test_scores_beyond_two_to_the_31(dtype):
    """q and k of +-2^13, 64 wide: a query's own key scores 2^32 before scaling, every other at least 2^29 less, all
    exact in fp32."""
    g = torch.Generator(device=DEV).manual_seed(22)
    q = (torch.randint(0, 2, (150, 1, 64), generator=g, device=DEV) * 2 - 1).to(dtype) * 8192
    _, _, v, do = inputs(150, 1, 1, 64, dtype, seed=23)
    own = q[:, 0].double() @ q[:, 0].double().T
    own.fill_diagonal_(-math.inf)
    assert float(own.max()) < 2.0 ** 32 - 2.0 ** 29
    check(q, q.clone(), v, do, cum([150]), causal=False)


def test_fp16_gradients_of_small_upstream_gradients():
    """4096 keys, upstream gradients of 1e-5: a gradient of one score is of the size 2e-9, below what fp16 holds, and
    the sums of 4096 of them are not."""
    g = torch.Generator(device=DEV).manual_seed(24)
    n = 4096
    q, v = torch.randn(n, 1, 64, generator=g, device=DEV), torch.randn(n, 1, 64, generator=g, device=DEV)
    do = q * 1e-5
    q, v, do = q.half(), v.half(), do.half()
    k = v.clone()                            # sums that add up: dq follows do, dk follows v
    got = run(q, k, v, do, cum([n]), causal=False, scale=0.05)
    ref, mag = reference(q, k, v, do, cum([n]), cum([n]), False, 0.05)
    assert float(ref["dq"].abs().mean()) > 2.0 ** -22 and float(ref["dk"].abs().mean()) > 2.0 ** -22
    for name in ("o", "dq", "dk", "dv"):
        close(name, got[name], ref[name], mag[name], U[torch.float16], 2.0 ** -25)


@pytest.mark.parametrize("size", [1e-6, 1.0, 300.0])
@pytest.mark.parametrize("heads", [(2, 1), (1, 1)])
def test_fp16_gradients_of_any_size(size, heads):
    """Sequences whose upstream gradients and values differ by powers of ten, side by side."""
    lens = [300, 1, 0, 140, 500]
    q, k, v, do = inputs(sum(lens), *heads, 64, torch.float16, seed=25)
    do[:300] *= size
    v[301:441] *= 1e-3
    cu = cum(lens)
    for causal in (True, False):
        got = run(q, k, v, do, cu, causal=causal)
        ref, mag = reference(q, k, v, do, cu, cu, causal, 0.125)
        for name in ("o", "dq", "dk", "dv"):
            close(name, got[name], ref[name], mag[name], U[torch.float16], 2.0 ** -25)


def test_fp16_probabilities_of_a_million_keys():
    q, k, v, do = inputs(8, 1, 1, 64, torch.float16, Tk=1 << 20, seed=26)
    do = do * 64
    cu, cuk = cum([8]), cum([1 << 20])
    got = run(q, k, v, do, cu, cuk, causal=False)
    ref, mag = reference(q, k, v, do, cu, cuk, False, 0.125)
    for name in ("o", "dq", "dk", "dv"):
        close(name, got[name], ref[name], mag[name], U[torch.float16], 2.0 ** -25)


@pytest.mark.parametrize("dtype", list(U))
def test_extreme_neighbours_change_no_bit(dtype):
    """The range of one sequence is no other's: the same bits beside a sequence, or rows of none, of the largest
    numbers and of NaN."""
    q, k, v, do = inputs(300, 2, 1, 64, dtype, seed=27)
    do = do * 1e-4
    want = run(q[100:200], k[100:200], v[100:200], do[100:200], cum([100]))
    for value in (60000.0, math.nan):
        wild = [t.clone() for t in (q, k, v, do)]
        for t in wild:
            t[:100] = value
            t[200:] = -value
        for cu in (cum([100, 100, 100]), cum([100]) + 100):
            got = run(*wild, cu)
            assert all(torch.equal(got[n][100:200], want[n]) for n in ("o", "dq", "dk", "dv"))


@pytest.mark.parametrize("D", [64, 128])
def test_one_row_or_one_head_of_any_stride(D):
    """The stride of a dimension of size one says nothing."""
    g = torch.Generator(device=DEV).manual_seed(28)
    buf = torch.randn(4, 3000, generator=g, device=DEV).bfloat16()
    row = lambda i: buf.as_strided((1, 6, D), (1003, D, 1), 3000 * i)  # noqa: E731
    want = run(*(row(i).clone() for i in range(4)), cum([1]))
    got = run(*(row(i) for i in range(4)), cum([1]))
    assert all(torch.equal(got[n], want[n]) for n in want)
    head = lambda i: buf.as_strided((20, 1, D), (136, 3, 1), 3000 * i)  # noqa: E731
    want = run(*(head(i).clone(memory_format=torch.contiguous_format).view(20, 1, D) for i in range(4)), cum([15, 5]))
    got = run(*(head(i) for i in range(4)), cum([15, 5]))
    assert all(torch.equal(got[n], want[n]) for n in want)
    both = lambda i: buf.as_strided((1, 1, D), (5, 7, 1), 3000 * i)  # noqa: E731
    want = run(*(both(i).clone().view(-1).view(1, 1, D) for i in range(4)), cum([1]))
    got = run(*(both(i) for i in range(4)), cum([1]))
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_a_wait_that_ran_out_is_reported():
    """A rehearsal: a wait that nothing ends sets the error 2 s later, without a synchronisation of the caller's; then
    forward and backward refuse, until the error is cleared."""
    import concord_b200
    from concord_b200 import _abi, packed_attention
    lib = _abi.load()
    q, k, v, do = inputs(300, 2, 2, 64, seed=30)
    cu = cum([100, 200])
    want = run(q, k, v, do, cu)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = packed_attention(*leaves, cu)
    word = lib.concord_attention_error_word()
    assert word[0] == 0 and concord_b200.attention_error() == 0
    try:
        assert lib.concord_attention_wait_check(torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert word[0] == 99 and concord_b200.attention_error() == 99
        with pytest.raises(RuntimeError, match="a wait inside an earlier attention kernel ran out .code 99."):
            packed_attention(q, k, v, cu)
        with pytest.raises(RuntimeError, match="ran out"):
            torch.autograd.grad(o, leaves, do, retain_graph=True)
        assert lib.concord_attention_wait_check(None) == -8
    finally:
        assert concord_b200.attention_error(reset=True) == 99
    assert word[0] == 0 and concord_b200.attention_error() == 0
    again = run(q, k, v, do, cu)
    assert all(torch.equal(again[n], want[n]) for n in want)
    word[0] = 5                          # another program's handler, or a kernel, wrote the host's word alone
    try:
        with pytest.raises(RuntimeError, match="code 5"):
            packed_attention(q, k, v, cu)
    finally:
        assert concord_b200.attention_error(reset=True) == 5
    assert torch.equal(packed_attention(q, k, v, cu), want["o"])


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("lq,lk", [([400], [5]), ([300, 20], [20, 300]), ([260, 1, 700], [3, 0, 200]), ([1], [1000]),
                                   ([5, 7], [0, 400])])
def test_wide_heads_with_keys_of_other_lengths(dtype, lq, lk):
    """Heads of 128: pairs of query tiles of which the first, or both, see no key."""
    q, k, v, do = inputs(sum(lq), 4, 2, 128, dtype, Tk=sum(lk), seed=29)
    for causal in (True, False):
        check(q, k, v, do, cum(lq), cum(lk), causal=causal)


@pytest.mark.parametrize("Tk", [0, 30])
def test_rows_of_no_sequence_without_any_keys(Tk):
    """Sequences without keys, whether or not k holds rows of none: o 0 and lse -inf, and lse 0 outside of them."""
    q, k, v, do = inputs(40, 2, 1, 64, Tk=Tk, seed=31)
    cu = torch.tensor([3, 10, 10, 33], dtype=torch.int32, device=DEV)
    got = run(q, k, v, do, cu, torch.full((4,), Tk, dtype=torch.int32, device=DEV))
    assert all(bool((got[n] == 0).all()) for n in ("o", "dq", "dk", "dv"))
    want = torch.zeros(2, 40, device=DEV)
    want[:, 3:33] = -math.inf
    assert torch.equal(got["lse"], want)
