"""packed_attention against a 64-bit implementation, forward and backward.

Tolerances, element by element, u being the operands' unit (2^-8 for bf16,
2^-10 for fp16: twice the largest rounding error): an output is rounded once
(u |result| at most), and the probabilities, or their gradients, are rounded
to the operands' type before they are summed (u / 2 times the sum of the
magnitudes that the product adds up, at most).  The fp32 arithmetic before
that (scores of magnitude S in base 2: S 2^-23 relative in p; sums) is under
u / 8 of the same magnitudes for every input here; u times the magnitudes is
granted in all.  delta carries the same errors as dp, summed over the row.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}


def reference(q, k, v, do, cu, cuk, causal, scale):
    """Outputs, gradients and the magnitudes that their sums add up, in 64 bits."""
    T, H, D = q.shape
    Tk, Hk, _ = k.shape
    f = dict(dtype=torch.float64, device=q.device)
    out = dict(o=torch.zeros(T, H, D, **f), lse=torch.zeros(H, T, **f), dq=torch.zeros(T, H, D, **f),
               dk=torch.zeros(Tk, Hk, D, **f), dv=torch.zeros(Tk, Hk, D, **f))
    mag = {n: torch.zeros_like(x) for n, x in out.items()}
    cu, cuk = cu.tolist(), cuk.tolist()
    for b in range(len(cu) - 1):
        i, j = slice(cu[b], cu[b + 1]), slice(cuk[b], cuk[b + 1])
        n, m = cu[b + 1] - cu[b], cuk[b + 1] - cuk[b]
        if n == 0:
            continue
        see = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril_(m - n)
        for h in range(H):
            g = h // (H // Hk)
            Q, K, V, G = q[i, h].double(), k[j, g].double(), v[j, g].double(), do[i, h].double()
            s = ((Q @ K.T) * scale).masked_fill(~see, -math.inf)
            lse = torch.logsumexp(s, 1) if m else torch.full((n,), -math.inf, **f)
            p = torch.where(see, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[:, None]), 0.0)
            o = p @ V
            dp = G @ V.T
            delta = (G * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            out["o"][i, h], out["lse"][h, i] = o, lse
            out["dq"][i, h] = scale * ds @ K
            out["dk"][j, g] += scale * ds.T @ Q
            out["dv"][j, g] += p.T @ G
            a = p * (dp.abs() + delta.abs() + (p * dp.abs()).sum(1, keepdim=True))
            mag["o"][i, h] = p @ V.abs()
            mag["dq"][i, h] = scale * a @ K.abs()
            mag["dk"][j, g] += scale * a.T @ Q.abs()
            mag["dv"][j, g] += p.T @ G.abs()
    return out, mag


def close(name, got, ref, mag, u):
    err = (got.double() - ref).abs()
    lim = u * (ref.abs() + mag) + 1e-7
    bad = ~(err <= lim)
    assert not bool(bad.any()), (name, int(bad.sum()), float((err / lim)[bad].max()))


def inputs(T, H, Hk, D, dtype=torch.bfloat16, Tk=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
    Tk = T if Tk is None else Tk
    return r(T, H, D), r(Tk, Hk, D), r(Tk, Hk, D), r(T, H, D)


def cum(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(DEV)


def run(q, k, v, do, cu, cuk=None, causal=True, scale=None):
    from concord_b200 import _abi, packed_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o, lse = packed_attention(*leaves, cu, cuk, causal=causal, scale=scale, return_lse=True)
    grads = torch.autograd.grad(o, leaves, do)
    torch.cuda.synchronize()
    assert _abi.load().concord_attention_error(0) == 0
    return dict(o=o.detach(), lse=lse, dq=grads[0], dk=grads[1], dv=grads[2])


def check(q, k, v, do, cu, cuk=None, causal=True, scale=None):
    got = run(q, k, v, do, cu, cuk, causal, scale)
    ref, mag = reference(q, k, v, do, cu, cu if cuk is None else cuk, causal, scale or q.shape[-1] ** -0.5)
    u = U[q.dtype]
    for name in ("o", "dq", "dk", "dv"):
        assert got[name].dtype == q.dtype
        close(name, got[name], ref[name], mag[name], u)
    fin = ref["lse"].isfinite()
    assert torch.equal(fin, got["lse"].isfinite())
    assert bool((got["lse"][fin].double() - ref["lse"][fin]).abs().max() <= 1e-4 if bool(fin.any()) else True)
    return got


# lengths of one and none, around the tiles of 128 and 256 rows, and several of them
@pytest.mark.parametrize("lens", [[1], [2, 1, 1], [127], [128], [129], [255, 1], [256, 257], [0, 5, 0, 0, 300, 0],
                                  [640], [64] * 37, [1] * 70, [1000, 3, 513], [1, 0, 2, 5] * 90,
                                  [0] * 300 + [140, 3]])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(lens, causal):
    check(*inputs(sum(lens), 2, 2, 64, seed=len(lens)), cum(lens), causal=causal)


@pytest.mark.parametrize("D", [8, 32, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize("dtype", list(U))
def test_head_sizes_and_types(D, dtype):
    check(*inputs(450, 2, 1, D, dtype, seed=D), cum([300, 150]))


@pytest.mark.parametrize("H,Hk", [(1, 1), (6, 6), (8, 2), (5, 1), (12, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_heads(H, Hk, D):
    check(*inputs(333, H, Hk, D, seed=H * Hk), cum([200, 133]))


def test_shared_heads_in_uneven_parts():
    """Five query heads of one key head, at 110 key blocks: parts of two, two and one."""
    from concord_b200 import _abi
    lens = [128] * 100 + [1, 0, 127, 300, 90, 130, 128, 60]
    q, k, v, do = inputs(sum(lens), 5, 1, 64, seed=11)
    p = _abi.AttentionParams(cu_q=1, cu_k=1, seqs=1, tokens_q=len(q), tokens_k=len(k), heads=5, kv_heads=1, head_dim=64,
                             type=_abi.BF16, causal=1, scale=1.0)
    assert _abi.load().concord_attention_bwd_workspace_bytes(p) == 3 * 2 * len(k) * 64 * 4
    check(q, k, v, do, cum(lens))


@pytest.mark.parametrize("lq,lk", [([5], [400]), ([400], [5]), ([130, 1, 300], [77, 500, 140]), ([0, 7], [9, 0]),
                                   ([1, 1, 1], [1000, 129, 0]), ([300, 20], [300, 700])])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_other_lengths(lq, lk, causal):
    """Cross attention, a later chunk of a prompt, queries that see no key."""
    q, k, v, do = inputs(sum(lq), 4, 2, 64, Tk=sum(lk), seed=7)
    got = check(q, k, v, do, cum(lq), cum(lk), causal=causal)
    if causal and lq == [400]:
        assert bool((got["o"][:395] == 0).all()) and bool((got["lse"][:, :395] == -math.inf).all())
        assert bool((got["dq"][:395] == 0).all())


def test_no_keys_and_no_queries():
    q, k, v, do = inputs(10, 2, 2, 64, Tk=0)
    got = run(q, k, v, do, cum([4, 6]), cum([0, 0]))
    assert bool((got["o"] == 0).all()) and bool((got["lse"] == -math.inf).all()) and bool((got["dq"] == 0).all())
    q, k, v, do = inputs(0, 2, 2, 64, Tk=9)
    got = run(q, k, v, do, cum([0, 0]), cum([4, 5]))
    assert got["o"].shape == (0, 2, 64) and bool((got["dk"] == 0).all()) and bool((got["dv"] == 0).all())


def test_strides():
    """Views of one projection, heads before tokens, every other token, broadcast heads, rows off 16 bytes."""
    T, H, D = 300, 4, 64
    cu = cum([170, 130])
    g = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    qkv = r(T, 3, H, D)
    do = r(T, H, D)
    want = run(*(qkv[:, i].contiguous() for i in range(3)), do, cu)

    def same(q, k, v, do):
        got = run(q, k, v, do, cu)
        assert all(torch.equal(got[n], want[n]) for n in want)
    same(qkv[:, 0], qkv[:, 1], qkv[:, 2], do)
    heads = qkv.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3)        # [3, H, T, D] in memory
    same(heads[:, 0], heads[:, 1], heads[:, 2], do.transpose(0, 1).contiguous().transpose(0, 1))
    apart = torch.stack([qkv, qkv * 0 + float("nan")], 1).flatten(0, 1)[::2]
    same(apart[:, 0], apart[:, 1], apart[:, 2], do)
    odd = torch.empty(T * 3 * H * D + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, 3, H, D).copy_(qkv)
    same(odd[:, 0], odd[:, 1], odd[:, 2], do)
    apart = torch.zeros(T, 3, H, D + 3, dtype=torch.bfloat16, device=DEV)
    apart[..., :D] = qkv
    same(apart[:, 0, :, :D], apart[:, 1, :, :D], apart[:, 2, :, :D], do)
    one = qkv[:, 1, :1].expand(T, H, D)                                      # one head shown as four
    a = run(qkv[:, 0], one, one, do[:, :1].expand(T, H, D), cu)
    b = run(qkv[:, 0], one.contiguous(), one.contiguous(), do[:, :1].repeat(1, H, 1), cu)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_neighbours_and_gaps_may_hold_anything(causal, D):
    """Rows of no sequence (before, after) are NaN, and so is a whole neighbouring sequence: the others' results
    are what they are without them, and rows of no sequence give zeros."""
    lens = [150, 40, 201]
    q, k, v, do = inputs(sum(lens), 2, 1, D, seed=5)
    want = run(q, k, v, do, cum(lens), causal=causal)
    pad = 23

    def wrapped(t):
        x = torch.full((pad + t.shape[0] + 60, *t.shape[1:]), float("nan"), dtype=t.dtype, device=DEV)
        x[pad:pad + t.shape[0]] = t
        return x
    cu = cum(lens) + pad
    got = run(*(wrapped(t) for t in (q, k, v, do)), cu, causal=causal)
    for n in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[n][pad:-60], want[n]), n
        assert bool((got[n][:pad] == 0).all()) and bool((got[n][-60:] == 0).all()), n
    assert torch.equal(got["lse"][:, pad:-60], want["lse"])
    bad = [t.clone() for t in (q, k, v, do)]
    for t in bad:
        t[150:190] = float("inf")
    got = run(*bad, cum(lens), causal=causal)
    for n in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[n][:150], want[n][:150]) and torch.equal(got[n][190:], want[n][190:]), n


def test_hidden_keys_may_be_infinite():
    """A key that a query does not see weighs nothing, whatever its scores are."""
    q, k, v, do = inputs(200, 1, 1, 64, seed=6)
    want = run(q, k, v, do, cum([200]))
    k2 = k.clone()
    k2[150] = float("nan")
    got = run(q, k2, v, do, cum([200]))
    assert torch.equal(got["o"][:150], want["o"][:150]) and torch.equal(got["lse"][:, :150], want["lse"][:, :150])
    assert bool(got["o"][150:].isnan().all())


def test_large_scores_and_scales():
    q, k, v, do = inputs(300, 2, 2, 64, seed=8)
    check(q, k, v, do, cum([300]), scale=0.01)
    check(q * 4, k, v, do, cum([300]), scale=0.3)
    # scores of +-1000 and more: the running maximum moves far, nothing overflows
    big = run(q * 16, k * 4, v, do, cum([300]))
    assert all(bool(t.isfinite().all()) for t in big.values())
    # rising scores: the maximum moves in every key block
    rise = (torch.arange(700, device=DEV) / 20.0)[:, None, None] * torch.ones(1, 1, 64, device=DEV)
    q, k, v, do = inputs(700, 1, 1, 64, seed=9)
    check(torch.ones_like(q), rise.bfloat16(), v, do, cum([700]), causal=False, scale=0.02)
    check(torch.ones_like(q), rise.flip(0).bfloat16(), v, do, cum([700]), causal=False, scale=0.02)


def test_int64_bounds_and_bounds_outside_the_tensor():
    q, k, v, do = inputs(100, 1, 1, 64)
    a, b = run(q, k, v, do, cum([60, 40])), run(q, k, v, do, cum([60, 40]).long())
    assert all(torch.equal(a[n], b[n]) for n in a)
    over = torch.tensor([0, 60, 1000], dtype=torch.int32, device=DEV)      # clamped to the tensors
    c = run(q, k, v, do, over)
    assert all(torch.equal(a[n], c[n]) for n in a)


def test_same_bits_every_time_and_on_another_stream():
    q, k, v, do = inputs(3000, 4, 2, 128, seed=2)
    cu = cum([1100, 900, 1000])
    first = run(q, k, v, do, cu)
    with torch.cuda.stream(torch.cuda.Stream()):
        second = run(q, k, v, do, cu)
    assert all(torch.equal(first[n], second[n]) for n in first)


def test_long_sequence():
    """More key blocks than the rings have slots, and a token offset of 2^31 elements and more in a strided view."""
    check(*inputs(2300, 1, 1, 128, seed=1), cum([2300]))
    T, wide = 2200, 1 << 20                                                # 2200 x 2^20 elements: 4.6 GB
    far = torch.empty(T, wide, dtype=torch.bfloat16, device=DEV)
    q, k, v, do = inputs(T, 1, 1, 64, seed=4)
    want = run(q, k, v, do, cum([T]))
    for i, t in enumerate((q, k, v, do)):
        far[:, i * 64:(i + 1) * 64] = t[:, 0]
    got = run(*(far[:, None, i * 64:(i + 1) * 64] for i in range(4)), cum([T]))
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_gradient_against_differences():
    """Central differences of the 64-bit formula along random directions, against the kernel's gradients: the step's
    error h^2 and the kernel's rounding, summed over the direction as independent errors of at most u times the
    magnitudes (four standard deviations of them)."""
    q, k, v, do = inputs(90, 2, 1, 64, seed=10)
    cu = cum([50, 40])
    got = run(q, k, v, do, cu)
    _, mag = reference(q, k, v, do, cu, cu, True, 0.125)
    for i, name in enumerate(("dq", "dk", "dv")):
        u = torch.randn(q.shape if i == 0 else k.shape, device=DEV).double()
        u /= u.norm()
        h = 1e-4

        def at(s):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + s * u
            return (reference(*x, do, cu, cu, True, 0.125)[0]["o"] * do.double()).sum()
        diff = float((at(h) - at(-h)) / (2 * h))
        rounding = U[q.dtype] * float(((mag[name] + got[name].double().abs()) * u).norm())
        assert abs(diff - float((got[name].double() * u).sum())) <= 4 * rounding + 1e-5, name


def test_captured_in_a_graph():
    from concord_b200 import packed_attention
    q, k, v, do = inputs(300, 2, 2, 64)
    cu = cum([100, 200])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]

    def once():
        o = packed_attention(*leaves, cu)
        return (o,) + torch.autograd.grad(o, leaves, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = once()
        cu.copy_(cum([250, 50]))                   # other lengths, the same graph
        g.replay()
        eager = once()
    torch.cuda.synchronize()
    assert all(torch.equal(p, r) for p, r in zip(out, eager))


def test_refusals():
    from concord_b200 import packed_attention as f
    q, k, v, _ = inputs(20, 4, 2, 64)
    cu = cum([20])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        f(q, k, v, cu.cpu())
    with pytest.raises(TypeError, match="q must be"):
        f(q.float(), k.float(), v.float(), cu)
    with pytest.raises(TypeError, match="k must have q's type"):
        f(q, k.half(), v, cu)
    with pytest.raises(ValueError, match=r"\[T, H, D\]"):
        f(q[None], k, v, cu)
    with pytest.raises(ValueError, match="multiple of k's"):
        f(q[:, :3], k, v, cu)
    with pytest.raises(ValueError, match="multiple of 8"):
        f(q[..., :60], k[..., :60], v[..., :60], cu)
    with pytest.raises(ValueError, match="multiple of 8"):
        f(*(torch.zeros(20, 2, 136, dtype=torch.bfloat16, device=DEV) for _ in range(3)), cu)
    with pytest.raises(TypeError, match="cu_seqlens must be"):
        f(q, k, v, cu.float())
    with pytest.raises(ValueError, match="B >= 1"):
        f(q, k, v, cu[:1])
    with pytest.raises(ValueError, match="one length"):
        f(q, k, v, cu, cum([10, 10]))
    with pytest.raises(ValueError, match="pass cu_seqlens_k"):
        f(q, k[:10], v[:10], cu)
    with pytest.raises(ValueError, match="scale"):
        f(q, k, v, cu, scale=-1.0)
