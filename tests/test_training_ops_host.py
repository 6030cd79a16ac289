"""CPU-only checks of the training operators: the extension builds and loads,
arguments are refused before anything reaches a device, sizes of workspaces, and
the measured cases' definitions."""
import random

import pytest
import torch


@pytest.fixture(scope="module")
def built():
    from concord_b200 import build
    build.build()
    return build


def test_extension_loads_and_offers_the_operators(built):
    from concord_b200 import _ops
    native = _ops.native()
    for name in ("layer_norm", "distill_loss", "distill_loss_and_grad", "attention"):
        assert callable(getattr(native, name))


def test_cpu_tensors_are_refused(built):
    import concord_b200 as c
    x = torch.zeros(4, 8)
    for call in (lambda: c.layer_norm(x), lambda: c.distill_loss(x, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2)),
                 lambda: c.distill_loss_and_grad(x, torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2)),
                 lambda: c.packed_attention(*(torch.zeros(4, 1, 8, dtype=torch.bfloat16) for _ in range(3)),
                                            torch.tensor([0, 4]))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(TypeError, match="x must be a tensor"):
        c.layer_norm([1.0])


def test_c_entries_refuse_bad_arguments(built):
    """Status codes, not crashes, and nothing launched: these all return before the first CUDA call."""
    import ctypes

    from concord_b200 import _abi
    lib = _abi.load()
    p = _abi.DistillParams(temperature=1.0, alpha=1.0, grad_scale=1.0)
    one = ctypes.c_void_p(16)

    def loss(N=4, V=8, K=2, ldz=8, kind=0, params=p, ws=one, nbytes=10 ** 6, z=one):
        return lib.concord_distill_loss(params, z, kind, ldz, one, one, None, one, None, None, None, N, V, K, ws, nbytes, None)
    assert loss(V=0) == -2 and loss(ldz=7) == -2 and loss(K=0) == -2
    assert loss(K=513) == -7 and loss(kind=3) == -1 and loss(params=None) == -1 and loss(z=None) == -1
    assert loss(nbytes=8) == -4 and loss(ws=None) == -4
    assert loss(params=_abi.DistillParams(temperature=0.0)) == -1
    assert lib.concord_distill_workspace_bytes(10) == 128 * 4 + 80

    assert lib.concord_layer_norm_fwd(one, 0, 8, None, None, one, 5, None, None, 4, 8, 1e-5, None) == -1
    assert lib.concord_layer_norm_fwd(one, 0, 7, None, None, one, 0, None, None, 4, 8, 1e-5, None) == -2
    assert lib.concord_layer_norm_fwd(one, 0, 20000, None, None, one, 0, None, None, 4, 20000, 1e-5, None) == -7
    assert lib.concord_layer_norm_fwd(None, 0, 8, None, None, one, 0, None, None, 4, 8, 1e-5, None) == -1
    assert lib.concord_layer_norm_fwd(one, 0, 8, None, None, one, 0, one, None, 4, 8, 1e-5, None) == -1
    assert lib.concord_layer_norm_fwd(one, 0, 8, None, None, one, 0, None, None, 0, 8, 1e-5, None) == 0

    def attend(o=one, q=one, ts=64, **kw):
        a = dict(cu_q=16, cu_k=16, seqs=1, tokens_q=4, tokens_k=4, heads=2, kv_heads=1, head_dim=32, type=_abi.BF16,
                 causal=1, scale=0.1)
        a.update(kw)
        return lib.concord_attention_fwd(_abi.AttentionParams(**a), q, ts, 32, one, 32, 32, one, 32, 32, o, None, one, None)
    assert attend(type=_abi.F32) == -1 and attend(kv_heads=3) == -2 and attend(head_dim=36) == -2
    assert attend(head_dim=136) == -2 and attend(scale=0.0) == -1 and attend(seqs=0) == -2 and attend(cu_q=None) == -1
    assert attend(q=ctypes.c_void_p(8)) == -3 and attend(ts=65) == -3 and attend(ts=0) == -2 and attend(o=None) == -1
    assert attend(tokens_k=0) == -2 and attend(tokens_q=0) == 0 and attend(tokens_q=2 ** 31) == -2
    assert b"concord_attention_fwd" in lib.concord_last_error()


def test_measured_cases():
    from perf import operators as M
    cases = M.listed()
    assert 4 <= len(cases) <= 12 and len({c["name"] for c in cases}) == len(cases)
    most = {op: max(M.work(c)["flops"] for c in cases if c["op"] == op) for op in ("norm", "distill", "attend")}
    rng = random.Random(5)
    for c in cases + [M.draw(rng) for _ in range(200)]:
        w = M.work(c)
        assert w["bytes"] > 0 and w["flops"] > 0 and w["flops"] <= 1.05 * most[c["op"]]
        if c["op"] == "attend":
            lens = M._lengths(c)
            assert sum(lens) == c["total"] and min(lens) >= 0 and len(lens) == c["seqs"]
