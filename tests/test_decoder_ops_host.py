"""CPU-only checks of the decoder's operators: the extension offers them, arguments are refused before anything reaches a
device, sizes of workspaces and saved forms, the shares of the weight gradient's tiles, the measured cases."""
import ctypes
import random

import pytest
import torch

ONE = ctypes.c_void_p(64)


@pytest.fixture(scope="module")
def lib():
    from concord_b200 import _abi, build
    build.build()
    return _abi.load()


def test_extension_offers_the_operators(lib):
    from concord_b200 import _ops
    for name in ("embedding", "qk_norm_rope", "save8", "dense8", "grad_weight8", "gated_unit"):
        assert callable(getattr(_ops.native(), name))


def test_cpu_tensors_are_refused(lib):
    import concord_b200 as c
    x = torch.zeros(4, 8)
    for call in (lambda: c.embedding(torch.zeros(2, dtype=torch.long), x), lambda: c.qk_norm_rope(x[None], None),
                 lambda: c.save8(x), lambda: c.gated_unit(x, x)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(TypeError, match="must be a tensor"):
        c.embedding([1], x)
    with pytest.raises(TypeError, match="must be a Saved8"):
        c.grad_weight8(x, x)


def test_tables_stay_in_fp32():
    from concord_b200 import QKNormRope, rope_tables
    m = torch.nn.Sequential(QKNormRope(64, 100, rot=32))
    want = rope_tables(100, 32, device="cpu")
    for cast in (lambda: m.bfloat16(), lambda: m.half(), lambda: m.to(torch.float64), lambda: m.float()):
        cast()
        assert torch.equal(m[0].cos, want[0]) and torch.equal(m[0].sin, want[1]) and m[0].cos.dtype == torch.float32
    assert m.half()[0].q_weight.dtype == torch.float16 and sorted(m.state_dict()) == ["0.k_weight", "0.q_weight"]


def test_embedding_from_a_table():
    from concord_b200 import Embedding
    w = torch.randn(7, 5)
    m = Embedding.from_pretrained(w, padding_idx=-1, scale=2.0)
    assert m.weight.data_ptr() == w.data_ptr() and torch.equal(m.weight, w) and not m.weight.requires_grad
    assert (m.num_embeddings, m.embedding_dim, m.padding_idx, m.scale) == (7, 5, 6, 2.0)
    assert Embedding.from_pretrained(w, freeze=False).weight.requires_grad
    with pytest.raises(ValueError, match=r"must be \[V, D\]"):
        Embedding.from_pretrained(w[0])


def test_layers_pickled_before_there_was_save8():
    from concord_b200 import ConcordLinearPackedB
    lay = ConcordLinearPackedB.__new__(ConcordLinearPackedB)          # (as unpickling makes them)
    torch.nn.Module.__init__(lay)
    assert lay.save8 is False
    lay.save8 = True
    assert lay.save8 and not ConcordLinearPackedB.save8


def test_embedding_entries_refuse(lib):
    def forward(ids=ONE, w=ONE, wt=0, ldw=8, yt=0, T=4, V=5, D=8):
        return lib.concord_embedding_fwd(ids, 1, w, wt, ldw, ONE, yt, T, V, D, 1.0, None)
    assert forward(wt=3) == -1 and forward(yt=-1) == -1 and forward(ids=None) == -1 and forward(w=None) == -1
    assert forward(ldw=7) == -2 and forward(V=0) == -2 and forward(D=0) == -2 and forward(T=-1) == -2
    assert forward(T=2 ** 30 + 1) == -7 and forward(V=2 ** 31) == -7 and forward(D=2 ** 21, ldw=2 ** 21) == -7
    assert forward(T=0) == 0
    size = lib.concord_embedding_bwd_workspace_bytes(100, 5, 8)
    assert size > 2 * 100 * 8 and lib.concord_embedding_bwd_workspace_bytes(0, 5, 8) == 0
    assert lib.concord_embedding_bwd_workspace_bytes(2 ** 31, 5, 8) == 0

    def backward(dy=ONE, ld=8, dw=ONE, T=100, ws=ONE, nbytes=size):
        return lib.concord_embedding_bwd(ONE, 0, dy, 0, ld, dw, 0, T, 5, 8, 1.0, -1, ws, nbytes, None)
    assert backward(dy=None) == -1 and backward(dw=None) == -1 and backward(ld=4) == -2
    assert backward(ws=None) == -4 and backward(nbytes=size - 1) == -4 and backward(ws=ctypes.c_void_p(8)) == -4


def test_rotation_entries_refuse(lib):
    from concord_b200 import _abi

    def forward(q=ONE, k=ONE, out=ONE, ts=64, **kw):
        a = dict(cos=64, sin=64, pos=None, tokens=4, heads=2, kv_heads=1, head_dim=32, rot=32, positions=10, type=0, norm=1, eps=0.1)
        a.update(kw)
        return lib.concord_qk_norm_rope_fwd(_abi.QKParams(**a), q, ts, 32, k, 32, 32, None, None, out, out, None)
    assert lib.concord_qk_norm_rope_fwd(None, ONE, 64, 32, ONE, 32, 32, None, None, ONE, ONE, None) == -1
    assert forward(type=3) == -1 and forward(eps=-1.0) == -1 and forward(eps=float("nan")) == -1 and forward(cos=None) == -1
    assert forward(rot=31) == -2 and forward(rot=34) == -2 and forward(heads=0, kv_heads=0) == -2 and forward(positions=0) == -2
    assert forward(head_dim=257) == -7 and forward(heads=2 ** 17) == -7 and forward(tokens=2 ** 31) == -7
    assert forward(q=None) == -1 and forward(k=None) == -1 and forward(out=None) == -1 and forward(ts=-1) == -2
    assert forward(tokens=0) == 0
    p = _abi.QKParams(tokens=4, heads=2, kv_heads=1, head_dim=32, norm=1)
    size = lib.concord_qk_norm_rope_bwd_workspace_bytes(p)
    assert size >= 32 * 4 and lib.concord_qk_norm_rope_bwd_workspace_bytes(_abi.QKParams(tokens=4, heads=2, head_dim=32)) == 0

    def backward(dy=ONE, x=ONE, ws=ONE, nbytes=size, norm=1):
        p = _abi.QKParams(tokens=4, heads=2, kv_heads=1, head_dim=32, norm=norm)
        return lib.concord_qk_norm_rope_bwd(p, x, 64, 32, x, 32, 32, None, None, dy, 64, 32, dy, 32, 32, ONE, ONE, ONE, ONE, ws,
                                            nbytes, None)
    assert backward(dy=None) == -1 and backward(x=None) == -1 and backward(ws=None) == -4 and backward(nbytes=size - 1) == -4


def test_saved_entries_refuse(lib):
    assert lib.concord_saved8_bytes(64, 128) == 64 * 128 + 256 and lib.concord_saved8_bytes(1, 1) == 66 * 16
    assert lib.concord_saved8_bytes(65, 130) == 2 * 66 * 144 and lib.concord_saved8_bytes(0, 5) == 0
    assert lib.concord_saved8_bytes(5, 2 ** 21) == 0

    def save(x=ONE, t=0, ld=8, out=ONE, M=4, K=8):
        return lib.concord_save8(x, t, ld, out, M, K, None)
    assert save(x=None) == -1 and save(out=None) == -1 and save(t=3) == -1 and save(ld=7) == -2 and save(K=0) == -2
    assert save(M=-1) == -2 and save(K=2 ** 21, ld=2 ** 21) == -7 and save(out=ctypes.c_void_p(48)) == -3 and save(M=0) == 0
    assert lib.concord_dense8(None, ONE, 0, 8, 4, 8, None) == -1 and lib.concord_dense8(ONE, ONE, 0, 4, 4, 8, None) == -2

    size = lib.concord_gemm_dw8_workspace_bytes(4096, 64, 64)          # one tile, cut
    assert size > 0 and lib.concord_gemm_dw8_workspace_bytes(64, 64, 64) == 0 and lib.concord_gemm_dw8_workspace_bytes(0, 8, 8) == 0

    def dw(dy=ONE, ld=64, s=ONE, out=ONE, M=4096, N=64, K=64, ws=ONE, nbytes=size):
        return lib.concord_gemm_dw8(dy, ld, s, out, M, N, K, ws, nbytes, None)
    assert dw(dy=None) == -1 and dw(s=None) == -1 and dw(out=None) == -1 and dw(N=60) == -2 and dw(ld=60) == -2 and dw(ld=68) == -2
    assert dw(M=-1) == -2 and dw(K=2 ** 21) == -7 and dw(M=2 ** 31) == -7 and dw(nbytes=size - 1) == -4 and dw(ws=None) == -4
    assert dw(dy=ctypes.c_void_p(8)) == -3 and dw(s=ctypes.c_void_p(48)) == -3

    def gated(gate=ONE, h=ONE, t=0, act=0, ld=8, M=4, K=8, s=None):
        return lib.concord_gated_fwd(gate, ld, ONE, 8, t, act, h, s, s, None, M, K, None)
    assert gated(gate=None) == -1 and gated(h=None) == -1 and gated(t=5) == -1 and gated(act=2) == -1 and gated(ld=7) == -2
    assert gated(s=ctypes.c_void_p(16)) == -3 and gated(M=0) == 0

    def back(gate=ONE, up=ONE, sg=None, su=None, dh=ONE, ld=8):
        return lib.concord_gated_bwd(gate, ld, up, 8, sg, su, 0, 0, dh, 8, ONE, 8, ONE, 8, 4, 8, None)
    assert back(gate=None) == -1 and back(dh=None) == -1 and back(sg=ONE) == -1 and back(su=ONE) == -1 and back(ld=7) == -2


def _plan(tiles, stages, resident):
    """The shares that gemm8.cu's share_out and Pieces give, restated."""
    pairs = min(resident, max(tiles, tiles * stages // 4))
    rest = tiles % pairs
    full, cut = tiles - rest, (stages * rest + pairs - 1) // pairs
    if stages - cut <= 16:
        cut = stages
    helpers, ends = min(pairs - rest, rest * (stages - cut)), rest * (stages - cut)
    pieces = []
    for p in range(pairs):
        for t in range(p, full + rest, pairs):
            last = stages if t < full else cut
            pieces.append((t, 0, last, -1 if last == stages else t - full))
        h = p - rest
        if 0 <= h < helpers:
            at, end = h * ends // helpers, (h + 1) * ends // helpers
            while at < end:
                j, off = divmod(at, stages - cut)
                stop = min(stages, cut + off + end - at)
                pieces.append((full + j, cut + off, stop, rest + j + h))
                at += stop - cut - off
    return pairs, pieces


def test_every_stage_of_every_tile_is_done_once():
    rng = random.Random(0)
    for _ in range(1500):
        tiles, stages = rng.choice([rng.randint(1, 12), rng.randint(1, 300)]), rng.choice([1, 2, 17, 18, rng.randint(1, 300)])
        pairs, pieces = _plan(tiles, stages, rng.choice([74, 72, 3, 1]))
        done = {}
        for t, a, b, slot in pieces:
            assert a < b
            done.setdefault(t, []).append((a, b, slot))
        slots = [p[3] for p in pieces if p[3] >= 0]
        assert len(set(slots)) == len(slots) and all(s < 2 * pairs for s in slots) and sorted(done) == list(range(tiles))
        for parts in done.values():
            parts.sort()
            assert parts[0][0] == 0 and parts[-1][1] == stages and all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
            # what the joining kernel goes by: the pieces behind the first stand side by side in the workspace
            assert [s for _, _, s in parts[1:]] == list(range(parts[1][2], parts[1][2] + len(parts) - 1)) if len(parts) > 1 else True


def test_measured_cases():
    from perf import more_operators as M
    cases = M.listed()
    assert 4 <= len(cases) <= 12 and len({c["name"] for c in cases}) == len(cases)
    most = {op: max(M.work(c)["flops"] for c in cases if c["op"] == op) for op in ("embed", "qk", "gated", "dw")}
    rng = random.Random(5)
    for c in cases + [M.draw(rng) for _ in range(200)]:
        w = M.work(c)
        assert w["bytes"] > 0 and w["flops"] > 0 and w["flops"] <= 1.05 * most[c["op"]]
        if c["op"] == "qk":
            lens = M._lengths(c)
            assert sum(lens) == c["tokens"] and min(lens) >= 1 and len(lens) == c["seqs"]
