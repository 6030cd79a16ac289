"""The decoder on packed documents: embedding, norms, heads normed and turned, packed attention, gated unit and
activations in 8 bits, together around the packed layers."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _asked():
    """Bytes that tensors asked for (a block of the allocator may be up to 1 MB larger)."""
    return torch.cuda.memory_stats()["requested_bytes.all.current"]

SMALL = dict(vocab=300, d=128, n_layer=2, n_head=4, kv_heads=2, ffn=200)


def test_batches_are_whole_documents():
    import workloads
    gen = torch.Generator().manual_seed(0)
    ids, pos, labels, cu = workloads.packed_tokens(500, 40, 300, gen, DEV)
    bounds = sorted(set(cu.tolist()))
    assert bounds[0] == 0 and bounds[-1] == 500 and all(1 <= b - a <= 40 for a, b in zip(bounds, bounds[1:]))
    for a, b in zip(bounds, bounds[1:]):
        assert pos[a:b].tolist() == list(range(b - a))
        assert torch.equal(labels[a:b - 1], ids[a + 1:b]) and int(labels[b - 1]) == -100


def _plain_logits(m, idx):
    """One document through the same weights in torch's operations and 32 bits."""
    T = len(idx)
    x = m.emb.weight[idx] * m.emb.scale
    for b in m.blocks:
        norm = lambda t, ln: F.layer_norm(t, (t.shape[-1],), ln.weight, None, ln.eps)  # noqa: E731
        a = norm(x, b.attn_norm)
        q, k, v = (F.linear(a, lin.weight).view(T, -1, b.hd) for lin in (b.wq, b.wk, b.wv))
        heads = []
        for t, w in ((q, b.qk.q_weight), (k, b.qk.k_weight)):
            t = t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + b.qk.eps) * w
            lo, hi = t.chunk(2, -1)
            c, s = b.qk.cos[:T, None], b.qk.sin[:T, None]
            heads.append(torch.cat((lo * c - hi * s, lo * s + hi * c), -1))
        group = q.shape[1] // k.shape[1]
        q, k, v = heads[0].transpose(0, 1), heads[1].transpose(0, 1).repeat_interleave(group, 0), \
            v.transpose(0, 1).repeat_interleave(group, 0)
        score = (q @ k.transpose(1, 2)) * b.hd ** -0.5
        score = score.masked_fill(torch.ones(T, T, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
        y = (score.softmax(-1) @ v).transpose(0, 1).reshape(T, -1)
        x = x + F.linear(y, b.wo.weight)
        f = norm(x, b.ffn_norm)
        x = x + F.linear(F.silu(F.linear(f, b.w_gate.weight)) * F.linear(f, b.w_up.weight), b.w_down.weight)
    return F.linear(norm(x, m.norm), m.lm_head.weight)


def test_packed_model_matches_plain_operations():
    """bf16 inputs of every matrix product leave 2^-8 relative each; over two blocks and a head 32 of them are granted."""
    import workloads
    torch.manual_seed(0)
    m = workloads.PackedLlama(**SMALL, positions=64, device=DEV)
    for b in m.blocks:
        with torch.no_grad():
            b.qk.q_weight.uniform_(0.5, 1.5)
            b.qk.k_weight.uniform_(0.5, 1.5)
    lens = [40, 1, 64, 17]
    cu = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
    x = torch.randint(0, 300, (sum(lens),), device=DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(x, pos, cu).float()
    with torch.no_grad():
        for i, n in enumerate(lens):
            ref = _plain_logits(m, x[cu[i]:cu[i + 1]])
            err = (got[cu[i]:cu[i + 1]] - ref).norm() / ref.norm()
            assert float(err) <= 32 * 2.0 ** -8, (n, float(err))


def test_gradients_match_plain_operations():
    """Ordinary layers: every parameter's gradient beside that of plain operations in 32 bits, bf16's 2^-8 over twice as
    many products; gate and up kept in 8 bits add at most 2^-7 of their blocks' largest."""
    import workloads
    torch.manual_seed(1)
    m = workloads.PackedLlama(**SMALL, positions=64, device=DEV)
    x = torch.randint(0, 300, (50,), device=DEV)
    cu, pos = torch.tensor([0, 50], dtype=torch.int32, device=DEV), torch.arange(50, dtype=torch.int32, device=DEV)
    up = torch.randn(50, 300, device=DEV)
    params = dict(m.named_parameters())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = m(x, pos, cu)
    got = torch.autograd.grad(logits.float(), list(params.values()), up)
    ref = torch.autograd.grad(_plain_logits(m, x), list(params.values()), up)
    for name, a, b in zip(params, got, ref):
        err = float((a - b).norm() / b.norm())
        assert err <= 64 * 2.0 ** -8, (name, err)


@pytest.mark.parametrize("save8", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_training_runs(save8, graph):
    """Packed layers stepping inside the backward; the same numbers on every run, captured or not."""
    import workloads
    run = lambda g: workloads.train_packed_llama(steps=4, warmup=3, tokens=512, longest=64, save8=save8, graph=g, **SMALL)  # noqa: E731
    r = run(graph)
    assert len(r["ms"]) == 4 and all(v == v and abs(v) < 100 for v in r["losses"])
    assert run(False)["losses"] == r["losses"]


def test_8_bits_take_less_memory():
    """What a forward leaves for the backward: of every token and block, inputs of 2 d and the unit's 3 ffn values in 66 / 64
    bytes in place of 2 (widths are multiples of 16); a twentieth is granted to the allocator's pieces."""
    import workloads
    from concord_b200.convert import concordify
    tokens, d, ffn, blocks = 4096, 512, 1536, 3
    ids, pos, _, cu = workloads.packed_tokens(tokens, 512, 300, torch.Generator().manual_seed(0), DEV)
    held = []
    for save8 in (False, True):
        m = workloads.PackedLlama(300, d, blocks, 8, 4, ffn, 512, save8, device=DEV)
        concordify(m, lr=1e-4, skip=lambda name, _: name == "lm_head")
        with torch.autocast("cuda", dtype=torch.bfloat16):
            with torch.no_grad():
                m(ids, pos, cu)                              # (buffers and workspaces made)
            torch.cuda.synchronize()
            before = _asked()
            out = m(ids, pos, cu)
        held.append(_asked() - before)
        del out, m
    want = tokens * blocks * (2 * d + 3 * ffn) * (2 - 66 / 64)
    assert abs(held[0] - held[1] - want) <= want / 20, (held, want)
