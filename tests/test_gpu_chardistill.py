"""The char GPT student on packed documents: layer norm, packed attention and
distillation loss together around the packed layers."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_batches_are_whole_documents():
    import workloads
    b = workloads.PackedDocuments(workloads.MarkovChars(n_chains=32, length=200, device=DEV), docs=7, block=32, top=4)
    x, pos, y, ids, t, cu = b.batch()
    cu = cu.tolist()
    assert cu[0] == 0 and all(1 <= n - m <= 32 for m, n in zip(cu, cu[1:]))
    for m, n in zip(cu, cu[1:]):
        assert pos[m:n].tolist() == list(range(n - m))
        assert torch.equal(y[m:n - 1], x[m + 1:n])
        assert bool((ids[m] == -1).all()) and bool((ids[m + 1:n] >= 0).all())
    assert bool((y[cu[-1]:] == -100).all()) and bool((ids[cu[-1]:] == -1).all())


def test_packed_student_matches_the_padded_model():
    """The same weights in CharGPT, one document at a time, torch's norm and attention in fp32: bf16 inputs of
    every matrix product leave 2^-9 relative each, over two blocks and a head; 32 of them are granted."""
    import workloads
    torch.manual_seed(0)
    packed = workloads.PackedCharGPT(n_layer=2, block=64).to(DEV)
    plain = workloads.CharGPT(n_layer=2, block=64).to(DEV)
    for b, c in zip(packed.blocks, plain.blocks):
        c.attn.c_attn.weight, c.attn.c_proj.weight = b.c_attn.weight, b.c_proj.weight
        c.c_fc.weight, c.mlp_proj.weight = b.c_fc.weight, b.mlp_proj.weight
    plain.wte.weight, plain.wpe.weight, plain.lm_head.weight = packed.wte.weight, packed.wpe.weight, packed.lm_head.weight
    lens = [40, 1, 64, 17]
    cu = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
    x = torch.randint(0, 65, (sum(lens),), device=DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).to(DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        got = packed(x, pos, cu).float()
    for i, n in enumerate(lens):
        idx = x[cu[i]:cu[i + 1]][None]
        with torch.no_grad():
            h = plain.wte(idx) + plain.wpe(torch.arange(n, device=DEV))[None]
            for b in plain.blocks:
                h = b(h)
            ref = plain.lm_head(plain.ln_f(h))[0]
        err = (got[cu[i]:cu[i + 1]] - ref).norm() / ref.norm()
        assert float(err) <= 32 * 2.0 ** -9, (n, float(err))


@pytest.mark.parametrize("graph", [False, True])
def test_training_lowers_the_loss(graph):
    import workloads
    r = workloads.train_chardistill(steps=60, docs=16, block=64, n_layer=2, lr=2e-3, graph=graph)
    first, last = sum(r["losses"][:5]) / 5, sum(r["losses"][-5:]) / 5
    assert all(l == l for l in r["losses"]) and last < first - 0.01, (first, last)
