"""The embedding's gradient where the sort in memory takes its rarer ways: runs of tokens that double in length, a fourth
digit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T", [4096 * 512 - 1, 4096 * 512, 4096 * 512 + 1, 4096 * 1024 + 33])
@pytest.mark.parametrize("V", [7, 1500])
def test_many_tokens(T, V):
    """Up to and beyond 512 sorting blocks of 4096 tokens: whole numbers whose sums stay below 2^24 are exact in any order."""
    from concord_b200 import embedding
    g = torch.Generator(device=DEV).manual_seed(T + V)
    ids = torch.randint(-1, V + 1, (T,), generator=g, device=DEV, dtype=torch.int32)             # a few outside on either side
    dy = torch.randint(-3, 4, (T, 1), generator=g, device=DEV).float()
    w = torch.randn(V, 1, generator=g, device=DEV, requires_grad=True)
    y = embedding(ids, w)
    inside = (ids >= 0) & (ids < V)
    assert torch.equal(y.detach(), torch.where(inside[:, None], w.detach()[ids.clamp(0, V - 1)], 0.0))
    (dw,) = torch.autograd.grad(y, w, dy)
    want = torch.zeros(V, 1, dtype=torch.float64, device=DEV)
    want.index_add_(0, ids[inside].long(), dy[inside].double())
    assert float(want.abs().max()) < 2 ** 24 and torch.equal(dw.double(), want)


@pytest.mark.parametrize("T", [70001, 300])
@pytest.mark.parametrize("V", [2 ** 27, 2 ** 27 + 5])
def test_many_rows(T, V):
    """Rows whose numbers take four digits, in memory and in one cluster: the touched rows' sums, and zeros elsewhere."""
    from concord_b200 import embedding
    g = torch.Generator(device=DEV).manual_seed(T)
    few = torch.randint(0, V, (max(T // 3, 1),), generator=g, device=DEV)
    few[:4] = torch.tensor([0, V - 1, 2 ** 27 - 1, 2 ** 18], device=DEV)
    ids = few[torch.randint(0, len(few), (T,), generator=g, device=DEV)]
    ids[:4] = few[:4]
    dy = torch.randint(-3, 4, (T, 1), generator=g, device=DEV).bfloat16()
    w = torch.zeros(V, 1, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    (dw,) = torch.autograd.grad(embedding(ids, w), w, dy)
    rows, where = ids.unique(return_inverse=True)
    want = torch.zeros(len(rows), 1, dtype=torch.float64, device=DEV).index_add_(0, where, dy.double())
    assert float(want.abs().max()) <= 256 and torch.equal(dw[rows].double(), want)               # (bf16 holds whole numbers to 256)
    assert int(torch.count_nonzero(dw)) == int(torch.count_nonzero(want))
