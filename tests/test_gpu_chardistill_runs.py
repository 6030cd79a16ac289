"""What a run of the packed distillation workload goes by, and what it reports."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_a_seed_is_a_run(graph):
    """The same losses whatever ran before: the stochastic rounding of the packed steps starts from the seed too."""
    import workloads
    run = lambda seed: workloads.train_chardistill(steps=12, docs=16, block=64, n_layer=2, lr=2e-3, graph=graph,  # noqa: E731
                                                   seed=seed)["losses"]
    first, other = run(3), run(4)
    assert run(3) == first and other != first


def test_the_documents_tokens_count():
    """Rows that belong to no document are none of the tokens, nor are the eager steps' documents."""
    import workloads
    r = workloads.train_chardistill(steps=7, docs=16, block=64, n_layer=1, warmup=3, graph=False)
    assert len(r["ms"]) == 7 and r["tokens_per_step"] == 16 * 64
    assert 7 * 16 <= r["document_tokens"] < 7 * 16 * 64
    again = workloads.train_chardistill(steps=7, docs=16, block=64, n_layer=1, warmup=3, graph=True)
    assert again["tokens_per_step"] == 16 * 64 and 7 * 16 <= again["document_tokens"] < 7 * 16 * 64
