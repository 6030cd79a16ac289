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
