"""packed_attention at the ends of its types' ranges, in layouts of one row or one head, and after a wait that ran
out.  Tolerances as in test_gpu_attention.py, with half of fp16's smallest number as the absolute part where results
are that small."""
import math

import pytest
import torch

from test_gpu_attention import DEV, U, check, cum, inputs, run

pytestmark = pytest.mark.gpu


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
