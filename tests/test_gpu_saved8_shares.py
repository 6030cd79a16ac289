"""The shares of the weight gradient's tiles, as the library works them out: its workspace against the plan that is restated
beside the host tests, and what is written behind it."""
import ctypes
import random

import pytest
import torch

from test_decoder_ops_host import _plan

DEV = "cuda"


@pytest.fixture(scope="module")
def lib():
    from concord_b200 import _abi, build
    build.build()
    return _abi.load()


def test_workspace_is_what_the_plan_stores(lib):
    """Without a device the library plans for 74 pairs: pieces of 256 x 256 sums, as many as the plan's slots, none to spare;
    146 at most, as is documented."""
    if torch.cuda.is_available():
        pytest.skip("a device's own number of pairs")
    rng = random.Random(1)
    most = 0
    for _ in range(3000):
        M, N, K = (int(2 ** rng.uniform(0, top)) for top in (17, 13, 14))
        N = max(8, N // 8 * 8)
        _, pieces = _plan(-(-N // 256) * -(-K // 256), -(-M // 64), 74)
        slots = 1 + max(s for _, _, _, s in pieces)
        assert lib.concord_gemm_dw8_workspace_bytes(M, N, K) == slots * 256 * 256 * 4, (M, N, K)
        most = max(most, slots)
    assert 100 < most <= 146
    assert lib.concord_gemm_dw8_workspace_bytes(80512, 18688, 256) == 146 * 256 * 1024          # 73 tiles on 74 pairs


@pytest.mark.gpu
def test_nothing_is_written_behind_the_workspace(lib):
    """Random sizes, most of them with tiles that are cut: sums of whole numbers are exact, and the bytes behind the workspace
    and the result stay as they were."""
    rng = random.Random(2)
    g = torch.Generator(device=DEV).manual_seed(3)
    cut = 0
    for _ in range(40):
        M, N, K = int(2 ** rng.uniform(6, 14)), 8 * int(2 ** rng.uniform(0, 7.5)), int(2 ** rng.uniform(0, 11))
        from concord_b200 import save8
        x = torch.randint(-30, 31, (M, K), generator=g, device=DEV).bfloat16()
        dy = torch.randint(-4, 5, (M, N), generator=g, device=DEV).bfloat16()
        s = save8(x)
        need = lib.concord_gemm_dw8_workspace_bytes(M, N, K)
        cut += need > 0
        ws = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device=DEV)
        dw = torch.full((N * K + 256,), -7.0, dtype=torch.bfloat16, device=DEV)
        ptr = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
        assert lib.concord_gemm_dw8(ptr(dy), N, ptr(s.data), ptr(dw), M, N, K, ptr(ws), need,
                                    ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        want = (dy.double().t() @ x.double()).float().bfloat16()
        assert torch.equal(dw[:N * K].view(N, K), want), (M, N, K)
        assert bool((dw[N * K:] == -7).all()) and bool((ws[need:] == 0x5a).all()), (M, N, K)
    assert cut > 10
