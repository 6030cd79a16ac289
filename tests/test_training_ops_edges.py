"""CPU-only checks of the training operators: what the C entries answer at the ends of their ranges, before anything
reaches a device, and what the extension is built for."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from concord_b200 import _abi, build
    build.build()
    return _abi.load()


ONE = ctypes.c_void_p(16)


def _loss(lib, N=4, V=8, K=2, ldz=None, loss=ONE, row_loss=None):
    from concord_b200 import _abi
    p = _abi.DistillParams(temperature=1.0, alpha=1.0, grad_scale=1.0)
    return lib.concord_distill_loss(p, ONE, 0, ldz or V, ONE, ONE, None, loss, row_loss, None, None, N, V, K, ONE, 10 ** 6,
                                    None)


def test_a_loss_per_row_of_no_rows_has_no_address(lib):
    assert _loss(lib, N=0, loss=None) == 0
    assert _loss(lib, N=1, loss=None) == -1


@pytest.mark.parametrize("V", [2 ** 31 - 1024, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
def test_rows_beyond_32_bits_of_columns_are_refused(lib, V):
    """A thread steps from column to column by up to 1024: beyond these widths the step would pass 32 bits and the
    gradient be written in front of its tensor."""
    assert _loss(lib, V=V) == -7
    from concord_b200 import _abi
    p = _abi.DistillParams(temperature=1.0, alpha=1.0, grad_scale=1.0)
    assert lib.concord_distill_grad(p, ONE, 0, V, ONE, ONE, None, ONE, None, 0, ONE, 4, V, 2, None) == -7


def test_extension_follows_the_installed_torch(lib, tmp_path, monkeypatch):
    """Built for another torch, it is neither kept by a build nor loaded."""
    from concord_b200 import _ops, build
    assert build.stamp() == build.built_for()
    commands = []
    monkeypatch.setattr(build, "STAMP", str(tmp_path / "stamp"))
    monkeypatch.setattr(build.subprocess, "check_call", commands.append)
    (tmp_path / "stamp").write_text("torch 1.0.0, cpython-30\n")
    monkeypatch.setattr(_ops, "_NATIVE", None)
    with pytest.raises(RuntimeError, match="built for torch 1.0.0"):
        _ops.native()
    build.build(extension=False)
    assert commands == []
    build.build()
    assert len(commands) == 1 and commands[0][0] == "g++" and build.stamp() == build.built_for()
    build.build()
    assert len(commands) == 1
    assert callable(_ops.native().layer_norm)


def test_library_without_the_extension(lib, tmp_path, monkeypatch):
    """The C ABI's users need no torch headers."""
    from concord_b200 import build
    monkeypatch.setattr(build, "NATIVE", str(tmp_path / "none.so"))
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd: pytest.fail(f"ran {cmd[0]}"))
    assert build.build(extension=False) == build.OUT
