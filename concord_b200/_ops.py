"""What the training operators (layer norm, packed attention, distillation
loss) share: checks of arguments, and the extension that runs them."""
import importlib.machinery
import importlib.util
import os

import torch

from . import _abi

TYPES = {torch.float32: _abi.F32, torch.bfloat16: _abi.BF16, torch.float16: _abi.F16}
NATIVE_PATH = os.path.join(os.path.dirname(_abi.LIB_PATH), "_native.so")
_NATIVE = None


def native():
    """The extension of csrc/torch_ops.cpp (raises if it was not built)."""
    global _NATIVE
    if _NATIVE is None:
        _abi.load()
        if not os.path.exists(NATIVE_PATH):
            raise RuntimeError(f"concord_b200 extension not built: {NATIVE_PATH} is missing "
                               "(run `python -m concord_b200.build`); there is no CPU fallback")
        from . import build
        if build.stamp() not in (None, build.built_for()):
            raise RuntimeError(f"concord_b200 extension built for {build.stamp()}, this is {build.built_for()}: "
                               "run `python -m concord_b200.build`")
        loader = importlib.machinery.ExtensionFileLoader("_native", NATIVE_PATH)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_native", loader))
        loader.exec_module(module)
        _NATIVE = module
    return _NATIVE


def need_cuda(*named):
    """Every tensor on one CUDA device; (name, tensor or None) pairs."""
    dev = None
    for name, t in named:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"concord_b200 runs on CUDA tensors only (no CPU fallback); {name} is on {t.device}")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"{name} is on {t.device}, the other tensors are on {dev}")


def need_type(name, t, types):
    if t.dtype not in types:
        raise TypeError(f"{name} must be one of {[str(x) for x in types]}, got {t.dtype}")
