"""What the training operators (layer norm, packed attention, distillation
loss) share: type codes of the C ABI, checks of arguments, the call itself."""
import ctypes

import torch

from . import _abi

TYPES = {torch.float32: _abi.F32, torch.bfloat16: _abi.BF16, torch.float16: _abi.F16}


def ptr(t):
    return None if t is None else t.data_ptr()


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
    return dev


def need_type(name, t, types):
    if t.dtype not in types:
        raise TypeError(f"{name} must be one of {[str(x) for x in types]}, got {t.dtype}")


_FN = {}
_raw_stream = torch._C._cuda_getCurrentRawStream     # current_stream(...).cuda_stream without the Stream object


def call(name, index, *args):
    """Call `name` of the C ABI on CUDA device `index` and its current stream
    (appended as the last argument)."""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(_abi.load(), name)
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    else:
        status = fn(*args, _raw_stream(index))
    if status != 0:
        _abi.check(status, name)


byref = ctypes.byref
