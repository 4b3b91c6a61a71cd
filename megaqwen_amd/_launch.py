"""What the tensor-level entry points (w4, kv4, logprobs) share: argument checks and the call."""
from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.MQ_DTYPE_BF16, torch.float16: _lib.MQ_DTYPE_F16,
          torch.float32: _lib.MQ_DTYPE_F32}

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = torch._C._cuda_getCurrentRawStream


def no_grad(what: str, *tensors) -> None:
    """These operators have no backward pass: a result that silently cut the gradient would train
    something else than its caller means."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no backward pass: call it under torch.no_grad()")


def call(fn, dev: int, *args) -> None:
    """fn(*args, stream) on device `dev`'s current stream; no device guard when it is the current
    one, and the raw stream handle: a short kernel's call is as fast as this code."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc != 0:
        _lib.check(rc)
