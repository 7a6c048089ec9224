"""Helpers shared by the op wrappers: pointers, streams, parameter gradient sinks."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from ..kernels import native


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def use_native(*tensors: torch.Tensor) -> bool:
    """CUDA bf16 tensors run on the sm_100a kernels; anything else on the PyTorch reference.
    On a CUDA device a missing library raises instead of falling back."""
    t = tensors[0]
    if not t.is_cuda:
        return False
    if t.dtype != torch.bfloat16:
        return False
    native.lib()
    return True


MAX_ROWS = 2 ** 31 - 1024      # row counts are 32-bit integers in the kernels, rounded up to whole blocks

_DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def dtype_code(t: torch.Tensor) -> int | None:
    """Type argument of the kernels that take bf16, fp16 and fp32 CUDA tensors; None: the reference runs."""
    if not t.is_cuda:
        return None
    return _DTYPE_CODES.get(t.dtype)


_HERE = contextlib.nullcontext()


def on_device(t: torch.Tensor):
    """Makes the tensor's device the current one for a launch on it."""
    if t.get_device() == torch._C._cuda_getDevice():
        return _HERE
    return torch.cuda.device(t.device)


def stream_of(t: torch.Tensor) -> int:
    """The current stream of the tensor's device."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def refuse_twice(what: str) -> None:
    """For a backward pass made of kernels: with create_graph its results would silently carry no graph."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} cannot be differentiated twice")


def refuse_tangents(what: str, *tensors: torch.Tensor | None) -> None:
    """For a call of kernels outside of an autograd function, which would drop a forward-mode tangent (a dual tensor does not
    require a gradient)."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def grad_sink(param: torch.Tensor):
    """Returns (buffer, accumulate) when `param` owns a slice of a flat gradient buffer
    (`param.main_grad`), else (None, False). The first write of a step overwrites, later
    writes accumulate, so the flat buffer never needs zeroing."""
    mg = getattr(param, "main_grad", None)
    if mg is None:
        return None, False
    acc = bool(getattr(param, "grad_acc", False))
    return mg, acc


def mark_grad_written(param: torch.Tensor) -> None:
    param.grad_acc = True


_scratch: dict = {}


def scratch(device: torch.device, nfloats: int, key: str = "f32") -> torch.Tensor:
    """A per-device fp32 scratch buffer that only grows (kernel partial sums and the like)."""
    k = (device, key)
    buf = _scratch.get(k)
    if buf is None or buf.numel() < nfloats:
        buf = torch.empty(max(nfloats, 1 << 16), dtype=torch.float32, device=device)
        _scratch[k] = buf
    return buf
