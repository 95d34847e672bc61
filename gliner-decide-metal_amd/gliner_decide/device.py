"""Device-buffer plumbing: torch tensors supply HIP memory and streams.

The arithmetic is in the HIP library; torch is only the allocator and the
stream handle.  Every helper refuses CPU tensors so a call can never run
anywhere but the GPU.
"""

from __future__ import annotations

import torch

from . import _native as N


def require_gpu() -> torch.device:
    if not torch.cuda.is_available():
        raise RuntimeError("a ROCm GPU is required (torch.cuda.is_available() is False)")
    return torch.device("cuda", torch.cuda.current_device())


def ptr(t: torch.Tensor | None) -> int | None:
    """Device address of a contiguous GPU tensor (None passes through)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a GPU tensor")
    return t.data_ptr()


# The current stream's handle and device alone, where this torch has such calls
# (they are not part of its public interface): a torch.cuda.Stream object costs
# more than the rest of a small call's arguments (2.8 against 0.2 us).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def stream_handle(stream: torch.cuda.Stream | None = None) -> int:
    if stream is None:
        if _raw_stream is not None:
            return _raw_stream(_current_device())
        stream = torch.cuda.current_stream()
    return stream.cuda_stream


def as_f16(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if t.dtype != torch.float16:
        raise TypeError(f"{name} must be float16 (got {t.dtype})")
    return t if t.is_contiguous() else t.contiguous()


def as_i32(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an integer tensor (got {t.dtype})")
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


_DTYPES_16 = {torch.float16: N.GD_F16, torch.bfloat16: N.GD_BF16}


def dtype16(t: torch.Tensor, name: str) -> int:
    """gd_dtype of an fp16 or bf16 GPU tensor."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    code = _DTYPES_16.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float16 or bfloat16 (got {t.dtype})")
    return code


def same_kind(t: torch.Tensor, like: torch.Tensor, name: str, dtype: torch.dtype | None = None) -> None:
    """Refuses a tensor on another device than `like`, or of another type than
    `dtype` (None: that of `like`)."""
    if t.get_device() != like.get_device():
        raise ValueError(f"{name} must be on {like.device} (got {t.device})")
    dtype = dtype or like.dtype
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")


def call_on(t: torch.Tensor, fn, *args) -> None:
    """fn(*args, current stream) on t's device, whichever device is current."""
    index = t.get_device()
    if index == _current_device():
        status = fn(*args, stream_handle() if _raw_stream is None else _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, stream_handle())
    if status != N.GD_OK:
        N.check(status)
