"""What the modules share on the host side of a launch: dtype codes, streams and the device error word."""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from qwenquest_b200 import _lib
from qwenquest_b200._lib import QQ_BF16, QQ_F32, check

__all__ = ["DeviceError", "dtype_code", "host_device_pointer", "stream_of"]


def dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return QQ_BF16
    if dtype == torch.float32:
        return QQ_F32
    raise ValueError(f"unsupported dtype {dtype}: the kernels take bfloat16 or float32")


def stream_of(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def host_device_pointer(t: torch.Tensor) -> int:
    """Device address of a pinned host tensor (``cudaHostGetDevicePointer``)."""
    if not t.is_pinned():
        raise ValueError("the host tier must be pinned memory")
    out = ctypes.c_void_p()
    check(_lib.load().qq_host_device_pointer(t.data_ptr(), ctypes.byref(out)), "host_device_pointer")
    return int(out.value)


@dataclass
class DeviceError:
    word: torch.Tensor  # pinned host int32 [1]; kernels OR error bits into it
    dev_ptr: int = 0

    def ptr(self) -> int:
        if not self.dev_ptr:
            self.dev_ptr = host_device_pointer(self.word)
        return self.dev_ptr

    def take(self) -> int:
        bits = int(self.word[0])
        if bits:
            self.word.zero_()
        return bits
