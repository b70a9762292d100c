"""Device plumbing shared by the API modules: run on the current ROCm device,
hand results back on the caller's device."""
from __future__ import annotations

import torch

from . import _lib as L


def to_gpu(t: torch.Tensor, dtype=None) -> torch.Tensor:
    L.lib()   # verifies the kernel library and the GPU
    if dtype is not None:
        t = t.to(dtype)
    if not t.is_cuda:
        t = t.to(torch.device("cuda", torch.cuda.current_device()))
    return t.contiguous()


def int32_on(t: torch.Tensor, device) -> torch.Tensor:
    """Whole numbers as a contiguous int32 tensor on the device, those beyond 32 bits as the nearest
    that has them: a number outside a range stays outside on its side, where narrowing alone
    would wrap 2^32 + 5 to 5."""
    if t.dtype is torch.int64:
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(device=device, dtype=torch.int32).contiguous()


def back(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return t if like.is_cuda else t.to(like.device)
