"""What every wrapper of a kernel checks its arguments with."""
from __future__ import annotations

from typing import Optional

import torch

GB_F32, GB_BF16 = 0, 1
_TAG = {torch.float32: GB_F32, torch.bfloat16: GB_BF16}


class KernelError(RuntimeError):
    pass


def _tag(t: torch.Tensor, what: str) -> int:
    try:
        return _TAG[t.dtype]
    except KeyError:
        raise KernelError(f"{what}: dtype {t.dtype} is not supported (float32 or bfloat16)") from None


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise KernelError(msg)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()
