"""Operand checks and layouts of the row-wise operators (criterions.py, blocks.py).  Their smallest calls are a few microseconds on the device:
nothing here does more than it has to when the operands are what they should be."""
from __future__ import annotations

import torch

from ._lib import FC_PREC_BF16, FC_PREC_FP32, FedcolaHipError

_CODES = {torch.bfloat16: FC_PREC_BF16, torch.float32: FC_PREC_FP32}


def operand_type(what, t, *others):
    """(type code, device) that the tensors share; raises where they do not."""
    try:
        dtype, dev = t.dtype, t.device
        if dev.type == "cuda" and dtype in _CODES:
            for u in others:
                if u.dtype is not dtype or u.device != dev:
                    break
            else:
                return _CODES[dtype], dev
    except AttributeError:
        pass
    for u in (t, *others):
        if not torch.is_tensor(u):
            raise ValueError(f"{what}: a tensor is expected, not {type(u).__name__}")
        if not u.is_cuda:
            raise FedcolaHipError(f"{what}: needs its tensors on an MI355X (cuda) device: the operator is HIP-only (no CPU fallback)")
        if u.dtype != t.dtype or u.device != t.device:
            raise ValueError(f"{what}: operands of one type on one device are expected: {t.dtype} on {t.device}, {u.dtype} on {u.device}")
    raise ValueError(f"{what}: {t.dtype}: bfloat16 or float32")


def as_rows(t):
    """(2-D view or copy of t with its last dimension contiguous, row stride in elements)"""
    D = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, D) if t.numel() else t.new_empty(t.shape[:-1].numel(), D)
    ld, one = t.stride()
    if t.shape[0] <= 1 and (D == 1 or one == 1):
        return t, D
    if (D > 1 and one != 1) or not D <= ld < 1 << 21:
        t = t.contiguous()
        return t, D
    return t, ld


def check_sizes(what, rows, D, most_D, N, most_N):
    """refuses sizes past the library's: its arguments are 32 bits wide, and a larger number would arrive as another one"""
    if rows > 1 << 28 or D > most_D or N > most_N:
        raise ValueError(f"{what}: {rows} rows, width {D}, {N} classes or hidden units: at most {1 << 28}, {most_D} and {most_N}")


def in_place(t, ld, rows):
    """whether the tiled products of `rows` rows read this matrix where it is (include/fedcola_hip.h)"""
    if t.element_size() == 4:
        return rows <= 512 and ld < 1 << 20
    return ld % 8 == 0 and t.shape[1] % 8 == 0 and t.data_ptr() % 16 == 0


class on_device:
    """``with on_device(dev) as stream``: the device current, and its current stream's handle"""
    __slots__ = ("dev", "back")

    def __init__(self, dev):
        self.dev = dev

    def __enter__(self):
        cur = torch.cuda.current_device()
        self.back = None
        if cur != self.dev.index:
            self.back = cur
            torch.cuda.set_device(self.dev)
        return torch._C._cuda_getCurrentRawStream(self.dev.index)

    def __exit__(self, *exc):
        if self.back is not None:
            torch.cuda.set_device(self.back)


def address(t):
    """a tensor's address for the C ABI, or None"""
    return None if t is None else t.data_ptr()
