"""What the Dense, dropout and beam operators share on the host: element types, the current stream, a dropout's arguments."""
from __future__ import annotations

import torch

from . import _lib

DTYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def stream(device) -> int:
    """The current stream of `device` as an integer; a Stream object for every call costs more than the call."""
    if _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def on_device(device):
    """Makes `device` current for a launch where it is not already."""
    return _ALREADY if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


class _Already:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_ALREADY = _Already()


def dtype_code(what: str, t) -> int:
    code = DTYPE_CODE.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16 expected, got {t.dtype}")
    return code


def need_gpu(what: str, **tensors):
    """All tensors (None skipped) on one MI355X device, which is returned."""
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a tensor")
        d = t.device
        if dev is None:
            if d.type != "cuda":
                raise ValueError(f"{what}: {name} must live on an MI355X device (there is no CPU path)")
            dev = d
        elif d != dev:
            if d.type != "cuda":
                raise ValueError(f"{what}: {name} must live on an MI355X device (there is no CPU path)")
            raise ValueError(f"{what}: {name} lives on {d}, the others on {dev}")
    return dev


def drop16(what: str, rate) -> int:
    """A dropout rate in the steps the generator has, 2^-16."""
    rate = float(rate)
    if not 0.0 <= rate < 1.0:
        raise ValueError(f"{what}: a dropout rate lies in [0, 1), got {rate}")
    d = round(rate * 65536)
    if d > 65535:
        raise ValueError(f"{what}: a dropout rate of {rate} keeps less than one element in 65536")
    return d


def seed_offset(what: str, seed, offset, device):
    """(seed, offset, offset tensor or None) with the ranges of the generator's key and counter."""
    seed = int(seed)
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"{what}: seed must lie in [0, 2^64)")
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1 or offset.device != device:
            raise ValueError(f"{what}: an offset tensor is one int64 on the device of the data")
        return seed, 0, offset
    offset = int(offset)
    if not 0 <= offset < 1 << 64:
        raise ValueError(f"{what}: offset must lie in [0, 2^64)")
    return seed, offset, None


def check(rc: int, what: str) -> None:
    if rc != _lib.OK:
        _lib.check(rc, what)
