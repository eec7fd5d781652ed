"""What the Dense and dropout operators share on the host: a dropout's arguments."""
from __future__ import annotations

import torch


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
