"""Shared by the kv8 tests: codes to and from torch, caches with poison in every place that no call may
look at."""
import numpy as np
import torch

import kv8_oracle as o

TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ELEM = {"bf16": torch.bfloat16, "f32": torch.float32}
#: bytes that no write makes / that turn what reads them into NaN
POISON = {"int8": 0x80, "e4m3": 0x7f}


def to_dev(codes, fmt, dev):
    return torch.from_numpy(np.ascontiguousarray(codes)).to(dev).view(TORCH[fmt])


def numbers_of(cache, fmt):
    return o.numbers(cache.view(torch.uint8).cpu().numpy(), fmt)


def rounded(rng, shape, dtype, sigma=1.0):
    """normal values that the dtype holds exactly: (torch CPU tensor, float64 array)"""
    t = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * np.float32(sigma)).to(ELEM[dtype])
    return t, t.double().numpy()


def random_codes(rng, shape, fmt):
    c = rng.integers(0, 256, shape, dtype=np.uint8)
    if fmt == "int8":
        return np.where(c == 0x80, 0x81, c).astype(np.uint8)
    return np.where((c & 0x7f) == 0x7f, c ^ 1, c).astype(np.uint8)


def gentle_codes(rng, shape, fmt):
    """normal-distributed codes over most of the range"""
    x = np.clip(rng.standard_normal(shape) * 0.26 * o.TOP[fmt], -o.TOP[fmt], o.TOP[fmt])
    t = torch.from_numpy(np.rint(x)).to(torch.int8) if fmt == "int8" else torch.from_numpy(x).to(torch.float8_e4m3fn)
    return t.view(torch.uint8).numpy()
