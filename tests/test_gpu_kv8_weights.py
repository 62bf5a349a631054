"""How finely attention over an 8-bit cache weighs: V exact and the weights in f16 wherever the V scales are powers of
two from 2^-15 to 2^5, so that only the output's own rounding to bf16 is left to see.

Tolerance per output value, in the terms of test_gpu_kv8_attention: scores, exp and sums as there; a weight is off by
2^-11 of itself, or, where f16 does not hold it in full (below 2^-14, the largest being 2^7 at least; half a step of
2^-24), by 2^-32 of the largest, that is 2^-32 |v| summed over the keys at most:
  |err| <= half |out| + A (2 ((D + 8) u S + 8 u + n u) + 2^-11) (1 + 2^-6) + 2^-32 n max |v|."""
import math

import numpy as np
import pytest
import torch

import kv8_oracle as o
from test_gpu_kv8_attention import FMT, call, make

pytestmark = pytest.mark.gpu
#: new tokens (8 and 2 heads): decode kernel with one, two and three query tiles, tile kernel with half and whole tiles
TOKENS = [1, 6, 12, 13, 40]


def compare_fine(got, host, scale, weight=2.0 ** -11):
    qx, kn, vn, ks, vs, tables, lens = host
    want, mean, reach = o.attend(qx, kn, vn, ks, vs, tables, lens, scale)
    D, n, u = qx.shape[-1], max(lens), 2.0 ** -24
    used = np.unique(np.concatenate([tables[i][:-(-m // vn.shape[1])] for i, m in enumerate(lens)]))
    top = np.nanmax(np.abs(vn[used]) * vs[used][:, None, :, None])
    got = got.double().cpu().numpy().reshape(want.shape)
    tol = 2.0 ** -8 * np.abs(want) + mean * (2 * ((D + 8) * u * reach + 8 * u + n * u) + weight) * (1 + 2.0 ** -6)
    off = np.abs(got - want) - (tol + 2.0 ** -32 * n * top)
    assert np.isfinite(got).all() and off.max() <= 0, (np.unravel_index(off.argmax(), off.shape), off.max())


def set_cache(on, fmt, kn=None, vn=None, ks=None, vs=None):
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    dev = on["k"].device
    for name, x in (("k", kn), ("v", vn)):
        if x is not None:
            on[name] = torch.from_numpy(np.where(np.isnan(x), 0.0, x)).to(dt).to(dev)
    for name, x in (("ks", ks), ("vs", vs)):
        if x is not None:
            on[name] = torch.from_numpy(x).float().to(dev)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("exponent", [-15, -12, -6, 0, 5])
def test_values_that_cancel(dev, fmt, T, exponent):
    """v and -v in turn, so that the output is small next to the weights' errors; scales over the range that is exact"""
    rng = np.random.default_rng(T)
    on, host = make(rng, fmt, "bf16", [T + 1, T + 40, 700, 1500], T, 8, 2, 128, 16, dev)
    qx, kn, vn, ks, vs, tables, lens = host
    vn[:, 1::2] = -vn[:, 0::2]
    vs[np.isfinite(vs)] = 2.0 ** exponent
    for i, n in enumerate(lens):  # (a context that ends inside a pair keeps its last value)
        vn[tables[i, n // 16], n % 16:] = 0.0
    set_cache(on, fmt, vn=vn, vs=vs)
    compare_fine(call(on, 128 ** -0.5), host, 128 ** -0.5)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("below", [3, 10, 18, 22, 25, 28])
@pytest.mark.parametrize("sink", [0, 500])
def test_one_key_takes_nearly_all_the_weight(dev, fmt, T, below, sink):
    """and has nothing in V, so that what is left is the sum of many small weights, at 2^-below of it each"""
    rng = np.random.default_rng(below)
    on, host = make(rng, fmt, "bf16", [900 + T, 600 + T], T, 8, 2, 128, 16, dev)
    qx, kn, vn, ks, vs, tables, lens = host
    qx[..., 0] = 1.0
    kn[:] = 0.0
    ks[np.isfinite(ks)] = 2.0 ** -5
    vn[:] = np.rint(rng.uniform(4, 8, vn.shape)) * 8
    for i in range(2):
        at = tables[i, sink // 16], sink % 16
        kn[at[0], at[1], :, 0], vn[at] = 64.0, 0.0
    set_cache(on, fmt, kn, vn, ks)
    on["q"] = torch.from_numpy(qx).to(torch.bfloat16).to(dev)
    scale = below * math.log(2.0) / 2.0
    compare_fine(call(on, scale), host, scale)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("every", [1, 9])
def test_scales_that_are_no_powers_of_two(dev, fmt, T, every):
    """from a calibration: all blocks, or some of them.  The decode kernel weighs as finely there (48 query rows a kv head
    at most); the tile kernel rounds weights times scale to bf16"""
    rng = np.random.default_rng(T + every)
    on, host = make(rng, fmt, "bf16", [T, 1700, 333 + T], T, 8, 2, 128, 16, dev)
    vs, tables = host[4], host[5]
    for i, n in enumerate(host[6]):
        for j in range(every // 2, -(-n // 16), every):
            vs[tables[i, j]] = np.float32(rng.uniform(0.001, 0.1, 2))
    set_cache(on, fmt, vs=vs)
    compare_fine(call(on, 128 ** -0.5), host, 128 ** -0.5, weight=2.0 ** (-11 if 4 * T <= 48 else -8))
