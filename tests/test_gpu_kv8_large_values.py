"""Attention over 8-bit caches whose blocks are far apart in size: V scales up to 2^121, where the weights
times the scale leave little room below f32's largest number, next to ordinary ones.

The tolerance is test_gpu_kv8_attention's, which is relative to the weighted mean of |v| of each output value,
so a large value in one dim excuses nothing in another."""
import math

import numpy as np
import pytest
import torch

import kv8_oracle as o
from kv8_helpers import gentle_codes
from test_gpu_kv8_attention import FMT, call, compare, make

pytestmark = pytest.mark.gpu

#: (T, Hq, H, D, block size, dtype): decode kernel with one, two and three query tiles, tile kernel with
#: half and whole tiles, generic kernel
SHAPES = [(1, 8, 2, 128, 16, "bf16"), (6, 8, 2, 128, 16, "bf16"), (12, 8, 2, 128, 16, "bf16"),
          (13, 8, 2, 128, 16, "bf16"), (40, 8, 2, 128, 16, "bf16"), (3, 4, 2, 64, 8, "f32")]
LAG = 7.65  # of the large value's score over the others, as a power of two


def far_apart(fmt, T, Hq, H, D, bs, dtype, exponent, every, dev, seed=20):
    """Sequences with `every`-th block from one that moves from sequence to sequence holding a single row that is
    not zero, of the scale 2^exponent, with a score LAG above the others' (which are all 0)."""
    rng = np.random.default_rng(seed)
    lens = [2100 + T, 1200 + T, 900 + T, 640 + T, 400 + T, 333 + T, 2000 + T, 1500 + T]
    on, host = make(rng, fmt, dtype, lens, T, Hq, H, D, bs, dev)
    qx, kn, vn, ks, vs, tables, lens = host
    kn[:], qx[..., 0] = 0.0, 1.0
    ks[np.isfinite(ks)] = 2.0 ** -5
    codes = np.where(np.isnan(vn), 0.0, vn)
    for i, n in enumerate(lens):
        for j in range(3 + 2 * i, n // bs - 2 * T // bs - 2, every):
            b = tables[i, j]
            codes[b] = 0.0
            codes[b, 1, :, 0] = min(64.0, 2.0 ** (127 - exponent)) * (1 if every > 999 else rng.choice([-1.0, 1.0]))
            kn[b, 1, :, 0] = 64.0
            vs[b] = 2.0 ** exponent
    vn[:] = codes
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    for name, x in (("k", kn), ("v", vn)):
        on[name] = torch.from_numpy(x).to(dt).to(dev)
    on["ks"], on["vs"] = (torch.from_numpy(x).float().to(dev) for x in (ks, vs))
    on["q"] = torch.from_numpy(qx).to(on["q"].dtype).to(dev)
    return on, host, LAG * math.log(2.0) / 2.0


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T,Hq,H,D,bs,dtype", SHAPES)
@pytest.mark.parametrize("exponent", [40, 63, 64, 65, 110, 118, 121])
@pytest.mark.parametrize("splits", [0, 1])
def test_one_value_near_the_largest(dev, policy, fmt, T, Hq, H, D, bs, dtype, exponent, splits):
    """one key, in another place of each sequence, with a value up to 2^127 and a score a little above the rest"""
    policy.setenv("NVLLM_PAGED_SPLITS", splits)
    on, host, scale = far_apart(fmt, T, Hq, H, D, bs, dtype, min(exponent, 121 if fmt == "int8" else 119), 1000, dev)
    compare(call(on, scale), host, scale, dtype)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T,Hq,H,D,bs,dtype", SHAPES)
@pytest.mark.parametrize("exponent", [-126, -60, 30, 64, 105, 118, 121])
def test_every_seventh_block_of_another_size(dev, fmt, T, Hq, H, D, bs, dtype, exponent):
    """up to several keys of 2^127 and equal weight, whose sum is past f32's range while their mean is not"""
    on, host, scale = far_apart(fmt, T, Hq, H, D, bs, dtype, min(exponent, 121 if fmt == "int8" else 119), 7, dev)
    compare(call(on, scale), host, scale, dtype)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T,Hq,H,D,bs,dtype", SHAPES)
def test_scales_over_the_whole_range(dev, fmt, T, Hq, H, D, bs, dtype):
    """every block with a V scale of its own from 2^-126 to 2^110, scores as they fall"""
    rng = np.random.default_rng(21)
    on, host = make(rng, fmt, dtype, [1300 + T, 90 + T, T], T, Hq, H, D, bs, dev)
    vs = host[4]
    some = np.isfinite(vs)
    vs[some] = 2.0 ** rng.integers(-126, 111, int(some.sum()))
    on["vs"].copy_(torch.from_numpy(vs))
    compare(call(on, D ** -0.5), host, D ** -0.5, dtype)


@pytest.mark.parametrize("fmt", FMT)
def test_written_by_the_cache_itself(dev, fmt):
    """a context of ordinary values, then one of 2^127 through the quantising write; the rest of its block is
    zeros at that scale and must stay so in the output"""
    import nano_vllm_rs_amd as nv
    rng = np.random.default_rng(22)
    H, D, bs, n = 2, 128, 16, 700
    at = 500
    k = torch.zeros((n, H, D), dtype=torch.bfloat16)
    v = torch.from_numpy(rng.standard_normal((n, H, D))).to(torch.bfloat16)
    k[at, :, 0] = 2.0
    v[at, :, 0] = 2.0 ** 127
    nb = -(-n // bs)
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    cache = [torch.zeros((nb, bs, H, D), dtype=dt, device=dev) for _ in range(2)]
    scales = [torch.zeros((nb, H), device=dev) for _ in range(2)]
    nv.reshape_and_cache_kv8(k.to(dev), v.to(dev), *cache, *scales, torch.arange(n, device=dev))
    numbers, sc = np.zeros((2, nb, bs, H, D)), np.zeros((2, nb, H))
    o.write(numbers[0], sc[0], k.double().numpy(), list(range(n)), fmt)
    o.write(numbers[1], sc[1], v.double().numpy(), list(range(n)), fmt)
    for T, Hq in ((1, 8), (12, 8), (16, 8), (40, 8)):
        q = torch.zeros((1, T, Hq, D), dtype=torch.bfloat16)
        q[..., 0] = 1.0
        tables = np.arange(nb, dtype=np.int32)[None]
        scale = LAG * math.log(2.0) / 2.0
        got = nv.paged_attention_kv8(q.to(dev), *cache, *scales, torch.from_numpy(tables).to(dev),
                                     torch.tensor([n], dtype=torch.int32, device=dev), scale)
        compare(got, (q.double().numpy(), *numbers, *sc, tables, [n]), scale, "bf16")
