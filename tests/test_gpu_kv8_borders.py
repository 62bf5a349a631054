"""Scales of rotated keys that lie next to a scale's border: K of the producer is known in 64 bits, and the
scale is the smallest power of two for that value, not for its rounding to 32 bits."""
import numpy as np
import pytest
import torch

import kv8_oracle as o
import nano_vllm_rs_amd as nv
from kv8_helpers import ELEM, TORCH, numbers_of

pytestmark = pytest.mark.gpu


def row_at_the_border(rng, D, fmt, above):
    """x, w (f32) with the largest |x w / rms| above (or below) a border by less than 2^-26 of it, so that f32
    rounds it to the border, and by more than 2^-40, which 64-bit arithmetic keeps apart by far"""
    for _ in range(1000):
        x = rng.standard_normal(D).astype(np.float32)
        d = int(rng.integers(D))
        norm = np.float64(x[d]) / np.sqrt((x.astype(np.float64) ** 2).mean() + 1e-6)
        w = (rng.uniform(0.5, 1, D) * 0.01).astype(np.float32)
        border = o.TOP[fmt] * 2.0 ** -4
        w[d] = np.float32(border / abs(norm))
        off = abs(norm) * np.float64(w[d]) / border - 1.0
        if 2.0 ** -40 < (off if above else -off) < 2.0 ** -26:
            return x, w, d
    raise AssertionError("no such row")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("above", [True, False])
@pytest.mark.parametrize("D,bs", [(64, 8), (128, 16), (10, 4)])
def test_scale_of_a_rotated_key(dev, fmt, above, D, bs):
    rng = np.random.default_rng(D)
    for _ in range(6):
        x, w, d = row_at_the_border(rng, D, fmt, above)
        k = torch.from_numpy(x).view(1, 1, D).to(dev)
        one = torch.ones(D, device=dev)
        rot = nv.RotaryEmbedding(D, 4, 1e6, ELEM["f32"], dev)  # position 0: cos 1, sin 0
        kc, vc = (torch.zeros((2, bs, 1, D), dtype=TORCH[fmt], device=dev) for _ in range(2))
        ks, vs = (torch.zeros((2, 1), device=dev) for _ in range(2))
        nv.qk_norm_rope_cache_kv8(k.clone(), k, k, one, torch.from_numpy(w).to(dev), 1e-6, rot,
                                  torch.zeros(1, dtype=torch.int32, device=dev), kc, vc, ks, vs,
                                  torch.tensor([bs], device=dev))
        want, scales = np.zeros((2, bs, 1, D)), np.zeros((2, 1))
        z = np.zeros((1, D))
        o.write(want, scales, o.rotate(x[None, None], w.astype(np.float64), z + 1.0, z, 1e-6), [bs], fmt)
        assert scales[1, 0] == 2.0 ** (-3 if above else -4)
        assert np.array_equal(ks.double().cpu().numpy(), scales)
        got = numbers_of(kc, fmt)
        assert got[1, 0, 0, d] == want[1, 0, 0, d] and np.abs(got - want).max() <= 1.0
