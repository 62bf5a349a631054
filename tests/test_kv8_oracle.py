"""The oracle of the 8-bit cache against torch's E4M3 and against the definition (CPU)."""
import numpy as np
import pytest
import torch

import kv8_oracle as o


def test_e4m3_table_is_torchs():
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(o.e4m3_table(), want, equal_nan=True)


def test_encode_is_the_nearest_number():
    y = np.random.default_rng(0).uniform(-448, 448, 4000) * 2.0 ** np.random.default_rng(1).integers(-14, 1, 4000)
    want = torch.from_numpy(y).to(torch.float8_e4m3fn).double().numpy()
    # (torch rounds f64 by way of f32: the same unless f32 lands on a tie, which none of these does)
    assert np.array_equal(o.encode(y, "e4m3"), want)
    got = o.encode(y, "int8")
    assert np.all(np.abs(got - np.clip(y, -127, 127)) <= 0.5) and np.all(got == np.rint(got))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_scale_is_the_smallest_power_of_two(fmt):
    for a in (1e-45, 1e-30, 0.3, 1.0, 127.0, 127.00001, 448.0, 448.0001, 1e30):
        s = o.scale_of(a, fmt)
        assert a <= o.TOP[fmt] * s and np.log2(s) == round(np.log2(s))
        assert s == 2.0 ** -126 or a > o.TOP[fmt] * s / 2


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_a_block_filled_token_by_token_is_off_by_less_than_a_step(fmt):
    """Growing scales: each kept code is rounded once more at a growth.  int8: less than one step of the
    final scale (1/2 + 1/4 + ...).  E4M3: the roundings after the first only touch values whose step is
    the smallest one, 2^-9 of the scale, so 2^-4 of the value or one such step."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((16, 1, 64)) * (1.5 ** np.arange(16))[:, None, None]
    cache, scales = np.zeros((1, 16, 1, 64)), np.zeros((1, 1))
    seen = set()
    for t in range(16):
        o.write(cache, scales, x[t:t + 1], [t], fmt)
        seen.add(scales[0, 0])
    assert len(seen) > 4
    err = np.abs(cache[0, :, 0] * scales[0, 0] - x[:, 0])
    s = scales[0, 0]
    bound = s if fmt == "int8" else np.maximum(np.abs(x[:, 0]) * 2.0 ** -4, s * 2.0 ** -9)
    assert np.all(err <= bound)
