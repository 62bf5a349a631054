"""Sizes past what the 8-bit cache's kernels count in 32 bits are refused (no call here launches)."""
import pytest

import nano_vllm_rs_amd as nv
from test_kv8_overlaps import CACHE
from test_kv8_refusals import gather, producer, write

C = nv.capi


@pytest.mark.parametrize("f", [write, producer])
@pytest.mark.parametrize("H", [65536, 1 << 27, 1 << 30, (1 << 31) - 1])
def test_kv_heads_of_the_writers(f, H):
    """a workgroup counts 32 H pairs of block and head (K and V, up to 16 blocks)"""
    assert f(**dict(CACHE, H=H, D=2 if H < 1 << 30 else 1, bs=1, nb=1)) == C.NVLLM_ERR_UNSUPPORTED


@pytest.mark.parametrize("Hq", [65536, (1 << 31) - 1])
def test_heads_of_the_producer(Hq):
    """a token has Hq + H rows"""
    assert producer(**dict(CACHE, Hq=Hq)) == C.NVLLM_ERR_UNSUPPORTED


@pytest.mark.parametrize("n", [1 << 31, 1 << 33, 1 << 62, (1 << 63) - 1])
def test_ids_of_the_read_back(n):
    """ids times values of a block are counted in 64 bits"""
    assert gather(n=n) == C.NVLLM_ERR_UNSUPPORTED
