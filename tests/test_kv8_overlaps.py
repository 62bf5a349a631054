"""What the 8-bit cache's writers refuse because waves of one launch would write what others read or write (no call
here launches)."""
import ctypes

import pytest

import nano_vllm_rs_amd as nv
from test_kv8_refusals import producer, write

C = nv.capi
P = ctypes.c_void_p
Q, QO, KO = 0x100000, 0x200000, 0x300000
Q_BYTES, K_BYTES = 4 * 16 * 128 * 2, 4 * 8 * 128 * 2
CACHE = dict(kc=P(0x400000), vc=P(0x500000), ks=P(0x600000), vs=P(0x700000))
CODES, SCALES = 4 * 16 * 8 * 128, 4 * 8 * 4


def refused(rc):
    return rc == C.NVLLM_ERR_CONFIG and "overlap" in C.last_error()


@pytest.mark.parametrize("f", [write, producer])
def test_k_and_v_of_the_cache(f):
    """two waves would write one block"""
    for a, b, n in (("kc", "vc", CODES), ("ks", "vs", SCALES)):
        at = CACHE[a].value
        for off in (0, n - 4, 4 - n):
            assert refused(f(**dict(CACHE, **{b: P(at + off)}))), (b, off)


def test_outputs_of_the_producer():
    """rows of q are read while rows of q_out and k_out are written: q_out is q itself or somewhere else, k_out is
    neither"""
    free = dict(CACHE, q=P(Q), q_out=P(QO), k_out=P(KO))
    for off in (256, 2, Q_BYTES - 2, 2 - Q_BYTES, -256):
        assert refused(producer(**dict(free, q_out=P(Q + off)))), off
    for at in (Q, QO):
        for off in (0, 256, Q_BYTES - 2, 2 - K_BYTES):
            assert refused(producer(**dict(free, k_out=P(at + off)))), (at, off)
    for off in (0, 256, 2 - K_BYTES):
        assert refused(producer(**dict(free, q_out=P(Q), k_out=P(Q + off)))), off
