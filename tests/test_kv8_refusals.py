"""What the 8-bit cache's entries refuse, and what they answer without a GPU (no call here launches)."""
import ctypes

import pytest
import torch

import nano_vllm_rs_amd as nv

C = nv.capi
FAKE, ODD = ctypes.c_void_p(0x10000), ctypes.c_void_p(0x10001)
KEY, VALUE = ctypes.c_void_p(0x80000), ctypes.c_void_p(0xa0000)


def write(**kw):
    a = dict(key=FAKE, value=ctypes.c_void_p(0x20000), kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, slots=FAKE, ws=None, wsb=0, n=4, H=8,
             D=128, bs=16, nb=4, fmt=0, dt=0)
    a.update(kw)
    return C.lib().nvllm_reshape_and_cache_kv8(*a.values(), None)


def producer(**kw):
    a = dict(q=FAKE, k=KEY, v=VALUE, q_out=FAKE, k_out=None, qw=FAKE, kw=FAKE, eps=1e-6, cos=FAKE, sin=FAKE, maxp=64, pos=FAKE, kc=FAKE,
             vc=FAKE, ks=FAKE, vs=FAKE, slots=FAKE, ws=None, wsb=0, n=4, Hq=16, H=8, D=128, bs=16, nb=4, fmt=0, dt=0)
    a.update(kw)
    return C.lib().nvllm_qk_norm_rope_cache_kv8(*a.values(), None)


def gather(**kw):
    a = dict(kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, ids=FAKE, n=4, ko=FAKE, vo=FAKE, nb=4, bs=16, H=8, D=128, fmt=0, dt=0)
    a.update(kw)
    return C.lib().nvllm_gather_cache_blocks_kv8(*a.values(), None)


def attend(**kw):
    a = dict(q=FAKE, kc=FAKE, vc=FAKE, ks=FAKE, vs=FAKE, bt=FAKE, cl=FAKE, out=FAKE, ws=FAKE, wsb=1 << 40, N=2, T=1, Hq=16, H=8, D=128,
             bs=16, mb=4, nb=8, scale=0.1, fmt=0, dt=0)
    a.update(kw)
    return C.lib().nvllm_paged_attn_kv8(*a.values(), None)


GEOMETRY = [("H", 0), ("H", -1), ("D", 0), ("bs", 0), ("nb", 0)]


@pytest.mark.parametrize("f", [write, producer, gather, attend])
def test_geometry_formats_and_alignment(f):
    for name, x in GEOMETRY:
        assert f(**{name: x}) == C.NVLLM_ERR_CONFIG, name
    for name, x in (("fmt", 2), ("fmt", -1), ("dt", 2), ("D", 257), ("D", 258), ("bs", 257),
                    ("H", 1 << 24)):
        assert f(**{name: x}) == C.NVLLM_ERR_UNSUPPORTED, (name, x)
    assert f(ks=ODD) == C.NVLLM_ERR_CONFIG and "aligned" in C.last_error()
    for name in ("kc", "ks"):
        assert f(**{name: None}) == C.NVLLM_ERR_NULL, name


def test_write():
    assert write(n=0, key=None) == C.NVLLM_OK
    assert write(n=-1) == C.NVLLM_ERR_CONFIG
    for n in (1 << 62, (1 << 30) + 1):
        for f in (write, producer):
            assert f(n=n, wsb=1 << 40, ws=FAKE) == C.NVLLM_ERR_UNSUPPORTED
    for name in ("key", "value", "vc", "vs", "slots"):
        assert write(**{name: None}) == C.NVLLM_ERR_NULL
    assert write(key=ODD) == C.NVLLM_ERR_CONFIG and write(dt=1, value=ctypes.c_void_p(0x10002)) == C.NVLLM_ERR_CONFIG
    assert write(slots=ctypes.c_void_p(0x10004)) == C.NVLLM_ERR_CONFIG


def test_write_workspace():
    need = C.lib().nvllm_kv8_write_workspace_bytes
    assert need(1024, 16, 100) == 0 and need(1025, 16, 100) == 6400 and need(0, 16, 100) == 0 and need(9999, 0, 5) == 0
    assert need(4097, 16, 1 << 28) == 1 << 34
    assert write(n=4097, nb=100) == C.NVLLM_ERR_CONFIG and "needs 6400" in C.last_error()
    assert write(n=4097, nb=100, ws=FAKE, wsb=6399) == C.NVLLM_ERR_CONFIG
    assert write(n=4097, nb=100, ws=ctypes.c_void_p(0x10004), wsb=6400) == C.NVLLM_ERR_CONFIG
    assert "16-byte aligned" in C.last_error()


def test_producer():
    assert producer(n=0) == C.NVLLM_OK
    for name, x in (("n", -1), ("Hq", 0), ("maxp", 0), ("maxp", 1 << 31), ("D", 127)):
        assert producer(**{name: x}) == C.NVLLM_ERR_CONFIG, name
    for name in ("q", "k", "v", "q_out", "qw", "kw", "cos", "sin", "pos", "vc", "vs", "slots"):
        assert producer(**{name: None}) == C.NVLLM_ERR_NULL, name
    last = 4 * 8 * 128 * 2 - 2  # offset of the last element of k, v
    for at in (KEY, VALUE):
        for name in ("k_out", "q_out"):
            for off in (0, last):
                assert producer(**{name: ctypes.c_void_p(at.value + off)}) == C.NVLLM_ERR_CONFIG and "overlap" in C.last_error()
        assert producer(q_out=ctypes.c_void_p(at.value - 4 * 16 * 128 * 2 + 2)) == C.NVLLM_ERR_CONFIG
        assert "overlap" in C.last_error()
    assert producer(pos=ODD) == C.NVLLM_ERR_CONFIG and producer(cos=ODD) == C.NVLLM_ERR_CONFIG


def test_gather():
    assert gather(n=0) == C.NVLLM_ERR_CONFIG and "empty" in C.last_error()
    for name in ("ids", "ko", "vc", "vs"):
        assert gather(**{name: None}) == C.NVLLM_ERR_NULL


def test_attend():
    assert attend(N=0) == C.NVLLM_OK
    for name, x in (("N", -1), ("T", 0), ("Hq", 0), ("Hq", 17), ("mb", 0)):
        assert attend(**{name: x}) == C.NVLLM_ERR_CONFIG, name
    for name, x in (("N", 65536), ("T", 1 << 30), ("mb", (1 << 26) + 1)):
        assert attend(**{name: x}) == C.NVLLM_ERR_UNSUPPORTED, name
    assert attend(Hq=1 << 17, H=1 << 17, D=8) == C.NVLLM_ERR_UNSUPPORTED
    for name in ("q", "vc", "vs", "bt", "cl", "out"):
        assert attend(**{name: None}) == C.NVLLM_ERR_NULL
    assert attend(q=ODD) == C.NVLLM_ERR_CONFIG and attend(dt=1, out=ctypes.c_void_p(0x10002)) == C.NVLLM_ERR_CONFIG


def test_path_and_sizes():
    assert nv.paged_attention_kv8_path(4, 1, 4, 2, 8, 4, 3) == "generic"
    assert nv.paged_attention_kv8_path(4, 1, 16, 8, 128, 16, 3, dtype=torch.float32) == "generic"
    for T, Hq in ((1, 8), (1, 32), (4, 32), (12, 32), (48, 8)):
        assert nv.paged_attention_kv8_path(4, T, Hq, 8, 128, 16, 3) == "decode"
    for T, Hq in ((13, 32), (49, 8), (4, 128), (1024, 16)):
        assert nv.paged_attention_kv8_path(4, T, Hq, 8, 128, 16, 3) == "tile"
        assert nv.paged_attention_kv8_path(4, T, Hq, 8, 128, 8, 3) == "generic"
    with pytest.raises(nv.ConfigError):
        nv.paged_attention_kv8_path(4, 1, 17, 8, 128, 16, 3)
    L = C.lib()
    assert L.nvllm_paged_attn_kv8_workspace_bytes(4, 1, 4, 2, 8, 4, 3, 0) == 0
    assert L.nvllm_paged_attn_kv8_workspace_bytes(4, 1, 5, 2, 8, 4, 3, 0) == 0
    need = L.nvllm_paged_attn_kv8_workspace_bytes(2, 1, 16, 8, 128, 16, 64, 0)
    assert need > 0 and attend(mb=64, wsb=need - 1) == C.NVLLM_ERR_CONFIG and "needs %d" % need in C.last_error()
    assert attend(mb=64, ws=None) == C.NVLLM_ERR_CONFIG
    assert attend(mb=64, ws=ctypes.c_void_p(0x10008)) == C.NVLLM_ERR_CONFIG
    for name in ("q", "kc", "vc", "out"):
        assert attend(**{name: ctypes.c_void_p(0x10008)}) == C.NVLLM_ERR_CONFIG, name
    assert L.nvllm_kv_cache_kv8_layer_bytes(10, 16, 8, 128) == 10 * 8 * (16 * 128 + 4)
    assert L.nvllm_kv_cache_kv8_layer_bytes(10, -1, 8, 128) == -1
    for dt in (torch.int8, torch.float8_e4m3fn):
        cfg = nv.KVCacheConfig(10, 16, 8, 128, 3, dt)
        assert cfg.layer_cache_size_bytes() == 10 * 8 * 2052 and cfg.total_cache_size_bytes() == 6 * 10 * 8 * 2052


def test_python_refuses_before_the_library():
    """shapes, dtypes and devices; the wide operators refuse an 8-bit cache (they would misread it)"""
    k = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    kc = torch.zeros((4, 16, 2, 128), dtype=torch.int8)
    ks = torch.zeros((4, 2))
    sm = torch.zeros(3, dtype=torch.int64)
    ok = [k, k, kc, kc, ks, ks, sm]

    def bad(i, x, err=nv.ConfigError):
        args = list(ok)
        args[i] = x
        with pytest.raises(err):
            nv.reshape_and_cache_kv8(*args)

    bad(0, k, RuntimeError)                                   # not on a device
    bad(0, k[:, :1])
    bad(1, k[:2])
    bad(2, kc.float())
    bad(3, kc.view(torch.float8_e4m3fn))
    bad(4, ks.double())
    bad(5, ks[:3])
    bad(6, sm.int())
    bad(6, sm[:2])
    bad(0, k.half())
    bt, cl = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros((1, 1, 4, 128), dtype=torch.bfloat16)
    for args in ((q[..., :64], kc, kc, ks, ks, bt, cl), (q, kc, kc, ks, ks, bt.long(), cl), (q, kc, kc, ks, ks, bt, cl[:0])):
        with pytest.raises(nv.ConfigError):
            nv.paged_attention_kv8(*args, 0.1)
    with pytest.raises(nv.ConfigError):
        nv.gather_cache_blocks_kv8(kc, kc, ks, ks, sm)
    with pytest.raises(nv.ConfigError):
        nv.gather_cache_blocks_kv8(kc, kc, ks, ks, cl, torch.float16)
