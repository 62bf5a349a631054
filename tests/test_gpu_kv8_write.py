"""The quantising write, the producer and the read-back of the 8-bit cache against the 64-bit oracle.

A plain write is exact by construction (power-of-two scales): codes and scales are compared bit for
bit.  The producer's K is computed in f64 before its one rounding; its tolerance is derived at the test."""
import numpy as np
import pytest
import torch

import kv8_oracle as o
import nano_vllm_rs_amd as nv
from kv8_helpers import ELEM, POISON, TORCH, numbers_of, random_codes, rounded, to_dev

pytestmark = pytest.mark.gpu
FMT = ["int8", "e4m3"]


def _cache(rng, nb, bs, H, D, fmt, dev, spread=3):
    codes = random_codes(rng, (nb, bs, H, D), fmt)
    scales = 2.0 ** rng.integers(-8, -8 + spread, (nb, H))
    return to_dev(codes, fmt, dev), torch.from_numpy(scales).float().to(dev), o.numbers(codes, fmt), scales.copy()


def _same(cache, scales, want, want_scales, fmt):
    assert np.array_equal(scales.double().cpu().numpy(), want_scales)
    got = numbers_of(cache, fmt)
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (np.isnan(got) & np.isnan(want))))[:5]


def _write_both(rng, fmt, dtype, nb, bs, H, D, slots, dev, sigma=1.0, make=None, workspace=None):
    n = len(slots)
    k, kx = rounded(rng, (n, H, D), dtype, sigma)
    v, vx = rounded(rng, (n, H, D), dtype, 0.5 * sigma)
    if make is not None:
        k = make(k)
        kx = k.double().numpy()
    kc, ks, kw, ksw = _cache(rng, nb, bs, H, D, fmt, dev)
    vc, vs, vw, vsw = _cache(rng, nb, bs, H, D, fmt, dev)
    sm = torch.tensor(slots, dtype=torch.int64, device=dev)
    nv.reshape_and_cache_kv8(k.to(dev), v.to(dev), kc, vc, ks, vs, sm, workspace=workspace)
    o.write(kw, ksw, kx, slots, fmt)
    o.write(vw, vsw, vx, slots, fmt)
    _same(kc, ks, kw, ksw, fmt)
    _same(vc, vs, vw, vsw, fmt)
    return kc, vc, ks, vs


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bs,H,D", [(16, 8, 128), (16, 1, 128), (16, 3, 128), (8, 2, 64), (4, 2, 8), (1, 1, 1), (5, 3, 7),
                                    (256, 1, 32), (16, 2, 256)])
def test_sequence_in_order(dev, fmt, dtype, bs, H, D):
    """a first chunk that ends inside a block, and a second one that goes on there"""
    rng = np.random.default_rng(bs * 1000 + H * 10 + D)
    nb = 9
    blocks = rng.permutation(nb)
    slots = [int(blocks[p // bs]) * bs + p % bs for p in range(min(5 * bs, 600))]
    cut = max(1, len(slots) // 2 - 1)
    _write_both(rng, fmt, dtype, nb, bs, H, D, slots[:cut], dev)
    _write_both(rng, fmt, dtype, nb, bs, H, D, slots[cut:], dev, sigma=3.0)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("bs,D", [(16, 128), (8, 64)])
def test_decode_steps_grow_the_scale(dev, fmt, bs, D):
    """one block per sequence filled token by token, values growing: kept rows follow the scale"""
    rng = np.random.default_rng(5)
    nb, H, n = 12, 2, 7
    blocks = rng.permutation(nb)[:n]
    state = [_cache(rng, nb, bs, H, D, fmt, dev) for _ in range(2)]
    for t in range(bs):
        slots = [int(b) * bs + t for b in blocks]
        sm = torch.tensor(slots, dtype=torch.int64, device=dev)
        (k, kx), (v, vx) = (rounded(rng, (n, H, D), "bf16", 1.4 ** t * f) for f in (1.0, 0.01))
        (kc, ks, kw, ksw), (vc, vs, vw, vsw) = state
        nv.reshape_and_cache_kv8(k.to(dev), v.to(dev), kc, vc, ks, vs, sm)
        o.write(kw, ksw, kx, slots, fmt)
        o.write(vw, vsw, vx, slots, fmt)
        _same(kc, ks, kw, ksw, fmt)
        _same(vc, vs, vw, vsw, fmt)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 300, 1024, 1025, 4097, 6001])
def test_any_order_skips_and_repeats(dev, fmt, n):
    """random slots: negative ones and ones past the pool are skipped, of repeats the last wins; both
    ways of finding a block's tokens (1024 is the last that scans), the workspace full of rubbish"""
    rng = np.random.default_rng(n)
    bs, H, D = 16, 2, 128
    nb = max(3, n // 12)
    slots = rng.integers(-20, nb * bs + 20, n).tolist()
    need = nv.capi.lib().nvllm_kv8_write_workspace_bytes(n, bs, nb)
    assert (need > 0) == (n > 1024)
    ws = torch.from_numpy(rng.integers(-5, n + 5, max(need // 4, 4)).astype(np.int32)).to(dev).view(torch.uint8)
    _write_both(rng, fmt, "bf16", nb, bs, H, D, slots, dev, workspace=ws)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("H", [1, 3, 8, 9, 20])
@pytest.mark.parametrize("blocks", [3, 40, 700])
def test_few_rows_of_a_block(dev, fmt, H, blocks):
    """one, two, three or all rows of blocks that hold others, mixed in one call; some begin, some grow"""
    rng = np.random.default_rng(H + blocks)
    bs, D = 16, 128
    slots = []
    for b in rng.permutation(blocks + 2)[:blocks].tolist():
        rows = rng.permutation(bs)[:rng.choice([1, 1, 2, 2, 3, 16])]
        slots += [b * bs + int(r) for r in rows]
    rng.shuffle(slots)
    _write_both(rng, fmt, "bf16", blocks + 2, bs, H, D, slots, dev, sigma=4.0)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [128, 64])
def test_values_at_the_edges(dev, fmt, dtype, D):
    """zeros, subnormals, the largest finite values, infinities, NaN, ties, amax on a scale's border"""
    rng = np.random.default_rng(17)
    bs, H = 16, 4
    top = o.TOP[fmt]

    def make(k):
        k = k.clone()
        k[0:16, 0] = 0.0                                    # a block of zeros
        k[0:16, 1] = 1e-40                                  # subnormal
        k[16:32, 0, 0] = float("inf")
        k[16:32, 1, 0] = float("-inf")
        k[16:32, 2, 3] = float("nan")
        k[32:48, 0, 5] = 3e38
        k[32:48, 1, 5] = -2.0 ** 127
        k[32:48, 2] = top * 2.0 ** -3                       # on the border
        k[48:64, 0] = torch.arange(16)[:, None].to(k.dtype) + 0.5  # ties
        k[48, 0, 0] = 100.0
        k[48:64, 1] = float("inf")                          # nothing finite
        k[48:64, 2, 1] = 0.0
        return k

    _write_both(rng, fmt, dtype, 6, bs, H, D, list(range(16, 80)), dev, make=make)


@pytest.mark.parametrize("n", [60, 3000])
def test_nothing_is_written_outside(dev, n):
    """a pool between guards, outputs and workspace with a tail: only what the call names changes"""
    rng = np.random.default_rng(n)
    bs, H, Hq, D, nb = 16, 2, 4, 128, 300
    edge = bs * H * D
    mem = [torch.full(((nb + 2) * edge,), 0x55, dtype=torch.uint8, device=dev) for _ in range(2)]
    scale_mem = [torch.full(((nb + 2) * H,), 3.0, device=dev) for _ in range(2)]
    kc, vc = (m[edge:-edge].view(nb, bs, H, D).view(torch.int8) for m in mem)
    ks, vs = (m[H:-H].view(nb, H) for m in scale_mem)
    q = torch.randn((n, Hq, D), device=dev).to(torch.bfloat16)
    k, v = (torch.randn((n, H, D), device=dev).to(torch.bfloat16) for _ in range(2))
    q_mem, k_mem = (torch.full((n + 1, h, D), 7.0, dtype=torch.bfloat16, device=dev) for h in (Hq, H))
    need = nv.capi.lib().nvllm_kv8_write_workspace_bytes(n, bs, nb)
    ws = torch.full((need + 4096,), 0xa5, dtype=torch.uint8, device=dev)
    slots = torch.from_numpy(rng.permutation((nb // 2) * bs)[:n] + (nb // 2) * bs if n < 1000 else
                             rng.permutation(nb * bs)[:n]).to(dev)
    slots[0], slots[1] = -1, nb * bs
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    rot = nv.RotaryEmbedding(D, 64, 1e6, torch.bfloat16, dev)
    pos = torch.from_numpy(rng.integers(0, 64, n).astype(np.int32)).to(dev)
    nv.qk_norm_rope_cache_kv8(q, k, v, w, w, 1e-6, rot, pos, kc, vc, ks, vs, slots, k_out=k_mem[:n], q_out=q_mem[:n],
                              workspace=ws[:need] if need else None)
    assert bool((q_mem[n] == 7.0).all()) and bool((k_mem[n] == 7.0).all()) and bool((ws[need:] == 0xa5).all())
    for m in mem:
        assert bool((m[:edge] == 0x55).all()) and bool((m[-edge:] == 0x55).all())
    for m in scale_mem:
        assert bool((m[:H] == 3.0).all()) and bool((m[-H:] == 3.0).all())
    touched = torch.zeros(nb, dtype=torch.bool, device=dev)
    live = slots[(slots >= 0) & (slots < nb * bs)]
    touched[live // bs] = True
    for c, s in ((kc, ks), (vc, vs)):
        assert bool((c[~touched].view(torch.uint8) == 0x55).all()) and bool((s[~touched] == 3.0).all())


def test_empty_call_and_untouched_blocks(dev):
    rng = np.random.default_rng(1)
    kc, ks, kw, ksw = _cache(rng, 4, 16, 2, 128, "int8", dev)
    e = torch.empty((0, 2, 128), dtype=torch.bfloat16, device=dev)
    nv.reshape_and_cache_kv8(e, e, kc, kc.clone(), ks, ks.clone(), torch.empty(0, dtype=torch.int64, device=dev))
    _same(kc, ks, kw, ksw, "int8")


def test_slots_past_32_bits_of_bytes(dev):
    """a pool whose codes pass 2^32 bytes: the last block is written and read back"""
    bs, H, D = 16, 8, 128
    nb = (1 << 32) // (bs * H * D) + 3
    kc, vc = (torch.zeros((nb, bs, H, D), dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((nb, H), device=dev) for _ in range(2))
    k = torch.randn((bs, H, D), device=dev).to(torch.bfloat16)
    sm = torch.arange((nb - 1) * bs, nb * bs, device=dev)
    nv.reshape_and_cache_kv8(k, k, kc, vc, ks, vs, sm)
    ids = torch.tensor([nb - 1, 0], dtype=torch.int32, device=dev)
    got, _ = nv.gather_cache_blocks_kv8(kc, vc, ks, vs, ids, torch.float32)
    assert bool((got[0] - k.float()).abs().max() <= ks[-1].max() / 2) and float(got[1].abs().max()) == 0.0
    assert int((kc != 0).flatten(1).any(1).sum()) == 1


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bs,H,D", [(16, 8, 128), (8, 2, 64), (5, 3, 7), (4, 1, 8)])
def test_read_back_is_exact(dev, fmt, dtype, bs, H, D):
    rng = np.random.default_rng(7)
    nb = 20
    kc, ks, kw, ksw = _cache(rng, nb, bs, H, D, fmt, dev, spread=9)
    vc, vs, vw, vsw = _cache(rng, nb, bs, H, D, fmt, dev, spread=9)
    ids = np.array([3, 0, 19, 3, -1, 20, 7, 2 ** 31 - 1], dtype=np.int32)
    k, v = nv.gather_cache_blocks_kv8(kc, vc, ks, vs, torch.from_numpy(ids).to(dev), ELEM[dtype])
    for got, num, sc in ((k, kw, ksw), (v, vw, vsw)):
        for i, b in enumerate(ids):
            want = num[b] * sc[b][None, :, None] if 0 <= b < nb else np.zeros((bs, H, D))
            assert np.array_equal(got[i].double().cpu().numpy(), want)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [128, 6])
def test_read_back_of_the_smallest_and_largest_scales(dev, fmt, dtype, D):
    """every code at the scales' ends: exact in f32; in bf16 rounded to nearest where it has no such number"""
    codes = np.arange(256, dtype=np.uint8)
    codes[[0x7f, 0xff]] = 0  # E4M3's NaN
    raw = np.resize(codes, (2, 16, 2, D))
    raw[1] = np.resize(codes[::-1], (16, 2, D))
    scales = np.array([[2.0 ** -126, 2.0 ** -124], [2.0 ** -120, 2.0 ** 119]])
    on = to_dev(raw, fmt, dev)
    s = torch.from_numpy(scales).float().to(dev)
    k, v = nv.gather_cache_blocks_kv8(on, on, s, s, torch.arange(2, dtype=torch.int32, device=dev), ELEM[dtype])
    want = torch.from_numpy(o.numbers(raw, fmt) * scales[:, None, :, None]).float().to(ELEM[dtype])
    assert torch.equal(k.cpu(), want) and torch.equal(v, k)


@pytest.mark.parametrize("fmt", FMT)
def test_layer_cache_and_gather(dev, fmt):
    cfg = nv.KVCacheConfig(16, 16, 8, 128, 2, TORCH[fmt])
    cache = nv.KVCache(cfg, dev)
    layer = cache.layer(0)
    assert layer.key_cache().dtype == TORCH[fmt] and tuple(layer.key_scales().shape) == (16, 8)
    k = torch.randn((32, 8, 128), device=dev).to(torch.bfloat16)
    nv.reshape_and_cache_kv8(k, 2 * k, layer.key_cache(), layer.value_cache(), layer.key_scales(),
                             layer.value_scales(), torch.arange(32, device=dev) + 48)
    ids = torch.tensor([3, 4], dtype=torch.int32, device=dev)
    want = nv.gather_cache_blocks_kv8(layer.key_cache(), layer.value_cache(), layer.key_scales(),
                                      layer.value_scales(), ids)
    assert torch.equal(layer.gather_keys([3, 4]), want[0]) and torch.equal(layer.gather_values([3, 4]), want[1])
    assert torch.equal(want[1], 2 * want[0])
    assert cfg.layer_cache_size_bytes() == layer.key_cache().numel() + 4 * layer.key_scales().numel()


# ---------------------------------------------------------------------------------- producer

def _producer(rng, fmt, dtype, n, Hq, H, D, bs, dev, slots, nb, k_out=True):
    q, qx = rounded(rng, (n, Hq, D), dtype)
    k, kx = rounded(rng, (n, H, D), dtype)
    v, vx = rounded(rng, (n, H, D), dtype)
    qw, qwx = rounded(rng, (D,), dtype)
    kw, kwx = rounded(rng, (D,), dtype)
    rot = nv.RotaryEmbedding(D, 512, 1e6, ELEM[dtype], dev)
    pos = rng.integers(0, 512, n).astype(np.int32)
    kc, ks, kn, ksn = _cache(rng, nb, bs, H, D, fmt, dev)
    vc, vs, vn, vsn = _cache(rng, nb, bs, H, D, fmt, dev)
    qd = q.to(dev)
    q_out = torch.empty_like(qd)
    ko = torch.full((n, H, D), float("nan"), dtype=ELEM[dtype], device=dev) if k_out else None
    sm = torch.tensor(slots, dtype=torch.int64, device=dev)
    r = nv.qk_norm_rope_cache_kv8(qd, k.to(dev), v.to(dev), qw.to(dev), kw.to(dev), 1e-6, rot,
                                  torch.from_numpy(pos).to(dev), kc, vc, ks, vs, sm, k_out=ko, q_out=q_out)
    assert r is q_out and torch.equal(qd.cpu(), q)
    cos, sin = (t.double().cpu().numpy()[pos] for t in (rot.cos_cache(), rot.sin_cache()))
    return dict(q=o.rotate(qx, qwx, cos, sin, 1e-6), vx=vx,
                q_out=q_out, k_out=ko, k=(kc, ks, kn, ksn), v=(vc, vs, vn, vsn), krot=o.rotate(kx, kwx, cos, sin, 1e-6))


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,Hq,H,D,bs", [(1, 16, 8, 128, 16), (37, 16, 8, 128, 16), (19, 4, 2, 64, 8), (9, 6, 3, 10, 4),
                                         (5, 2, 1, 256, 16), (4100, 2, 1, 128, 16)])
@pytest.mark.parametrize("step", [1, 17])
def test_producer(dev, fmt, dtype, n, Hq, H, D, bs, step):
    """q_out and k_out: f32 arithmetic of some ten operations (each off by 2^-24 of terms no larger than
    |a| + |b| of the pair), the sum of squares (relative D * 2^-24 at worst), one rounding.  Codes: V is
    exact.  K is computed in f64, its value known to some (D / 2 + 12) 2^-53 of its pair: a code may differ
    by one step where a border lies that near, its scale only where amax lies within 2^-24 of a border of
    its own, which none of these inputs does."""
    rng = np.random.default_rng(n * 7 + D)
    nb = n * step // bs + 6
    at = np.arange(n) * step  # 1: in order; 17: a row of every block
    slots = (rng.permutation(nb)[at // bs] * bs + at % bs).tolist()
    if n > 4:
        slots[2] = -1
    r = _producer(rng, fmt, dtype, n, Hq, H, D, bs, dev, slots, nb)
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    err = (D / 2 + 12) * 2.0 ** -24
    kx = r["krot"]

    def pair(x):  # |a| + |b| of each value's rotation pair
        h = D // 2
        return np.concatenate([np.abs(x[..., :h]) + np.abs(x[..., h:])] * 2, -1) * 2

    for got, want in ((r["q_out"], r["q"]), (r["k_out"], kx)):
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= half * np.abs(want) + err * pair(want) + 1e-37)
    vc, vs, vn, vsn = r["v"]
    o.write(vn, vsn, r["vx"], slots, fmt)
    _same(vc, vs, vn, vsn, fmt)
    kc, ks, kn, ksn = r["k"]
    o.write(kn, ksn, kx, slots, fmt)
    assert np.array_equal(ks.double().cpu().numpy(), ksn)
    got = numbers_of(kc, fmt)
    at = np.argwhere(got != kn)
    err = (D / 2 + 12) * 2.0 ** -53
    token = {s: t for t, s in enumerate(slots)}
    for b, row, h, d in at:
        t = token[b * bs + row]
        y, tol = kx[t, h, d] / ksn[b, h], err * pair(kx)[t, h, d] / ksn[b, h]
        assert o.encode(y - tol, fmt) <= got[b, row, h, d] <= o.encode(y + tol, fmt)
    assert len(at) <= 1 + 1e-3 * got.size


def test_producer_in_place_without_k_out(dev):
    """q_out = q (the default), no k_out; the same bits as with separate tensors"""
    rng = np.random.default_rng(2)
    n, Hq, H, D, bs, nb = 33, 16, 8, 128, 16, 5
    q, k, v = (rounded(rng, (n, h, D), "bf16")[0].to(dev) for h in (Hq, H, H))
    w = rounded(rng, (D,), "bf16")[0].to(dev)
    rot = nv.RotaryEmbedding(D, 64, 1e6, torch.bfloat16, dev)
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    outs = []
    for in_place in (False, True):
        kc, vc = (torch.zeros((nb, bs, H, D), dtype=torch.int8, device=dev) for _ in range(2))
        ks, vs = (torch.zeros((nb, H), device=dev) for _ in range(2))
        qq = q.clone()
        y = nv.qk_norm_rope_cache_kv8(qq, k, v, w, w, 1e-6, rot, pos, kc, vc, ks, vs, torch.arange(n, device=dev),
                                      q_out=None if in_place else torch.empty_like(qq),
                                      k_out=None if in_place else torch.empty_like(k))
        outs.append((y, kc, vc, ks, vs))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [128, 64])
def test_producer_q_is_the_wide_producers(dev, D):
    """q_out and k_out of the producer with a bf16 cache and of this one: the same operation on the same
    inputs, each within its rounding of the other"""
    rng = np.random.default_rng(3)
    n, Hq, H, bs, nb = 40, 8, 2, 16, 4
    q, k, v = (rounded(rng, (n, h, D), "bf16")[0].to(dev) for h in (Hq, H, H))
    w = rounded(rng, (D,), "bf16")[0].to(dev)
    rot = nv.RotaryEmbedding(D, 64, 1e6, torch.bfloat16, dev)
    pos, sm = torch.arange(n, dtype=torch.int32, device=dev), torch.arange(n, device=dev)
    kc, vc = (torch.zeros((nb, bs, H, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    q1, k1, q2, k2 = (torch.empty_like(x) for x in (q, k, q, k))
    nv.qk_norm_rope_cache(q, k, v, w, w, 1e-6, rot, pos, kc, vc, sm, k_out=k1, q_out=q1)
    c8 = [torch.zeros((nb, bs, H, D), dtype=torch.int8, device=dev) for _ in range(2)]
    s8 = [torch.zeros((nb, H), device=dev) for _ in range(2)]
    nv.qk_norm_rope_cache_kv8(q, k, v, w, w, 1e-6, rot, pos, *c8, *s8, sm, k_out=k2, q_out=q2)
    for a, b in ((q1, q2), (k1, k2)):
        # both round the same value, known to 2^-16 at worst: at most one bf16 step apart
        assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * a.float().abs() + 2.0 ** -16).all())


# ------------------------------------------------------------------------- streams, graphs

def test_other_stream_and_graph_replays(dev):
    """captured write and read-back replayed on changing inputs, eager work in between, against an
    eager cache that makes the same calls; both ways of finding the tokens"""
    rng = np.random.default_rng(9)
    for n in (40, 5000):
        bs, H, D, nb = 16, 2, 128, 400
        k, v = (torch.zeros((n, H, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
        slots = torch.zeros(n, dtype=torch.int64, device=dev)
        ids = torch.arange(nb, dtype=torch.int32, device=dev)
        mk = lambda: [torch.zeros((nb, bs, H, D), dtype=torch.int8, device=dev) for _ in range(2)] + \
            [torch.zeros((nb, H), device=dev) for _ in range(2)]
        a, b = mk(), mk()
        ws = torch.empty(max(16, nv.capi.lib().nvllm_kv8_write_workspace_bytes(n, bs, nb)), dtype=torch.uint8, device=dev)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):  # warm-up outside the capture; what it writes is written again below
            nv.reshape_and_cache_kv8(k, v, *a, slots - 1, workspace=ws)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            nv.reshape_and_cache_kv8(k, v, *a, slots, workspace=ws)
            out = nv.gather_cache_blocks_kv8(*a, ids)
        for step in range(4):
            k.copy_(torch.from_numpy(rng.standard_normal((n, H, D)) * 1.7 ** step))
            v.copy_(torch.from_numpy(rng.standard_normal((n, H, D))))
            slots.copy_(torch.from_numpy(rng.permutation(nb * bs)[:n]))
            nv.reshape_and_cache_kv8(k, v, *b, slots)
            want = nv.gather_cache_blocks_kv8(*b, ids)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(list(out) + a, list(want) + b):
                assert torch.equal(x, y), (n, step)
