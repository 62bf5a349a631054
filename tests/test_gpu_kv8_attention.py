"""Attention over the 8-bit cache against the 64-bit oracle.

Every place that no call may look at holds poison: rows past a context (E4M3 NaN codes, int8's unused
-128), blocks no table names, their scales (NaN), table entries past a sequence's blocks.

Tolerance per output value, with A = the attention-weighted mean of |v|, S = the largest sum |q||k| times
the softmax scale of the row, u = 2^-24:
  scores      (D + 8) u S absolute (products and sums of D terms, the two scale products, the exp2 domain)
  exp         8 u relative (the hardware's exp2 and expf are within a few ulp)
  p rounded   2^-8 relative, bf16 only (the matrix unit takes bf16)
  sums        n u relative over n keys, for numerator and denominator
  output      2^-8 relative in bf16, 2^-24 in f32
so |err| <= half |out| + A (2 ((D + 8) u S + 8 u + n u) + [bf16] 2^-8) (1 + 2^-6)."""
import numpy as np
import pytest
import torch

import kv8_oracle as o
import nano_vllm_rs_amd as nv
from kv8_helpers import ELEM, POISON, gentle_codes, rounded, to_dev

pytestmark = pytest.mark.gpu
FMT = ["int8", "e4m3"]


def tolerance(want, mean, reach, n, D, dtype):
    u = 2.0 ** -24
    half = 2.0 ** -8 if dtype == "bf16" else u
    return half * np.abs(want) + mean * (2 * ((D + 8) * u * reach + 8 * u + n * u)
                                         + (2.0 ** -8 if dtype == "bf16" else 0)) * (1 + 2.0 ** -6) + 1e-37


def make(rng, fmt, dtype, lens, T, Hq, H, D, bs, dev, slack=2, spread=3, shared=0, sigma=1.0):
    N = len(lens)
    used = [max(0, -(-n // bs)) for n in lens]
    width = max(max(used), 1) + slack
    nb = sum(used) + 4
    perm = rng.permutation(nb).tolist()
    k, v = (np.full((nb, bs, H, D), POISON[fmt], dtype=np.uint8) for _ in range(2))
    ks, vs = (np.full((nb, H), np.nan) for _ in range(2))
    tables = np.full((N, width), -7, dtype=np.int32)
    tables[:, -1] = 2 ** 31 - 1
    first = None
    for i, n in enumerate(lens):
        for j in range(used[i]):
            if first is not None and j < shared and j < len(first):
                tables[i, j] = first[j]
                continue
            b = perm.pop()
            tables[i, j] = b
            live = min(bs, n - j * bs) if j >= shared else bs
            k[b, :live] = gentle_codes(rng, (live, H, D), fmt)
            v[b, :live] = gentle_codes(rng, (live, H, D), fmt)
            base = -5 if fmt == "int8" else -7
            ks[b] = 2.0 ** rng.integers(base - spread + 2, base + 1, H)
            vs[b] = 2.0 ** rng.integers(base - spread + 2, base + 1, H)
        if first is None and shared:
            first = tables[i, :used[i]].copy()
    q, qx = rounded(rng, (N, T, Hq, D), dtype, sigma)
    on = dict(q=q.to(dev), k=to_dev(k, fmt, dev), v=to_dev(v, fmt, dev), ks=torch.from_numpy(ks).float().to(dev),
              vs=torch.from_numpy(vs).float().to(dev), tables=torch.from_numpy(tables).to(dev),
              lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    return on, (qx, o.numbers(k, fmt), o.numbers(v, fmt), ks, vs, tables, lens)


def call(on, scale, **kw):
    return nv.paged_attention_kv8(on["q"], on["k"], on["v"], on["ks"], on["vs"], on["tables"], on["lens"], scale, **kw)


def compare(got, host, scale, dtype):
    qx, kn, vn, ks, vs, tables, lens = host
    N, T, Hq, D = qx.shape
    want, mean, reach = o.attend(qx, kn, vn, ks, vs, tables, lens, scale)
    got = got.double().cpu().numpy().reshape(want.shape)
    assert np.isfinite(got).all()
    tol = tolerance(want, mean, reach, max(max(lens), 1), D, dtype)
    off = np.abs(got - want) - tol
    assert off.max() <= 0, (np.unravel_index(off.argmax(), off.shape), off.max())


def check(rng, fmt, dtype, lens, T, Hq, H, D, bs, dev, **kw):
    on, host = make(rng, fmt, dtype, lens, T, Hq, H, D, bs, dev, **kw)
    got = call(on, D ** -0.5)
    assert got.shape == (len(lens), T, Hq * D) and got.dtype == ELEM[dtype]
    compare(got, host, D ** -0.5, dtype)
    return on, host, got


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,H,D,bs,T", [(4, 2, 8, 4, 1), (8, 2, 64, 8, 3), (6, 3, 7, 5, 2), (4, 4, 256, 16, 1),
                                         (2, 1, 96, 4, 17), (3, 1, 130, 1, 1), (16, 8, 128, 16, 2), (4, 2, 128, 32, 5),
                                         (2, 2, 36, 256, 1)])
def test_small_shapes(dev, fmt, dtype, Hq, H, D, bs, T):
    rng = np.random.default_rng(D + T)
    check(rng, fmt, dtype, [T, T + 1, 5 * bs, 5 * bs + 1, 63 + T, 64 + T, 65 + T, 300], T, Hq, H, D, bs, dev)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("Hq,H", [(16, 8), (32, 8), (8, 8), (24, 8), (16, 1), (6, 3), (28, 4), (5, 5)])
@pytest.mark.parametrize("T", [1, 2, 4, 7, 16, 33, 70])
def test_head_layouts_and_query_counts(dev, fmt, Hq, H, T):
    rng = np.random.default_rng(Hq * 100 + H + T)
    check(rng, fmt, "bf16", [T, T + 15, 16 * 5, 129 + T], T, Hq, H, 128, 16, dev)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", [1, 4, 12, 13, 16, 17, 32, 33, 100])
def test_lengths_around_the_tiles(dev, fmt, T):
    rng = np.random.default_rng(T)
    lens = [n for n in (1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 255, 257, 1023, 1025) if n >= T]
    check(rng, fmt, "bf16", lens, T, 8, 2, 128, 16, dev)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype,D,bs", [("bf16", 128, 16), ("f32", 64, 8)])
@pytest.mark.parametrize("T", [1, 3, 6, 20, 70])
def test_rows_that_see_no_key_are_zero(dev, fmt, dtype, D, bs, T):
    """context 0, negative, and shorter than the queries: those rows are zeros, the others right"""
    rng = np.random.default_rng(T)
    lens = [0, 1, max(1, T - 1), T, 40]
    on, host = make(rng, fmt, dtype, lens, T, 4, 2, D, bs, dev)
    on["lens"][0] = -2 ** 31 if T % 2 else -3
    got = call(on, 0.1)
    compare(got, host, 0.1, dtype)
    g = got.view(len(lens), T, -1)
    for i, n in enumerate(lens):
        if n < T:
            assert float(g[i, :T - n].float().abs().max()) == 0.0


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", [1, 4, 30, 40, 200])
def test_long_contexts(dev, fmt, T):
    """one sequence over 8192 keys and a short neighbour"""
    rng = np.random.default_rng(T)
    check(rng, fmt, "bf16", [8192 - 3, 100], T, 4, 2, 128, 16, dev)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", [1, 4, 20])
def test_many_sequences_with_a_shared_prefix(dev, fmt, T):
    rng = np.random.default_rng(T)
    check(rng, fmt, "bf16", [64 + T + int(x) for x in rng.integers(0, 200, 70)], T, 4, 2, 128, 16, dev, shared=4)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", [1, 40])
def test_scales_far_apart_and_zero(dev, fmt, T):
    """scales from 2^-22 up, blocks of scale 0 (zeros), large scores"""
    rng = np.random.default_rng(11)
    on, host = make(rng, fmt, "bf16", [200 + T, 90 + T], T, 4, 2, 128, 16, dev, spread=18, sigma=4.0)
    ks, vs, tables = host[3], host[4], host[5]
    ks[tables[0, 3]] = 0.0
    vs[tables[0, 5]] = 0.0
    on["ks"].copy_(torch.from_numpy(ks))
    on["vs"].copy_(torch.from_numpy(vs))
    compare(call(on, 128 ** -0.5), host, 128 ** -0.5, "bf16")


@pytest.mark.parametrize("D,bs", [(128, 16), (64, 8)])
@pytest.mark.parametrize("T", [2, 6, 20, 70])
def test_a_nan_reaches_only_the_queries_that_see_it(dev, T, D, bs):
    """an E4M3 NaN in a new token's key or value: rows before that token are as without it, rows from it
    on are NaN (all dims for a key, the one dim for a value)"""
    rng = np.random.default_rng(T)
    n, H, Hq = 100 + T, 2, 8
    on, host = make(rng, "e4m3", "bf16", [n, 40 + T], T, Hq, H, D, bs, dev)
    clean = call(on, 0.1).view(2, T, H, Hq // H, D)
    assert bool(torch.isfinite(clean).all())
    t = T // 2
    pos = n - T + t
    at = (int(host[5][0][pos // bs]), pos % bs)
    for name, dims in (("k", slice(None)), ("v", slice(5, 6))):
        bad = dict(on, **{name: on[name].clone()})
        bad[name].view(torch.uint8)[at[0], at[1], 1, 5] = 0xff
        got = call(bad, 0.1).view(2, T, H, Hq // H, D)
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[0, t:, 1, :, dims] = True
        assert torch.equal(got.isnan(), hit), name
        assert torch.equal(got[~hit], clean[~hit]), name


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", [1, 40])
def test_tables_out_of_the_pool_and_lengths_past_the_row(dev, fmt, T):
    """ids outside the pool are clamped and lengths past the table row cut off: finite, and right for the
    sequences whose tables are right"""
    rng = np.random.default_rng(12)
    on, host = make(rng, fmt, "bf16", [100 + T, 70 + T], T, 4, 2, 128, 16, dev, slack=0)
    for s in (on["ks"], on["vs"]):
        s.copy_(torch.where(s.isnan(), torch.full_like(s, 0.01), s))
    for c in (on["k"], on["v"]):
        u = c.view(torch.uint8)
        u.copy_(torch.where((u == POISON[fmt]), torch.zeros_like(u), u))
    want = call(on, 0.1)
    bad = dict(on, tables=on["tables"].clone(), lens=on["lens"].clone())
    bad["tables"][1, 1], bad["tables"][1, 2] = -2 ** 31, 2 ** 31 - 1
    bad["lens"][1] = 2 ** 31 - 1
    got = call(bad, 0.1)
    assert bool(torch.isfinite(got).all()) and torch.equal(got[0], want[0])


@pytest.mark.parametrize("fmt", FMT)
def test_blocks_past_32_bits_of_bytes(dev, fmt):
    rng = np.random.default_rng(13)
    on, host = make(rng, fmt, "bf16", [70, 33], 1, 16, 8, 128, 16, dev)
    nb = (1 << 32) // (16 * 8 * 128) + 40
    big = torch.zeros((nb, 16, 8, 128), dtype=torch.uint8, device=dev)
    at = nb - on["k"].shape[0]
    want = call(on, 0.1)
    big[at:] = on["k"].view(torch.uint8)
    s = torch.zeros((nb, 8), device=dev)
    s[at:] = on["ks"]
    sv = torch.zeros((nb, 8), device=dev)
    sv[at:] = on["vs"]
    far = dict(on, k=big.view(on["k"].dtype), ks=s, vs=sv, tables=torch.where(on["tables"] >= 0, on["tables"] + at, 0).int())
    v = torch.zeros_like(big)
    v[at:] = on["v"].view(torch.uint8)
    far["v"] = v.view(on["v"].dtype)
    assert torch.equal(call(far, 0.1), want)
    call(dict(far, lens=torch.zeros_like(on["lens"])), 0.1)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
@pytest.mark.parametrize("T", [1, 5, 13, 40])
def test_any_number_of_parts(dev, policy, fmt, splits, T):
    """the key walk in a forced number of parts: lengths that end in every part, parts without keys"""
    policy.setenv("NVLLM_PAGED_SPLITS", splits)
    rng = np.random.default_rng(splits)
    check(rng, fmt, "bf16", [n for n in (0, 1, T, 700, 1023, 1024, 1025, 2500) if n == 0 or n >= T], T, 8, 2, 128, 16,
          dev)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("T", [1, 4, 13, 30])
def test_tables_that_reach_past_the_caches(dev, fmt, T):
    """rows of the table wide enough that the launch streams its loads (more than 256 MiB in reach)"""
    rng = np.random.default_rng(15)
    check(rng, fmt, "bf16", [T, 300, 1111], T, 16, 8, 128, 16, dev, slack=3000)


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("dtype,D,bs", [("bf16", 128, 16), ("f32", 64, 8)])
@pytest.mark.parametrize("T", [1, 6, 20, 70])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_softmax_scales_without_a_plus(dev, fmt, dtype, D, bs, T, scale):
    rng = np.random.default_rng(16)
    on, host = make(rng, fmt, dtype, [T, 90, 500], T, 8, 4, D, bs, dev)
    compare(call(on, scale), host, scale, dtype)


@pytest.mark.parametrize("splits", [0, 2, 5])
@pytest.mark.parametrize("T", [1, 6, 12, 13, 50])
def test_nothing_is_written_outside_output_and_workspace(dev, policy, T, splits):
    """rows behind the last sequence and bytes behind the workspace that the entry asks for keep what they held"""
    policy.setenv("NVLLM_PAGED_SPLITS", splits)
    rng = np.random.default_rng(17)
    Hq, H, D, N = 8, 2, 128, 3
    on, host = make(rng, "e4m3", "bf16", [T, 600, 1500], T, Hq, H, D, 16, dev)
    L, width = nv.capi.lib(), on["tables"].shape[1]
    need = L.nvllm_paged_attn_kv8_workspace_bytes(N, T, Hq, H, D, 16, width, 0)
    assert need > 0 or splits == 0
    ws = torch.full((need + 4096,), 0xa5, dtype=torch.uint8, device=dev)
    out = torch.full((N + 1, T, Hq * D), 7.0, dtype=torch.bfloat16, device=dev)
    rc = L.nvllm_paged_attn_kv8(on["q"].data_ptr(), on["k"].data_ptr(), on["v"].data_ptr(), on["ks"].data_ptr(),
                                on["vs"].data_ptr(), on["tables"].data_ptr(), on["lens"].data_ptr(), out.data_ptr(),
                                ws.data_ptr(), need, N, T, Hq, H, D, 16, width, on["k"].shape[0], 0.1, 1, 0,
                                torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    compare(out[:N], host, 0.1, "bf16")
    assert bool((out[N] == 7.0).all()) and bool((ws[need:] == 0xa5).all())


@pytest.mark.parametrize("T,lens", [(1, [70, 300]), (1, [5000]), (5, [800, 9]), (40, [500, 77])])
def test_same_bits_again_on_another_stream_and_in_a_graph(dev, T, lens):
    """no result depends on the order of anything: repeated, side by side on two streams, replayed from a
    graph while the lengths grow"""
    rng = np.random.default_rng(14)
    on, host = make(rng, "int8", "bf16", lens, T, 16, 8, 128, 16, dev)
    want = call(on, 0.1)
    for _ in range(3):
        assert torch.equal(call(on, 0.1), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(call(on, 0.1))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for x in outs)
    need = nv.capi.lib().nvllm_paged_attn_kv8_workspace_bytes(len(lens), T, 16, 8, 128, 16, on["tables"].shape[1], 0)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    now = on["lens"].clone()
    moving = dict(on, lens=now)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(moving, 0.1, workspace=ws)
    for cut in (0, 3, 1):
        now.copy_(on["lens"] - cut)
        ws.fill_(255)
        eager = call(moving, 0.1)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), cut


def test_two_graphs_share_a_workspace(dev, policy):
    """replayed in turn, with eager work of either shape between the replays"""
    policy.setenv("NVLLM_PAGED_SPLITS", 3)
    rng = np.random.default_rng(18)
    cases = [make(rng, "int8", "bf16", lens, T, 16, 8, 128, 16, dev)[0] for T, lens in ((1, [900, 2000]), (20, [1500, 64]))]
    need = max(nv.capi.lib().nvllm_paged_attn_kv8_workspace_bytes(2, c["q"].shape[1], 16, 8, 128, 16,
                                                                 c["tables"].shape[1], 0) for c in cases)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    want = [call(c, 0.1) for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c, 0.1, workspace=ws))
        graphs.append(g)
    for _ in range(3):
        for i in (0, 1, 1, 0):
            outs[i].zero_()
            call(cases[1 - i], 0.1, workspace=ws)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], want[i])


@pytest.mark.parametrize("fmt", FMT)
def test_one_sequence_through_the_layer_cache(dev, fmt):
    """the reference-shaped operator on an 8-bit LayerKVCache: write, attend, extend, attend"""
    rng = np.random.default_rng(15)
    H, Hq, D, bs = 8, 16, 128, 16
    layer = nv.LayerKVCache(nv.KVCacheConfig(16, bs, H, D, 1, torch.int8 if fmt == "int8" else torch.float8_e4m3fn), dev)
    table = nv.BlockTable(bs)
    for b in (5, 2, 9):
        table.append_block(b)
    kn, vn = np.zeros((16, bs, H, D)), np.zeros((16, bs, H, D))
    ks, vs = np.zeros((16, H)), np.zeros((16, H))
    done = 0
    for n in (30, 1, 1, 7):
        k, kx = rounded(rng, (n, H, D), "bf16")
        v, vx = rounded(rng, (n, H, D), "bf16")
        q, qx = rounded(rng, (1, n, Hq, D), "bf16")
        slots = table.get_slot_mapping(done + n)[done:]
        nv.reshape_and_cache_kv8(k.to(dev), v.to(dev), layer.key_cache(), layer.value_cache(), layer.key_scales(),
                                 layer.value_scales(), torch.tensor(slots, device=dev))
        o.write(kn, ks, kx, slots, fmt)
        o.write(vn, vs, vx, slots, fmt)
        done += n
        got = nv.paged_attention(q.to(dev), layer, table, done, Hq, H, D, 0.1)
        compare(got, (qx, kn, vn, ks, vs, np.array([table.get_physical_block_ids()]), [done]), 0.1, "bf16")
    with pytest.raises(nv.TensorError):
        nv.paged_attention(q.to(dev), layer, table, 49, Hq, H, D, 0.1)
    with pytest.raises(nv.TensorError):
        nv.paged_attention(q.to(dev), layer, table, 3, Hq, H, D, 0.1)


@pytest.mark.parametrize("fmt", FMT)
def test_serving_steps(dev, fmt):
    """the set as a loop uses it: producer writes prompts, then decode steps through the batch metadata;
    every step's attention against the oracle fed with the cache read back"""
    rng = np.random.default_rng(16)
    Hq, H, D, bs, nb = 8, 2, 128, 16, 64
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    layer = nv.LayerKVCache(nv.KVCacheConfig(nb, bs, H, D, 1, dt), dev)
    cache = (layer.key_cache(), layer.value_cache(), layer.key_scales(), layer.value_scales())
    mgr = nv.BlockManager(nb, bs)
    rot = nv.RotaryEmbedding(D, 256, 1e6, torch.bfloat16, dev)
    w = rounded(rng, (D,), "bf16")[0].to(dev)
    tables, lens = [nv.BlockTable(bs) for _ in range(3)], [0, 0, 0]
    for new in (21, 1, 1, 1, 4, 1):
        meta = nv.BatchMetadata(8)
        for i, t in enumerate(tables):
            lens[i] += new
            while t.num_blocks() * bs < lens[i]:
                t.append_block(mgr.allocate())
            meta.add_sequence(t, lens[i], new)
        bt, cl, sm, _, pos = meta.upload(dev)
        n = 3 * new
        q, k, v = (rounded(rng, (n, h, D), "bf16")[0].to(dev) for h in (Hq, H, H))
        nv.qk_norm_rope_cache_kv8(q, k, v, w, w, 1e-6, rot, pos, *cache, sm)
        got = nv.paged_attention_kv8(q.view(3, new, Hq, D), *cache, bt, cl, D ** -0.5)
        every = torch.arange(nb, dtype=torch.int32, device=dev)
        kk, vv = (x.double().cpu().numpy() for x in nv.gather_cache_blocks_kv8(*cache, every, torch.float32))
        one = np.ones((nb, H))
        compare(got, (q.double().cpu().numpy().reshape(3, new, Hq, D), kk, vv, one, one, bt.cpu().numpy(), lens),
                D ** -0.5, "bf16")
