"""Cases of the 8-bit KV cache: quantised write, read-back, producer and attention over it.

The cache holds one byte a value and one power-of-two scale for each (block of tokens, kv head),
K and V apart:

    value = code * scale,   scale = 2^e, the smallest with  max|x| <= top * 2^e  (0 for a block of zeros)

with top = 127 and code an integer (format "int8"), or top = 448 and code an OCP E4M3 number (format
"e4m3").  A call that writes slot 0 of a block begins the block: its scale comes from the rows of that
call.  Any other call keeps the rows it does not write; when its rows need a larger scale, the kept
codes are rounded to it.  Scales being powers of two, no step but these roundings (to nearest, ties to
even) is inexact, and a write has one right answer, bit for bit.

`run` is one call as a serving loop makes it.  Where a case writes, it reads the written blocks back
as well, so that what the cache holds is returned as the values that it stands for.
"""
import math

import torch

own = False

TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ELEM = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS, THETA = 1e-6, 1e6


# ------------------------------------------------------------------------------------- the cases

def _case(name, kind, fmt, dtype, heads, kv_heads, head_dim, block_size, seqs, new, past, ragged):
    """past: tokens of the longest sequence that the cache holds already, new: tokens of the call
    (for "read": past tokens are read).  ragged: the sequences differ in length."""
    c = dict(kind=kind, format=fmt, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             block_size=block_size, seqs=seqs, new=new, past=past, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token for each of 256 running sequences goes into the middle of its last block
        _case("write decode 256", "write", "int8", "bf16", 32, 8, 128, 16, 256, 1, 2047, True),
        # eight fresh prompts of 4096 tokens
        _case("write prompt 8x4096", "write", "e4m3", "bf16", 32, 8, 128, 16, 8, 4096, 0, False),
        # second chunks of three prompts that ended inside a block, f32 activations, small heads
        _case("write chunk f32", "write", "int8", "f32", 4, 2, 64, 8, 3, 211, 93, True),
        # sixteen sequences handed over as contiguous K/V
        _case("read 16x2048", "read", "int8", "bf16", 32, 8, 128, 16, 16, 0, 2048, False),
        # one sequence whose last block is part full
        _case("read 1x517 f32", "read", "e4m3", "f32", 16, 8, 128, 16, 1, 0, 517, False),
        # the whole producer step (norm, rotation, quantised write) of a decode batch
        _case("producer decode 256", "producer", "e4m3", "bf16", 32, 8, 128, 16, 256, 1, 2047, True),
        # and of a prefill batch
        _case("producer prompt 4x2048", "producer", "int8", "bf16", 16, 8, 128, 16, 4, 2048, 0, False),
        # a lone user's next token: latency
        _case("attend 1x300", "attend", "int8", "bf16", 16, 8, 128, 16, 1, 1, 299, False),
        # the full decode batch: bandwidth
        _case("attend decode 256x2048", "attend", "int8", "bf16", 32, 8, 128, 16, 256, 1, 2047, False),
        # long verify of drafted tokens over ragged contexts
        _case("attend verify 64x4096 T13", "attend", "e4m3", "bf16", 32, 8, 128, 16, 64, 13, 4083, True),
        # chunked prefill against a long cached prefix: compute
        _case("attend chunk 4x1024 of 8192", "attend", "e4m3", "bf16", 16, 8, 128, 16, 4, 1024, 7168, False),
        # f32 activations, small heads, small blocks
        _case("attend f32 9x777 T3", "attend", "int8", "f32", 8, 2, 64, 8, 9, 3, 774, True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(("write", "read", "producer", "attend", "attend"))
    fmt = rng.choice(("int8", "e4m3"))
    f32 = rng.random() < 0.2
    heads, kv_heads = rng.choice(((32, 8), (16, 8), (8, 8), (24, 8), (32, 4), (16, 1)))
    head_dim, block_size = 128, 16
    small = f32 or rng.random() < 0.1
    if small:  # shapes of the small kind: few tokens
        heads, kv_heads = rng.choice(((8, 2), (4, 2), (6, 3)))
        head_dim, block_size = rng.choice(((64, 8), (64, 16), (128, 16), (96, 4)))
    dtype = "f32" if f32 else "bf16"
    if kind == "attend":
        new = rng.choice((1, 1, _log(rng, 2, 12), _log(rng, 13, 64), _log(rng, 65, 1024)))
        if small:
            new = min(new, 16)
        past = _log(rng, 1, 777 if small else 8192 - new)
        room = min(4 * 1024 * 8192 * 16 // (new * (past + new) * heads),  # work of the largest chunk
                   256 * 2048 // (past + new), 9 if small else 256)
        seqs = _log(rng, 1, max(1, room))
    elif kind == "read":
        past = _log(rng, 1, 600 if small else 8192)
        seqs, new = _log(rng, 1, max(1, (2400 if small else 32768) // past)), 0
    elif rng.random() < 0.5:  # a decode step
        new, past, seqs = 1, _log(rng, 1, 4095), _log(rng, 1, 256)
    else:
        new = _log(rng, 2, 400 if small else 4096)
        past = rng.choice((0, _log(rng, 1, 1000)))
        seqs = _log(rng, 1, max(1, (1200 if small else 16384) // new))
    return _case(None, kind, fmt, dtype, heads, kv_heads, head_dim, block_size, seqs, new, past,
                 rng.random() < 0.6)


def _past(case):
    """Cached tokens of each sequence: from all of `past` down to half of it where ragged."""
    p, span = case["past"], case["past"] // 2 + 1
    return [p - (i * 7919 % span if case["ragged"] else 0) for i in range(case["seqs"])]


def work(case):
    past, new, bs = _past(case), case["new"], case["block_size"]
    row, d = case["kv_heads"] * case["head_dim"], case["head_dim"]
    elt, n = 2 if case["dtype"] == "bf16" else 4, case["seqs"] * case["new"]
    blocks = sum(-(-(p + new) // bs) for p in past)
    if case["kind"] == "attend":
        tokens = sum(p + new for p in past)
        pairs = sum(new * p + new * (new + 1) // 2 for p in past)
        return {"bytes": 2 * tokens * row + 8 * blocks * case["kv_heads"] + 4 * blocks + 4 * len(past)
                + 2 * n * case["heads"] * d * elt, "flops": 4 * pairs * case["heads"] * d}
    if case["kind"] == "read":
        return {"bytes": 2 * blocks * bs * row * (1 + elt) + 8 * blocks * case["kv_heads"] + 4 * blocks,
                "flops": 2 * blocks * bs * row}
    touched = sum(-(-(p + new) // bs) - p // bs for p in past)
    moved = 2 * n * row * (elt + 1) + 8 * n + 16 * touched * case["kv_heads"]
    moved += 2 * touched * bs * row * (1 + elt)  # the read-back
    flops = 6 * n * row + 2 * touched * bs * row
    if case["kind"] == "producer":
        moved += 2 * n * case["heads"] * d * elt + 4 * n + 2 * d * elt * min(n, 2 * max(past) + 2 * new)
        flops += 10 * n * d * (case["heads"] + case["kv_heads"])
    return {"bytes": moved, "flops": flops}


# ----------------------------------------------------------------------------------- the inputs

class _Rotary:
    """cos / sin tables [positions, head_dim], each row a half-row twice."""

    def __init__(self, dim, positions, dtype, device):
        inv = THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
        a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
        a = torch.cat([a, a], 1)
        self._cos, self._sin = a.cos().to(dtype), a.sin().to(dtype)

    def cos_cache(self):
        return self._cos

    def sin_cache(self):
        return self._sin


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    dtype, fmt, bs = ELEM[case["dtype"]], case["format"], case["block_size"]
    heads, kvh, d, new = case["heads"], case["kv_heads"], case["head_dim"], case["new"]
    past = torch.tensor(_past(case), device=dev)
    seqs = case["seqs"]
    used = (past + new + bs - 1) // bs
    width = int(used.max())
    pool = int(used.sum()) + 3
    order = torch.randperm(pool, generator=g, device=dev)
    start = used.cumsum(0) - used
    col = torch.arange(width, device=dev)
    live = col < used[:, None]
    tables = torch.where(live, order[(start[:, None] + col).clamp(max=pool - 1)], 0).to(torch.int32)

    # what earlier calls left in the cache: codes over most of the format's range, scales that differ
    # from block to block and head to head
    def codes():
        x = randn(pool, bs, kvh, d).mul_(0.26 * TOP[fmt]).clamp_(-TOP[fmt], TOP[fmt])
        return x.round_().to(torch.int8) if fmt == "int8" else x.to(torch.float8_e4m3fn)

    def scales():
        e = torch.randint(-1, 2, (pool, kvh), generator=g, device=dev).float()
        return torch.exp2(e - (5 if fmt == "int8" else 7))

    s = dict(case=case, tables=tables, lens=(past + new).to(torch.int32), k_cache=codes(), v_cache=codes(),
             k_scales=scales(), v_scales=scales(), scale=1.0 / math.sqrt(d))
    if case["kind"] == "attend":
        s["query"] = randn(seqs, new, heads, d).to(dtype)
        return s
    if case["kind"] == "read":
        s["ids"] = tables[live]
        return s
    s["ids"] = tables[live & (col >= (past // bs)[:, None])]  # the blocks that the call writes
    pos = (past[:, None] + torch.arange(new, device=dev)).reshape(-1)
    seq = torch.arange(seqs, device=dev).repeat_interleave(new)
    s["slots"] = tables[seq, pos // bs].long() * bs + pos % bs
    n = seqs * new
    # a few channels stand out, as the keys of a trained model have them
    s["key"] = (randn(n, kvh, d) * (1 + 3 * (torch.arange(d, device=dev) % 32 == 5))).to(dtype)
    s["value"] = (0.7 * randn(n, kvh, d)).to(dtype)
    if case["kind"] == "producer":
        s["query"] = randn(n, heads, d).to(dtype)
        s["positions"] = pos.to(torch.int32)
        s["q_weight"] = (1 + 0.2 * randn(d)).to(dtype)
        s["k_weight"] = (1 + 0.2 * randn(d)).to(dtype)
        s["rotary"] = _Rotary(d, int(pos.max()) + 1, dtype, dev)
    return s


# ------------------------------------------------------------------------------- the plain forms

def _take(cache, ids):
    return cache.view(torch.uint8)[ids].view(cache.dtype)


def _scale_of(amax, fmt):
    """The smallest power of two s with amax <= top * s, in f32; 0 for 0."""
    m, e = torch.frexp(amax.double() / TOP[fmt])
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(m), e), 0.0).float()


def _encode(y, fmt):
    """y = x / scale to the nearest code, ties to even."""
    y = y.clamp(-TOP[fmt], TOP[fmt])
    return y.round().to(torch.int8) if fmt == "int8" else _e4m3(y)


def _e4m3(y):
    """Through 32 bits (24 of significand) only where y has no more of them: a second rounding could
    fall on the other side of a border."""
    if y.dtype == torch.float64:
        step = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp(min=-5) - 4)  # of E4M3 at y
        y = (y / step).round() * step
    return y.to(torch.float8_e4m3fn)


def _write(cache, scales, x, slots, ids, fmt, bs):
    """x [tokens, kv_heads, D] into the slots of the blocks `ids`."""
    at = torch.full((cache.shape[0] * bs,), -1, dtype=torch.int64, device=x.device)
    at[slots] = torch.arange(slots.numel(), device=x.device)
    token = at.view(-1, bs)[ids]                                          # [blocks, bs], -1: not written
    new = (token >= 0)[:, :, None, None]
    rows = torch.where(new, x[token.clamp(min=0)], 0.0)                   # [blocks, bs, kv_heads, D]
    begins = (token[:, 0] >= 0)[:, None]
    old = torch.where(begins, 0.0, scales[ids])
    s = torch.maximum(old, _scale_of(rows.abs().amax(dim=(1, 3)), fmt))
    safe = torch.where(s > 0, s, 1.0)
    was = _take(cache, ids).float()
    kept = torch.where(begins[:, :, None, None], was, was * (old / safe)[:, None, :, None])
    codes = _encode(torch.where(new, rows / safe[:, None, :, None], kept), fmt)
    cache.view(torch.uint8)[ids] = codes.view(torch.uint8)
    scales[ids] = s


def _read(cache, scales, ids, dtype):
    return (_take(cache, ids).float() * scales[ids][:, None, :, None]).to(dtype)


def _rotate(x, weight, cos, sin):
    """In x's type: 64 bits for what is quantised, whose values may lie next to a code's border."""
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)
    h = x.shape[-1] // 2
    turned = torch.cat([-x[..., h:], x[..., :h]], -1)
    return x * cos[:, None].to(x.dtype) + turned * sin[:, None].to(x.dtype)


def _attend(s, bs):
    q, tables, lens = s["query"].float(), s["tables"].long(), s["lens"].long()
    n, t, heads, d = q.shape
    kvh, width = s["k_cache"].shape[2], tables.shape[1] * bs

    def rows(cache, scales):
        x = _take(cache, tables).float() * scales[tables][:, :, None, :, None]   # [n, blocks, bs, kvh, d]
        return x.reshape(n, width, kvh, d).transpose(1, 2).contiguous()   # [n, kvh, keys, d]

    qg = q.view(n, t, kvh, heads // kvh, d).permute(0, 2, 1, 3, 4).reshape(n, kvh, -1, d)
    score = torch.matmul(qg, rows(s["k_cache"], s["k_scales"]).transpose(2, 3).contiguous()) * s["scale"]
    last = lens[:, None] - t + torch.arange(t, device=q.device)           # the last key that a query sees
    seen = torch.arange(width, device=q.device) <= last[:, :, None]       # [n, t, keys]
    seen = seen.repeat_interleave(heads // kvh, 1)[:, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows(s["v_cache"], s["v_scales"])) / torch.where(total == 0, 1.0, total)
    o = o.view(n, kvh, t, heads // kvh, d).permute(0, 2, 1, 3, 4)
    return o.reshape(n, t, heads * d).to(s["query"].dtype)


def _plain(s):
    c = s["case"]
    fmt, bs, dtype, ids = c["format"], c["block_size"], ELEM[c["dtype"]], s.get("ids")
    if c["kind"] == "attend":
        return {"out": _attend(s, bs)}
    ids = ids.long()
    out = {}
    if c["kind"] != "read":
        key = s["key"].float()
        if c["kind"] == "producer":
            cos, sin = s["rotary"].cos_cache()[s["positions"].long()], s["rotary"].sin_cache()[s["positions"].long()]
            key = _rotate(s["key"].double(), s["k_weight"], cos, sin)
            out["q"] = _rotate(s["query"].float(), s["q_weight"], cos, sin).to(dtype)
        _write(s["k_cache"], s["k_scales"], key, s["slots"], ids, fmt, bs)
        _write(s["v_cache"], s["v_scales"], s["value"].float(), s["slots"], ids, fmt, bs)
    out["k"] = _read(s["k_cache"], s["k_scales"], ids, dtype)
    out["v"] = _read(s["v_cache"], s["v_scales"], ids, dtype)
    return out


# -------------------------------------------------------------------------- the framework's calls

def _own(s):
    import nano_vllm_rs_amd as nv
    c = s["case"]
    cache = (s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"])
    if c["kind"] == "attend":
        return {"out": nv.paged_attention_kv8(s["query"], *cache, s["tables"], s["lens"], s["scale"])}
    out = {}
    if c["kind"] == "write":
        nv.reshape_and_cache_kv8(s["key"], s["value"], *cache, s["slots"])
    elif c["kind"] == "producer":
        out["q"] = nv.qk_norm_rope_cache_kv8(s["query"], s["key"], s["value"], s["q_weight"], s["k_weight"],
                                             EPS, s["rotary"], s["positions"], *cache, s["slots"],
                                             q_out=torch.empty_like(s["query"]))
    out["k"], out["v"] = nv.gather_cache_blocks_kv8(*cache, s["ids"], ELEM[c["dtype"]])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------- the definition, once more, in 64 bits

def _exact_codes(y, fmt):
    """The nearest code to y, as a number: the grid of the format, ties to the even multiple."""
    if fmt == "int8":
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_write(cache, scales, x, case, tables, past, fmt):
    """Sequence by sequence, block by block of the call; returns the blocks' values in call order."""
    bs, new, got = case["block_size"], case["new"], []
    for i, p in enumerate(past):
        rows = x[i * new:(i + 1) * new]                       # [new, kvh, d]
        first, lastb = p // bs, (p + new - 1) // bs
        n = lastb - first + 1
        ids = tables[i, first:lastb + 1].long()
        full = torch.zeros((n * bs,) + rows.shape[1:], dtype=torch.float64, device=x.device)
        full[p - first * bs:p - first * bs + new] = rows
        full = full.view(n, bs, *rows.shape[1:])
        written = torch.zeros(n * bs, dtype=torch.bool, device=x.device)
        written[p - first * bs:p - first * bs + new] = True
        written = written.view(n, bs)
        big = full.abs().amax(dim=(1, 3))                     # [n, kvh]
        e = torch.ceil(torch.log2(big.clamp(min=1e-300) / TOP[fmt]))
        e = torch.where(big > TOP[fmt] * torch.exp2(e), e + 1, e)
        e = torch.where(big <= TOP[fmt] * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        s = torch.where(big > 0, torch.exp2(e), torch.zeros_like(e))
        held = _take(cache, ids).double()
        if p % bs:                                            # the first block goes on
            s[0] = torch.maximum(s[0], scales[ids[0]].double())
            held[0] = _exact_codes(held[0] * (scales[ids[0]].double() / s[0])[None, :, None], fmt)
        unit = torch.where(s > 0, s, torch.ones_like(s))[:, None, :, None]
        code = torch.where(written[:, :, None, None], _exact_codes(full / unit, fmt), held)
        got.append(code * s[:, None, :, None])
    return torch.cat(got)


def exact(case, seed):
    if case["seqs"] > 300:
        return None
    s = prepare(case, seed)
    fmt, bs, d = case["format"], case["block_size"], case["head_dim"]
    past, new = _past(case), case["new"]
    if case["kind"] == "read":
        ids = s["ids"].long()
        return {x: _take(s[x + "_cache"], ids).double() * s[x + "_scales"][ids].double()[:, None, :, None] for x in "kv"}
    if case["kind"] == "attend":
        group, outs = case["heads"] // case["kv_heads"], []
        for i, p in enumerate(past):
            ids = s["tables"][i, :-(-(p + new) // bs)].long()
            k, v = ((_take(s[x + "_cache"], ids).double() * s[x + "_scales"][ids].double()[:, None, :, None])
                    .flatten(0, 1)[:p + new].transpose(0, 1).repeat_interleave(group, 0) for x in "kv")
            score = torch.matmul(s["query"][i].double().transpose(0, 1), k.transpose(1, 2).contiguous())
            score = score / math.sqrt(d)
            hidden = torch.ones(new, p + new, dtype=torch.bool, device=k.device).triu(p + 1)
            score.masked_fill_(hidden, -math.inf)
            outs.append(torch.matmul(torch.softmax(score, -1), v).transpose(0, 1).reshape(new, -1))
        return {"out": torch.stack(outs)}
    out, key = {}, s["key"].double()
    if case["kind"] == "producer":
        pos = s["positions"].long()
        c, w = (t[pos].double()[:, None, :d // 2] for t in (s["rotary"].cos_cache(), s["rotary"].sin_cache()))

        def turn(x, weight):
            x = x.double()
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / d + EPS) * weight.double()
            a, b = x[..., :d // 2], x[..., d // 2:]
            return torch.cat([a * c - b * w, b * c + a * w], -1)

        key, out["q"] = turn(s["key"], s["k_weight"]), turn(s["query"], s["q_weight"])
    out["k"] = _exact_write(s["k_cache"], s["k_scales"], key, case, s["tables"], past, fmt)
    out["v"] = _exact_write(s["v_cache"], s["v_scales"], s["value"].double(), case, s["tables"], past, fmt)
    return out
