"""The 8-bit KV cache in 64 bits, token by token, from its definition (include/nvllm_attn.h): the
oracle of the kv8 tests.  numpy only; a cache is codes as float64 numbers and scales [blocks, heads]."""
import numpy as np

TOP = {"int8": 127.0, "e4m3": 448.0}


def e4m3_table():
    """code 0 .. 255 -> number (NaN at 0x7f and 0xff)"""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    x = np.where(e > 0, np.ldexp(1 + m / 8.0, e - 7), np.ldexp(m / 8.0, -6))
    x = np.where((c & 127) == 127, np.nan, x)
    return np.where(c >> 7, -x, x)


def numbers(codes, fmt):
    """uint8 codes -> the numbers they stand for (before the scale)"""
    codes = np.asarray(codes)
    return codes.view(np.int8).astype(np.float64) if fmt == "int8" else e4m3_table()[codes]


def scale_of(amax, fmt):
    if amax == 0:
        return 0.0
    e = -126
    while amax > TOP[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def encode(y, fmt):
    """y = x / scale -> the nearest number of the format, ties to even; infinities saturate; NaN is 0 in
    int8 and NaN in E4M3"""
    y = np.asarray(y, dtype=np.float64)
    nan = np.isnan(y)
    y = np.clip(np.where(nan, 0.0, y), -TOP[fmt], TOP[fmt])
    if fmt == "int8":
        return np.rint(y)
    _, e = np.frexp(y)
    step = np.ldexp(1.0, np.maximum(e, -5) - 4)
    return np.where(nan, np.nan, np.rint(y / step) * step)


def write(cache, scales, x, slots, fmt):
    """One call, in place: cache [nb, bs, H, D] numbers, scales [nb, H], x [n, H, D], slots [n]."""
    nb, bs, H, _ = cache.shape
    last = {}
    for t, s in enumerate(slots):
        if 0 <= s < nb * bs:
            last[int(s)] = t
    for b in sorted({s // bs for s in last}):
        rows = {s % bs: t for s, t in last.items() if s // bs == b}
        for h in range(H):
            v = np.stack([np.asarray(x[t, h], dtype=np.float64) for t in rows.values()])
            ok = np.abs(v) <= 2.0 ** 127
            need = scale_of(np.abs(np.where(ok, v, 0.0)).max(), fmt)
            s = need if 0 in rows else max(scales[b, h], need)
            if 0 not in rows and s > scales[b, h]:
                for o in range(bs):
                    if o not in rows:
                        cache[b, o, h] = encode(cache[b, o, h] * (scales[b, h] / s), fmt)
            for o, t in rows.items():
                cache[b, o, h] = encode(np.asarray(x[t, h], dtype=np.float64) / (s if s > 0 else 1.0), fmt)
            scales[b, h] = s


def rotate(x, w, cos, sin, eps):
    """norm and rotation of x [n, H, D] with tables' rows cos, sin [n, D]"""
    x = np.asarray(x, dtype=np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    c, s = cos[:, None], sin[:, None]
    return np.concatenate([a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:]], -1)


def attend(q, k, v, ks, vs, tables, lens, scale):
    """q [N, T, Hq, D]; k, v [nb, bs, H, D] numbers -> (out, weighted mean of |v|, largest sum |q||k|
    scale): the last two, per output value and per row, are what error bounds need."""
    N, T, Hq, D = q.shape
    nb, bs, H, _ = k.shape
    G = Hq // H
    out = np.zeros((N, T, Hq, D))
    mean = np.zeros((N, T, Hq, D))
    reach = np.zeros((N, T, Hq, 1))
    for i in range(N):
        n = int(lens[i])
        if n <= 0:
            continue
        ids = np.asarray(tables[i])[:-(-n // bs)]
        kk = (k[ids] * ks[ids][:, None, :, None]).reshape(-1, H, D)[:n]
        vv = (v[ids] * vs[ids][:, None, :, None]).reshape(-1, H, D)[:n]
        for t in range(T):
            see = n - T + t + 1
            if see <= 0:
                continue
            for h in range(Hq):
                s = kk[:see, h // G] @ q[i, t, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, t, h] = p @ vv[:see, h // G]
                mean[i, t, h] = p @ np.abs(vv[:see, h // G])
                reach[i, t, h] = (np.abs(kk[:see, h // G]) @ np.abs(q[i, t, h]) * abs(scale)).max()
    return out, mean, reach
