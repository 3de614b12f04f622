"""Plain forms of the INT8 key/value cache's operators, on the host: fp32 where the codes are decided (numpy rounds every
operation), 64 bits elsewhere."""
import numpy as np


def held(rows):
    """Codes and scales of fp32 rows [..., dim]: quantization.cpp:22-78 per row."""
    rows = np.asarray(rows, np.float32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        a = np.fmax.reduce(np.abs(rows), axis=-1, initial=np.float32(1e-8))
        v = rows * (np.float32(127.0) / a)[..., None]
        t = np.trunc(v)
        r = np.where(np.abs(v - t) >= np.float32(0.5), t + np.copysign(np.float32(1.0), v), t)
        codes = np.clip(np.where(np.isnan(r), np.float32(127.0), r), -127, 127).astype(np.int8)
        return codes, (a / np.float32(127.0)).astype(np.float32)


def turned(x, cos, sin):
    """Rotary pairs (d, d + dim / 2) of x [..., dim], cos / sin [..., dim / 2], in the inputs' precision."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    with np.errstate(invalid="ignore", over="ignore"):
        return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


def tables(rows, dim, base=10000.0):
    angle = np.arange(rows)[:, None] * base ** (-2.0 * np.arange(dim // 2) / dim)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def attend(q, keys, values):
    """softmax(q k^T / sqrt(dim)) v for q [G, dim], keys / values [T, dim], in 64 bits."""
    s = q.astype(np.float64) @ keys.astype(np.float64).T / np.sqrt(q.shape[-1])
    w = np.exp(s - s.max(-1, keepdims=True))
    return (w / w.sum(-1, keepdims=True)) @ values.astype(np.float64)


def decode(qkv, cache, cos, sin, pos, heads, prefix=None, prefix_len=0):
    """One decode step: qkv [B, (heads + 2 kv) * dim], cache = dict of k_codes, k_scales, v_codes, v_scales (copied, not
    changed).  Returns out [B, heads * dim] in 64 bits, the cache afterwards, and a bound on |out - fp32 evaluation|.

    The bound: the query's rotation rounds three times and its fixed point by half of 1 / 8355000 of its largest value, that
    is 4 * 2^-24 of that value together, and the score is rounded when it is scaled (twice), when the maximum is
    subtracted (once) and by the key's scale (once): a score is off by at most e = 8 * 2^-24 * max |q| sum |k| / sqrt(dim).
    Weights are off by 2 e (their sum as well, hence the 2), by the exponential (2 ulp: 4 * 2^-24) and by their own fixed point
    (half of 1 / 4194000 of the largest: 2 * 2^-24), 6 * 2^-24 together.  Sums over n positions round once per 32-position tile of
    a warp, with one rescaling each, and when warps, CTAs and prefix parts are joined (at most 39 times; or 16 times inside
    the tensor core, whose sums may be cut off at 2 * 2^-24, and 7 times behind it): (3 n / 256 + 39) * 2^-24 of the largest
    value."""
    cache = {k: v.copy() for k, v in cache.items()}
    B, kv, S, dim = cache["k_codes"].shape
    G = heads // kv
    out, tol = np.zeros((B, heads * dim)), np.zeros((B, heads * dim))
    for b in range(B):
        p = int(pos[b] if len(pos) > 1 else pos[0])
        if not 0 <= p < S:
            continue
        rows = qkv[b].reshape(heads + 2 * kv, dim)
        c, s = cos[prefix_len + p], sin[prefix_len + p]
        q = turned(rows[:heads].astype(np.float64), c.astype(np.float64), s.astype(np.float64))
        for name, new in (("k", turned(rows[heads:heads + kv], c, s)), ("v", rows[heads + kv:])):
            codes, scales = held(new)
            cache[name + "_codes"][b, :, p], cache[name + "_scales"][b, :, p] = codes, scales
        for h in range(kv):
            read = []
            for name in "kv":
                own = cache[name + "_codes"][b, h, :p + 1].astype(np.float64) * cache[name + "_scales"][b, h, :p + 1, None].astype(np.float64)
                if prefix is not None:
                    first = prefix[name + "_codes"][0, h, :prefix_len].astype(np.float64) * prefix[name + "_scales"][0, h, :prefix_len, None]
                    own = np.concatenate([first, own])
                read.append(own)
            at = slice((h * G) * dim, (h + 1) * G * dim)
            qh = q[h * G:(h + 1) * G]
            out[b, at] = attend(qh, *read).reshape(-1)
            e = 8 * 2.0 ** -24 * np.abs(qh).max(-1) * np.abs(read[0]).sum(-1).max() / np.sqrt(dim)            # [G]
            n = read[0].shape[0]
            tol[b, at] = np.repeat(np.abs(read[1]).max() * (2 * e + (3 * n / 256 + 39 + 6) * 2.0 ** -24), dim)
    return out, cache, tol
