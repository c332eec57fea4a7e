"""The 4-bit KV cache in numpy and 64 bits: quantisation, the packed pool and
ragged causal attention, each from the definition in include/lunelette_cuda.h."""
import numpy as np

PAGE, GROUP = 64, 32


def block_bytes(dim):
    return PAGE * dim + 4 * PAGE * (dim // GROUP)


def scale_of(m):
    """m / -8 to 8 significant bits, on the grid of 2^-24, at most 8160 in magnitude."""
    x = np.asarray(m, np.float64) / -8
    _, e = np.frexp(x)
    unit = np.ldexp(1.0, np.maximum(e - 8, -24))
    with np.errstate(invalid="ignore"):
        d = np.clip(np.rint(x / unit) * unit, -8160, 8160)
    return np.where(np.isfinite(x), d, np.nan)


def quantise(r):
    """[..., dim] -> codes (0..15) and scales [..., dim / 32], both float64."""
    r = np.asarray(r, np.float64)
    g = r.reshape(r.shape[:-1] + (r.shape[-1] // GROUP, GROUP))
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    high, low = g.max(-1), g.min(-1)
    d = scale_of(np.where(high >= -low, high, low))
    zero = (d == 0)[..., None]
    c = np.clip(np.rint(g / np.where(zero, 1.0, d[..., None])), -8, 7)
    c = np.where(zero, 0.0, c) + 8
    return c.reshape(r.shape), np.where(bad, np.nan, d)


def dequantise(codes, d):
    c = codes.reshape(d.shape + (GROUP,)) - 8
    return (c * d[..., None]).reshape(codes.shape)


def k_byte(slot, dim_index, dim):
    word = (dim_index % 32 // 8) * (dim // 32) + dim_index // 32
    return slot * (dim // 2) + 4 * word + dim_index % 8 // 2


def k_scale_byte(slot, group, dim):
    return PAGE * dim // 2 + 2 * (slot * (dim // GROUP) + group)


def v_byte(slot, dim_index, dim):
    n = slot * (dim // 8) + dim_index // 8
    n = n ^ (8 * ((n >> 5) & (3 if dim == 128 else 1)))
    return PAGE * dim // 2 + 2 * PAGE * (dim // GROUP) + 4 * n + dim_index % 8 // 2


def v_scale_byte(slot, group, dim):
    return PAGE * dim + 2 * PAGE * (dim // GROUP) + 2 * ((slot // 2 * (dim // GROUP) + group) * 2 + slot % 2)


def store(pool, dim, page, slot, codes, d, kind):
    """Write one position's rows ([heads, dim] codes, [heads, groups] scales) into pool
    [pages, heads, block bytes] (one layer)."""
    byte = (k_byte, v_byte)[kind]
    scale = (k_scale_byte, v_scale_byte)[kind]
    even = np.arange(0, dim, 2)
    codes = codes.astype(np.uint8)
    pool[page][:, byte(slot, even, dim)] = codes[:, even] | codes[:, even + 1] << 4
    half = d.astype(np.float16).view(np.uint16)
    half = np.where(np.isnan(d), 0x7FFF, half)
    for g in range(dim // GROUP):
        at = scale(slot, g, dim)
        pool[page][:, at] = half[:, g] & 255
        pool[page][:, at + 1] = half[:, g] >> 8


def fetch(pool, dim, page, slot, kind):
    """[heads, dim] values held at one position."""
    d_index = np.arange(dim)
    byte = (k_byte, v_byte)[kind](slot, d_index, dim)
    c = (pool[page][:, byte] >> (4 * (d_index & 1))) & 15
    at = np.array([(k_scale_byte, v_scale_byte)[kind](slot, g, dim) for g in range(dim // GROUP)])
    bits = pool[page][:, at].astype(np.uint16) | pool[page][:, at + 1].astype(np.uint16) << 8
    return dequantise(c.astype(np.float64), bits.view(np.float16).astype(np.float64))


def rotate(x, cos, sin):
    """Split-half rotation of [..., dim] in float64; cos, sin [dim]."""
    half = x.shape[-1] // 2
    x = np.asarray(x, np.float64)
    turned = np.concatenate([-x[..., half:], x[..., :half]], -1)
    return x * cos + turned * sin


def query_scale(position):
    return 1 + 0.1 * np.log(1.0 + position // 16384)


def attention(q, k, v, scale, first_position):
    """Rows q [n, query heads, dim] at first_position.. over k, v [length, heads, dim]. Returns the
    output and, for error bounds, per row and head the largest sum |q_d k_d| * |scale| over visible
    keys, and sum p |v| and sum |v| per dim."""
    n, qh, dim = q.shape
    group = qh // k.shape[1]
    out, spread, weight, total = np.zeros((n, qh, dim)), np.zeros((n, qh)), np.zeros((n, qh, dim)), np.zeros((n, qh, dim))
    for i in range(n):
        seen = min(first_position + i + 1, k.shape[0])
        if seen <= 0:
            continue
        for h in range(qh):
            kk, vv = k[:seen, h // group], v[:seen, h // group]
            s = scale * (kk @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vv
            spread[i, h] = abs(scale) * (np.abs(kk) @ np.abs(q[i, h])).max()
            weight[i, h] = p @ np.abs(vv)
            total[i, h] = np.abs(vv).sum(0)
    return out, spread, weight, total
