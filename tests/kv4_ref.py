"""Plain restatements for the 4-bit cache tests, apart from the kernels: the byte order of a tile from its description in
include/agxc.h (dim by dim), quantisation in fp32 numpy, and attention in 64 bits."""
import numpy as np

LOG2E = 1.4426950408889634


def offsets(hd):
    """(k, v): the byte of [token 0..15][dim] in a tile, for K and for V."""
    G = hd // 64
    k, v = np.empty((16, hd), np.int64), np.empty((16, hd), np.int64)
    for t in range(16):
        for d in range(hd):
            g, i = d // 64, d % 64 // 2
            k[t, d] = t * 32 * G + i // 8 * 8 * G + 8 * g + i % 8
            v[t, d] = 8 * hd + t // 8 * 256 * G + (4 * (i // 4) + t % 8 // 2) * 8 * G + t % 2 * 4 * G + 4 * g + i % 4
    return k, v


def tile_bytes(hd):
    return 16 * (hd + 8 * (hd // 64))


def pack_tiles(kc, vc, ksb, vsb):
    """uint8 [..., tiles, bytes] of codes [..., tiles, 16, hd] and fp16 pairs [..., tiles, 16, G, 2]."""
    hd = kc.shape[-1]
    out = np.zeros(kc.shape[:-2] + (tile_bytes(hd),), np.uint8)
    for c, off in zip((kc, vc), offsets(hd)):
        for d in range(hd):
            out[..., off[:, d]] |= (c[..., d] << (4 * (d & 1))).astype(np.uint8)
    sb = np.ascontiguousarray(np.stack([ksb, vsb], -3)).astype(np.float16)      # [..., 16, 2, G, 2]
    out[..., 16 * hd:] = sb.reshape(sb.shape[:-4] + (-1,)).view(np.uint8)
    return out


def quantise(x):
    """(codes, pairs fp16 [..., G, 2]) of fp32 [..., hd]: every step an IEEE fp32 operation."""
    g = np.asarray(x, np.float32).reshape(x.shape[:-1] + (-1, 64))
    lo, hi = g.min(-1), g.max(-1)
    s = np.where(hi > lo, (hi - lo) * np.float32(1 / 15), np.float32(1)).astype(np.float16)
    b = lo.astype(np.float16)
    with np.errstate(all="ignore"):
        q = np.rint((g - b.astype(np.float32)[..., None]) / s.astype(np.float32)[..., None])
    q = np.clip(np.where(np.isfinite(q), q, 0), 0, 15).astype(np.uint8)
    return q.reshape(x.shape), np.stack([s, b], -1)


def values(codes, pairs):
    """code * scale + bias in 64 bits (exact), [..., hd]."""
    g = codes.reshape(codes.shape[:-1] + (codes.shape[-1] // 64, 64)).astype(np.float64)
    p = pairs.astype(np.float64)
    return (g * p[..., 0:1] + p[..., 1:2]).reshape(codes.shape)


def attention(q, K, V, length):
    """out [n, H, hd] and the weights' spread of q [n, H, hd] over K, V [length, KVH, hd], in 64 bits."""
    n, H, hd = q.shape
    out = np.zeros((n, H, hd))
    KVH = K.shape[1]
    for i in range(n):
        keys = length - n + i + 1
        if keys <= 0:
            continue
        for h in range(H):
            j = h // (H // KVH)
            s = K[:keys, j] @ q[i, h].astype(np.float64)
            p = np.exp2(s - s.max())
            out[i, h] = p @ V[:keys, j] / p.sum()
    return out


def attention_bound(q, K, V, out, pairs_k, pairs_v, out_ulp):
    """How far a kernel that rounds each weight times scale to 11 bits may be off, per [n, H] row: the weight's rounding
    (2^-11 of half a code range, 7.5 scales, averaged with weights that add to one), the scores' fp32 sums (2^-19 of
    sum |q| times the largest term of a code's affine form, through p's derivative ln 2, against the spread of v), and
    the output's own rounding (added per element by the caller as out_ulp * |out|)."""
    n, H, hd = q.shape
    KVH = K.shape[1]
    if not K.shape[0]:
        return np.zeros((n, H, 1))
    term = max(1e-9, float((np.abs(pairs_k.astype(np.float64)) * [15, 1]).max()))
    vs = pairs_v.astype(np.float64)[..., 0].max(axis=(0, 2))          # per KV head
    vm = np.abs(V).max(axis=(0, 2))
    j = np.arange(H) // (H // KVH)
    ds = 2.0 ** -19 * np.abs(q.astype(np.float64)).sum(-1) * term
    return (2.0 ** -11 * 7.5 * vs[j] + 2 * np.log(2) * ds * vm[j] + 2.0 ** -20 * vm[j])[..., None]
