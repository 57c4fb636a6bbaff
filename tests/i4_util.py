"""FlatI4 in numpy: the row format, quantizer, scores and top-k, in whole
numbers (int64) and the float32 steps that the format defines."""
import numpy as np

import oracle

GROUP = 32


def groups(dim):
    return (dim + GROUP - 1) // GROUP


def quantize(v):
    """float32 rows [n, dim] -> codes [n, G, 16], mults [n, G], scales [n]."""
    v = np.asarray(v, np.float32)
    n, dim = v.shape
    G = groups(dim)
    x = np.zeros((n, G * GROUP), np.float32)
    x[:, :dim] = v
    x = x.reshape(n, G, GROUP)
    one = np.float32(1)
    with np.errstate(all="ignore"):
        gmax = np.fmax.reduce(np.abs(x), axis=2, initial=np.float32(0))
        rmax = gmax.max(1)
        zero = rmax == 0
        scale = np.where(zero, one, rmax / np.float32(1785)).astype(np.float32)
        up = np.where(zero, np.float32(0), np.float32(255) / rmax).astype(np.float32)
        t = np.ceil(gmax * up[:, None])
        mult = np.where(gmax == 0, 0, np.where(t <= 255, t, 255)).astype(np.float32)
        inv = one / (mult * scale[:, None])
        y = (x * inv[:, :, None]).astype(np.float64)
        c = np.copysign(np.floor(np.abs(y) + 0.5), y)
        c = np.clip(np.where(np.isnan(c), 0, c), -7, 7)
    c = np.where(mult[:, :, None] == 0, 0, c).astype(np.int64)
    u = (c + 8).astype(np.uint8)
    return u[:, :, :16] | (u[:, :, 16:] << 4), mult.astype(np.uint8), scale


def numbers(codes, mults):
    """The whole numbers m * c [n, G * 32]."""
    c = np.concatenate([codes & 15, codes >> 4], 2).astype(np.int64) - 8
    return (c * mults.astype(np.int64)[:, :, None]).reshape(len(codes), -1)


def scores(codes, mults, scales, q):
    """float32(dot) * qscale * scale for float32 queries q [M, dim]."""
    q = np.ascontiguousarray(q, np.float32)
    q8, qs = oracle.quantize_queries(q)
    w = numbers(codes, mults)[:, : q.shape[1]]
    # the products stay below 2^53, so the float64 product is the whole number
    dot = np.rint(q8.astype(np.float64) @ w.astype(np.float64).T)
    with np.errstate(all="ignore"):
        s = dot.astype(np.float32) * qs[:, None] * np.asarray(scales, np.float32)
    return np.where(qs[:, None] == 0, np.float32(0), s).astype(np.float32)


def topk(score, k, keep=None, id_base=0):
    """(ids [M, k], scores [M, k]) by (score desc, index asc), NaN excluded, -1 padded."""
    M, n = score.shape
    ids = np.full((M, k), -1, np.int64)
    out = np.zeros((M, k), np.float32)
    for m in range(M):
        ok = ~np.isnan(score[m])
        if keep is not None:
            ok &= np.asarray(keep, bool)[id_base : id_base + n]
        at = np.flatnonzero(ok)
        best = at[np.lexsort((at, -score[m, at]))][:k]
        ids[m, : len(best)] = best + id_base
        out[m, : len(best)] = score[m, best]
    return ids, out
