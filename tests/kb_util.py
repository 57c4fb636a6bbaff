"""KeyBlocks in numpy and 64 bits: block rows, the choice of blocks, attention,
and how far a kernel that rounds its weights and outputs may be from it."""
import numpy as np

import i4_util


def block_rows(keys, block):
    """keys [heads, tokens, D] (float) -> rows of the full blocks: codes
    [heads, blocks, G, 16], mults [heads, blocks, G], scales [heads, blocks]."""
    heads, tokens, D = keys.shape
    full = tokens // block
    mean = keys[:, : full * block].astype(np.float64).reshape(heads, full, block, D).sum(2) / block
    parts = [i4_util.quantize(m.astype(np.float32)) for m in mean]
    return tuple(np.stack([p[i] for p in parts]) for i in range(3))


def order(score):
    """float32 -> ranks that order as the scores do, NaN below everything."""
    b = (score + np.float32(0)).view(np.int32).astype(np.int64)
    r = np.where(b < 0, -b - 1, b + (1 << 31))
    return np.where(np.isnan(score), 0, r)


def select(rows, q, length, block, k, first, last):
    """rows = block rows of one slot, q [q_heads, D] float32 -> [kv_heads, k]."""
    codes, mults, scales = rows
    heads = codes.shape[0]
    nb = -(-length // block)
    out = np.full((heads, k), -1, np.int64)
    for h in range(heads):
        if nb <= k:
            chosen = np.arange(nb)
        else:
            inner = np.arange(first, nb - last)
            qh = q.reshape(heads, -1, q.shape[1])[h]
            rank = order(i4_util.scores(codes[h][inner], mults[h][inner], scales[h][inner], qh)).max(0)
            best = inner[np.lexsort((inner, -rank))][: k - first - last]
            chosen = np.sort(np.concatenate([np.arange(first), best, np.arange(nb - last, nb)]))
        out[h, : len(chosen)] = chosen
    return out


def attend(keys, values, q, length, sel, block, scale):
    """keys, values [heads, tokens, D], q [q_heads, D], sel [heads, k] -> out
    [q_heads, D], lse [q_heads], and the tolerances' parts: sum of p|v|, the
    bound on a logit's size sum |q k| scale, and the tokens seen."""
    heads, _, D = keys.shape
    q = q.astype(np.float64).reshape(heads, -1, D)
    out = np.zeros_like(q)
    mass = np.zeros_like(q)
    lse = np.full(q.shape[:2], -np.inf)
    size = np.zeros(q.shape[:2])
    seen = 0
    nb = -(-length // block)
    for h in range(heads):
        t = [np.arange(b * block, min((b + 1) * block, length)) for b in sel[h] if 0 <= b < nb]
        t = np.concatenate(t) if t else np.zeros(0, np.int64)
        seen = max(seen, len(t))
        if len(t) == 0:
            continue
        k, v = keys[h][t].astype(np.float64), values[h][t].astype(np.float64)
        z = q[h] @ k.T * scale
        top = z.max(1, keepdims=True)
        p = np.exp(z - top)
        total = p.sum(1, keepdims=True)
        out[h] = p @ v / total
        mass[h] = p @ np.abs(v) / total
        lse[h] = (np.log(total) + top)[:, 0]
        size[h] = (np.abs(q[h]) @ np.abs(k).T).max(1) * abs(scale)
    return out.reshape(-1, D), lse.reshape(-1), mass.reshape(-1, D), size.reshape(-1), seen


def tolerances(out, lse, mass, size, seen, D, half, f16):
    """half: half a step of the cache's type (relative). A float32 logit of D
    products is off by (D + 8) 2^-24 of its terms' size (the products themselves
    are exact), a weight by twice that and by half a step when it enters the
    product (an f16 weight below 2^-14 by 2^-25), exp2 by 2^-21, a sum of n
    weights by n 2^-24, the joins of partial results by 32 more; the result is
    rounded once more."""
    logit = (D + 8) * 2.0**-24 * size + 2.0**-21
    rel = 2 * logit + (2 * seen + 64) * 2.0**-24
    low = seen * 2.0**-25 if f16 else 0.0
    big = np.abs(mass).max() if mass.size else 0.0
    tol = half * (mass + np.abs(out)) + 2 * rel[:, None] * mass + low * 4 * big + 2.0**-25
    tol_lse = logit + (seen + 64) * 2.0**-24 + 8 * 2.0**-24 * np.abs(np.where(np.isfinite(lse), lse, 0))
    return tol, tol_lse
