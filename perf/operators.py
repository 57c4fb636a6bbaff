"""Timed cases of the 4-bit row index (FlatI4) and of block-sparse attention over a key/value cache (KeyBlocks).

A FlatI4 row is a vector in 4 bits a value. Its dim values are padded with zeros to whole groups of 32. A group holds 32
codes c in [-7, 7], stored as the nibbles c + 8 (byte i of a group's 16 bytes: value i in the low nibble, value 16 + i
in the high one), and one multiplier m in [0, 255]; a row has one float32 scale s. The row stands for s * m * c.

  score(q, row) = float32(dot) * qscale * s,   dot = sum over the groups of m * sum(c * q8)

with q8, qscale the int8 query that FlatI8 uses too. The dot is a whole number, so its order of summation is free, and a
top-k, (score descending, index ascending), has one answer. Packed keys are those of the other indexes: the float32's
order-preserving image in the high word, 2^31 - 1 - index in bits 31..1.

KeyBlocks keeps one such row for every full block of a cache's keys: the mean key (summed in 64 bits) of that block, head
and slot. A query row, with a slot and the number of cached tokens it may see, scores the blocks it sees (the largest
score of the query heads that share a key/value head), takes the first and the last ones and the best of the others, and
attends to the tokens of those blocks alone.
"""
import math

import numpy as np
import torch

own = False

GROUP = 32
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _index(name, kind, n, dim, batch, k=0):
    return {"name": name, "kind": kind, "n": n, "dim": dim, "batch": batch, "k": k}


def _attend(name, q_heads, kv_heads, head_dim, block, slots, tokens, rows, k, dtype, layout="heads", short=False, update=False):
    return {"name": name, "kind": "attend", "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block,
            "slots": slots, "tokens": tokens, "rows": rows, "k": k, "dtype": dtype, "layout": layout, "short": short,
            "update": update}


def listed():
    return [
        # one question over a small library of passages: every score, latency counts
        _index("score one 100k x 384", "score", 100_000, 384, 1),
        # three questions at once over a ragged library with an odd dimension
        _index("score three 1000003 x 300", "score", 1_000_003, 300, 3),
        # a server's batch: the scores of eight questions, 1024 values a vector
        _index("score eight 2M x 1024", "score", 2_000_000, 1024, 8),
        # the passages that one question is answered with, over a small and a large library
        _index("top 10 of 100k x 384", "topk", 100_000, 384, 1, 10),
        _index("top 100 of 4M x 768", "topk", 4_000_000, 768, 1, 100),
        # sixteen questions at once, vectors of a small embedding model
        _index("top 10 of 1.5M x 256 sixteen", "topk", 1_500_000, 256, 16, 10),
        # one sequence's next token behind a prompt of 4096 tokens: latency counts
        _attend("one token 4k", 32, 8, 128, 64, 1, 4096, 1, 16, "bf16"),
        # a serving batch: the next token of sixteen sequences of up to 32768 tokens
        _attend("sixteen tokens 32k", 32, 8, 128, 64, 16, 32768, 1, 32, "bf16"),
        # the next token of two sequences of half a million tokens, an odd length
        _attend("two tokens 500k", 32, 8, 128, 64, 2, 500_011, 1, 64, "f16"),
        # four drafted tokens for each of eight sequences, a key/value head for every query head, two slots next to empty
        _attend("drafts 12 heads of 64", 12, 12, 64, 32, 8, 5000, 4, 12, "f16", "tokens", True),
        # a chunk of a long prompt: its keys' blocks are made first
        _attend("prompt chunk 2048 of 16k", 32, 8, 128, 64, 1, 16384, 2048, 16, "bf16", "tokens", False, True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["score", "topk", "attend", "attend"])
    if kind != "attend":
        dim = rng.choice([64, 96, 128, 200, 256, 384, 500, 768, 1000, 1024, rng.randrange(33, 1024)])
        batch = rng.choice([1, 1, 2, 3, 4, 6, 8, 11, 16])
        n = _log(rng, 3000, 2.4e9 / dim / (1 + batch / 8))
        return {"kind": kind, "n": n, "dim": dim, "batch": batch, "k": 0 if kind == "score" else rng.choice([1, 7, 10, 50, 100, 200])}
    q_heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (16, 16, 64), (28, 4, 128), (24, 8, 96), (12, 4, 64), (64, 8, 128), (20, 5, 80), (8, 1, 256)])
    block = rng.choice([16, 32, 64, 128])
    rows = rng.choice([1, 1, 1, 2, 3, 5, 8, _log(rng, 16, 512)])
    slots = _log(rng, 1, 32 if rows <= 8 else 2)
    update = rng.random() < 0.3
    # a single row reads its blocks alone, more rows or an update most of the cache
    most = min(500_000, (4.0e9 if rows == 1 and not update else 1.2e9) / (slots * kv_heads * head_dim * 4))
    tokens = _log(rng, max(2 * block, rows + 1), max(4 * block, most if rows == 1 else min(most, 65536)))
    k = rng.choice([4, 8, 16, 24, 32])
    while rows * slots * k * block * q_heads * head_dim > 8.0e9:
        k //= 2
    return {"kind": kind, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "slots": slots, "tokens": tokens,
            "rows": rows, "k": max(k, 2), "dtype": rng.choice(["bf16", "f16"]), "layout": rng.choice(["heads", "tokens"]),
            "short": rng.random() < 0.3, "update": update}


# ---------------------------------------------------------------------------------------------------------------------
# the plain form: 4-bit rows, int8 queries, keys
# ---------------------------------------------------------------------------------------------------------------------
def _half_away(x):
    """Round half away from zero; the half is added in 64 bits, where it is exact."""
    y = x.double()
    return torch.sign(y) * torch.floor(y.abs() + 0.5)


def _over(a, b):
    """a / b, rounded once (a tensor over a number may be taken as a product with the number's inverse)."""
    return a / torch.full_like(a, b)


def _padded(x, dim):
    return torch.nn.functional.pad(x, (0, -(-dim // GROUP) * GROUP - dim))


def _quantize_rows(x):
    """float32 rows [..., dim] -> packed codes [..., G, 16], multipliers [..., G] (uint8), scales [...]."""
    x = _padded(x, x.shape[-1])
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    gmax = g.abs().amax(-1)
    rmax = gmax.amax(-1)
    some = rmax > 0
    scale = torch.where(some, _over(rmax, 1785.0), torch.ones_like(rmax))
    up = torch.where(some, torch.full_like(rmax, 255.0) / rmax, torch.zeros_like(rmax))
    mult = torch.clamp(torch.ceil(gmax * up[..., None]), max=255.0)
    inv = torch.reciprocal(mult * scale[..., None])
    c = torch.where(mult[..., None] > 0, torch.clamp(_half_away(g * inv[..., None]), -7, 7), torch.zeros((), dtype=torch.float64, device=x.device))
    u = (c + 8).to(torch.uint8)
    return u[..., :16] | (u[..., 16:] << 4), mult.to(torch.uint8), scale


def _values(codes, mult):
    """The whole numbers m * c of packed rows, in 64 bits: [..., G * 32]."""
    c = torch.cat([codes & 15, codes >> 4], -1).double()
    c -= 8
    c *= mult[..., None]
    return c.flatten(-2)


def _quantize_queries(q):
    """float32 queries [..., dim] -> int8 values as float64, padded to whole groups, and scales [...] (0 for a zero query)."""
    q = _padded(q, q.shape[-1])
    top = q.abs().amax(-1)
    scale = _over(top, 127.0)
    inv = torch.where(top > 0, torch.reciprocal(scale), torch.zeros_like(scale))
    return torch.clamp(_half_away(q * inv[..., None]), -127, 127), scale


def _ordered(score):
    """The float32's order-preserving image (-0 as +0), as a whole number in [0, 2^32)."""
    b = (score + 0.0).view(torch.int32).long()
    return torch.where(b < 0, -b - 1, b + (1 << 31))


def _index_scores(s):
    q8, qscale = _quantize_queries(s["q"])
    dot = q8 @ _values(s["codes"], s["mult"]).T
    return dot.float() * qscale[:, None] * s["scale"]


def _plain_topk(s):
    score = _index_scores(s)
    n = score.shape[1]
    keys = ((_ordered(score) - (1 << 31)) << 32) + ((((1 << 31) - 1) - torch.arange(n, device=score.device)) << 1)
    best = torch.topk(keys, min(s["k"], n), dim=1).values
    return best ^ (-(1 << 63))


# ---------------------------------------------------------------------------------------------------------------------
# the plain form: blocks, selection, attention
# ---------------------------------------------------------------------------------------------------------------------
def _block_rows(keys, block):
    """keys [slots, heads, tokens, D] -> the rows of their full blocks."""
    full = keys.shape[2] // block
    x = keys[:, :, : full * block].unflatten(2, (full, block)).double().sum(3) / block
    return _quantize_rows(x.float())


def _plain_select(s):
    q, slot, length, k, block = s["q"].float(), s["slot"].long(), s["length"].long(), s["k"], s["block"]
    q8, qscale = _quantize_queries(q)
    slots, kv_heads = s["keys"].shape[:2]
    blocks = -(-length // block)
    w = _values(s["codes"], s["mult"])  # [slots, kv_heads, blocks, D padded]; the query rows are in their slots' order
    by_slot = q8.reshape(slots, -1, kv_heads, q8.shape[1] // kv_heads, q8.shape[2]).transpose(1, 2)
    dot = by_slot.flatten(2, 3) @ w.transpose(-1, -2)
    dot = dot.unflatten(2, by_slot.shape[2:4]).transpose(1, 2).flatten(0, 1)  # [rows, kv_heads, query heads, blocks]
    score = dot.float() * qscale.unflatten(1, (kv_heads, -1))[..., None] * s["scale"][slot][:, :, None]
    rank = _ordered(score.amax(2))
    most = -(-s["keys"].shape[2] // block)
    rank = torch.nn.functional.pad(rank, (0, most - rank.shape[2]))
    b = torch.arange(most, device=q.device)
    always = (b < s["first"]) | (b >= blocks[:, None] - s["last"])
    rank = torch.where(always[:, None], (1 << 32) - 1, rank)
    rank = torch.where((b < blocks[:, None])[:, None], rank, -1)
    key = (rank << 30) + ((1 << 30) - 1 - b)
    best = torch.topk(key, min(k, most), dim=2).values
    picked = torch.where(best >= 0, (1 << 30) - 1 - (best & ((1 << 30) - 1)), 1 << 30).sort(2).values
    picked = torch.where(picked == 1 << 30, -1, picked)
    return torch.nn.functional.pad(picked, (0, k - picked.shape[2]), value=-1).to(torch.int32)


def _plain_attend(s, picked):
    q, slot, length, block = s["q"].float(), s["slot"].long(), s["length"].long(), s["block"]
    kv_heads = s["keys"].shape[1]
    token = (picked.long()[..., None] * block + torch.arange(block, device=q.device)).flatten(2)  # [rows, kv_heads, k * block]
    seen = (token >= 0) & (token < length[:, None, None]) & (picked >= 0).repeat_interleave(block, 2)
    at = torch.where(seen, token, 0)
    head = torch.arange(kv_heads, device=q.device)[None, :, None]
    where = (slot[:, None, None], head, at)
    logit = (q.unflatten(1, (kv_heads, -1)) @ s["keys"][where].float().transpose(-1, -2)) * s["softmax_scale"]
    logit = torch.where(seen[:, :, None], logit, -math.inf)
    top = logit.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(logit - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ s["values"][where].float()) / torch.where(total > 0, total, 1.0)
    lse = (torch.log(total) + top)[..., 0]
    return out.flatten(1, 2).to(s["keys"].dtype), lse.flatten(1, 2)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _vectors(gen, rows, centres):
    """Clustered vectors whose values differ in size from group to group, as embeddings' do."""
    dim = centres.shape[1]
    c = torch.randint(centres.shape[0], (rows,), device="cuda", generator=gen)
    return centres[c] + 0.6 * torch.randn(rows, dim, device="cuda", generator=gen)


def _prepare_index(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    n, dim, batch, k = case["n"], case["dim"], case["batch"], case["k"]
    spread = torch.exp(0.5 * torch.randn(dim, device="cuda", generator=gen))
    centres = torch.randn(200, dim, device="cuda", generator=gen) * spread
    s = {"kind": case["kind"], "k": k, "n": n, "batch": batch, "q": _vectors(gen, batch, centres)}
    groups = -(-dim // GROUP)
    if own:
        from aikit_b200.ann import B200Backend
        s["index"] = B200Backend(torch.cuda.current_device()).NewI4IndexEmpty(n, dim)
        s["keys"] = torch.empty(batch, k, dtype=torch.int64, device="cuda")
        s["scores"] = torch.empty(batch if case["kind"] == "score" else 0, n, device="cuda")
    else:
        s["codes"] = torch.empty(n, groups, 16, dtype=torch.uint8, device="cuda")
        s["mult"] = torch.empty(n, groups, dtype=torch.uint8, device="cuda")
        s["scale"] = torch.empty(n, device="cuda")
    step = 1 << 18
    for a in range(0, n, step):
        x = _vectors(gen, min(step, n - a), centres)
        if own:
            s["index"].set_rows_async(a, x.data_ptr(), x.shape[0], torch.cuda.current_stream().cuda_stream)
        else:
            s["codes"][a : a + step], s["mult"][a : a + step], s["scale"][a : a + step] = _quantize_rows(x)
    return s


def _prepare_attend(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, block, slots, heads, dim = TYPES[case["dtype"]], case["block"], case["slots"], case["kv_heads"], case["head_dim"]
    tokens, per = case["tokens"], case["rows"]
    shape = (slots, heads, tokens, dim) if case["layout"] == "heads" else (slots, tokens, heads, dim)
    lay = (lambda t: t) if case["layout"] == "heads" else (lambda t: t.transpose(1, 2))
    keys, values = (lay(torch.randn(shape, device="cuda", generator=gen, dtype=dtype)) for _ in range(2))
    # neighbouring tokens' keys are alike, so that blocks differ from one another
    full = tokens // block
    topic = torch.randn(slots, heads, full, 1, dim, device="cuda", generator=gen, dtype=dtype)
    keys[:, :, : full * block].unflatten(2, (full, block)).add_(topic)
    ends = torch.randint(max(per, int(0.4 * tokens)), tokens + 1, (slots,), device="cuda", generator=gen)
    ends[0] = tokens
    if case["short"]:
        ends[-1] = per - 1  # its first row sees nothing
        ends[slots // 2] = per
    length = (ends[:, None] - per + 1 + torch.arange(per, device="cuda")).flatten()
    length = length if not case["short"] else torch.clamp(length, min=0)
    s = {"kind": "attend", "keys": keys, "values": values, "block": block, "k": case["k"], "first": 1, "last": 1, "update": case["update"],
         "q": torch.randn(slots * per, case["q_heads"], dim, device="cuda", generator=gen, dtype=dtype),
         "slot": torch.arange(slots, device="cuda", dtype=torch.int32).repeat_interleave(per), "length": length.to(torch.int32),
         "softmax_scale": 1 / math.sqrt(dim)}
    rows = slots * per
    if own:
        from aikit_b200.ann import B200Backend
        s["blocks"] = B200Backend(torch.cuda.current_device()).NewKeyBlocks(
            keys.data_ptr(), values.data_ptr(), dtype=case["dtype"], slots=slots, kv_heads=heads, q_heads=case["q_heads"],
            head_dim=dim, capacity=tokens, block=block, max_rows=rows, max_select=case["k"],
            slot_stride=keys.stride(0), head_stride=keys.stride(1), token_stride=keys.stride(2))
        s["every_slot"] = torch.arange(slots, device="cuda", dtype=torch.int32)
        s["from"], s["to"] = torch.zeros_like(s["every_slot"]), torch.full_like(s["every_slot"], tokens)
        s["picked"] = torch.empty(rows, heads, case["k"], dtype=torch.int32, device="cuda")
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(rows, case["q_heads"], device="cuda")
        s["tokens"], s["slots"], s["rows"] = tokens, slots, rows
        if not case["update"]:
            _own_update(s, torch.cuda.current_stream().cuda_stream)
    elif not case["update"]:
        s["codes"], s["mult"], s["scale"] = _block_rows(keys, block)
    return s


def prepare(case, seed):
    return _prepare_attend(case, seed) if case["kind"] == "attend" else _prepare_index(case, seed)


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _own_update(s, stream):
    s["blocks"].update_async(s["every_slot"].data_ptr(), s["from"].data_ptr(), s["to"].data_ptr(), s["slots"], s["tokens"], stream)


def _own(s):
    stream = torch.cuda.current_stream().cuda_stream
    if s["kind"] == "score":
        s["index"].score_async(s["q"].data_ptr(), s["batch"], s["scores"].data_ptr(), stream)
        return {"scores": s["scores"]}
    if s["kind"] == "topk":
        s["index"].topk_async(s["q"].data_ptr(), s["batch"], s["k"], s["keys"].data_ptr(), stream)
        return {"keys": s["keys"]}
    if s["update"]:
        _own_update(s, stream)
    s["blocks"].query_async(s["q"].data_ptr(), s["slot"].data_ptr(), s["length"].data_ptr(), s["rows"], s["k"], s["softmax_scale"],
                            s["picked"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(), first=s["first"], last=s["last"], stream=stream)
    return {"picked": s["picked"], "out": s["out"], "lse": s["lse"]}


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "score":
        return {"scores": _index_scores(s)}
    if s["kind"] == "topk":
        return {"keys": _plain_topk(s)}
    if s["update"]:
        s["codes"], s["mult"], s["scale"] = _block_rows(s["keys"], s["block"])
    picked = _plain_select(s)
    out, lse = _plain_attend(s, picked)
    return {"picked": picked, "out": out, "lse": lse}


def work(case):
    if case["kind"] != "attend":
        n, dim, batch = case["n"], case["dim"], case["batch"]
        groups = -(-dim // GROUP)
        out = 4 * n * batch if case["kind"] == "score" else 8 * case["k"] * batch
        return {"bytes": n * (17 * groups + 4) + 4 * dim * batch + out, "flops": 2 * n * dim * batch}
    block, heads, dim, rows = case["block"], case["kv_heads"], case["head_dim"], case["slots"] * case["rows"]
    blocks = -(-case["tokens"] // block)
    picked = min(case["k"], blocks)
    row = 17 * -(-dim // GROUP) + 4
    used = min(blocks, case["rows"] * picked)  # of a slot and head: its rows pick their own blocks
    b = case["slots"] * heads * (used * block * dim * 4 + blocks * row) + rows * case["q_heads"] * (dim * 4 + 4) + rows * heads * case["k"] * 4
    f = rows * case["q_heads"] * (4 * picked * block * dim + 2 * blocks * dim)
    if case["update"]:
        b += case["slots"] * heads * blocks * (block * dim * 2 + row)
        f += case["slots"] * heads * blocks * block * dim
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_query(q):
    """What an int8 query stands for: float32 arithmetic decides the codes, the rest is 64 bits."""
    q = q.cpu().numpy().astype(np.float32)
    scale = (np.abs(q).max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(scale > 0, np.float32(1) / scale, np.float32(0)).astype(np.float32)
    t = (q * inv[..., None]).astype(np.float32).astype(np.float64)
    code = np.clip(np.copysign(np.floor(np.abs(t) + 0.5), t), -127, 127)
    return code, scale


def _exact_rows(keys, block):
    """The whole numbers m * c of the blocks' rows and the rows' scales: float32 arithmetic decides them."""
    slots, heads, tokens, dim = keys.shape
    full = tokens // block
    mean = np.stack([keys[:, :, b * block : (b + 1) * block].double().mean(2).cpu().numpy() for b in range(full)], 2).astype(np.float32)
    mean = np.pad(mean, [(0, 0)] * 3 + [(0, -dim % GROUP)]).reshape(slots, heads, full, -1, GROUP)
    gmax = np.abs(mean).max(-1)
    rmax = gmax.max(-1, keepdims=True)
    scale = rmax / np.float32(1785)
    mult = np.minimum(np.ceil(gmax * (np.float32(255) / rmax)), np.float32(255))
    t = (mean * (np.float32(1) / (mult * scale))[..., None]).astype(np.float64)
    code = np.clip(np.copysign(np.floor(np.abs(t) + 0.5), t), -7, 7)
    return (code * mult[..., None]).reshape(slots, heads, full, -1)[..., :dim], scale[..., 0]


def _exact_attend(case, seed):
    s = prepare(case, seed)
    block, k, heads = case["block"], case["k"], case["kv_heads"]
    per = case["q_heads"] // heads
    code, qscale = _exact_query(s["q"].float())
    slot, length = s["slot"].tolist(), s["length"].tolist()
    if case["update"]:
        number, row_scale = _exact_rows(s["keys"], block)
    else:
        c = s["codes"].cpu().numpy().astype(np.int64)
        number = (np.concatenate([c % 16, c // 16], -1) - 8) * s["mult"].cpu().numpy().astype(np.int64)[..., None]
        number = number.reshape(*number.shape[:3], -1)[..., : case["head_dim"]].astype(np.float64)
        row_scale = s["scale"].cpu().numpy()
    out, lse = [], []
    for r in range(len(slot)):
        o = torch.zeros(heads, per, case["head_dim"], dtype=torch.float64, device="cuda")
        l = torch.full((heads, per), -math.inf, dtype=torch.float64, device="cuda")
        blocks = -(-length[r] // block)
        if blocks:
            tokens = torch.zeros(heads, min(k, blocks), block, dtype=torch.int64)
            for h in range(heads):
                inner = np.arange(1, blocks - 1)
                dot = number[slot[r], h, inner] @ code[r, h * per : (h + 1) * per, : case["head_dim"]].T  # whole numbers
                score = (dot.astype(np.float32) * qscale[r, h * per : (h + 1) * per] * row_scale[slot[r], h, inner][:, None]).max(1) if len(inner) else inner
                best = inner[np.lexsort((inner, -score))][: max(0, k - 2)]
                chosen = np.unique(np.concatenate([[0, blocks - 1], best])).astype(np.int64)
                tokens[h] = torch.from_numpy(chosen)[:, None] * block + torch.arange(block)
            t = tokens.flatten(1).cuda()
            seen = t < length[r]
            t = torch.where(seen, t, 0)[..., None].expand(-1, -1, case["head_dim"])
            keys, values = (x[slot[r]].gather(1, t).double() for x in (s["keys"], s["values"]))
            z = torch.einsum("hgd,htd->hgt", s["q"][r].double().unflatten(0, (heads, per)), keys) / math.sqrt(case["head_dim"])
            z = z.masked_fill(~seen[:, None], -math.inf)
            l = torch.logsumexp(z, -1)
            o = torch.einsum("hgt,htd->hgd", torch.exp(z - l[..., None]), values)
        out.append(o.flatten(0, 1))
        lse.append(l.flatten(0, 1))
    return {"picked": None, "out": torch.stack(out), "lse": torch.stack(lse)}


def exact(case, seed):
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    if case["kind"] == "topk":
        return None  # keys are whole numbers
    s = prepare(case, seed)
    code, qscale = _exact_query(s["q"])
    q = torch.from_numpy(code * qscale[:, None].astype(np.float64)).cuda()
    out = torch.empty(case["batch"], case["n"], dtype=torch.float64, device="cuda")
    step = 1 << 18
    for a in range(0, case["n"], step):
        low, high = (s["codes"][a : a + step] & 15).double() - 8, (s["codes"][a : a + step] >> 4).double() - 8
        size = s["mult"][a : a + step].double() * s["scale"][a : a + step, None].double()
        row = (torch.cat([low, high], -1) * size[..., None]).flatten(1)[:, : case["dim"]]
        out[:, a : a + step] = q @ row.T
    return {"scores": out}
