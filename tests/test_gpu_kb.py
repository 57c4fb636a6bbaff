"""KeyBlocks on the device: block rows and chosen blocks equal the numpy
statement exactly; attention is within the bounds that kb_util derives."""
import numpy as np
import pytest

import i4_util
import kb_util
from aikit_b200._ffi import DeclinedError, Fi8Error

pytestmark = pytest.mark.gpu


class Cache:
    """A cache on the device and its values in float64 on the host."""

    def __init__(self, backend, *, q_heads, kv_heads, D, block, capacity, lens, dtype="bf16", layout="heads", seed=0, max_rows=64,
                 max_select=64, fill=None, pad=0):
        import torch
        self.torch, self.type = torch, {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
        self.q_heads, self.kv_heads, self.D, self.block, self.capacity, self.f16 = q_heads, kv_heads, D, block, capacity, dtype == "f16"
        slots = len(lens)
        gen = torch.Generator("cuda").manual_seed(seed)
        def tensor():
            shape = (slots, kv_heads, capacity, D + pad) if layout == "heads" else (slots, capacity, kv_heads, D + pad)
            t = torch.randn(shape, device="cuda", generator=gen).to(self.type)
            t = t if layout == "heads" else t.transpose(1, 2)
            return t[..., :D]
        self.k, self.v = tensor(), tensor()
        topic = torch.randn(slots, kv_heads, -(-capacity // block), D, device="cuda", generator=gen).to(self.type)
        self.k += topic.repeat_interleave(block, 2)[:, :, :capacity]
        if fill is not None:
            for s, n in enumerate(lens):
                self.k[s, :, n:], self.v[s, :, n:] = fill, fill
        assert self.k.stride() == self.v.stride()
        self.kb = backend.NewKeyBlocks(self.k.data_ptr(), self.v.data_ptr(), dtype=dtype, slots=slots, kv_heads=kv_heads,
                                       q_heads=q_heads, head_dim=D, capacity=capacity, block=block, max_rows=max_rows,
                                       max_select=max_select, slot_stride=self.k.stride(0), head_stride=self.k.stride(1),
                                       token_stride=self.k.stride(2))
        self.lens = lens
        self.hk, self.hv = self.host()
        self.gen = gen

    def host(self):
        return self.k.double().cpu().numpy(), self.v.double().cpu().numpy()

    def ints(self, x):
        return self.torch.tensor(x, dtype=self.torch.int32, device="cuda")

    def update(self, slots, a, b, stream=0):
        t = [self.ints(x) for x in (slots, a, b)]
        self.kb.update_async(*(x.data_ptr() for x in t), len(slots), max(y - x for x, y in zip(a, b)), stream)
        self.torch.cuda.synchronize()

    def update_all(self):
        self.update(list(range(len(self.lens))), [0] * len(self.lens), list(self.lens))

    def queries(self, rows, scale=1.0):
        q = self.torch.randn(rows, self.q_heads, self.D, device="cuda", generator=self.gen) * scale
        return q.to(self.type)

    def check(self, q, slot, length, k, first=1, last=1, scale=None):
        """query_async against the statement; returns the chosen blocks and outputs."""
        torch = self.torch
        rows = len(slot)
        scale = self.D**-0.5 if scale is None else scale
        ds, dl = self.ints(slot), self.ints(length)
        sel = torch.full((rows, self.kv_heads, k), -7, dtype=torch.int32, device="cuda")
        out = torch.full((rows, self.q_heads, self.D), float("nan"), dtype=self.type, device="cuda")
        lse = torch.full((rows, self.q_heads), float("nan"), device="cuda")
        self.kb.query_async(q.data_ptr(), ds.data_ptr(), dl.data_ptr(), rows, k, scale, sel.data_ptr(), out.data_ptr(),
                            lse.data_ptr(), first=first, last=last, q_stride=q.stride(0))
        self.kb.sync()
        self.compare(q, slot, length, k, first, last, scale, sel, out, lse)
        again, out2, lse2 = torch.zeros_like(sel), torch.zeros_like(out), torch.zeros_like(lse)
        self.kb.select_async(q.data_ptr(), ds.data_ptr(), dl.data_ptr(), rows, k, again.data_ptr(), first=first, last=last,
                             q_stride=q.stride(0))
        self.kb.attend_async(q.data_ptr(), ds.data_ptr(), dl.data_ptr(), rows, k, scale, again.data_ptr(), out2.data_ptr(),
                             lse2.data_ptr(), q_stride=q.stride(0))
        self.kb.sync()
        assert torch.equal(again, sel) and torch.equal(out2, out) and torch.equal(lse2, lse)
        return sel, out

    def compare(self, q, slot, length, k, first, last, scale, sel, out, lse):
        qh = q.float().cpu().numpy()
        sel, out, lse = sel.cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
        half = float(self.torch.finfo(self.type).eps) / 2
        rows_of = {s: kb_util.block_rows(np.nan_to_num(self.hk[s][:, : self.lens[s]]), self.block) for s in set(slot)}
        for r in range(len(slot)):
            want = kb_util.select(rows_of[slot[r]], qh[r], length[r], self.block, k, first, last)
            np.testing.assert_array_equal(sel[r], want)
            parts = kb_util.attend(self.hk[slot[r]], self.hv[slot[r]], qh[r], length[r], want, self.block, scale)
            tol, tol_lse = kb_util.tolerances(*parts, self.D, half, self.f16)
            off = np.abs(out[r] - parts[0])
            assert (off <= tol).all(), (r, float((off / tol).max()))
            if length[r] == 0:
                assert (lse[r] == -np.inf).all() and (out[r] == 0).all()
            else:
                assert (np.abs(lse[r] - parts[1]) <= tol_lse).all(), (r, np.abs(lse[r] - parts[1]).max())


SHAPES = [(8, 2, 128, 64, "bf16", "heads"), (4, 4, 64, 32, "f16", "tokens"), (40, 2, 80, 16, "bf16", "tokens"),
          (16, 1, 256, 128, "bf16", "heads"), (6, 2, 16, 16, "f16", "heads"), (64, 1, 96, 32, "f16", "heads"),
          (5, 5, 192, 64, "bf16", "tokens")]


@pytest.mark.parametrize("q_heads,kv_heads,D,block,dtype,layout", SHAPES)
def test_block_rows(backend, q_heads, kv_heads, D, block, dtype, layout):
    """Rows appear for full blocks alone, range by range."""
    n = 5 * block + 3
    c = Cache(backend, q_heads=q_heads, kv_heads=kv_heads, D=D, block=block, capacity=6 * block, lens=[n, 2 * block, block - 1],
              dtype=dtype, layout=layout, pad=8)
    want = [kb_util.block_rows(c.hk[s], block) for s in range(3)]

    def rows(s, have):
        got = c.kb.read_rows(s)
        for g, w in zip(got, want[s]):
            np.testing.assert_array_equal(g[:, :have], w[:, :have])
            assert not g[:, have:].any()

    c.update([0, 1, 2], [0, 0, 0], [block + 1, 2 * block, block - 1])
    rows(0, 1), rows(1, 2), rows(2, 0)
    c.update([0], [block + 1], [2 * block - 1])
    rows(0, 1)
    c.update([0], [2 * block - 1], [2 * block])
    rows(0, 2)
    c.update([0], [2 * block], [n])
    rows(0, 5), rows(1, 2), rows(2, 0)
    c.kb.Close()


@pytest.mark.parametrize("q_heads,kv_heads,D,block,dtype,layout", SHAPES)
@pytest.mark.parametrize("k", [2, 5, 9])
def test_query(backend, q_heads, kv_heads, D, block, dtype, layout, k):
    """Lengths from nothing to full, rows that share slots, tokens past each
    sequence's end that are NaN."""
    n = 11 * block + 5
    lens = [n, 3 * block, 1, 0, 7 * block + 1]
    c = Cache(backend, q_heads=q_heads, kv_heads=kv_heads, D=D, block=block, capacity=n, lens=lens, dtype=dtype, layout=layout,
              seed=k, fill=float("nan"))
    c.update_all()
    slot = [4, 0, 0, 0, 1, 2, 3, 0, 0, 0, 4, 0]
    length = [lens[4], n, n - 1, n - 2, lens[1], 1, 0, 0, 16, block + 1, 6 * block, 10 * block]
    c.check(c.queries(len(slot)), slot, length, k)
    c.kb.Close()


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("first,last,k", [(0, 1, 1), (0, 1, 7), (2, 3, 8), (4, 4, 8), (1, 1, 64)])
def test_first_and_last(backend, rows, first, last, k):
    c = Cache(backend, q_heads=8, kv_heads=2, D=64, block=16, capacity=1500, lens=[1500, 900], seed=rows)
    c.update_all()
    rng = np.random.default_rng(rows)
    slot = [int(s) for s in rng.integers(0, 2, rows)]
    length = [int(rng.integers(0, c.lens[s] + 1)) for s in slot]
    c.check(c.queries(rows), slot, length, k, first, last)
    c.kb.Close()


def test_many_blocks_and_ties(backend):
    """Thousands of blocks; then all blocks alike, where the lowest numbers win."""
    c = Cache(backend, q_heads=4, kv_heads=2, D=32, block=16, capacity=100_000, lens=[100_000, 65_000], dtype="f16", max_select=1024)
    c.update_all()
    for k in (3, 100, 1024):
        c.check(c.queries(3), [0, 1, 0], [100_000, 65_000, 30_001], k)
    c.k[:] = 1
    c.hk, c.hv = c.host()
    c.update_all()
    sel, _ = c.check(c.queries(1), [0], [100_000], 50)
    want = list(range(49)) + [6249]
    assert sel[0, 0].tolist() == want and sel[0, 1].tolist() == want
    c.kb.Close()


@pytest.mark.parametrize("D,block,k", [(256, 128, 64), (128, 64, 128), (64, 16, 1024), (80, 128, 300)])
def test_one_row_and_many_blocks(backend, D, block, k):
    """One row's blocks split over as many CTAs as there can be."""
    n = block * (k + 20) + 3
    c = Cache(backend, q_heads=2, kv_heads=1, D=D, block=block, capacity=n, lens=[n], seed=D, max_select=1024)
    c.update_all()
    c.check(c.queries(1), [0], [n], k)
    c.check(c.queries(1), [0], [n - block * 19], k)
    c.kb.Close()


@pytest.mark.parametrize("blocks", [257, 258, 259, 1500])
@pytest.mark.parametrize("order", ["few", "rising", "every 256th", "every 128th"])
def test_lists_out_of_order(backend, blocks, order):
    """Equal scores at the last place, scores in order, and all of the best at one remainder of their number."""
    c = Cache(backend, q_heads=2, kv_heads=1, D=32, block=16, capacity=blocks * 16, lens=[blocks * 16], seed=blocks, max_select=80)
    j = np.arange(blocks)
    level = {"few": np.random.default_rng(blocks).integers(0, 4, blocks), "rising": j // 7,
             "every 256th": (j % 256 == 5) * (j + 1), "every 128th": (j % 128 == 70) * (j + 1)}[order]
    c.k[:] = c.torch.tensor(level * 0.01, device="cuda").repeat_interleave(16)[None, None, :, None].to(c.type)
    c.hk, c.hv = c.host()
    c.update_all()
    for k in (6, 65, 66, 67):
        c.check(c.queries(1), [0], [blocks * 16], k)
        c.check(c.queries(1), [0], [blocks * 16], k, 0, 1)
    c.kb.Close()


@pytest.mark.parametrize("q_heads,kv_heads,D,block,dtype", [(8, 1, 128, 16, "bf16"), (3, 1, 48, 64, "f16"), (6, 2, 256, 16, "bf16")])
@pytest.mark.parametrize("blocks", [1, 127, 128, 129])
def test_few_rows_of_short_caches(backend, q_heads, kv_heads, D, block, dtype, blocks):
    """Where a query's two steps become one launch, and just beyond."""
    n = blocks * block
    c = Cache(backend, q_heads=q_heads, kv_heads=kv_heads, D=D, block=block, capacity=n, lens=[n, n], dtype=dtype, seed=blocks, max_select=130)
    c.update_all()
    for k, first, last in ((1, 0, 1), (7, 3, 4), (9, 0, 3), (126, 1, 1), (130, 1, 1)):
        c.check(c.queries(2), [1, 0], [n, n - block // 2], k, first, last)
        c.check(c.queries(1), [1], [min(n, 37 * block + 1)], k, first, last, scale=-0.2)
        c.check(c.queries(2), [0, 1], [0, 1], k, first, last)
    c.kb.Close()


def test_prompt_over_long_and_short_lists(backend):
    """Rows that share a CTA, some with more than a thousand blocks to choose from beside some with few."""
    rows = 160
    c = Cache(backend, q_heads=8, kv_heads=8, D=32, block=16, capacity=18_000, lens=[18_000], max_rows=rows)
    c.update_all()
    length = [18_000 if i % 3 == 0 else 16_390 + i if i % 3 == 1 else 40 * i + 1 for i in range(rows)]
    c.check(c.queries(rows), [0] * rows, length, 9)
    c.kb.Close()


def test_large_and_small_scores(backend):
    """Scores far apart (one token takes all the weight) and a scale of 0, a negative one."""
    c = Cache(backend, q_heads=8, kv_heads=2, D=128, block=64, capacity=700, lens=[700], seed=3)
    c.update_all()
    for size, scale in ((30.0, None), (1e-3, None), (1.0, 0.0), (1.0, -0.3)):
        c.check(c.queries(2, size), [0, 0], [700, 333], 4, scale=scale)
    c.kb.Close()


def test_infinities_and_nan(backend):
    """A NaN or infinite key that is visible reaches the rows that read it, and
    no others; NaN rows rank below every other block."""
    import torch
    c = Cache(backend, q_heads=2, kv_heads=2, D=64, block=16, capacity=320, lens=[320], seed=4)
    c.k[0, 0, 16 * 7 + 2, 5] = float("nan")
    c.v[0, 1, 319, 3] = float("inf")
    c.update_all()
    q = c.queries(1)
    slot, length = c.ints([0]), c.ints([320])
    sel = torch.zeros(1, 2, 8, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(1, 2, device="cuda")
    c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 1, 8, 0.1, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    c.kb.sync()
    codes, mults, _ = c.kb.read_rows(0)
    assert i4_util.numbers(codes[0], mults[0])[7, 5] == 0  # a NaN mean is a zero code
    assert (7 in sel[0, 0].tolist()) == bool(torch.isnan(out[0, 0]).any())
    bad = torch.isinf(out[0, 1])
    assert bad[3] and bad.sum() == 1 and torch.isfinite(lse[0, 1])
    sel[:] = torch.tensor([0, 7, 19, -1, 3, 55, -4, 2], device="cuda")
    c.kb.attend_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 1, 8, 0.1, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    c.kb.sync()
    assert torch.isnan(out[0, 0]).all() and torch.isnan(lse[0, 0]) and torch.isfinite(lse[0, 1])
    c.kb.Close()


def test_given_blocks(backend):
    """Chosen blocks in any order, absent and foreign numbers skipped, a repeated one counted again."""
    import torch
    c = Cache(backend, q_heads=4, kv_heads=2, D=64, block=32, capacity=1000, lens=[1000], seed=5)
    q = c.queries(2)
    lists = [[9, 0, 31, 4, -1, 77], [5, 5, 2, -3, 1 << 30, -(1 << 31)]]
    sel = torch.tensor([[l, l] for l in lists], dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(2, 4, device="cuda")
    slot, length = c.ints([0, 0]), c.ints([999, 170])
    c.kb.attend_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 2, 6, 0.2, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    c.kb.sync()
    for r in range(2):
        n = int(length[r])
        parts = kb_util.attend(c.hk[0], c.hv[0], q[r].float().cpu().numpy(), n, np.array([lists[r]] * 2), 32, 0.2)
        tol, tol_lse = kb_util.tolerances(*parts, 64, 2.0**-8, False)
        assert (np.abs(out[r].double().cpu().numpy() - parts[0]) <= tol).all()
        assert (np.abs(lse[r].double().cpu().numpy() - parts[1]) <= tol_lse).all()
    c.kb.Close()


def test_rows_outside_the_cache(backend):
    """A slot or length outside the cache makes its row see nothing and is reported once."""
    import torch
    c = Cache(backend, q_heads=4, kv_heads=2, D=64, block=32, capacity=300, lens=[300, 200], seed=6)
    c.update_all()
    q = c.queries(6)
    slot, length = c.ints([0, 2, -1, 1, 1, 0]), c.ints([300, 10, 10, 301, -1, 7])
    sel = torch.zeros(6, 2, 4, dtype=torch.int32, device="cuda")
    out, lse = torch.full_like(q, float("nan")), torch.zeros(6, 4, device="cuda")
    c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 6, 4, 0.2, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    with pytest.raises(Fi8Error, match="outside the cache"):
        c.kb.sync()
    c.kb.sync()
    assert not out[1:5].any() and torch.isinf(lse[1:5]).all() and (sel[1:5] == -1).all()
    assert torch.isfinite(out).all() and torch.isfinite(lse[[0, 5]]).all()
    for t in (([0], [-1], [5]), ([2], [0], [5]), ([0], [5], [301]), ([1], [50], [40])):
        slots, a, b = (c.ints(x) for x in t)
        c.kb.update_async(slots.data_ptr(), a.data_ptr(), b.data_ptr(), 1, 300)
        with pytest.raises(Fi8Error, match="outside the cache"):
            c.kb.sync()
    c.kb.Close()


def test_far_offsets_and_query_strides(backend):
    """A cache whose last slot lies past 2^31 values; query rows inside wider rows."""
    import torch
    far = 1_200_000_000
    store = [torch.empty(2 * far + 2 * 400 * 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    c = Cache(backend, q_heads=4, kv_heads=2, D=64, block=32, capacity=400, lens=[400, 400, 400], seed=7)
    views = [torch.as_strided(t, (3, 2, 400, 64), (far, 400 * 64, 64, 1)) for t in store]
    views[0].copy_(c.k), views[1].copy_(c.v)
    c.kb.Close()
    c.kb = backend.NewKeyBlocks(store[0].data_ptr(), store[1].data_ptr(), dtype="bf16", slots=3, kv_heads=2, q_heads=4, head_dim=64,
                                capacity=400, block=32, max_rows=8, max_select=8, slot_stride=far, head_stride=400 * 64,
                                token_stride=64)
    c.update_all()
    wide = torch.zeros(5, 4 * 64 + 72, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 8 : 8 + 256].unflatten(1, (4, 64))
    q.copy_(c.queries(5))
    c.check(q, [2, 0, 1, 2, 2], [400, 399, 77, 33, 1], 4)
    c.kb.Close()


def test_decoding_run(backend):
    """A decoding run of both operators: tokens are appended and their blocks
    made as they fill, on a side stream in one captured graph; the chosen blocks
    are those that a FlatI4 index of the block rows answers."""
    import torch
    steps, start, block, k = 40, 250, 16, 6
    c = Cache(backend, q_heads=4, kv_heads=4, D=64, block=block, capacity=start + steps, lens=[start + steps] * 2, seed=8)
    c.update([0, 1], [0, 0], [start, start - 1])
    stream = torch.cuda.Stream()
    slot, to = c.ints([0, 1]), c.ints([start, start - 1])
    q, out = c.queries(2), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    sel, lse = torch.zeros(2, 4, k, dtype=torch.int32, device="cuda"), torch.zeros(2, 4, device="cuda")
    frm = torch.zeros_like(to)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s = torch.cuda.current_stream().cuda_stream
        frm.copy_(to)
        to.add_(1)
        c.kb.update_async(slot.data_ptr(), frm.data_ptr(), to.data_ptr(), 2, 1, s)
        c.kb.query_async(q.data_ptr(), slot.data_ptr(), to.data_ptr(), 2, k, 0.125, sel.data_ptr(), out.data_ptr(), lse.data_ptr(), stream=s)
    for step in range(steps):
        with torch.cuda.stream(stream):
            q.copy_(torch.randn(2, 4, 64, device="cuda", generator=c.gen))
            graph.replay()
        stream.synchronize()
        n = [start + step + 1, start + step]
        assert to.tolist() == n
        if step % 13 == 0 or step == steps - 1:
            c.compare(q, [0, 1], n, k, 1, 1, 0.125, sel, out, lse)
            codes, mults, scales = c.kb.read_rows(1)
            nb = -(-n[1] // block)
            for h in range(4):
                ix = backend.NewI4Index(codes[h, 1 : nb - 1], mults[h, 1 : nb - 1], scales[h, 1 : nb - 1], nb - 2, 64, id_base=1)
                ids, _ = ix.topk_arrays(q[1, h : h + 1].float().cpu().numpy(), k - 2)
                assert sorted(ids[0].tolist()) == sel[1, h, 1:-1].tolist()
                ix.Close()
    c.kb.sync()
    del graph
    c.kb.Close()


def test_refusals(backend):
    import torch
    c = Cache(backend, q_heads=4, kv_heads=2, D=64, block=32, capacity=64, lens=[64], max_rows=4, max_select=3)
    ok = dict(dtype="bf16", slots=1, kv_heads=2, q_heads=4, head_dim=64, capacity=64, block=32, max_rows=4, max_select=3,
              slot_stride=8192, head_stride=4096, token_stride=64)
    k = c.k.data_ptr()
    for change in (dict(slots=0), dict(capacity=0), dict(q_heads=3), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=72),
                   dict(head_dim=272), dict(block=48), dict(block=256), dict(capacity=36864 * 32 + 1), dict(max_rows=0),
                   dict(max_rows=65536), dict(max_select=0), dict(max_select=1025), dict(token_stride=56), dict(token_stride=68),
                   dict(head_stride=4), dict(slot_stride=-8), dict(q_heads=130)):
        with pytest.raises(Fi8Error):
            backend.NewKeyBlocks(k, k, **{**ok, **change})
    for a, b in ((0, k), (k, 0), (k + 2, k), (k, k + 8)):
        with pytest.raises(Fi8Error):
            backend.NewKeyBlocks(a, b, **ok)
    with pytest.raises(DeclinedError):
        backend.NewKeyBlocks(k, k, **{**ok, "block": 17})
    q, n = c.queries(5), c.ints([0] * 5)
    sel, out = torch.zeros(5, 2, 3, dtype=torch.int32, device="cuda"), torch.zeros_like(q)
    p = [x.data_ptr() for x in (q, n, n, sel, out)]
    kb = c.kb
    for call in (lambda: kb.select_async(p[0], p[1], p[2], 5, 3, p[3]), lambda: kb.select_async(p[0], p[1], p[2], -1, 3, p[3]),
                 lambda: kb.select_async(p[0], p[1], p[2], 1, 4, p[3]), lambda: kb.select_async(p[0], p[1], p[2], 1, 0, p[3]),
                 lambda: kb.select_async(p[0], p[1], p[2], 1, 3, p[3], first=-1), lambda: kb.select_async(p[0], p[1], p[2], 1, 3, p[3], last=0),
                 lambda: kb.select_async(p[0], p[1], p[2], 1, 3, p[3], first=2, last=2), lambda: kb.select_async(0, p[1], p[2], 1, 3, p[3]),
                 lambda: kb.select_async(p[0] + 2, p[1], p[2], 1, 3, p[3]), lambda: kb.select_async(p[0], p[1], p[2], 1, 3, p[3], q_stride=248),
                 lambda: kb.select_async(p[0], p[1], p[2], 1, 3, p[3], q_stride=260), lambda: kb.select_async(p[0], p[1], p[2], 1, 3, 0),
                 lambda: kb.attend_async(p[0], p[1], p[2], 1, 3, float("nan"), p[3], p[4]),
                 lambda: kb.attend_async(p[0], p[1], p[2], 1, 3, 1.0, p[3], 0), lambda: kb.query_async(p[0], p[1], 0, 1, 3, 1.0, p[3], p[4]),
                 lambda: kb.query_async(p[0], p[1], p[2], 1, 3, float("inf"), p[3], p[4]), lambda: kb.update_async(p[1], p[1], p[1], -1, 1),
                 lambda: kb.update_async(p[1], p[1], p[1], 1, -1), lambda: kb.update_async(0, p[1], p[1], 1, 1),
                 lambda: kb.update_async(p[1], p[1], p[1], 65536, 1), lambda: kb.read_rows(1)):
        with pytest.raises(Fi8Error):
            call()
    kb.query_async(0, 0, 0, 0, 3, 1.0, 0, 0)
    kb.update_async(0, 0, 0, 0, 0)
    kb.sync()
    kb.Close()


@pytest.mark.parametrize("q_heads,kv_heads,D,block,dtype,layout", SHAPES)
@pytest.mark.parametrize("rows,k", [(64, 12), (150, 5)])
def test_many_rows(backend, q_heads, kv_heads, D, block, dtype, layout, rows, k):
    """A chunk of one sequence, rows of another one in between, some that see
    nothing or one token."""
    n = 7 * block + 5 + rows
    c = Cache(backend, q_heads=q_heads, kv_heads=kv_heads, D=D, block=block, capacity=n, lens=[n, 2 * block + 7], dtype=dtype,
              layout=layout, seed=rows, max_rows=rows, fill=float("nan"))
    c.update_all()
    slot = [0] * rows
    length = list(range(n - rows + 1, n + 1))
    for i, (s, m) in enumerate([(1, 2 * block + 7), (0, 0), (1, 1), (1, 0), (0, block), (0, 3 * block + 1)]):
        slot[7 * i + 3], length[7 * i + 3] = s, m
    c.check(c.queries(rows), slot, length, k, scale=-0.2 if k == 5 else None)
    c.kb.Close()


@pytest.mark.parametrize("D,block", [(64, 16), (128, 64), (96, 32)])
def test_many_rows_and_hidden_values(backend, D, block):
    """Infinite and NaN keys and values reach the rows that see them and no
    others, in one call of 100 rows as in two of 50."""
    import torch
    rows, n, k = 100, 6 * block + 3, 6
    c = Cache(backend, q_heads=4, kv_heads=2, D=D, block=block, capacity=n, lens=[n, n], seed=1, max_rows=rows)
    c.update_all()
    at = [block + 3, 4 * block + 2, 5 * block + 1]
    c.v[0, 0, at[0], 3], c.v[0, 1, at[1], 1], c.k[1, 0, at[2], 0], c.v[1, 1, at[2] + 3, 5] = float("nan"), float("inf"), float("nan"), -float("inf")
    rng = np.random.default_rng(2)
    slot, length = c.ints(rng.integers(0, 2, rows)), c.ints(rng.integers(0, n + 1, rows))
    q = c.queries(rows)
    sel, out, lse = torch.zeros(rows, 2, k, dtype=torch.int32, device="cuda"), torch.zeros_like(q), torch.zeros(rows, 4, device="cuda")
    c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), rows, k, 0.1, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    sel2, out2, lse2 = torch.zeros_like(sel), torch.zeros_like(out), torch.zeros_like(lse)
    for i in (0, 50):
        c.kb.query_async(q[i:].data_ptr(), slot[i:].data_ptr(), length[i:].data_ptr(), 50, k, 0.1, sel2[i:].data_ptr(), out2[i:].data_ptr(),
                         lse2[i:].data_ptr())
    c.kb.sync()
    assert torch.equal(sel, sel2)
    for a, b, tol in ((out, out2, 2.0**-6), (lse, lse2, 1e-4)):  # each is within its own bound of the truth; these cover both
        a, b = a.float(), b.float()
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        ok = torch.isfinite(a)
        assert ((a - b)[ok].abs() <= tol * (1 + b[ok].abs())).all()
    assert torch.isnan(out).any() and torch.isinf(out).any() and torch.isfinite(out).float().mean() > 0.5
    c.kb.Close()


def test_thousands_of_rows(backend):
    """Every row of 5000 equals its own in a smaller call."""
    import torch
    rows, n, block, k = 5000, 900, 16, 40
    c = Cache(backend, q_heads=8, kv_heads=8, D=32, block=block, capacity=n, lens=[n, n, n], seed=1, max_rows=rows, dtype="f16")
    c.update_all()
    rng = np.random.default_rng(5)
    slot, length = c.ints(np.sort(rng.integers(0, 3, rows))), c.ints(rng.integers(0, n + 1, rows))
    q = c.queries(rows)
    sel, out, lse = torch.zeros(rows, 8, k, dtype=torch.int32, device="cuda"), torch.zeros_like(q), torch.zeros(rows, 8, device="cuda")
    for _ in range(2):
        c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), rows, k, 0.2, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    sel2, out2, lse2 = torch.zeros_like(sel), torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(0, rows, 50):
        c.kb.query_async(q[i:].data_ptr(), slot[i:].data_ptr(), length[i:].data_ptr(), 50, k, 0.2, sel2[i:].data_ptr(), out2[i:].data_ptr(),
                         lse2[i:].data_ptr())
    c.kb.sync()
    assert torch.equal(sel, sel2)
    # weights near 1 differ by a half step of f16 each, results once more
    assert ((out.float() - out2.float()).abs() <= 4 * 2.0**-11 * (1 + out2.float().abs())).all()
    seen = length > 0
    assert torch.equal(torch.isinf(lse).all(1), ~seen) and (lse - lse2)[seen].abs().max() < 1e-5
    c.kb.Close()


@pytest.mark.parametrize("dtype,value", [("f16", 30000.0), ("bf16", 200 * 4096.0)])
@pytest.mark.parametrize("q_heads,D,capacity", [(2, 64, 100), (12, 80, 3000), (3, 256, 3000)])
@pytest.mark.parametrize("scale", [0.37, 1.0, -0.2])
def test_largest_scores(backend, dtype, value, q_heads, D, capacity, scale):
    """Scores from 10^10 on, whose rounding is far more than a factor of the softmax: equal ones still share the weight, smaller
    ones have none."""
    import torch
    c = Cache(backend, q_heads=q_heads, kv_heads=1, D=D, block=16, capacity=capacity, lens=[capacity], dtype=dtype, max_select=200, seed=D)
    c.k[:] = value if scale > 0 else -value
    c.k[:, :, ::3] *= -1
    c.hk, c.hv = c.host()
    q = torch.full((2, q_heads, D), value, device="cuda", dtype=c.type)
    slot, length = c.ints([0, 0]), c.ints([capacity, 39])
    sel = torch.zeros(2, 1, 200, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(2, q_heads, device="cuda")
    c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 2, 200, scale, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    c.kb.sync()
    half = float(torch.finfo(c.type).eps) / 2
    for r, n in enumerate((capacity, 39)):
        seen = [t for t in range(n) if t % 3]
        v = c.hv[0, 0, seen]
        # weights of exactly 1: what is left are sums of n terms, and the result's own rounding
        tol = half * np.abs(v.mean(0)) + (2 * n + 64) * 2.0**-24 * np.abs(v).mean(0) + 2.0**-25
        assert (np.abs(out[r].double().cpu().numpy() - v.mean(0)) <= tol).all()
        want = abs(scale) * D * value**2 + np.log(len(seen))
        assert (np.abs(lse[r].double().cpu().numpy() - want) <= (D + 16) * 2.0**-24 * want).all()
    c.kb.Close()


@pytest.mark.parametrize("q_heads", [1, 12])
@pytest.mark.parametrize("depth,value", [(25.5, 6400), (27, 6400), (30, 60000)])
def test_long_tails(backend, q_heads, depth, value):
    """131,008 f16 tokens whose weights lie 2^-depth under the largest, but whose values are large: they stay in the result."""
    import torch
    n, tops = 131_072, 64
    c = Cache(backend, q_heads=q_heads, kv_heads=1, D=64, block=128, capacity=n, lens=[n], dtype="f16", max_select=1024)
    c.k[:], c.v[:] = 0, value
    c.k[..., 0] = -16
    at = torch.arange(0, 16 * tops, 16, device="cuda")  # a largest weight for every warp that shares the row
    c.k[0, 0, at, 0], c.v[0, 0, at] = 0, 1
    q = torch.zeros(1, q_heads, 64, device="cuda", dtype=c.type)
    q[..., 0] = 1
    slot, length = c.ints([0]), c.ints([n])
    sel = torch.zeros(1, 1, 1024, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(1, q_heads, device="cuda")
    c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 1, 1024, depth * np.log(2) / 16, sel.data_ptr(), out.data_ptr(),
                     lse.data_ptr())
    c.kb.sync()
    tail = (n - tops) * 2.0**-depth
    want = (tops + tail * value) / (tops + tail)
    parts = np.full((q_heads, 64), want), np.full(q_heads, np.log(tops + tail)), np.full((q_heads, 64), want), np.full(q_heads, depth)
    tol, tol_lse = kb_util.tolerances(*parts, n, 64, 2.0**-11, False)  # no allowance for weights that vanish
    assert (np.abs(out[0].double().cpu().numpy() - want) <= tol).all() and (tol < 0.04 * want).all()
    assert (np.abs(lse[0].double().cpu().numpy() - parts[1]) <= tol_lse).all()
    c.kb.Close()


@pytest.mark.parametrize("at", [3, 33, 36])
def test_infinite_score_and_no_scale(backend, at):
    """A visible score of -inf times a scale of 0 is a NaN, in a block's whole pieces as in the sequence's last, ragged one."""
    import torch
    c = Cache(backend, q_heads=2, kv_heads=1, D=64, block=16, capacity=100, lens=[100])
    c.k[0, 0, at, 5] = -float("inf")
    q = c.queries(2).abs()
    slot, length, sel = c.ints([0, 0]), c.ints([37, at]), torch.zeros(2, 1, 8, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(2, 2, device="cuda")
    c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 2, 8, 0.0, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    c.kb.sync()
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert torch.isfinite(out[1]).all() and torch.isfinite(lse[1]).all()  # the row that ends before it
    c.kb.Close()


def test_every_report_arrives(backend):
    """A bad row straight behind a report, on a stream that waits for no other, is reported again."""
    import torch
    c = Cache(backend, q_heads=2, kv_heads=1, D=64, block=16, capacity=100, lens=[100])
    q, slot, length = c.queries(1), c.ints([1]), c.ints([5])
    sel, out = torch.zeros(1, 1, 4, dtype=torch.int32, device="cuda"), torch.zeros_like(q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(300):
        c.kb.query_async(q.data_ptr(), slot.data_ptr(), length.data_ptr(), 1, 4, 0.1, sel.data_ptr(), out.data_ptr(), stream=stream.cuda_stream)
        with pytest.raises(Fi8Error, match="outside the cache"):
            c.kb.sync()
    c.kb.sync()
    c.kb.Close()


@pytest.mark.parametrize("D,block", [(64, 16), (128, 64), (96, 32)])
@pytest.mark.parametrize("at_once", [100, 2])
def test_hidden_values_by_row(backend, D, block, at_once):
    """Which outputs an infinite or NaN key or value reaches, derived from the chosen blocks and lengths; all others are right."""
    import torch
    rows, n, k = 100, 6 * block + 3, 6
    c = Cache(backend, q_heads=4, kv_heads=2, D=D, block=block, capacity=n, lens=[n, n], seed=2, max_rows=rows)
    c.update_all()
    # (slot, head, token, channel, value); a key's reaches all channels and the sum
    planted = [(c.v, 0, 0, block + 3, 3, float("nan")), (c.v, 0, 1, 4 * block + 2, 1, float("inf")),
               (c.k, 1, 0, 5 * block + 1, 0, float("nan")), (c.v, 1, 1, 5 * block + 4, 5, -float("inf"))]
    for t, s, h, at, d, x in planted:
        t[s, h, at, d] = x
    rng = np.random.default_rng(3)
    slot, length = rng.integers(0, 2, rows), rng.integers(0, n + 1, rows)
    for i, (_, s, _, at, _, _) in enumerate(planted):  # the rows that end before the token and right behind it
        slot[2 * i : 2 * i + 2], length[2 * i : 2 * i + 2] = s, (at, at + 1)
    ds, dl, q = c.ints(slot), c.ints(length), c.queries(rows)
    sel, out, lse = torch.zeros(rows, 2, k, dtype=torch.int32, device="cuda"), torch.zeros_like(q), torch.zeros(rows, 4, device="cuda")
    for i in range(0, rows, at_once):
        c.kb.query_async(q[i:].data_ptr(), ds[i:].data_ptr(), dl[i:].data_ptr(), at_once, k, 0.1, sel[i:].data_ptr(), out[i:].data_ptr(),
                         lse[i:].data_ptr())
    c.kb.sync()
    sel, out, lse = sel.cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    hit = 0
    for r in range(rows):
        want, want_lse, mass, size, seen = kb_util.attend(c.hk[slot[r]], c.hv[slot[r]], q[r].float().cpu().numpy(), int(length[r]), sel[r], block, 0.1)
        tol, tol_lse = kb_util.tolerances(want, want_lse, mass, size, seen, D, 2.0**-8, False)
        for t, s, h, at, d, x in planted:
            if s == slot[r] and at < length[r] and at // block in sel[r, h]:
                hit += 1
                heads = slice(2 * h, 2 * h + 2)
                want[heads, slice(None) if t is c.k else d] = x
                if t is c.k:
                    want_lse[heads] = x
        np.testing.assert_array_equal(np.isnan(out[r]), np.isnan(want))
        np.testing.assert_array_equal(np.isnan(lse[r]), np.isnan(want_lse))
        inf = np.isinf(want)
        np.testing.assert_array_equal(out[r][inf], want[inf])
        ok = np.isfinite(want)
        assert (np.abs(out[r][ok] - want[ok]) <= tol[ok]).all()
        ok = np.isfinite(want_lse)
        assert (np.abs(lse[r][ok] - want_lse[ok]) <= tol_lse[ok]).all()
    assert hit > 40
    c.kb.Close()


def test_thousands_of_rows_by_row(backend):
    """Rows out of 5000 against the statement: the first and last ones and some in between."""
    import torch
    rows, n, block, k = 5000, 900, 16, 40
    c = Cache(backend, q_heads=8, kv_heads=8, D=32, block=block, capacity=n, lens=[n, n, n], seed=1, max_rows=rows, dtype="f16")
    c.update_all()
    rng = np.random.default_rng(6)
    slot, length = np.sort(rng.integers(0, 3, rows)), rng.integers(0, n + 1, rows)
    q = c.queries(rows)
    sel, out, lse = torch.zeros(rows, 8, k, dtype=torch.int32, device="cuda"), torch.zeros_like(q), torch.zeros(rows, 8, device="cuda")
    ds, dl = c.ints(slot), c.ints(length)
    c.kb.query_async(q.data_ptr(), ds.data_ptr(), dl.data_ptr(), rows, k, 0.2, sel.data_ptr(), out.data_ptr(), lse.data_ptr())
    c.kb.sync()
    at = np.unique(np.concatenate([np.arange(8), np.arange(rows - 8, rows), rng.integers(0, rows, 80)]))
    c.compare(q[at], slot[at].tolist(), length[at].tolist(), k, 1, 1, 0.2, sel[at], out[at], lse[at])
    c.kb.Close()


@pytest.mark.parametrize("rows,kv_heads,D,blocks", [(16, 1, 256, 64), (2, 8, 256, 128), (4, 4, 208, 128), (15, 1, 256, 200), (10, 5, 64, 128),
                                                   (5, 5, 128, 300), (53, 2, 128, 40)])
def test_rows_around_what_runs_at_once(backend, rows, kv_heads, D, blocks):
    """Numbers of rows at which a row's split over a cluster changes, in one launch and in two."""
    block = 16
    n = blocks * block - 3
    c = Cache(backend, q_heads=2 * kv_heads, kv_heads=kv_heads, D=D, block=block, capacity=n, lens=[n, n], seed=rows)
    c.update_all()
    for m in (rows - 1, rows, rows + 1):
        c.check(c.queries(m), [r % 2 for r in range(m)], [n - 7 * r for r in range(m)], 32)
    c.kb.Close()


def test_cache_shorter_than_a_block(backend):
    """A cache that never fills a block has no rows, and its one block is read."""
    c = Cache(backend, q_heads=4, kv_heads=2, D=64, block=64, capacity=37, lens=[37, 5])
    c.update_all()
    assert [x.shape[:2] for x in c.kb.read_rows(1)] == [(2, 0)] * 3
    c.check(c.queries(4), [0, 1, 1, 0], [37, 5, 0, 1], 1, 0, 1)
    c.kb.Close()
