"""FlatI4 on the device against its numpy statement (i4_util): every result is
whole-number arithmetic followed by two rounded products, so all comparisons
are exact."""
import numpy as np
import pytest

import i4_util
from aikit_b200.ann import unpack_keys
from aikit_b200._ffi import DeclinedError, Fi8Error

pytestmark = pytest.mark.gpu


def rows(n, dim, seed):
    rng = np.random.default_rng(seed)
    spread = np.exp(0.5 * rng.standard_normal(dim))
    return (rng.standard_normal((n, dim)) * spread).astype(np.float32)


def same(a, b):
    a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    assert a.shape == b.shape
    np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dim", [1, 31, 32, 33, 64, 100, 384, 768, 1000, 4096])
@pytest.mark.parametrize("n", [1, 7, 1003])
def test_rows_and_scores(backend, n, dim):
    v, q = rows(n, dim, dim + n), rows(9, dim, 5)
    ix = backend.NewI4IndexFromFloats(v)
    want = i4_util.quantize(v)
    got = ix.read_rows()
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
    for M in (1, 2, 3, 4, 5, 6, 7, 8, 9):
        dst = np.full(M * n, np.nan, np.float32)
        ix.ScoreBatch(q[:M], dst)
        same(dst.reshape(M, n), i4_util.scores(*want, q[:M]))
    iy = backend.NewI4Index(*want, n, dim)
    dst = np.empty(n, np.float32)
    iy.Score(q[0], dst)
    same(dst, i4_util.scores(*want, q[:1])[0])
    ix.Close()
    iy.Close()


@pytest.mark.parametrize("dim,M", [(1537, 16), (3000, 16), (3100, 16), (2000, 9), (64, 16), (130, 12)])
def test_wide_batches(backend, dim, M):
    """Batches that share a pass at dimensions around its limits."""
    n = 333
    v, q = rows(n, dim, dim), rows(M, dim, 5)
    ix = backend.NewI4IndexFromFloats(v)
    dst = np.full(M * n, np.nan, np.float32)
    ix.ScoreBatch(q, dst)
    want = i4_util.scores(*i4_util.quantize(v), q)
    same(dst.reshape(M, n), want)
    wi, ws = i4_util.topk(want, 21)
    idx, sc = ix.topk_arrays(q, 21)
    np.testing.assert_array_equal(idx, wi)
    same(sc, ws)
    ix.Close()


def test_set_rows_in_parts(backend):
    """Rows set in pieces that start and end inside the device's groups of rows."""
    import torch
    n, dim = 117, 45
    v = rows(n, dim, 9)
    dv = torch.from_numpy(v).cuda()
    ix = backend.NewI4IndexEmpty(n, dim)
    for a, b in ((3, 4), (60, 117), (4, 41), (41, 60), (0, 3)):
        ix.set_rows_async(a, dv[a:b].data_ptr(), b - a)
    for got, want in zip(ix.read_rows(), i4_util.quantize(v)):
        np.testing.assert_array_equal(got, want)
    ix.set_rows_async(10, dv[50:].data_ptr(), 5)
    v[10:15] = v[50:55]
    for got, want in zip(ix.read_rows(), i4_util.quantize(v)):
        np.testing.assert_array_equal(got, want)
    ix.Close()


@pytest.mark.parametrize("k", [1, 100, 2048])
def test_infinite_and_few_scores(backend, k):
    """Scores of both infinities, of two values, and of which nearly all are NaN."""
    n = 70_000
    codes, mults, _ = i4_util.quantize(np.ones((n, 32), np.float32))
    q = np.ones((2, 32), np.float32)
    q[1] = -1
    rng = np.random.default_rng(k)
    for scales in (np.where(rng.random(n) < 0.01, np.inf, rng.standard_normal(n)), np.where(rng.random(n) < 0.001, 2.0, -1.0),
                   np.where(rng.random(n) < 0.999, np.nan, 1.0), np.full(n, np.nan), rng.standard_normal(n) * 1e-38):
        scales = scales.astype(np.float32)
        ix = backend.NewI4Index(codes, mults, scales, n, 32)
        wi, ws = i4_util.topk(i4_util.scores(codes, mults, scales, q), k)
        idx, sc = ix.topk_arrays(q, k)
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
        ix.Close()


@pytest.mark.parametrize("n", [262_144, 262_145])
@pytest.mark.parametrize("k", [1, 32, 33, 50, 51])
def test_close_scores(backend, n, k):
    """Scores some roundings apart, equal but for a few, and tied at the last place, at the sizes where the selection changes its form."""
    codes, mults, _ = i4_util.quantize(np.ones((n, 64), np.float32))
    q = np.ones((1, 64), np.float32)
    rng = np.random.default_rng(n + k)
    some = rng.permutation(n)[: k + 40]
    few = np.ones(n)
    few[some] = 1 + np.arange(k + 40) // 2 * 2.0**-20
    for scales in (1 + rng.integers(0, 64, n) * 2.0**-23, -1 - rng.integers(0, 9000, n) * 2.0**-23, few, np.where(few > 1, 5.0, -few)):
        scales = scales.astype(np.float32)
        ix = backend.NewI4Index(codes, mults, scales, n, 64)
        wi, ws = i4_util.topk(i4_util.scores(codes, mults, scales, q), k)
        idx, sc = ix.topk_arrays(q, k)
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
        ix.Close()


def test_odd_rows_and_queries(backend):
    """Zero, NaN, infinite, tiny and huge rows and queries; every nibble and multiplier."""
    v = rows(40, 70, 1)
    v[0] = 0
    v[1] = np.nan
    v[2, 3] = np.inf
    v[3] = 0
    v[3, 0] = 1e-44
    v[4] *= np.float32(1e30)
    v[5, 64:] = 0
    v[6, ::2] = np.nan
    v[7, :32] *= np.float32(1e-30)
    q = rows(4, 70, 2)
    q[1] = 0
    q[2] *= np.float32(1e25)
    q[3, 5] = np.nan
    ix = backend.NewI4IndexFromFloats(v)
    want = i4_util.quantize(v)
    for a, b in zip(ix.read_rows(), want):
        np.testing.assert_array_equal(a, b)
    dst = np.empty(4 * 40, np.float32)
    ix.ScoreBatch(q, dst)
    same(dst.reshape(4, 40), i4_util.scores(*want, q))
    idx, sc = ix.topk_arrays(q, 39)
    wi, ws = i4_util.topk(i4_util.scores(*want, q), 39)
    np.testing.assert_array_equal(idx, wi)
    same(sc, ws)
    rng = np.random.default_rng(3)
    codes, mults = rng.integers(0, 256, (300, 3, 16), np.uint8), rng.integers(0, 256, (300, 3), np.uint8)
    codes[0], mults[0] = 0, 255
    codes[1], mults[1] = 255, 255
    scales = rng.standard_normal(300).astype(np.float32)
    iy = backend.NewI4Index(codes, mults, scales, 300, 96)
    big = np.where(np.arange(96) % 2, 1, -1).astype(np.float32)[None].repeat(2, 0)
    big[1] = 1
    dst = np.empty(600, np.float32)
    iy.ScoreBatch(big, dst)
    same(dst.reshape(2, 300), i4_util.scores(codes, mults, scales, big))
    ix.Close()
    iy.Close()


def test_largest_dot(backend):
    """4096 values of the largest size: the dot stays whole in 32 bits."""
    codes, mults = np.zeros((2, 128, 16), np.uint8), np.full((2, 128), 255, np.uint8)
    codes[1] = 255
    ix = backend.NewI4Index(codes, mults, np.ones(2), 2, 4096)
    q = np.stack([np.ones(4096), -np.ones(4096)]).astype(np.float32)
    dst = np.empty(4, np.float32)
    ix.ScoreBatch(q, dst)
    same(dst.reshape(2, 2), i4_util.scores(codes, mults, np.ones(2, np.float32), q))
    ix.Close()


@pytest.mark.parametrize("n,dim,M,k", [(2, 32, 1, 1), (500, 33, 3, 499), (5000, 64, 1, 10), (5000, 64, 8, 100),
                                       (40_000, 96, 5, 1000), (40_000, 32, 17, 2048), (1024, 40, 2, 1023),
                                       (1025, 40, 1, 7), (300_001, 32, 1, 2048), (300_001, 32, 8, 50)])
def test_topk(backend, n, dim, M, k):
    v, q = rows(n, dim, n), rows(M, dim, 3)
    ix = backend.NewI4IndexFromFloats(v)
    wi, ws = i4_util.topk(i4_util.scores(*i4_util.quantize(v), q), k)
    for _ in range(2):  # the scratch returns to rest
        idx, sc = ix.topk_arrays(q, k)
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
    hits = ix.TopKBatch(q, min(k, 3))
    assert [h.Index for h in hits[0]] == wi[0, : min(k, 3)].tolist()
    ix.Close()


@pytest.mark.parametrize("M", [1, 4])
def test_ties_and_order(backend, M):
    """All rows alike, few distinct scores, and rows ordered against the query."""
    v = np.ones((30_000, 32), np.float32)
    q = np.ones((M, 32), np.float32)
    ix = backend.NewI4IndexFromFloats(v)
    idx, _ = ix.topk_arrays(q, 777)
    np.testing.assert_array_equal(idx, np.tile(np.arange(777), (M, 1)))
    ix.Close()
    scales = (np.arange(30_000) // 100 + 1).astype(np.float32)
    for s in (scales, scales[::-1].copy()):
        codes, mults, _ = i4_util.quantize(v)
        ix = backend.NewI4Index(codes, mults, s, 30_000, 32)
        wi, ws = i4_util.topk(i4_util.scores(codes, mults, s, q), 250)
        idx, sc = ix.topk_arrays(q, 250)
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
        ix.Close()


def test_keep_and_id_base(backend):
    v, q = rows(20_000, 48, 1), rows(3, 48, 2)
    base = 1000
    ix = backend.NewI4IndexFromFloats(v, id_base=base)
    score = i4_util.scores(*i4_util.quantize(v), q)
    rng = np.random.default_rng(1)
    for keep in (rng.random(base + 20_000) < 0.5, rng.random(base + 9_000) < 0.001, np.zeros(base + 20_000, bool),
                 np.zeros(0, bool)):
        full = np.zeros(base + 20_000, bool)
        full[: len(keep)] = keep
        wi, ws = i4_util.topk(score, 60, full, base)
        idx, sc = ix.topk_arrays(q, 60, keep=keep)
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
    assert ix.QueryFilterBatch(q, 5, np.zeros(4, bool)) == [[], [], []]
    ix.Close()


def test_row_ranges_and_shards(backend):
    """More scores than the scratch holds at once, and the same rows as two
    shards whose keys are merged."""
    import torch
    n, dim, M, k = 2_300_000, 32, 8, 40
    gen = torch.Generator("cuda").manual_seed(1)
    v = torch.randn(n, dim, device="cuda", generator=gen)
    q = torch.randn(M, dim, device="cuda", generator=gen)
    torch.cuda.synchronize()
    ix = backend.NewI4IndexEmpty(n, dim)
    ix.set_rows_async(0, v.data_ptr(), n)
    keys = torch.zeros(M, k, dtype=torch.int64, device="cuda")
    ix.topk_async(q.data_ptr(), M, k, keys.data_ptr())
    scores = torch.empty(M, n, device="cuda")
    ix.score_async(q.data_ptr(), M, scores.data_ptr())
    torch.cuda.synchronize()
    wi, ws = i4_util.topk(scores.cpu().numpy(), k)
    idx, sc = unpack_keys(keys.cpu().numpy().view(np.uint64))
    np.testing.assert_array_equal(idx, wi)
    same(sc, ws)
    at = torch.cat([torch.arange(5), torch.arange(n - 5, n)])
    same(scores[:, at].cpu(), i4_util.scores(*i4_util.quantize(v[at].cpu().numpy()), q.cpu().numpy()))
    both = torch.zeros(2, M, k, dtype=torch.int64, device="cuda")
    cut = 2_299_980  # the second shard is smaller than k
    parts = []
    for i, (a, b) in enumerate(((0, cut), (cut, n))):
        part = backend.NewI4IndexEmpty(b - a, dim, id_base=a)
        part.set_rows_async(0, v[a:b].data_ptr(), b - a)
        part.topk_async(q.data_ptr(), M, k, both[i].data_ptr())
        parts.append(part)
    merged = torch.zeros_like(keys)
    backend.ctx.merge_keys_async(both.data_ptr(), 2, M, k, merged.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(merged, keys)
    for p in parts + [ix]:
        p.Close()


def test_far_rows(backend):
    """Rows past 2^31 bytes."""
    import torch
    n, dim = 4_300_000, 1024
    ix = backend.NewI4IndexEmpty(n, dim)
    v = torch.randn(3000, dim, device="cuda")
    q = torch.randn(1, dim, device="cuda")
    ix.set_rows_async(n - 3000, v.data_ptr(), 3000)
    dst = torch.empty(1, n, device="cuda")
    ix.score_async(q.data_ptr(), 1, dst.data_ptr())
    torch.cuda.synchronize()
    want = i4_util.scores(*i4_util.quantize(v.cpu().numpy()), q.cpu().numpy())
    same(dst[:, n - 3000:].cpu(), want)
    assert not dst[:, : n - 3000].any()
    ix.Close()


def test_streams_and_graph(backend):
    """Fill, score and search on a side stream; the same calls captured and
    replayed with other queries in place."""
    import torch
    n, dim, M, k = 50_000, 100, 3, 20
    v, q = rows(n, dim, 1), rows(2 * M, dim, 2)
    ix = backend.NewI4IndexEmpty(n, dim)
    stream = torch.cuda.Stream()
    dv, dq = torch.from_numpy(v).cuda(), torch.from_numpy(q[:M].copy()).cuda()
    keys = torch.zeros(M, k, dtype=torch.int64, device="cuda")
    scores = torch.zeros(M, n, device="cuda")
    torch.cuda.synchronize()
    s = stream.cuda_stream
    ix.set_rows_async(0, dv.data_ptr(), n, s)
    ix.score_async(dq.data_ptr(), M, scores.data_ptr(), s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ix.score_async(dq.data_ptr(), M, scores.data_ptr(), torch.cuda.current_stream().cuda_stream)
        ix.topk_async(dq.data_ptr(), M, k, keys.data_ptr(), torch.cuda.current_stream().cuda_stream)
    packed = i4_util.quantize(v)
    for part in (q[:M], q[M:], q[:M]):
        with torch.cuda.stream(stream):
            dq.copy_(torch.from_numpy(part.copy()))
            graph.replay()
        stream.synchronize()
        want = i4_util.scores(*packed, part)
        same(scores.cpu(), want)
        wi, ws = i4_util.topk(want, k)
        idx, sc = unpack_keys(keys.cpu().numpy().view(np.uint64))
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
    del graph
    ix.Close()


def test_refusals(backend):
    v = rows(100, 32, 1)
    ix = backend.NewI4IndexFromFloats(v)
    q = np.ones((1, 32), np.float32)
    for k in (0, -1, 100, 101):
        with pytest.raises(DeclinedError):
            ix.topk_arrays(q, k)
    with pytest.raises(DeclinedError):
        ix.topk_async(16, 1, 2049, 16)
    with pytest.raises(Fi8Error):
        ix.topk_async(0, 1, 5, 16)
    with pytest.raises(Fi8Error):
        ix.score_async(16, 1, 0)
    with pytest.raises(Fi8Error):
        ix.score_async(16, -1, 16)
    for row0, count in ((-1, 2), (99, 2), (0, 101), (0, -1)):
        with pytest.raises(Fi8Error):
            ix.set_rows_async(row0, 16, count)
    assert ix.topk_arrays(np.empty((0, 32)), 5)[0].shape == (0, 5)
    with pytest.raises(DeclinedError):
        backend.NewI4IndexEmpty(10, 4097)
    with pytest.raises(Fi8Error, match="31 bits"):
        backend.NewI4IndexEmpty(10, 32, id_base=2**31 - 5)
    with pytest.raises(Fi8Error, match="empty"):
        backend.NewI4IndexEmpty(0, 32)
    ix.Close()


@pytest.mark.parametrize("n,k", [(262_145, 1200), (262_145, 2048), (300_001, 2048), (591_000, 2048)])
def test_every_run_picked(backend, n, k):
    """So many picks that all runs of tiles are among them: the same answer, and the right one, call after call."""
    v, q = rows(n, 32, k), rows(8, 32, 4)
    ix = backend.NewI4IndexFromFloats(v)
    wi, ws = i4_util.topk(i4_util.scores(*i4_util.quantize(v), q), k)
    for _ in range(25):
        idx, sc = ix.topk_arrays(q, k)
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
    ix.Close()


def test_host_calls_behind_set_rows(backend):
    """The host forms answer over the rows that calls before them set, on whichever stream; of two calls for the same rows the
    later one stays."""
    import torch
    n, dim, k = 5000, 64, 10
    old, new, q = rows(n, dim, 1), rows(n, dim, 2), rows(2, dim, 3)
    d_old, d_new = torch.from_numpy(old).cuda(), torch.from_numpy(new).cuda()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    ix = backend.NewI4IndexEmpty(n, dim)
    torch.cuda.synchronize()
    for last, stream in ((old, one), (new, two), (old, one)):
        with torch.cuda.stream(one):
            torch.cuda._sleep(40_000_000)  # some 20 ms: longer than what follows
        ix.set_rows_async(0, d_new.data_ptr(), n, one.cuda_stream)
        ix.set_rows_async(0, (d_old if last is old else d_new).data_ptr(), n, stream.cuda_stream)
        want = i4_util.scores(*i4_util.quantize(last), q)
        dst = np.empty(2 * n, np.float32)
        ix.ScoreBatch(q, dst)
        same(dst.reshape(2, n), want)
        with torch.cuda.stream(one):
            torch.cuda._sleep(40_000_000)
        ix.set_rows_async(7, d_old[7:].data_ptr(), 100, one.cuda_stream)
        mixed = last.copy()
        mixed[7:107] = old[7:107]
        wi, ws = i4_util.topk(i4_util.scores(*i4_util.quantize(mixed), q), k)
        idx, sc = ix.topk_arrays(q, k)
        np.testing.assert_array_equal(idx, wi)
        same(sc, ws)
    ix.Close()


def test_captured_set_rows(backend):
    """Rows set by a captured call, replayed with other vectors in place."""
    import torch
    n, dim = 300, 40
    v, q = rows(2 * n, dim, 1), rows(1, dim, 2)
    dv, dq, dst = torch.from_numpy(v[:n]).cuda(), torch.from_numpy(q).cuda(), torch.zeros(1, n, device="cuda")
    ix = backend.NewI4IndexEmpty(n, dim)
    ix.set_rows_async(0, dv.data_ptr(), n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = torch.cuda.current_stream().cuda_stream
        ix.set_rows_async(0, dv.data_ptr(), n, s)
        ix.score_async(dq.data_ptr(), 1, dst.data_ptr(), s)
    for part in (v[n:], v[:n]):
        dv.copy_(torch.from_numpy(part.copy()))
        graph.replay()
        torch.cuda.synchronize()
        want = i4_util.scores(*i4_util.quantize(part), q)
        same(dst.cpu(), want)
        host = np.empty(n, np.float32)
        ix.Score(q[0], host)
        same(host, want[0])
    del graph
    ix.Close()


@pytest.mark.parametrize("n,k", [(8_500_000, 1), (8_500_000, 100), (34_000_000, 2048)])
@pytest.mark.parametrize("distinct", [3000, 1_000_000])
def test_topk_of_very_many_rows(backend, n, k, distinct):
    """Runs of 512, 64 and 32 tiles, those of the last more than fit shared memory, with ties within runs and across them."""
    import torch
    dim, M = 32, 2
    gen = torch.Generator("cuda").manual_seed(k + distinct)
    some = torch.randn(distinct, dim, device="cuda", generator=gen)
    q = torch.randn(M, dim, device="cuda", generator=gen)
    ix = backend.NewI4IndexEmpty(n, dim)
    stream = torch.cuda.current_stream().cuda_stream
    for a in range(0, n, 1 << 22):
        m = min(1 << 22, n - a)
        v = some[torch.randint(distinct, (m,), device="cuda", generator=gen)]
        ix.set_rows_async(a, v.data_ptr(), m, stream)
        torch.cuda.synchronize()
    keys, scores = torch.zeros(M, k, dtype=torch.int64, device="cuda"), torch.empty(M, n, device="cuda")
    ix.topk_async(q.data_ptr(), M, k, keys.data_ptr(), stream)
    ix.score_async(q.data_ptr(), M, scores.data_ptr(), stream)
    torch.cuda.synchronize()
    idx, sc = unpack_keys(keys.cpu().numpy().view(np.uint64))
    for m in range(M):
        # the scores in order, and where one is tied the rows in order: a stable sort
        want = torch.sort(scores[m], descending=True, stable=True)
        np.testing.assert_array_equal(idx[m], want.indices[:k].cpu().numpy())
        same(sc[m], want.values[:k].cpu())
        if distinct < n // 2048:  # more copies of the best row than there are picks
            assert want.values[0] == want.values[k]
    ix.Close()
