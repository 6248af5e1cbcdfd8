"""4-bit rows (cz_q4_*): quantising, decoding, products, exhaustive k-NN against plain implementations in 64 bits."""
import numpy as np
import pytest

from tests import table_ref as R

U32 = 2.0 ** -24  # half a step of f32, relative


def _table(n, dim, group, seed, kind="normal"):
    """random codes (-8 among them), scales and squared norms on the host"""
    rng = np.random.default_rng(seed)
    groups = -(-dim // group)
    c = rng.integers(-8, 8, (n, groups * group))
    c[:, dim:] = 0
    s = R.bf16_value(R.bf16_bits(np.exp(rng.uniform(-4, 2, (n, groups))).astype(np.float32)))
    codes = R.pack(c)
    x = R.decode(codes, s, dim)
    return codes, R.bf16_bits(s), (x ** 2).sum(1).astype(np.float32), x


def _q4(codes, scales, sq, dim):
    from cozo_amd.quantized import Q4Table
    return Q4Table(codes, scales, sq, dim)


def _gpu_table(codes, scales, sq, dim):
    import torch
    return _q4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales.view(np.int16)).cuda().view(torch.bfloat16),
               torch.from_numpy(sq).cuda(), dim)


# ---- on the CPU ----------------------------------------------------------------------------------------------------
def test_refusals():
    import ctypes as C
    from cozo_amd import _lib, quantized
    L = _lib.lib()
    x = np.zeros((4, 40), np.float32)
    for bad in (dict(group=16), dict(group=0)):
        with pytest.raises(ValueError):
            quantized.quantize(x, **bad)
    with pytest.raises(ValueError):
        quantized.quantize(np.zeros((4, 40), np.float64))
    with pytest.raises(ValueError):
        quantized.quantize(np.zeros(40, np.float32))
    codes, scales, sq, _ = _table(4, 40, 32, 0)
    with pytest.raises(ValueError):
        _q4(codes, scales, sq, 65)  # two groups of 32 hold 33..64
    with pytest.raises(ValueError):
        _q4(codes, scales, sq[:3], 40)
    with pytest.raises(ValueError):
        _q4(codes, scales.astype(np.float32), sq, 40)
    with pytest.raises(ValueError):
        _q4(codes[:, ::-1], scales, sq, 40)
    t = _q4(codes, scales, sq, 40)
    with pytest.raises(ValueError):
        t.dots(np.zeros((2, 41), np.float32))
    with pytest.raises(KeyError):
        t.knn(np.zeros((2, 40), np.float32), 3, distance="Hamming")
    with pytest.raises(ValueError):
        _q4(codes, scales, None, 40).knn(np.zeros((2, 40), np.float32), 3)
    # the C entries look at sizes before they look for a device
    buf = np.zeros(64, np.uint8)
    p = _lib.ptr(buf)
    assert L.cz_q4_quantize(p, 0, 1, 0, 0, 32, p, p, p, 0, None) == _lib.CZ_E_UNSUPPORTED
    assert L.cz_q4_quantize(p, 0, 1, 8193, 8193, 32, p, p, p, 0, None) == _lib.CZ_E_UNSUPPORTED
    assert L.cz_q4_quantize(p, 7, 1, 4, 4, 32, p, p, p, 0, None) == _lib.CZ_E_INVALID
    assert L.cz_q4_quantize(p, 0, 1, 4, 3, 32, p, p, p, 0, None) == _lib.CZ_E_INVALID
    assert L.cz_q4_quantize(p, 0, 1, 4, 4, 48, p, p, p, 0, None) == _lib.CZ_E_INVALID
    assert L.cz_q4_quantize(p, 0, 1 << 31, 4, 4, 32, p, p, p, 0, None) == _lib.CZ_E_INVALID
    assert L.cz_q4_dequantize(p, p, 2, 4, 32, None, 1, p, 0, None) == _lib.CZ_E_INVALID
    knn = lambda metric, k: L.cz_q4_knn(metric, p, p, p, 1, 4, 32, p, 1, k, 0, 0.0, p, p, p, None, 0, None, 0, None)  # noqa: E731
    assert knn(3, 1) == _lib.CZ_E_INVALID
    assert knn(0, 0) == _lib.CZ_E_UNSUPPORTED and knn(0, 1025) == _lib.CZ_E_UNSUPPORTED
    assert L.cz_q4_workspace(10, 4, 48, 1, 1) == 0 and L.cz_q4_workspace(10, 4, 32, 1, 1025) == 0
    assert L.cz_q4_workspace(10, 4, 32, 1, 1) > 0 and L.cz_q4_workspace(0, 4, 32, 1, 1) > 0


def test_no_device_no_answer():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    from cozo_amd import _lib, quantized
    with pytest.raises(_lib.CozoGpuError) as e:
        quantized.quantize(np.ones((2, 8), np.float32))
    assert e.value.code == _lib.CZ_E_NO_DEVICE


def test_reference_round_trip():
    """the restatement itself: an element is off by at most half a code step, plus what rounding the scale to 8 bits cuts off at the
    group's end (the largest element may be 7 + 7 * 2^-8 steps and is clamped to 7)"""
    x = np.random.default_rng(1).standard_normal((50, 70)).astype(np.float32)
    c, s = R.quantize(x, 32)
    step = np.repeat(s, 32, 1)[:, :70].astype(np.float64)
    back = R.decode(R.pack(c), s, 70)
    assert np.all(np.abs(back - x) <= step * (0.5 + 1e-5))
    assert np.array_equal(R.unpack(R.pack(c)), c)


# ---- on the GPU ----------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n,dim", [(1, 1), (5, 31), (3, 32), (257, 33), (64, 100), (1000, 128), (33, 200), (130, 768), (17, 1000), (3, 8192)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize(gpu_lib, n, dim, group, dtype):
    from cozo_amd import quantized
    rng = np.random.default_rng(n * dim + group)
    x = (rng.standard_normal((n, dim)) * np.exp(rng.uniform(-20, 20, (n, 1)))).astype(np.float32)
    x[0] = 0
    if n > 2:
        x[2] *= np.float32(2.0 ** -70 / max(np.abs(x[2]).max(), 1e-30))  # below what a scale is kept for
    arg = x
    if dtype == "bf16":
        arg = R.bf16_bits(x)
        x = R.bf16_value(arg)
    c, s = R.quantize(x, group)
    t = quantized.quantize(arg, group=group)
    assert np.array_equal(t.codes, R.pack(c))
    assert np.array_equal(t.scales, R.bf16_bits(s))
    want = R.decode(t.codes, s, dim)
    sq = (want ** 2).sum(1)
    assert np.allclose(t.sqnorms, sq, rtol=2 * U32, atol=0)  # one rounding of an f64 sum
    assert np.array_equal(t.dequantize(), want.astype(np.float32))  # 3 bits times 8 bits: exact
    if n > 1:
        rows = rng.integers(0, n, 7)
        assert np.array_equal(t.dequantize(rows), want[rows].astype(np.float32))


@pytest.mark.gpu
def test_quantize_strided_and_device(gpu_lib):
    import torch
    from cozo_amd import quantized
    x = torch.randn(100, 96, device="cuda")
    for view in (x[:, :70], x[:, 3:70], x[::2, 1:90], x.t(), x[:1].expand(4, 96), x[5:6, :]):
        for v in (view, view.to(torch.bfloat16)):
            a, b = quantized.quantize(v, group=32), quantized.quantize(v.contiguous().clone(), group=32)
            h = quantized.quantize(v.float().cpu().numpy(), group=32)
            assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.sqnorms, b.sqnorms)
            assert np.array_equal(a.codes.cpu().numpy(), h.codes) and np.array_equal(a.sqnorms.cpu().numpy(), h.sqnorms)
    wide = torch.randn(40, 200, device="cuda").to(torch.bfloat16)
    v = wide[:, :72]  # rows 400 bytes apart
    a, b = quantized.quantize(v), quantized.quantize(v.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.dequantize(), b.dequantize())
    rows = torch.tensor([3, 39, 40, -1, 0], device="cuda")
    got = a.dequantize(rows)
    assert torch.equal(got[[0, 1, 4]], a.dequantize()[[3, 39, 0]]) and bool(got[2:4].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_quantize_non_finite(gpu_lib, bad):
    from cozo_amd import quantized
    x = np.random.default_rng(3).standard_normal((6, 100)).astype(np.float32)
    x[1, 40] = bad
    t = quantized.quantize(x, group=32)
    back = t.dequantize()
    assert np.isnan(back[1, 32:64]).all() and np.isnan(t.sqnorms[1]) and np.isfinite(np.delete(back, 1, 0)).all()
    d = t.dots(np.ones((2, 100), np.float32))
    assert np.isnan(d[:, 1]).all() and np.isfinite(np.delete(d, 1, 1)).all()
    for metric in ("L2", "Cosine", "IP"):
        ids, dist, cnt = t.knn(x[:1], 6, distance=metric)
        assert ids[0, 5] == 1 and np.isnan(dist[0, 5]) and cnt[0] == 6 and np.isfinite(dist[0, :5]).all()


def _dots_tol(q, x):
    """f32 sums of dim terms, and a query held to 2^-31 of its largest element (half a step of a 31-bit fixed point)"""
    q, x = np.abs(np.asarray(q, np.float64)), np.abs(x)
    return (x.shape[1] + 64) * U32 * (q @ x.T) * 3 + 2.0 ** -30 * q.max(1)[:, None] * x.sum(1)[None, :] + 1e-37


@pytest.mark.gpu
@pytest.mark.parametrize("n,dim", [(1, 1), (15, 7), (16, 32), (33, 100), (257, 128), (1000, 200), (129, 768), (70, 1024), (40, 1999), (5, 8192)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B", [1, 3, 4, 5, 17, 70])
def test_dots(gpu_lib, n, dim, group, B):
    codes, scales, sq, x = _table(n, dim, group, n + dim)
    rng = np.random.default_rng(B)
    q = rng.standard_normal((B, dim)).astype(np.float32)
    q[0] *= np.float32(1e6)
    if B > 1:
        q[1, rng.random(dim) < 0.7] *= np.float32(1e-4)  # a wide range of magnitudes within a query
    if B > 2:
        q[2] = 0
    got = _gpu_table(codes, scales, sq, dim).dots(_cuda(q)).cpu().numpy()
    want = q.astype(np.float64) @ x.T
    assert got.shape == (B, n) and np.all(np.abs(got - want) <= _dots_tol(q, x))
    if B == 3:
        assert np.array_equal(got, _q4(codes, scales, sq, dim).dots(q))


def _cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.gpu
def test_dots_query_values(gpu_lib):
    """queries with nothing, with extremes and with values that are no numbers; one query does not touch another"""
    codes, scales, sq, x = _table(100, 90, 32, 5)
    t = _gpu_table(codes, scales, sq, 90)
    q = np.random.default_rng(1).standard_normal((6, 90)).astype(np.float32)
    clean = t.dots(_cuda(q)).cpu().numpy()
    q[1, 5], q[3, 80], q[4] = np.nan, -np.inf, 1e-40
    got = t.dots(_cuda(q)).cpu().numpy()
    assert np.isnan(got[1]).all() and np.isnan(got[3]).all()
    assert np.array_equal(got[[0, 2, 5]], clean[[0, 2, 5]])
    assert np.all(np.abs(got[4] - q[4].astype(np.float64) @ x.T) <= _dots_tol(q[4:5], x)[0])
    assert t.dots(_cuda(q[:0])).shape == (0, 100)
    big = np.full((1, 90), 3e38, np.float32)
    assert np.isfinite(t.dots(_cuda(big * np.float32(1e-4)))[0].cpu().numpy()).all()


METRICS = ["L2", "Cosine", "IP"]


def _check_knn(t, q, x, k, metric, radius=None, host=False, only=None):
    """the answer to the whole batch, looked at for all queries or for those that `only` names"""
    ids, dist, cnt = t.knn(q if host else _cuda(q), k, distance=metric, radius=radius)
    if not host:
        ids, dist, cnt = ids.cpu().numpy().view(np.uint32), dist.cpu().numpy(), cnt.cpu().numpy().view(np.uint32)
    if only is not None:
        q, ids, dist, cnt = q[only], ids[only], dist[only], cnt[only]
    all_d = R.distances(metric, q, x)
    _, wdist, wcnt = R.nearest(all_d, k, radius)
    assert np.array_equal(cnt, wcnt)
    # f64 sums of dim products: a distance is known to dim * 2^-53 of what its terms add up to (for a cosine: of 1 and of the dot's terms)
    if metric == "L2":
        tol = 4 * x.shape[1] * 2.0 ** -53 * wdist
    elif metric == "IP":
        tol = 4 * x.shape[1] * 2.0 ** -53 * (1 + np.nan_to_num(np.abs(q).astype(np.float64)) @ np.nan_to_num(np.abs(x)).T).max(1)[:, None]
    else:
        tol = np.full_like(wdist, 8 * x.shape[1] * 2.0 ** -53)
    tol = np.broadcast_to(tol, wdist.shape)
    for b in range(q.shape[0]):
        c = int(cnt[b])
        assert np.all(ids[b, c:] == 0xFFFFFFFF) and np.all(np.isinf(dist[b, c:]))
        got, want = dist[b, :c], wdist[b, :c]
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fin = ~np.isnan(want)
        assert np.all(np.abs(got[fin] - want[fin]) <= tol[b, :c][fin]), (metric, b)
        # every id has the distance that stands beside it, none comes twice, ties ascend by row
        assert np.unique(ids[b, :c]).size == c
        own = all_d[b, ids[b, :c].astype(np.int64)]
        assert np.all(np.abs(own[fin] - got[fin]) <= tol[b, :c][fin])
        same = got[1:] == got[:-1]
        assert np.all(ids[b, 1:c][same] > ids[b, :c - 1][same])
    return ids, dist


@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("n,dim,group,B,k", [(1, 1, 32, 1, 1), (5, 40, 32, 3, 9), (63, 33, 64, 2, 10), (1000, 128, 32, 5, 10), (4099, 96, 32, 40, 7),
                                             (20000, 200, 128, 3, 100), (70000, 64, 64, 1, 10), (70000, 64, 64, 33, 13), (6000, 768, 64, 130, 10),
                                             (3000, 8192, 64, 1, 5), (9000, 48, 32, 2, 1024)])
def test_knn(gpu_lib, metric, n, dim, group, B, k):
    codes, scales, sq, x = _table(n, dim, group, n + B)
    rng = np.random.default_rng(k)
    q = rng.standard_normal((B, dim)).astype(np.float32)
    near = rng.integers(0, n, B)
    q[::2] = x[near[::2]].astype(np.float32) + np.float32(0.1) * q[::2]  # near a row of the table
    _check_knn(_gpu_table(codes, scales, sq, dim), q, x, k, metric)


@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("n,B", [(3000, 3), (40000, 2), (40000, 70)])
def test_knn_ties(gpu_lib, metric, n, B):
    """many equal rows: the lowest row numbers win, in order"""
    codes, scales, sq, x = _table(50, 64, 32, 9)
    pick = np.random.default_rng(2).integers(0, 50, n)
    codes, scales, sq, x = codes[pick], scales[pick], sq[pick], x[pick]
    q = x[np.arange(B) % 50].astype(np.float32)
    t = _gpu_table(codes, scales, sq, 64)
    ids, dist = _check_knn(t, q, x, 20, metric)
    for b in range(B):
        first = np.flatnonzero(R.distances(metric, q[b:b + 1], x)[0] <= dist[b, 0] + 1e-9)
        want = first[:20]
        assert np.array_equal(ids[b, :want.size], want)


@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("n", [500, 30000])
def test_knn_hard_rows(gpu_lib, metric, n):
    """rows of zeros (their cosine is no number: last), rows that are not finite, norms over many orders of magnitude"""
    from cozo_amd.quantized import quantize
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((n, 80)) * np.exp(rng.uniform(-30, 20, (n, 1)))).astype(np.float32)
    x[::7] = 0
    x[3, 2] = np.inf
    x[11, 79] = np.nan
    t = quantize(_cuda(x), group=32)
    back = t.dequantize().cpu().numpy().astype(np.float64)
    q = np.concatenate([rng.standard_normal((3, 80)), x[[1, 8]], np.zeros((1, 80))]).astype(np.float32)
    for k in (1, 12, 400):
        _check_knn(t, q, back, k, metric)
    q[0, 0], q[1, 3] = np.nan, np.inf
    ids, dist, cnt = t.knn(_cuda(q), 4, distance=metric)
    assert int(cnt[0]) == 4 and bool(dist[0].isnan().all()) and ids[0].tolist() == [0, 1, 2, 3]
    _check_knn(t, q[2:], back, 4, metric)


@pytest.mark.gpu
def test_knn_all_rows_zero_or_gone(gpu_lib):
    codes = np.zeros((5000, 32), np.uint8)
    scales, sq = np.zeros((5000, 2), np.uint16), np.zeros(5000, np.float32)
    q = np.ones((2, 64), np.float32)
    t = _gpu_table(codes, scales, sq, 64)
    ids, dist, cnt = t.knn(_cuda(q), 6, distance="Cosine")
    assert ids.tolist() == [list(range(6))] * 2 and bool(dist.isnan().all()) and cnt.tolist() == [6, 6]
    ids, dist, cnt = t.knn(_cuda(q), 6, distance="L2")
    assert ids.tolist() == [list(range(6))] * 2 and bool((dist == 64).all())
    empty = _gpu_table(codes[:0], scales[:0], sq[:0], 64)
    ids, dist, cnt = empty.knn(_cuda(q), 3)
    assert bool((ids == -1).all()) and bool(dist.isinf().all()) and cnt.tolist() == [0, 0]
    assert empty.dots(_cuda(q)).shape == (2, 0) and empty.dequantize().shape == (0, 64)
    assert t.knn(_cuda(q[:0]), 3)[0].shape == (0, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("n", [900, 50000])
def test_knn_radius_and_host(gpu_lib, metric, n):
    codes, scales, sq, x = _table(n, 72, 32, 4)
    q = np.random.default_rng(8).standard_normal((6, 72)).astype(np.float32)
    t = _gpu_table(codes, scales, sq, 72)
    d = R.distances(metric, q, x)
    radius = float(np.sort(d, 1)[:, 5].mean())
    ids, dist = _check_knn(t, q, x, 12, metric, radius=radius)
    hids, hdist, hcnt = _q4(codes, scales, sq, 72).knn(q, 12, distance=metric, radius=radius)
    assert np.array_equal(hids, ids) and np.array_equal(hdist, dist)
    none, _, cnt = t.knn(_cuda(q), 12, distance=metric, radius=-1e30)
    assert bool((none == -1).all()) and int(cnt.sum()) == 0


@pytest.mark.gpu
def test_knn_many_queries(gpu_lib):
    """more queries than one launch takes"""
    codes, scales, sq, x = _table(300, 40, 32, 6)
    q = np.random.default_rng(0).standard_normal((4101, 40)).astype(np.float32)
    _check_knn(_gpu_table(codes, scales, sq, 40), q, x, 3, "L2")


@pytest.mark.gpu
def test_streams_graphs_and_scratch(gpu_lib):
    import torch
    from cozo_amd import _lib
    codes, scales, sq, x = _table(40000, 96, 32, 3)
    t = _gpu_table(codes, scales, sq, 96)
    q = torch.randn(9, 96, device="cuda")
    want_d, want = t.dots(q), t.knn(q, 5, distance="Cosine")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got_d, got = t.dots(q), t.knn(q, 5, distance="Cosine")
    by_handle = t.knn(q, 5, distance="Cosine", stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got_d, want_d) and all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(by_handle, want))
    # captured once, replayed on new queries, with eager work in between
    static = q.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cap_d, cap = t.dots(static), t.knn(static, 5, distance="Cosine")
    for seed in range(4):
        new = torch.randn(9, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        static.copy_(new)
        g.replay()
        eager_d, eager = t.dots(new), t.knn(new, 5, distance="Cosine")
        torch.cuda.synchronize()
        assert torch.equal(cap_d, eager_d) and all(torch.equal(a, b) for a, b in zip(cap, eager))
    # the C entry: scratch that is too small, unaligned or on the host is refused; without scratch the call waits
    L, P = _lib.lib(), _lib.ptr
    out = torch.full((9, 40000), 7.0, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    need = L.cz_q4_workspace(40000, 96, 32, 9, 0)
    call = lambda w, b, c=t.codes: L.cz_q4_dots((c if isinstance(c, int) else P(c)), P(t.scales), 40000, 96, 32, P(q), 9, P(out), w, b, 1, None)  # noqa: E731
    assert call(P(ws), need - 1) == _lib.CZ_E_INVALID
    assert call(ws.data_ptr() + 8, 1 << 19) == _lib.CZ_E_INVALID
    assert call(P(ws), need, t.codes.data_ptr() + 4) == _lib.CZ_E_INVALID
    assert call(P(ws), need, codes) == _lib.CZ_E_INVALID  # a host table with CZ_DEVICE_PTRS
    torch.cuda.synchronize()
    assert bool((out == 7).all())
    assert call(None, 0) == _lib.CZ_OK
    torch.cuda.synchronize()
    assert torch.equal(out, want_d)


@pytest.mark.gpu
def test_knn_cancelled(gpu_lib):
    from cozo_amd import _lib
    codes, scales, sq, _ = _table(100, 64, 32, 3)
    with pytest.raises(_lib.ProcessKilled):
        _q4(codes, scales, sq, 64).knn(np.ones((1, 64), np.float32), 3, poison=np.ones(1, np.uint8))


@pytest.mark.gpu
def test_mixed_places_are_refused(gpu_lib):
    codes, scales, sq, _ = _table(10, 64, 32, 3)
    t = _gpu_table(codes, scales, sq, 64)
    with pytest.raises(ValueError):
        t.dots(np.ones((1, 64), np.float32))
    with pytest.raises(ValueError):
        _q4(codes, t.scales, sq, 64)
    with pytest.raises(ValueError):
        t.dots(_cuda(np.ones((1, 64))))
