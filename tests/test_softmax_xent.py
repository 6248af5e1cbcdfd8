"""Softmax cross entropy over a whole table and its gradient, against plain implementations in 64 bits."""
import numpy as np
import pytest

from tests import table_ref as R

U32, UBF16 = 2.0 ** -24, 2.0 ** -8  # half a step, relative


def _case(T, V, dim, dtype, seed, ignored=True):
    """(queries, table) as arrays the call takes and as f64 values, targets, grad_loss"""
    rng = np.random.default_rng(seed)
    q = (rng.standard_normal((T, dim)) / np.sqrt(dim)).astype(np.float32)
    w = (rng.standard_normal((V, dim))).astype(np.float32)
    y = rng.integers(0, V, T)
    if ignored:
        y[1::3] = -1
    g = rng.standard_normal(T).astype(np.float32)
    if dtype == "bf16":
        q, w = R.bf16_bits(q), R.bf16_bits(w)
        return q, w, R.bf16_value(q).astype(np.float64), R.bf16_value(w).astype(np.float64), y, g
    return q, w, q.astype(np.float64), w.astype(np.float64), y, g


def _cuda(a):
    import torch
    if a.dtype == np.uint16:
        return torch.from_numpy(a.view(np.int16)).cuda().view(torch.bfloat16)
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _host(t):
    import torch
    return t.float().cpu().numpy().astype(np.float64) if t.dtype in (torch.bfloat16, torch.float32) else t.cpu().numpy()


def _z_err(q, w, scale):
    """how far an f32 logit may be off: sums of dim products, the factor and the exponent's argument (in units of log2 e) rounded"""
    a = scale * (np.abs(q) @ np.abs(w).T)
    return ((q.shape[1] + 8) * U32 * a).max(1) if a.size else np.zeros(q.shape[0])


def _lse_tol(q, w, scale):
    """the largest logit error; sums of positive terms in f32, 16 or more lanes to a sum; two ulp of exp2"""
    return _z_err(q, w, scale) + (w.shape[0] / 16 + 64) * U32 + 2.0 ** -21


def _check(q, w, q64, w64, y, g, scale, dtype, got):
    loss, lse, dq, dw = got
    wloss, wlse, z = R.softmax_xent(q64, w64, y, scale)
    tol = _lse_tol(q64, w64, scale)
    assert np.all(np.abs(lse - wlse) <= tol + U32 * np.abs(wlse))
    # the answer's own logit is summed in f64
    assert np.all(np.abs(loss - wloss) <= (tol + U32 * np.abs(wlse) + U32 * np.abs(wloss)) * (y >= 0))
    wdq, wdw, G = R.softmax_xent_grad(q64, w64, y, scale, g)
    p = np.exp(z - wlse[:, None])
    # of P: the logit's and lse's errors in the exponent; the subtraction of the one; for bf16 the rounding of G itself
    ep = 2 * tol + 4 * U32 * (np.abs(z).max(1) + np.abs(wlse)) + 2.0 ** -21
    live = (np.abs(g) * (y >= 0))[:, None]
    eG = live * (p * ep[:, None] + 2 * U32) + (2 * U32 + (UBF16 if dtype == "bf16" else 0)) * np.abs(G)
    out = UBF16 if dtype == "bf16" else U32
    V, T = w64.shape[0], q64.shape[0]
    tq = scale * (eG @ np.abs(w64)) + (V + 64) * U32 * scale * (np.abs(G) @ np.abs(w64)) + out * np.abs(wdq)
    tw = scale * (eG.T @ np.abs(q64)) + (T + 64) * U32 * scale * (np.abs(G).T @ np.abs(q64)) + out * np.abs(wdw)
    if dq is not None:
        assert np.all(np.abs(dq - wdq) <= tq * 1.01 + 1e-37)
        assert not dq[y < 0].any()
    if dw is not None:
        assert np.all(np.abs(dw - wdw) <= tw * 1.01 + 1e-37)


def _run(q, w, y, g, scale, **kw):
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    loss, lse = softmax_xent(q, w, y, scale=scale, **kw)
    return (loss, lse) + softmax_xent_grad(q, w, y, lse, g, scale=scale, **kw)


# ---- on the CPU ----------------------------------------------------------------------------------------------------
def test_reference_gradient_against_differences():
    q, w, q64, w64, y, g = _case(5, 11, 7, "f32", 0)
    dq, dw, _ = R.softmax_xent_grad(q64, w64, y, 1.7, g)
    f = lambda a, b: float(g.astype(np.float64) @ R.softmax_xent(a, b, y, 1.7)[0])  # noqa: E731
    h = 1e-5
    for a, da, at in ((q64, dq, 0), (w64, dw, 1)):
        for i in np.ndindex(a.shape):
            x = a[i]
            a[i] = x + h
            hi = f(q64, w64)
            a[i] = x - h
            lo = f(q64, w64)
            a[i] = x
            assert abs((hi - lo) / (2 * h) - da[i]) < 1e-7  # h^2 of the third derivative, and 2^-52 / h of rounding


def test_refusals():
    from cozo_amd import _lib
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    L = _lib.lib()
    q, w, y = np.zeros((3, 8), np.float32), np.zeros((5, 8), np.float32), np.zeros(3, np.int64)
    for a in ((q[:, :7], w, y), (q, w.astype(np.float64), y), (q, R.bf16_bits(w), y), (q[0], w, y), (q, w, y[:2]), (q, w, y.astype(float)),
              (q, w, y - 2)):
        with pytest.raises(ValueError):
            softmax_xent(*a)
    with pytest.raises(ValueError):
        softmax_xent_grad(q, w, y, np.zeros(2, np.float32), np.zeros(3, np.float32))
    p = _lib.ptr(np.zeros(64, np.uint8))
    call = lambda elem, T, V, dim, ld: L.cz_softmax_xent(p, ld, p, ld, elem, T, V, dim, p, 1.0, p, p, None, 0, 0, None)  # noqa: E731
    assert call(2, 1, 1, 4, 4) == _lib.CZ_E_INVALID
    assert call(0, 1, 0, 4, 4) == _lib.CZ_E_INVALID
    assert call(0, 1, 1, 0, 4) == _lib.CZ_E_UNSUPPORTED and call(0, 1, 1, 8193, 8193) == _lib.CZ_E_UNSUPPORTED
    assert call(0, 1, 1, 4, 3) == _lib.CZ_E_INVALID
    assert call(0, 1 << 24, 1, 4, 4) == _lib.CZ_E_UNSUPPORTED
    assert L.cz_softmax_xent_workspace(1, 0, 4, 0, 0) == 0 and L.cz_softmax_xent_workspace(1, 1, 4, 0, 1) > 0


def test_no_device_no_answer():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    from cozo_amd import _lib
    from cozo_amd.softmax import softmax_xent
    with pytest.raises(_lib.CozoGpuError) as e:
        softmax_xent(np.zeros((3, 8), np.float32), np.zeros((5, 8), np.float32), np.zeros(3, np.int64))
    assert e.value.code == _lib.CZ_E_NO_DEVICE


# ---- on the GPU ----------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("T,V,dim", [(1, 1, 1), (1, 2, 7), (3, 127, 64), (2, 129, 32), (16, 1000, 128), (64, 5003, 96), (130, 300, 130),
                                     (255, 257, 64), (257, 3001, 40), (5, 700, 768), (4, 90, 1999), (2, 33, 8192), (300, 2000, 256)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_loss_and_gradient(gpu_lib, T, V, dim, dtype):
    q, w, q64, w64, y, g = _case(T, V, dim, dtype, T + V)
    got = _run(_cuda(q), _cuda(w), _cuda(y), _cuda(g), 3.0)
    _check(q, w, q64, w64, y, g, 3.0, dtype, [_host(a) for a in got])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_several_pieces(gpu_lib, dtype):
    """a table that is worked on in more than one piece (the scratch bounds a piece by the wide of queries and rows)"""
    T, V, dim = 700, 150_000, 24
    q, w, q64, w64, y, g = _case(T, V, dim, dtype, 5)
    got = _run(_cuda(q), _cuda(w), _cuda(y), _cuda(g), 2.0)
    _check(q, w, q64, w64, y, g, 2.0, dtype, [_host(a) for a in got])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_types_and_host(gpu_lib, dtype):
    import torch
    q, w, q64, w64, y, g = _case(37, 211, 72, dtype, 1)
    tq, tw = _cuda(q), _cuda(w)
    want = _run(tq, tw, _cuda(y), _cuda(g), 1.5)
    wide_q = torch.cat([tq, torch.full_like(tq, float("nan"))], 1)[:, :72]
    wide_w = torch.cat([torch.full_like(tw[:, :3], float("nan")), tw, tw[:, :2]], 1)[:, 3:75]
    got = _run(wide_q, wide_w, _cuda(y.astype(np.int32)), _cuda(g), 1.5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = _run(tq.t().contiguous().t(), tw, _cuda(y), _cuda(np.stack([g, g], 1))[:, 0], 1.5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    host = _run(q, w, y, g, 1.5)
    for a, b in zip(host, want):
        b = b.view(torch.int16).cpu().numpy().view(np.uint16) if b.dtype == torch.bfloat16 else b.cpu().numpy()
        assert np.array_equal(a, b)
    from cozo_amd.softmax import softmax_xent_grad
    only_q = softmax_xent_grad(tq, tw, _cuda(y), want[1], _cuda(g), scale=1.5, want_table=False)
    only_w = softmax_xent_grad(tq, tw, _cuda(y), want[1], _cuda(g), scale=1.5, want_queries=False)
    assert only_q[1] is None and torch.equal(only_q[0], want[2]) and only_w[0] is None and torch.equal(only_w[1], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_without_an_answer(gpu_lib, dtype):
    import torch
    q, w, q64, w64, y, g = _case(40, 333, 64, dtype, 2, ignored=False)
    y[5] = y[20] = -1
    clean = _run(_cuda(q), _cuda(w), _cuda(y), _cuda(g), 1.0)
    tq = _cuda(q)
    tq[5], tq[20] = float("nan"), float("inf")
    tg = _cuda(g)
    tg[5] = float("nan")
    loss, lse, dq, dw = _run(tq, _cuda(w), _cuda(y), tg, 1.0)
    assert torch.equal(loss, clean[0]) and torch.equal(dq, clean[2]) and torch.equal(dw, clean[3])
    assert not bool(loss[[5, 20]].any()) and not bool(dq[[5, 20]].any())
    # a target that is no row: no loss that could be mistaken for one, no gradient
    bad = _cuda(y)
    bad[7] = 333
    loss, _, dq, dw = _run(_cuda(q), _cuda(w), bad, _cuda(g), 1.0)
    gone = y.copy()
    gone[7] = -1
    ref = _run(_cuda(q), _cuda(w), _cuda(gone), _cuda(g), 1.0)
    assert bool(loss[7].isnan()) and torch.equal(dq, ref[2]) and torch.equal(dw, ref[3])
    none = _run(_cuda(q), _cuda(w), _cuda(np.full(40, -1)), _cuda(g), 1.0)
    assert not bool(none[0].any()) and not bool(none[2].any()) and not bool(none[3].any())
    # no queries at all: the table's gradient is zeros
    none = _run(_cuda(q[:0]), _cuda(w), _cuda(y[:0]), _cuda(g[:0]), 1.0)
    assert none[0].shape == (0,) and none[2].shape == (0, 64) and none[3].shape == w.shape and not bool(none[3].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_extreme_logits(gpu_lib, dtype):
    """logits thousands apart: the largest decides, nothing overflows; rows at minus infinity weigh nothing"""
    import torch
    q, w, q64, w64, y, g = _case(20, 500, 64, dtype, 3, ignored=False)
    got = _run(_cuda(q), _cuda(w), _cuda(y), _cuda(g), 4000.0)
    assert all(bool(torch.isfinite(a).all()) for a in got)
    wloss, wlse, _ = R.softmax_xent(q64, w64, y, 4000.0)
    tol = _lse_tol(q64, w64, 4000.0)
    assert np.all(np.abs(_host(got[1]) - wlse) <= tol + U32 * np.abs(wlse))
    # one row of -inf products: as if it were not there
    tq, tw = _cuda(q).abs() + 0.5, _cuda(w)
    without = _run(tq, torch.cat([tw[:77], tw[78:]]), torch.zeros(20, dtype=torch.int64, device="cuda"), _cuda(g), 1.0)
    tw[77] = -float("inf")
    loss, lse = _run(tq, tw, torch.zeros(20, dtype=torch.int64, device="cuda"), _cuda(g), 1.0)[:2]
    # (another place in the sum's order)
    assert torch.allclose(lse, without[1], rtol=0, atol=float(_lse_tol(_host(tq), _host(tw[:77]), 1.0).max()))
    assert bool(torch.isfinite(loss).all())
    tw[78] = float("inf")
    assert bool((_run(tq, tw, torch.zeros(20, dtype=torch.int64, device="cuda"), _cuda(g), 1.0)[1] == float("inf")).all())
    tw[78] = float("nan")
    assert bool(_run(tq, tw, torch.zeros(20, dtype=torch.int64, device="cuda"), _cuda(g), 1.0)[1].isnan().all())
    only = torch.full((3, 64), -float("inf"), device="cuda").to(tq.dtype)
    assert bool((_run(tq, only, torch.zeros(20, dtype=torch.int64, device="cuda"), _cuda(g), 1.0)[1] == -float("inf")).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradient_against_differences(gpu_lib, dtype):
    """the loss the kernel gives, moved along the gradient the kernel gives: a central difference over a step whose cubic term and
    rounding are both below the bound.  bf16 inputs cannot be moved by small steps: the f64 loss is moved instead."""
    q, w, q64, w64, y, g = _case(12, 400, 48, dtype, 6)
    _, _, dq, dw = (_host(a) for a in _run(_cuda(q), _cuda(w), _cuda(y), _cuda(g), 2.0))
    rng = np.random.default_rng(1)
    for _ in range(3):
        aq, aw = rng.standard_normal(q64.shape), rng.standard_normal(w64.shape)
        h = 1e-4
        f = lambda s: float(g.astype(np.float64) @ R.softmax_xent(q64 + s * aq, w64 + s * aw, y, 2.0)[0])  # noqa: E731
        slope, own = (f(h) - f(-h)) / (2 * h), float((dq * aq).sum() + (dw * aw).sum())
        size = float((np.abs(dq) * np.abs(aq)).sum() + (np.abs(dw) * np.abs(aw)).sum())
        assert abs(slope - own) <= (3 * UBF16 if dtype == "bf16" else 1e-4) * size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_streams_and_graphs(gpu_lib, dtype):
    import torch
    from cozo_amd import _lib
    q, w, q64, w64, y, g = _case(70, 3000, 64, dtype, 8)
    tq, tw, ty, tg = _cuda(q), _cuda(w), _cuda(y), _cuda(g)
    want = _run(tq, tw, ty, tg, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(_run(tq, tw, ty, tg, 1.0), want))  # the same bits every time
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(tq, tw, ty, tg, 1.0)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sq = tq.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = _run(sq, tw, ty, tg, 1.0)
    for seed in range(4):
        new = torch.randn(70, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(tq.dtype)
        sq.copy_(new)
        graph.replay()
        eager = _run(new, tw, ty, tg, 1.0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cap, eager))
    L, P = _lib.lib(), _lib.ptr
    elem = 1 if dtype == "bf16" else 0
    need = L.cz_softmax_xent_workspace(70, 3000, 64, elem, 0)
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    loss, lse = torch.full((70,), 7.0, device="cuda"), torch.full((70,), 7.0, device="cuda")
    y32 = ty.to(torch.int32)
    call = lambda w_, n: L.cz_softmax_xent(P(tq), 64, P(tw), 64, elem, 70, 3000, 64, P(y32), 1.0, P(loss), P(lse), w_, n, 1, None)  # noqa: E731
    assert call(P(ws), need - 1) == _lib.CZ_E_INVALID and call(ws.data_ptr() + 8, need) == _lib.CZ_E_INVALID
    torch.cuda.synchronize()
    assert bool((loss == 7).all())
    assert call(P(ws), need) == _lib.CZ_OK
    torch.cuda.synchronize()
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
def test_trained_then_quantised_then_searched(gpu_lib):
    """the operators as they are used together: gradient steps on a table, its 4-bit form, the search over that form"""
    import torch
    from cozo_amd.quantized import quantize
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    gen = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(4000, 96, device="cuda", generator=gen)
    q = torch.randn(50, 96, device="cuda", generator=gen)
    y = torch.randint(0, 4000, (50,), device="cuda", generator=gen)
    g = torch.full((50,), 0.02, device="cuda")
    for _ in range(3):
        loss, lse = softmax_xent(q, w, y, scale=0.3)
        dq, dw = softmax_xent_grad(q, w, y, lse, g, scale=0.3)
        wdq, wdw, _ = R.softmax_xent_grad(_host(q), _host(w), y.cpu().numpy(), 0.3, _host(g))
        assert np.linalg.norm(_host(dq) - wdq) <= 1e-4 * np.linalg.norm(wdq) and np.linalg.norm(_host(dw) - wdw) <= 1e-4 * np.linalg.norm(wdw)
        w -= 5.0 * dw
        q -= 5.0 * dq
    t = quantize(w, group=32)
    rows = t.dequantize().cpu().numpy().astype(np.float64)
    ids, dist, cnt = t.knn(q, 8, distance="IP")
    want_ids, want, _ = R.nearest(R.distances("IP", q.cpu().numpy(), rows), 8)
    assert np.array_equal(ids.cpu().numpy().view(np.uint32), want_ids)
    assert np.allclose(dist.cpu().numpy(), want, rtol=1e-12, atol=1e-12)
    d = t.dots(q).cpu().numpy()
    best = np.take_along_axis(d, want_ids.astype(np.int64), 1)
    assert np.allclose(1 - best, want, rtol=0, atol=1e-4)
