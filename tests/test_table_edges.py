"""The operators over whole tables at their edges: what the documentation allows and ordinary use does not reach."""
import threading

import numpy as np
import pytest

from tests import table_ref as R
from tests.test_quantized import METRICS, _check_knn, _cuda, _dots_tol, _gpu_table, _q4, _table


def _bf16(a):
    import torch
    return a.to(torch.bfloat16)


def test_host_row_numbers_are_refused():
    codes, scales, sq, _ = _table(10, 40, 32, 0)
    t = _q4(codes, scales, sq, 40)
    for bad in ([10], [-1], [2**32 + 3], [0.5]):
        with pytest.raises(ValueError):
            t.dequantize(np.asarray(bad))


@pytest.mark.gpu
def test_row_numbers_beyond_32_bits(gpu_lib):
    import torch
    codes, scales, sq, _ = _table(10, 40, 32, 0)
    t = _gpu_table(codes, scales, sq, 40)
    got = t.dequantize(torch.tensor([2**32 + 3, -2**32 + 3, 3, 10], device="cuda"))
    assert bool(got[[0, 1, 3]].isnan().all()) and torch.equal(got[2], t.dequantize()[3])
    with pytest.raises(ValueError):
        t.dequantize(torch.tensor([1.0], device="cuda"))


@pytest.mark.gpu
def test_more_queries_than_a_turn(gpu_lib):
    codes, scales, sq, x = _table(70, 33, 32, 1)
    q = np.random.default_rng(0).standard_normal((4099, 33)).astype(np.float32)
    got = _gpu_table(codes, scales, sq, 33).dots(_cuda(q)).cpu().numpy()
    assert np.all(np.abs(got - q.astype(np.float64) @ x.T) <= _dots_tol(q, x))


@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("B", [40, 140, 300])
def test_many_queries_over_hard_rows(gpu_lib, metric, B):
    """scores in f16 (a large batch) over rows of zeros, rows that are not finite, norms over many orders of magnitude, queries alike"""
    from cozo_amd.quantized import quantize
    rng = np.random.default_rng(B)
    n = 33000
    x = (rng.standard_normal((n, 72)) * np.exp(rng.uniform(-30, 20, (n, 1)))).astype(np.float32)
    x[::9] = 0
    x[5, 2], x[17, 71] = np.inf, np.nan
    t = quantize(_cuda(x), group=32)
    back = t.dequantize().cpu().numpy().astype(np.float64)
    q = (rng.standard_normal((B, 72)) * np.exp(rng.uniform(-30, 30, (B, 1)))).astype(np.float32)
    q[1] = x[40]
    q[2] = 0
    q[3] = 1e-42
    look = np.concatenate([np.arange(12), rng.integers(12, B, 18)])
    for k in (1, 10, 100):
        _check_knn(t, q, back, k, metric, only=look)
    q[4, 7], q[6, 0] = np.nan, np.inf
    ids, dist, _ = t.knn(_cuda(q), 3, distance=metric)
    assert bool(dist[[4]].isnan().all()) and ids[4].tolist() == [0, 1, 2]
    _check_knn(t, q, back, 3, metric, only=np.setdiff1d(look, [4, 6]))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,group", [(31, 32), (95, 32), (160, 64), (200, 128), (1000, 128)])
@pytest.mark.parametrize("B", [1, 50, 129, 257])
def test_scores_at_odd_sizes(gpu_lib, dim, group, B):
    codes, scales, sq, x = _table(32900, dim, group, dim + B)
    rng = np.random.default_rng(B)
    q = rng.standard_normal((B, dim)).astype(np.float32)
    pick = rng.integers(0, B, min(B, 6))
    t = _gpu_table(codes, scales, sq, dim)
    for metric in METRICS:
        all_ids, all_dist, _ = t.knn(_cuda(q), 11, distance=metric)
        ids, dist = _check_knn(t, q[pick], x, 11, metric)  # (a few queries, by another path than the batch)
        assert np.array_equal(all_ids.cpu().numpy()[pick].view(np.uint32), ids)
        assert np.array_equal(all_dist.cpu().numpy()[pick], dist)


@pytest.mark.gpu
def test_large_launches_are_captured(gpu_lib):
    """the forms for large batches inside a graph, replayed with eager work in between"""
    import torch
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    codes, scales, sq, _ = _table(40000, 128, 64, 2)
    t = _gpu_table(codes, scales, sq, 128)
    w = _bf16(torch.randn(40000, 128, device="cuda"))
    q = torch.randn(300, 128, device="cuda")
    y = torch.randint(0, 40000, (300,), device="cuda")
    g = torch.rand(300, device="cuda")

    def all_of(q):
        knn = t.knn(q, 9, distance="L2")
        loss, lse = softmax_xent(_bf16(q), w, y, scale=0.2)
        return (*knn, loss, lse, *softmax_xent_grad(_bf16(q), w, y, lse, g, scale=0.2))
    static = q.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = all_of(static)
    for seed in range(4):
        new = torch.randn(300, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        static.copy_(new)
        graph.replay()
        eager = all_of(new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(cap, eager))


@pytest.mark.gpu
def test_two_threads_at_once(gpu_lib):
    import torch
    from cozo_amd.softmax import softmax_xent
    codes, scales, sq, _ = _table(40000, 96, 32, 3)
    t = _gpu_table(codes, scales, sq, 96)
    qs = [torch.randn(40, 96, device="cuda") for _ in range(2)]
    w = torch.randn(5000, 96, device="cuda")
    y = torch.arange(40, device="cuda")
    want = [(t.knn(q, 5), softmax_xent(q, w, y), _q4(codes, scales, sq, 96).dots(q.cpu().numpy())) for q in qs]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = (t.knn(qs[i], 5), softmax_xent(qs[i], w, y), _q4(codes, scales, sq, 96).dots(qs[i].cpu().numpy()))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    for a, b in zip(got, want):
        assert all(torch.equal(x, z) for x, z in zip(a[0], b[0])) and all(torch.equal(x, z) for x, z in zip(a[1], b[1]))
        assert np.array_equal(a[2], b[2])


@pytest.mark.gpu
def test_nothing_is_written_behind_an_output(gpu_lib):
    import torch
    from cozo_amd import _lib
    L, P = _lib.lib(), _lib.ptr
    C = _lib.C

    def guarded(count, dtype):
        return torch.full((count + 4096,), 77, dtype=dtype, device="cuda")

    def ws(n):
        assert n > 0
        return torch.empty(n, dtype=torch.uint8, device="cuda")
    held = []
    for n, dim, group, B, k in ((1, 1, 32, 1, 1), (65, 33, 32, 3, 7), (130, 200, 128, 5, 200), (33001, 48, 64, 40, 3), (33001, 40, 32, 9, 5)):
        x = torch.randn(n, dim, device="cuda")
        groups = -(-dim // group)
        codes, scales, sq = guarded(n * groups * group // 2, torch.uint8), guarded(n * groups, torch.int16), guarded(n, torch.float32)
        assert L.cz_q4_quantize(P(x), 0, n, dim, dim, group, P(codes), P(scales), P(sq), 1, None) == 0
        rows = guarded(n * dim, torch.float32)
        assert L.cz_q4_dequantize(P(codes), P(scales), n, dim, group, None, n, P(rows), 1, None) == 0
        q = torch.randn(B, dim, device="cuda")
        out = guarded(B * n, torch.float32)
        need = L.cz_q4_workspace(n, dim, group, B, 0)
        w = guarded(need, torch.uint8)
        assert L.cz_q4_dots(P(codes), P(scales), n, dim, group, P(q), B, P(out), P(w), need, 1, None) == 0
        ids, dist, cnt = guarded(B * k, torch.int32), guarded(B * k, torch.float64), guarded(B, torch.int32)
        need2 = L.cz_q4_workspace(n, dim, group, B, k)
        w2 = guarded(need2, torch.uint8)
        assert L.cz_q4_knn(1, P(codes), P(scales), P(sq), n, dim, group, P(q), B, k, 0, 0.0, P(ids), P(dist), P(cnt), P(w2), need2, None, 1,
                           None) == 0
        held += [(codes, n * groups * group // 2), (scales, n * groups), (sq, n), (rows, n * dim), (out, B * n), (w, need), (ids, B * k),
                 (dist, B * k), (cnt, B), (w2, need2)]
        # (a plain loop over the few sizes keeps one process and one set of kernels)
    for T, V, dim, elem in ((1, 1, 1, 0), (3, 65, 33, 0), (130, 300, 40, 1), (257, 2049, 64, 1), (40, 1000, 96, 0)):
        dt, es = (torch.bfloat16, 2) if elem else (torch.float32, 4)
        q, tab = torch.randn(T, dim, device="cuda").to(dt), torch.randn(V, dim, device="cuda").to(dt)
        y = torch.randint(0, V, (T,), device="cuda", dtype=torch.int32)
        loss, lse = guarded(T, torch.float32), guarded(T, torch.float32)
        need = L.cz_softmax_xent_workspace(T, V, dim, elem, 0)
        w = guarded(need, torch.uint8)
        one = C.c_float(1.0)
        assert L.cz_softmax_xent(P(q), dim, P(tab), dim, elem, T, V, dim, P(y), one, P(loss), P(lse), P(w), need, 1, None) == 0
        dq, dw = guarded(T * dim, dt), guarded(V * dim, dt)
        need2 = L.cz_softmax_xent_workspace(T, V, dim, elem, 1)
        w2 = guarded(need2, torch.uint8)
        assert L.cz_softmax_xent_grad(P(q), dim, P(tab), dim, elem, T, V, dim, P(y), one, P(lse), P(loss), P(dq), P(dw), P(w2), need2, 1, None) == 0
        held += [(loss, T), (lse, T), (w, need), (dq, T * dim), (dw, V * dim), (w2, need2)]
    torch.cuda.synchronize()
    for i, (buf, used) in enumerate(held):
        assert bool((buf[used:] == 77).all()), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -2.0])
def test_scales_of_any_sign(gpu_lib, dtype, scale):
    from tests.test_softmax_xent import _case, _check, _cuda as cuda, _host, _run
    q, w, q64, w64, y, g = _case(33, 700, 40, dtype, 4)
    got = [_host(a) for a in _run(cuda(q), cuda(w), cuda(y), cuda(g), scale)]
    # the bounds are in the logits' size: for a negative scale those of the table turned round
    _check(q, w, q64, np.sign(scale) * w64, y, g, abs(scale), dtype, got[:2] + [None, None])
    wdq, wdw, _ = R.softmax_xent_grad(q64, w64, y, scale, g)
    for a, b in zip(got[2:], (wdq, wdw)):
        assert np.linalg.norm(a - b) <= (2.0 ** -7 if dtype == "bf16" else 1e-5) * np.linalg.norm(b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_queries_than_rows_and_one_row_for_all(gpu_lib, dtype):
    """many queries answered by the same few rows: their terms meet in one row of the table's gradient, in one order"""
    import torch
    from tests.test_softmax_xent import _case, _check, _cuda as cuda, _host, _run
    q, w, q64, w64, y, g = _case(5000, 40, 24, dtype, 9, ignored=False)
    y[:] = np.where(np.arange(5000) % 3, 7, y)
    args = (cuda(q), cuda(w), cuda(y), cuda(g), 1.0)
    got = _run(*args)
    _check(q, w, q64, w64, y, g, 1.0, dtype, [_host(a) for a in got])
    assert all(torch.equal(a, b) for a, b in zip(got, _run(*args)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sure_answers(gpu_lib, dtype):
    """an answer that is all but certain: what is left of its gradient is the small difference, not the rounding of the large terms"""
    import torch
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    w = torch.eye(64, device="cuda").to(_bf16(torch.ones(1)).dtype if dtype == "bf16" else torch.float32)
    q = (w[:40].float() * 20).to(w.dtype)
    y = torch.arange(40, device="cuda")
    g = torch.full((40,), 0.37, device="cuda")
    loss, lse = softmax_xent(q, w, y)
    dq, dw = softmax_xent_grad(q, w, y, lse, g)
    wl, _, _ = R.softmax_xent(q.double().cpu().numpy(), w.double().cpu().numpy(), y.cpu().numpy(), 1.0)
    wdq, wdw, _ = R.softmax_xent_grad(q.double().cpu().numpy(), w.double().cpu().numpy(), y.cpu().numpy(), 1.0, g.double().cpu().numpy())
    # lse = 20 + 1.3e-7 is an f32: half a step of it is 2^-20, and so is what p - 1 may be off by
    assert np.all(np.abs(loss.cpu().numpy() - wl) <= 2.0 ** -19)
    assert np.abs(dq.double().cpu().numpy() - wdq).max() <= 0.37 * 2.0 ** -18 and np.abs(dw.double().cpu().numpy() - wdw).max() <= 20 * 0.37 * 2.0 ** -18


@pytest.mark.gpu
def test_tables_beyond_four_gigabytes(gpu_lib):
    """offsets that pass 32 bits: codes, products, the loss and its gradient"""
    import torch
    from cozo_amd.quantized import Q4Table
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    n, dim = 8_400_011, 1024
    gen = torch.Generator(device="cuda").manual_seed(3)
    codes = torch.randint(0, 256, (n, dim // 2), dtype=torch.uint8, device="cuda", generator=gen)  # 4.3e9 bytes
    scales = torch.rand(n, 8, device="cuda", generator=gen).to(torch.bfloat16)
    at = torch.tensor([0, 1, 4_194_303, 4_194_304, n - 65, n - 2, n - 1], device="cuda")
    part = Q4Table(codes[at].contiguous(), scales[at].contiguous(), None, dim).dequantize().double()
    # the norms from the codes' squares, by pieces
    sq = torch.empty(n, device="cuda")
    square = torch.tensor([(c - 16 if c > 7 else c) ** 2 for c in range(16)], dtype=torch.float32, device="cuda")
    for i in range(0, n, 400_000):
        c = codes[i:i + 400_000].long()
        s2 = (square[c & 15] + square[c >> 4]).view(c.shape[0], 8, 64).sum(2)
        sq[i:i + 400_000] = (s2 * scales[i:i + 400_000].float().square()).sum(1)
        del c, s2
    t = Q4Table(codes, scales, sq, dim)
    assert torch.equal(t.dequantize(at).double(), part)
    q = torch.randn(2, dim, device="cuda", generator=gen)
    q[1] = part[-1].float() * 2
    d = t.dots(q)
    assert bool(((d[:, at].double() - q.double() @ part.T).abs() <= 2e-4 * part.norm(dim=1)).all())
    ids, dist, _ = t.knn(q[1:], 3)
    assert int(ids[0, 0]) == n - 1 and abs(float(dist[0, 0])) <= 1e-12
    del t, codes, scales, sq, d
    V = 1_100_003
    w = torch.randn(V, dim, device="cuda", generator=gen) * 0.05  # 4.5e9 bytes
    q = torch.randn(3, dim, device="cuda", generator=gen)
    y = torch.tensor([V - 1, 5, 1_048_576], device="cuda")
    loss, lse = softmax_xent(q, w, y)
    g = torch.ones(3, device="cuda")
    dq, dw = softmax_xent_grad(q, w, y, lse, g)
    z = torch.cat([q.double() @ p.double().T for p in w.split(100_000)], 1)
    want = torch.logsumexp(z, 1)
    assert bool(((lse - want).abs() <= 1e-4).all()) and bool(((loss - (want - z.gather(1, y[:, None])[:, 0])).abs() <= 1e-4).all())
    p = torch.exp(z - want[:, None])
    p[torch.arange(3), y] -= 1
    wdq = sum(p[:, i:i + 100_000] @ w[i:i + 100_000].double() for i in range(0, V, 100_000))
    assert float((dq - wdq).norm() / wdq.norm()) <= 1e-4
    for rows in (at[:2], torch.arange(V - 300, V, device="cuda"), torch.tensor([1_048_575, 1_048_576, 1_048_577], device="cuda")):
        assert float((dw[rows] - p[:, rows].T @ q.double()).norm() / (p[:, rows].T @ q.double()).norm()) <= 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [4, 24, 72, 100, 200, 840])
@pytest.mark.parametrize("T", [3, 40, 200])
def test_rows_that_end_inside_a_step(gpu_lib, dtype, dim, T):
    """rows read where they are although they are no whole number of steps: what lies between two rows, or in the next one, is not seen"""
    import torch
    from tests.test_softmax_xent import _case, _check, _cuda as cuda, _host, _run
    V = 333
    q, w, q64, w64, y, g = _case(T, V, dim, dtype, dim + T)
    tw, tq = cuda(w), cuda(q)
    want = _run(tq, tw, cuda(y), cuda(g), 1.5)
    _check(q, w, q64, w64, y, g, 1.5, dtype, [_host(a) for a in want])
    wide = torch.full((V, dim + 24), float("nan"), device="cuda").to(tw.dtype)
    wide[:, :dim] = tw
    got = _run(tq, wide[:, :dim], cuda(y), cuda(g), 1.5)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a row that is not finite is its own affair: the logits of the row before it are not touched (its weight is nothing, as -inf)
    tw2, tq2 = tw.clone(), tq.abs() + 0.5
    y2 = torch.where(cuda(y) == 200, torch.full_like(cuda(y), 7), cuda(y))
    tw2[200] = -float("inf")
    rest = torch.cat([tw[:200], tw[201:]])
    y3 = torch.where(y2 > 200, y2 - 1, y2)
    a, b = _run(tq2, tw2, y2, cuda(g), 1.0)[:2], _run(tq2, rest, y3, cuda(g), 1.0)[:2]
    assert all(bool(((x - z).abs() <= 1e-4 + 1e-6 * z.abs()).all()) for x, z in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logits_without_fractions(gpu_lib, dtype, sign):
    """logits of 1e9 to 1e36, all of one query's alike or nearly so: lse stays as exact as f32 logits are, weights stay within 0 and 1"""
    import torch
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    T, V, dim = 5, 700, 40
    g = torch.Generator().manual_seed(3)
    q = torch.rand(T, dim, generator=g).add_(0.5) * torch.tensor([1e9, 3e10, 1e15, 1e30, 1e34])[:, None]
    w = sign * (1.0 + 1e-3 * torch.rand(V, dim, generator=g))
    w[300:] = w[7]
    q, w = (a.cuda() if dtype == "f32" else _bf16(a).cuda() for a in (q, w))
    y = torch.arange(T, dtype=torch.int32, device="cuda")
    loss, lse = softmax_xent(q, w, y)
    z = q.double().cpu() @ w.double().cpu().T
    # a product's f32 additions (dim of them), to base 2 and back, the sum (at most log V, far below an ulp of such a logit), the result's rounding
    tol = (dim + 4) * 2.0**-24 * (q.double().cpu().abs() @ w.double().cpu().abs().T).amax(1) + np.log(V)
    assert bool(((lse.double().cpu() - torch.logsumexp(z, 1)).abs() <= tol).all())
    assert bool(loss.isfinite().all())
    gl = torch.full((T,), 0.25, device="cuda")
    dq, dw = softmax_xent_grad(q, w, y, lse, gl)
    assert bool(dq.isfinite().all()) and bool(dw.isfinite().all())
    # |G| <= 0.25: a row's gradient is at most that share of all queries, whatever the rounding (of G, of the sum, of the result)
    most = 0.25 * q.double().cpu().abs().sum(0)
    assert bool((dw.double().cpu().abs() <= most * (1 + (2.0**-6 if dtype == "bf16" else 2.0**-20))).all())


@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("B,dim,k", [(500, 512, 50), (30, 4096, 45), (500, 512, 57)])
def test_hardly_more_tiles_than_results(gpu_lib, metric, B, dim, k):
    """58 tiles of 64 rows: scores say which of them can hold one of k results although there are few, or nearly none, to leave out"""
    n = 57 * 64 + 3
    codes, scales, sq, x = _table(n, dim, 64, k)
    q = np.random.default_rng(B).standard_normal((B, dim)).astype(np.float32)
    q[3] = x[n - 1]
    _check_knn(_gpu_table(codes, scales, sq, dim), q, x, k, metric, only=np.arange(0, B, 17 if B > 100 else 1))
