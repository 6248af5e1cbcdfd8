"""The operators over whole tables at the limits of their number ranges and lengths: tables that callers make themselves, products near
the end of the f32 range, tables long enough for a sum to forget, tables worked on in pieces."""
import numpy as np
import pytest

from tests import table_ref as R
from tests.test_quantized import METRICS, U32, _check_knn, _cuda, _gpu_table, _table

UBF16 = 2.0 ** -8  # half a step, relative


# ---- scores of a large batch ---------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("B", [5, 40, 300])
def test_groups_of_zeros_with_large_scales(gpu_lib, metric, B):
    """a group whose codes are all zero may have any scale, and what stands in the padding does not count: such rows, each the nearest one
    and alone in its tile, are found"""
    n, dim, group = 33000, 72, 32
    rng = np.random.default_rng(B)
    c = rng.integers(-7, 8, (n, 96))
    u = rng.integers(1, 8, 32)
    c[c[:, :32] @ u > 0] *= -1  # all others point away
    c[:, dim:] = rng.integers(-8, 8, (n, 96 - dim))  # the padding
    s = np.exp(rng.uniform(-1, 2, (n, 3)))
    at = np.array([70, 6400, 12801, 20031, 32999])
    # 1e-3 in all, beside a group of zeros with a scale up to the largest bfloat16 numbers
    c[at, :] = 0
    c[at, :32] = u
    s[at, 0] = 1e-3 / np.linalg.norm(u) * (1 + 0.05 * np.arange(5))
    s[at, 1] = [1.0, 1e30, 1.0, 3e38, 1.0]
    s[at, 2] = [1.0, 1.0, 1e30, 3e38, 1e6]
    c[at[2:], dim:] = 7
    c[at[3], dim:] = -8
    scales = R.bf16_bits(s.astype(np.float32))
    codes = R.pack(c)
    x = R.decode(codes, R.bf16_value(scales), dim)
    t = _gpu_table(codes, scales, (x ** 2).sum(1).astype(np.float32), dim)
    q = np.zeros((B, dim), np.float32)
    q[:, :32] = u * np.exp(rng.uniform(-1, 1, (B, 1))) * 1e-3 / np.linalg.norm(u)
    look = np.arange(0, B, max(1, B // 8))
    for k in (1, 5, 20):
        ids, _ = _check_knn(t, q, x, k, metric, only=look)
        assert np.isin(ids[:, :min(k, 5)], at).all()


@pytest.mark.gpu
def test_scores_beyond_the_range(gpu_lib):
    """products around -2^128, where the f16 score of the nearer of two rows overflows and that of the farther one does not: the query's first
    half is rounded down by its f16 form and the second half up, by half a step each"""
    n, half = 33000, 2.0 ** -11
    q1 = np.concatenate([np.full(32, 1 + half), np.full(32, 1 + 3 * half)])

    def row(total, scale, first):
        """32 codes that sum to -total, in the first or the second half, and a scale that puts their sum into [2^57, 2^58)"""
        c, part = np.zeros(64, np.int64), np.full(32, total // 32)
        part[:total % 32] += 1
        c[:32 if first else None][-32:] = -part
        return c, scale * 2.0 ** (57 - np.floor(np.log2(total * scale)))
    c = np.full((n, 64), -7)
    s = np.full((n, 2), 0.8125 * 2.0 ** 50)  # the others: no longer than the two, products of -1.4 times theirs
    near, far = 6000, 20000
    for at, (total, scale, first) in ((near, (155, 211, False)), (far, (137, 239, True))):
        c[at], v = row(total, scale, first)
        s[at] = v
    scales = R.bf16_bits(s.astype(np.float32))
    assert np.array_equal(R.bf16_value(scales), s)
    codes = R.pack(c)
    x = R.decode(codes, s, 64)
    q = np.tile(q1 * 2.0 ** 70, (40, 1)).astype(np.float32)
    assert np.array_equal(q[0], q1 * 2.0 ** 70)
    t = _gpu_table(codes, scales, (x ** 2).sum(1).astype(np.float32), 64)
    ids, _ = _check_knn(t, q, x, 1, "IP")
    assert (ids == near).all()
    _check_knn(t, q, x, 3, "IP", only=[0, 39])
    _check_knn(t, q, x, 2, "L2", only=[0, 39])


@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("B", [30, 40])
@pytest.mark.parametrize("size", [1e-25, 1e-30, 1e-38, 1e-43])
def test_tiny_queries(gpu_lib, metric, B, size):
    """queries so small that their products with small rows are below the f32 range, the nearest row among the small ones"""
    n, dim = 33000, 72
    codes, scales, _, x = _table(n, dim, 32, B)
    s = R.bf16_value(scales).astype(np.float64)
    s[6400:6464] *= 1.03e-15 / np.linalg.norm(x[6400:6464], axis=1)[:, None]  # (all of a tile)
    scales = R.bf16_bits(s.astype(np.float32))
    x = R.decode(codes, R.bf16_value(scales), dim)
    rng = np.random.default_rng(B)
    d = rng.standard_normal((B, dim))
    a = x[6400 + np.arange(B)] / np.linalg.norm(x[6400 + np.arange(B)], axis=1)[:, None]
    d -= (d * a).sum(1)[:, None] * a
    q = ((0.6 * a + 0.8 * d / np.linalg.norm(d, axis=1)[:, None]) * size).astype(np.float32)
    t = _gpu_table(codes, scales, (x ** 2).sum(1).astype(np.float32), dim)
    for k in (1, 7):
        _check_knn(t, q, x, k, metric, only=np.arange(0, B, 4))


# ---- products ------------------------------------------------------------------------------------------------------
def _dots_bound(q, x, group):
    """|q| |x|: a group's sum is joined with two roundings and added with one, to partial sums of at most that; the fixed point is off by
    2^-31 of twice the query's largest element; one rounding of the result; 2^-132 for each group where sums leave the f32 range"""
    groups = -(-x.shape[1] // group)
    a = np.abs(q.astype(np.float64)) @ np.abs(x).T
    return 1.01 * ((groups + 4) * U32 * a + 2.0 ** -30 * np.abs(q).max(1).astype(np.float64)[:, None] * np.abs(x).sum(1)[None, :]) + groups * 2.0 ** -132


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("B", [1, 6, 20])
def test_products_across_the_range(gpu_lib, group, B):
    """rows from 1e-30 to 1e36 with queries from 1e-44 to 1e30: whatever is finite comes back, with the same relative error"""
    n, dim = 200, 768
    codes, scales, sq, x = _table(n, dim, group, B)
    s = R.bf16_value(scales).astype(np.float64)
    s *= (10.0 ** np.linspace(-30, 34, n))[:, None]
    scales = R.bf16_bits(s.astype(np.float32))
    x = R.decode(codes, R.bf16_value(scales), dim)
    t = _gpu_table(codes, scales, sq, dim)
    rng = np.random.default_rng(group)
    for size in (1e-44, 1e-40, 1e-30, 1e-20, 1e-10, 1e-5, 1.0, 1e5, 1e20, 1e30):
        q = rng.standard_normal((B, dim)) * size
        q = q.astype(np.float32)
        want = q.astype(np.float64) @ x.T
        # partial sums within the range: a large sum of terms of both signs is a plain f32 sum's own limit
        fits = np.abs(q.astype(np.float64)) @ np.abs(x).T < 3e38
        got = t.dots(_cuda(q)).cpu().numpy()
        assert fits[:, :100].any() and np.isfinite(got[fits]).all(), size
        err = np.abs(got.astype(np.float64) - want)
        assert np.all((err <= _dots_bound(q, x, group))[fits]), size


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 20])
def test_products_that_cancel(gpu_lib, B):
    """partial sums beyond the f32 range whose total is not; the largest rows there are, with small queries"""
    dim, group = 1024, 32
    c = np.full((40, dim), 7)
    c[:, dim // 2:] = -7
    c[:, 0] = 6
    s = np.full((40, dim // group), 2.0 ** 122)  # 512 elements of 3.7e37 each, then as many of the other sign
    codes, scales = R.pack(c), R.bf16_bits(s.astype(np.float32))
    x = R.decode(codes, s, dim)
    sq = np.zeros(40, np.float32)
    t = _gpu_table(codes, scales, sq, dim)
    for size in (1.0, 0.75, 1e-3, 1e-20):
        q = np.full((B, dim), size, np.float32)
        got = t.dots(_cuda(q)).cpu().numpy()
        want = q.astype(np.float64) @ x.T
        assert np.all(np.abs(got - want) <= _dots_bound(q, x, group)), size
    top = R.bf16_bits(np.full((40, dim // group), 2.0 ** 127, np.float32))
    got = _gpu_table(R.pack(np.full((40, dim), 7)), top, sq, dim).dots(_cuda(np.full((B, dim), 1e-10, np.float32))).cpu().numpy()
    assert np.allclose(got, dim * 7 * 2.0 ** 127 * np.float64(np.float32(1e-10)), rtol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("n,dim,group,B", [(300, 768, 64, 1), (300, 768, 32, 17), (300, 200, 128, 7), (64, 8192, 64, 5), (100, 33, 32, 70)])
def test_products_keep_every_digit(gpu_lib, n, dim, group, B):
    """one large element in each query: the others live in the fixed point's lower digits"""
    codes, scales, sq, x = _table(n, dim, group, n + dim)
    rng = np.random.default_rng(B)
    for spread in (1.0, 1e-3, 1e-6):
        q = (rng.standard_normal((B, dim)) * spread).astype(np.float32)
        q[np.arange(B), rng.integers(0, dim, B)] = 1.0
        got = _gpu_table(codes, scales, sq, dim).dots(_cuda(q)).cpu().numpy()
        assert np.all(np.abs(got - q.astype(np.float64) @ x.T) <= _dots_bound(q, x, group))


# ---- the loss ------------------------------------------------------------------------------------------------------
def _typed(a, dtype):
    import torch
    return a.to(torch.bfloat16 if dtype == "bf16" else torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,V", [(40, 1_000_000), (1024, 1_000_000), (33000, 1_000_003)])
def test_long_sums(gpu_lib, dtype, T, V):
    """a million equal rows and one that outweighs each of them: the sum of their exponentials does not lose more with every row"""
    import torch
    from cozo_amd.softmax import softmax_xent
    w = torch.zeros(V, 8, device="cuda")
    w[V // 3, 0] = 1.0
    w = _typed(w, dtype)
    q = torch.zeros(T, 8, device="cuda")
    q[:, 0] = torch.linspace(0.125, 3.0, T, device="cuda")
    q = _typed(q, dtype)
    y = torch.full((T,), V // 3, dtype=torch.int32, device="cuda")
    loss, lse = softmax_xent(q, w, y)
    z = q[:, 0].double()
    want = torch.log(torch.exp(z) + (V - 1))
    # an exponential: 2 ulp, and its argument (at most 5 to base 2, of two products and a difference) 3 roundings; sums of at most 64 of them
    # before wider ones, 12 joins; lse's own rounding
    tol = (4 + 15 + 64 + 12) * U32 + U32 * want
    assert bool(((lse.double() - want).abs() <= tol).all()), float((lse.double() - want).abs().max())
    assert bool(((loss.double() - (want - z)).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,step", [(300, 2.0 ** -12), (300, 2.0 ** -7), (33000, 2.0 ** -8)])
def test_sums_whose_maximum_keeps_rising(gpu_lib, dtype, T, step):
    """every tile of the table beats the ones before it a little: taking the sum along does not cost a rounding each time"""
    import torch
    from cozo_amd.softmax import softmax_xent
    V = 400_000
    w = torch.zeros(V, 8, device="cuda")
    w[:, 0] = torch.floor(torch.arange(V, device="cuda") / 64.0) * step
    w[:, 1] = w[:, 0] - _typed(w[:, 0], dtype).float()
    w[:, 0] -= w[:, 1]
    w[:, 2] = w[:, 1] - _typed(w[:, 1], dtype).float()
    w[:, 1] -= w[:, 2]
    w = _typed(w, dtype)
    q = torch.zeros(T, 8, device="cuda")
    q[:, :3] = 1.0
    q = _typed(q, dtype)
    y = torch.zeros(T, dtype=torch.int32, device="cuda")
    loss, lse = softmax_xent(q, w, y)
    z = w.double().sum(1)
    want = float(torch.logsumexp(z, 0))
    # (arguments are differences from the maximum: what weighs is within 30 of it; logits of at most 2^7 are off by their roundings)
    top = float(z.max())
    tol = (4 + 64 + 12) * U32 + 8 * U32 * max(1.0, top) + U32 * want
    assert float((lse.double() - want).abs().max()) <= tol


def test_scales_that_are_no_factor_are_refused():
    from cozo_amd import _lib
    L = _lib.lib()
    p = _lib.ptr(np.zeros(64, np.uint8))
    for scale in (np.nan, np.inf, -np.inf, 2.0 ** 127, -2.0 ** 127):
        assert L.cz_softmax_xent(p, 4, p, 4, 0, 1, 1, 4, p, scale, p, p, None, 0, 0, None) == _lib.CZ_E_INVALID
        assert L.cz_softmax_xent_grad(p, 4, p, 4, 0, 1, 1, 4, p, scale, p, p, p, p, None, 0, 0, None) == _lib.CZ_E_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size,scale", [(1e18, 1e-36), (1e18, 1e-37), (1e18, -1e-37), (1e18, 2e-38), (1e-18, 1.5e38), (1e-18, -1.7e38)])
def test_scales_at_the_ends_of_the_range(gpu_lib, dtype, size, scale):
    """products near one end of the f32 range and a scale near the other"""
    import torch
    from cozo_amd.softmax import softmax_xent
    g = torch.Generator().manual_seed(5)
    q, w = torch.randn(9, 40, generator=g) * size, torch.randn(500, 40, generator=g) * size
    q, w = _typed(q, dtype).cuda(), _typed(w, dtype).cuda()
    y = torch.arange(9, dtype=torch.int32, device="cuda")
    loss, lse = softmax_xent(q, w, y, scale=scale)
    z = float(np.float32(scale)) * (q.double() @ w.double().T)
    want = torch.logsumexp(z, 1)
    # of a logit: 40 products, the factors and the argument; the sum of 500 exponentials; lse's own rounding
    tol = 48 * U32 * abs(scale) * (q.double().abs() @ w.double().abs().T).amax(1) + 128 * U32 + U32 * want.abs()
    assert bool(((lse.double() - want).abs() <= tol).all())
    answer = z.gather(1, y.long()[:, None])[:, 0]
    assert bool(((loss.double() - (want - answer)).abs() <= tol + U32 * (want - answer).abs()).all())


# ---- the gradient --------------------------------------------------------------------------------------------------
def _grad_bounds(q, w, y, g, scale, dtype):
    """the gradient in f64 (tensors on the GPU) and how far off each entry may be: as the bound of the other tests, but an answer's entry of G
    loses nothing to bf16"""
    import torch
    q, w, g = q.double(), w.double(), g.double()
    live = (y >= 0)
    at = y.clamp(min=0).long()[:, None]
    z = scale * (q @ w.T)
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    lz = ((q.shape[1] + 8) * U32 * scale) * (q.abs() @ w.abs().T).amax(1)
    ep = 2 * (lz + 128 * U32) + 4 * U32 * (z.abs().amax(1) + lse.abs()) + 2.0 ** -21
    weight = (g.abs() * live)[:, None]
    G = p.clone()
    G.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    G *= (g * live)[:, None]
    del z
    cut = G.abs() * (UBF16 if dtype == "bf16" else 0.0)
    cut.scatter_(1, at, 0.0)
    eG = weight * (p * ep[:, None] + 2 * U32) + 2 * U32 * G.abs() + cut
    del p, cut
    out = UBF16 if dtype == "bf16" else U32
    dq, dw = scale * (G @ w), scale * (G.T @ q)
    a = G.abs()
    tq = scale * (eG @ w.abs()) + (w.shape[0] + 64) * U32 * scale * (a @ w.abs()) + out * dq.abs()
    tw = scale * (eG.T @ q.abs()) + (q.shape[0] + 64) * U32 * scale * (a.T @ q.abs()) + out * dw.abs()
    return dq, dw, 1.01 * tq + 1e-37, 1.01 * tw + 1e-37


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,V,dim", [(3000, 100_003, 24), (3000, 100_003, 23), (700, 70_001, 4100)])
def test_gradient_in_pieces(gpu_lib, dtype, T, V, dim):
    """tables worked on in several pieces, the last one ragged, rows aligned and not, with answers in every piece and at the seams"""
    import torch
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    elem = 1 if dtype == "bf16" else 0
    size = lambda rows: gpu_lib.cz_softmax_xent_workspace(T, rows, dim, elem, 1)  # noqa: E731
    lo, hi = 1, V  # the rows of a piece: from there on the scratch no longer grows
    while lo < hi:
        mid = (lo + hi) // 2
        lo, hi = (lo, mid) if size(mid) == size(V) else (mid + 1, hi)
    piece = -(-lo // 256) * 256
    assert size(2 * V) == size(V) and V > piece + 1 and V % piece
    gen = torch.Generator(device="cuda").manual_seed(dim)
    q = _typed(torch.randn(T, dim, device="cuda", generator=gen) / dim ** 0.5, dtype)
    w = _typed(torch.randn(V, dim, device="cuda", generator=gen), dtype)
    y = torch.randint(0, V, (T,), device="cuda", generator=gen)
    y[1::7] = -1
    seams = [0, piece - 1, piece, piece + 1, V - 1] + [v for k in range(2, -(-V // piece)) for v in (k * piece - 1, k * piece)]
    y[2:2 + 2 * len(seams):2] = torch.tensor(seams, device="cuda")
    g = torch.randn(T, device="cuda", generator=gen)
    loss, lse = softmax_xent(q, w, y, scale=2.0)
    got_q, got_w = softmax_xent_grad(q, w, y, lse, g, scale=2.0)
    dq, dw, tq, tw = _grad_bounds(q, w, y, g, 2.0, dtype)
    assert bool(((got_q.double() - dq).abs() <= tq).all()) and bool(((got_w.double() - dw).abs() <= tw).all())
    assert not bool(got_q[y < 0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,dim", [(40, 700, 64), (300, 3000, 128), (5, 2000, 72)])
def test_answers_lose_nothing_to_rounding(gpu_lib, T, V, dim):
    """bf16: G is rounded to 8 bits before the products, but not at the answers, whose entries outweigh the others"""
    import torch
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    gen = torch.Generator(device="cuda").manual_seed(T)
    w = torch.randn(V, dim, device="cuda", generator=gen).to(torch.bfloat16)
    y = torch.randperm(V, device="cuda", generator=gen)[:T]
    q = (torch.randn(T, dim, device="cuda", generator=gen) * 0.05).to(torch.bfloat16)
    g = torch.full((T,), 171.45 / 512, device="cuda")  # (rounded to bf16: off by two thirds of what the result's own rounding may be)
    _, lse = softmax_xent(q, w, y)
    got_q, got_w = softmax_xent_grad(q, w, y, lse, g)
    dq, dw, tq, tw = _grad_bounds(q, w, y, g, 1.0, "bf16")
    assert bool(((got_q.double() - dq).abs() <= tq).all()) and bool(((got_w.double() - dw).abs() <= tw).all())


@pytest.mark.gpu
def test_answers_do_not_drown_the_rest(gpu_lib):
    """f32: a query's gradient is one large term, of the row that answers it, and a sum of many, each below half a step of that term"""
    import torch
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    T, V, dim = 60, 3001, 64
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = 0.07 + 0.005 * torch.rand(V, dim, device="cuda", generator=gen)
    y = torch.randperm(V, device="cuda", generator=gen)[:T]
    w[y] = 900.0 + 100.0 * torch.rand(T, dim, device="cuda", generator=gen)
    q = -torch.rand(T, dim, device="cuda", generator=gen) / dim  # (the answers' logits are far below the others: their weights are -1)
    g = torch.ones(T, device="cuda")
    _, lse = softmax_xent(q, w, y)
    got, _ = softmax_xent_grad(q, w, y, lse, g, want_table=False)
    z = q.double() @ w.double().T
    p = torch.exp(z - torch.logsumexp(z, 1)[:, None])
    # of a weight: its logit and lse, each rounded, an exponential; of the sum: V additions
    ep = 2 * (dim + 8) * U32 * (q.double().abs() @ w.double().abs().T) + 128 * U32 + 12 * U32 * np.log(V)
    at = torch.arange(T, device="cuda")
    small = p.clone()
    small[at, y] = 0
    hit = (p[at, y] - 1)[:, None] * w[y].double()
    want = small @ w.double() + hit
    tol = (small * (ep + (V + 64) * U32)) @ w.double().abs() + 4 * U32 * hit.abs() + 2 * U32 * want.abs()
    assert bool(((got.double() - want).abs() <= tol).all())


# ---- tensors that require a gradient -------------------------------------------------------------------------------
def test_tensors_that_require_a_gradient_are_refused():
    import torch
    from cozo_amd import softmax
    from cozo_amd._device import no_graph
    a, b = torch.zeros(3, 8), torch.zeros(5, 8, requires_grad=True)
    y = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="gradient"):
        softmax.softmax_xent(a, b, y)
    with pytest.raises(ValueError, match="gradient"):
        softmax.softmax_xent(b[:3], a, y)
    with pytest.raises(ValueError, match="gradient"):
        softmax.softmax_xent_grad(a, b, y, torch.zeros(3), torch.zeros(3))
    with pytest.raises(ValueError, match="gradient"):
        no_graph(None, np.zeros(3), b)
    with torch.no_grad():
        no_graph(b)
    no_graph(b.detach(), a, None)


@pytest.mark.gpu
def test_a_parameter_trains(gpu_lib):
    import torch
    from cozo_amd.quantized import quantize
    from cozo_amd.softmax import softmax_xent, softmax_xent_grad
    w = torch.nn.Parameter(torch.randn(300, 64, device="cuda"))
    q, y = torch.randn(5, 64, device="cuda"), torch.arange(5, device="cuda")
    with pytest.raises(ValueError, match="gradient"):
        softmax_xent(q, w, y)
    with torch.no_grad():
        loss, lse = softmax_xent(q, w, y)
        w.grad = softmax_xent_grad(q, w, y, lse, torch.ones(5, device="cuda"), want_queries=False)[1]
        t = quantize(w)
    ref = w.detach().double().requires_grad_()
    torch.nn.functional.cross_entropy(q.double() @ ref.T, y, reduction="sum").backward()
    # a weight's relative error: its logit's (64 products and 8 roundings), twice with lse's, and the sum's and the exponential's
    off = 2 * 72 * U32 * float((q.double().abs() @ ref.detach().abs().T).max()) + 128 * U32
    assert bool(((w.grad.double() - ref.grad).abs() <= off * q.double().abs().sum(0)).all())
    with pytest.raises(ValueError, match="gradient"):
        t.dots(q.clone().requires_grad_())
    with pytest.raises(ValueError, match="gradient"):
        t.knn(q.clone().requires_grad_(), 3)
