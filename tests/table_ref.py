"""64-bit restatements of the operators over whole tables (4-bit rows, softmax cross entropy), from their formulas."""
import numpy as np


def bf16_bits(x):
    """f32 -> bfloat16 bits, round to nearest even (finite values)"""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(b):
    return (np.asarray(b, dtype=np.uint32) << 16).view(np.float32)


def quantize(x, group):
    """codes int [n][groups * group], scales f32 [n][groups] (bfloat16 values); x finite"""
    x = np.asarray(x, dtype=np.float32)
    n, d = x.shape
    x = np.concatenate([x, np.zeros((n, -d % group), np.float32)], 1).reshape(n, -1, group)
    m = np.abs(x).max(2)
    s = bf16_value(bf16_bits((m / np.float32(7)).astype(np.float32)))
    s = np.where(m < np.float32(2.0 ** -60), np.float32(0), s)
    with np.errstate(divide="ignore"):
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
    c = np.clip(np.rint(x * inv[:, :, None]), -7, 7).astype(np.int64)
    return c.reshape(n, -1), s


def pack(c):
    c = np.asarray(c) & 15
    return (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)


def unpack(codes):
    b = np.asarray(codes).astype(np.int64)
    c = np.stack([b & 15, b >> 4], 2).reshape(b.shape[0], -1)
    return np.where(c > 7, c - 16, c)


def decode(codes, scale_values, dim):
    """the f64 rows that packed codes and scales (as numbers) stand for"""
    c = unpack(codes).astype(np.float64)
    s = np.asarray(scale_values, dtype=np.float64)
    n, groups = s.shape
    return (c.reshape(n, groups, -1) * s[:, :, None]).reshape(n, -1)[:, :dim]


def distances(metric, q, x):
    """f64 [B][n] of q [B][d], x [n][d], summed in numpy's long doubles"""
    q, x = np.asarray(q, dtype=np.longdouble), np.asarray(x, dtype=np.longdouble)
    out = np.empty((q.shape[0], x.shape[0]))
    with np.errstate(all="ignore"):
        for b in range(q.shape[0]):
            if metric == "L2":
                out[b] = ((q[b] - x) ** 2).sum(1)
            elif metric == "IP":
                out[b] = 1 - x @ q[b]
            else:
                out[b] = 1 - (x @ q[b]) / np.sqrt((q[b] ** 2).sum() * (x ** 2).sum(1))
    return out


def nearest(dist, k, radius=None):
    """(ids, distances, count) rows of dist [B][n]: ascending, ties to the lower row, NaN last, padded"""
    B, n = dist.shape
    ids = np.full((B, k), 0xFFFFFFFF, dtype=np.uint32)
    out = np.full((B, k), np.inf)
    cnt = np.zeros(B, dtype=np.uint32)
    for b in range(B):
        d = dist[b]
        order = np.lexsort((np.arange(n), np.where(np.isnan(d), np.inf, d), np.isnan(d)))[:k]
        if radius is not None:
            order = order[~(d[order] > radius)]
        cnt[b] = order.size
        ids[b, :order.size] = order
        out[b, :order.size] = d[order]
    return ids, out, cnt


def softmax_xent(q, w, y, scale):
    """(loss, lse, z) in f64; y = -1: no answer"""
    q, w, y = np.asarray(q, dtype=np.float64), np.asarray(w, dtype=np.float64), np.asarray(y, dtype=np.int64)
    z = scale * (q @ w.T)
    m = z.max(1)
    lse = m + np.log(np.exp(z - m[:, None]).sum(1))
    loss = np.where(y >= 0, lse - z[np.arange(y.size), np.maximum(y, 0)], 0.0)
    return loss, lse, z


def softmax_xent_grad(q, w, y, scale, grad_loss):
    """(grad_queries, grad_table, G) in f64"""
    q, w, y = np.asarray(q, dtype=np.float64), np.asarray(w, dtype=np.float64), np.asarray(y, dtype=np.int64)
    _, lse, z = softmax_xent(q, w, y, scale)
    g = np.exp(z - lse[:, None])
    g[np.arange(y.size), np.maximum(y, 0)] -= 1
    g *= (np.asarray(grad_loss, dtype=np.float64) * (y >= 0))[:, None]
    return scale * (g @ w), scale * (g.T @ q), g
