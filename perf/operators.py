"""What the operators over tables of embeddings are measured on: 4-bit rows (quantising them, products with them, k-NN over
them) and the softmax cross entropy over a whole table, forward and as a training step.

`run` computes a case in its plain form, in elementary torch operations, or (``own``) with the calls that a user makes of
`cozo_amd.quantized` and `cozo_amd.softmax`."""
import math

import torch

own = False

RANK = 16     # of the embeddings' latent factor
EXTRA = 24    # rows beyond k whose distances the plain k-NN computes again in 64 bits


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    return [
        # an index of the smallest configuration (10k x 128) quantised when it is loaded, and read back
        {"name": "quantize 10k x 128", "op": "quantize", "n": 10_000, "dim": 128, "group": 32, "dtype": "f32"},
        # the 1M x 768 configuration quantised once after training
        {"name": "quantize 1M x 768", "op": "quantize", "n": 1_000_000, "dim": 768, "group": 64, "dtype": "f32"},
        # one query against a small table: what a single tuple of a query plan asks for
        {"name": "dots 1 x 10k x 128", "op": "dots", "B": 1, "n": 10_000, "dim": 128, "group": 32},
        # one query against the 10M x 768 table: the product that reads every row
        {"name": "dots 1 x 10M x 768", "op": "dots", "B": 1, "n": 10_000_000, "dim": 768, "group": 64},
        # a few queries, a ragged table: rows that are no multiple of a tile, a dimension that is no multiple of a group
        {"name": "dots 7 x 1000003 x 200", "op": "dots", "B": 7, "n": 1_000_003, "dim": 200, "group": 128},
        # the smallest search
        {"name": "knn L2 1 x 10k x 128", "op": "knn", "B": 1, "n": 10_000, "dim": 128, "group": 32, "k": 10, "metric": "L2"},
        # one parent tuple against the whole 10M table
        {"name": "knn cosine 1 x 10M x 768", "op": "knn", "B": 1, "n": 10_000_000, "dim": 768, "group": 64, "k": 10, "metric": "Cosine"},
        # the benchmark's batch of 1024 queries against the 1M table
        {"name": "knn cosine 1024 x 1M x 768", "op": "knn", "B": 1024, "n": 1_000_000, "dim": 768, "group": 64, "k": 10, "metric": "Cosine"},
        # the loss of a few queries over the small table
        {"name": "xent f32 16 x 10k x 128", "op": "xent", "T": 16, "V": 10_000, "dim": 128, "dtype": "f32"},
        # evaluation of a batch over the 1M table
        {"name": "xent bf16 1024 x 1M x 768", "op": "xent", "T": 1024, "V": 1_000_000, "dim": 768, "dtype": "bf16"},
        # a training step in f32 at ragged sizes
        {"name": "step f32 255 x 100003 x 96", "op": "step", "T": 255, "V": 100_003, "dim": 96, "dtype": "f32"},
        # a training step of the benchmark's batch over the 1M table
        {"name": "step bf16 1024 x 1M x 768", "op": "step", "T": 1024, "V": 1_000_000, "dim": 768, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "dots", "dots", "knn", "knn", "xent", "step"])
    dim = rng.choice([rng.randint(33, 1024), 8 * rng.randint(5, 128), 128 * rng.randint(1, 8)])
    group = rng.choice([32, 64, 128])
    if op == "quantize":
        return {"op": op, "n": _spread(rng, 1_000, 700_000), "dim": dim, "group": group, "dtype": rng.choice(["f32", "bf16"])}
    if op == "dots":
        n = _spread(rng, 1_000, 3_000_000)
        return {"op": op, "B": min(_spread(rng, 1, 64), max(1, 30_000_000 // n)), "n": n, "dim": dim, "group": group}
    if op == "knn":
        n = _spread(rng, 1_000, 3_000_000)
        return {"op": op, "B": min(_spread(rng, 1, 1024), max(1, 500_000_000 // n)), "n": n, "dim": dim, "group": group,
                "k": rng.randint(1, 100), "metric": rng.choice(["L2", "Cosine", "IP"])}
    T, V, dtype = _spread(rng, 1, 1024), _spread(rng, 1_000, 500_000), rng.choice(["f32", "bf16"])
    return {"op": op, "T": T, "V": V, "dim": dim, "dtype": dtype}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _embeddings(g, n, dim):
    """rows as an embedding model gives them: a low-rank factor and a little isotropic noise (the benchmark's corpus)"""
    w = torch.randn(RANK, dim, generator=torch.Generator(device="cuda").manual_seed(12345), device="cuda")
    return torch.randn(n, RANK, generator=g, device="cuda") @ w + 0.1 * torch.randn(n, dim, generator=g, device="cuda")


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d = case["dim"]
    if case["op"] == "quantize":
        return {"case": case, "x": _embeddings(g, case["n"], d).to(_dtype(case))}
    if case["op"] in ("dots", "knn"):
        parts = [_quantize(_embeddings(g, min(1_000_000, case["n"] - at), d), case["group"]) for at in range(0, case["n"], 1_000_000)]
        codes, scales, sq = (torch.cat(p) for p in zip(*parts))
        return {"case": case, "codes": codes, "scales": scales, "sqnorms": sq, "q": _embeddings(g, case["B"], d)}
    T, V = case["T"], case["V"]
    w = torch.nn.functional.normalize(_embeddings(g, V, d), dim=1)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    # a query lies near the row that answers it, half way to a random direction
    q = torch.nn.functional.normalize(w[y] + torch.nn.functional.normalize(_embeddings(g, T, d), dim=1), dim=1)
    y[16::17] = -1  # padding of a ragged batch: no row answers it
    answered = (y >= 0).float()
    return {"case": case, "q": q.to(_dtype(case)), "w": w.to(_dtype(case)), "y": y.to(torch.int32), "scale": 20.0,
            "dloss": answered / answered.sum().clamp(min=1)}


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _quantize(x, group):
    """-> codes [n][groups * group / 2] u8, scales [n][groups] bf16, squared norms of the quantised rows f32 [n]"""
    n, d = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -d % group)).view(n, -1, group)
    m = x.abs().amax(2)
    s = (m.double() / 7).float().to(torch.bfloat16)
    s = torch.where(m < 2.0 ** -60, torch.zeros_like(s), s)
    inv = torch.where(s > 0, (1 / s.double()).float(), torch.zeros_like(m))
    c = (x * inv[:, :, None]).round_().clamp_(-7, 7)
    sq = (c.square().sum(2).double() * s.double().square()).sum(1).float()
    c = c.to(torch.int8).view(n, -1, 2)
    return ((c[:, :, 0] & 15) | (c[:, :, 1] << 4)).view(torch.uint8), s, sq


def _decode(codes, scales):
    """the rows that 4-bit codes and group scales stand for, f32, with the last group's padding"""
    n, groups = scales.shape
    c = torch.stack((codes << 4, codes & 0xF0), dim=-1).view(torch.int8) >> 4
    return (c.view(n, groups, -1).float() * scales.float()[:, :, None]).view(n, -1)


def _distance(metric, q, x):
    """distances of q [B][1][d] from x [B][m][d]"""
    if metric == "L2":
        return (q - x).square().sum(-1)
    dot = (q * x).sum(-1)
    return 1 - (dot / (q.square().sum(-1) * x.square().sum(-1)).sqrt() if metric == "Cosine" else dot)


def _nearest(dist, ids, k):
    """the k nearest in each row, ties to the lowest id"""
    ids, by_id = ids.sort(dim=1)
    dist, by = dist.gather(1, by_id).sort(dim=1, stable=True)
    return ids.gather(1, by)[:, :k].to(torch.int32), dist[:, :k].contiguous()


def _knn(s, case):
    q, d, k = s["q"], case["dim"], case["k"]
    rows = _decode(s["codes"], s["scales"])[:, :d]
    near = q @ rows.T
    if case["metric"] == "Cosine":
        near *= s["sqnorms"].rsqrt()
    if case["metric"] == "L2":
        near = near.mul_(2).sub_(s["sqnorms"])
    ids = near.topk(min(k + EXTRA, case["n"]), dim=1).indices
    dist = _distance(case["metric"], q.double()[:, None], rows[ids].double())
    ids, dist = _nearest(dist, ids, k)
    return {"ids": ids, "dist": dist}


def _xent(s):
    y = s["y"].long()
    z = (s["q"].float() @ s["w"].float().T) * s["scale"]
    lse = torch.logsumexp(z, 1)
    loss = torch.where(y >= 0, lse - z.gather(1, y.clamp(min=0)[:, None])[:, 0], torch.zeros_like(lse))
    return z, lse, loss


def _step(s):
    y = s["y"].long()
    z, lse, loss = _xent(s)
    p = z.sub_(lse[:, None]).exp_()
    weight = (torch.where(y >= 0, s["dloss"], torch.zeros_like(lse)) * s["scale"])[:, None]
    at, w, q = y.clamp(min=0)[:, None], s["w"].float(), s["q"].float()
    hit = (p.gather(1, at) - 1) * weight
    # dq is a long sum beside one term that outweighs the others: that one is added to the sum of the rest
    p = (p * weight).scatter_(1, at, 0.0)
    dq = p @ w + hit * w[at[:, 0]]
    dw = p.scatter_(1, at, hit).T @ q
    return {"loss": loss, "dq": dq.to(s["q"].dtype), "dw": dw.to(s["w"].dtype)}


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from cozo_amd import quantized, softmax
        if op == "quantize":
            t = quantized.quantize(s["x"], group=case["group"])
            return {"rows": t.dequantize(), "sqnorms": t.sqnorms}
        if op in ("dots", "knn"):
            t = quantized.Q4Table(s["codes"], s["scales"], s["sqnorms"], case["dim"])
            if op == "dots":
                return t.dots(s["q"])
            ids, dist, _ = t.knn(s["q"], case["k"], distance=case["metric"])
            return {"ids": ids, "dist": dist}
        loss, lse = softmax.softmax_xent(s["q"], s["w"], s["y"], scale=s["scale"])
        if op == "xent":
            return {"loss": loss, "lse": lse}
        dq, dw = softmax.softmax_xent_grad(s["q"], s["w"], s["y"], lse, s["dloss"], scale=s["scale"])
        return {"loss": loss, "dq": dq, "dw": dw}
    if op == "quantize":
        codes, scales, sq = _quantize(s["x"], case["group"])
        return {"rows": _decode(codes, scales)[:, :case["dim"]].contiguous(), "sqnorms": sq}
    if op == "dots":
        return (_decode(s["codes"], s["scales"])[:, :case["dim"]] @ s["q"].T).T.contiguous()
    if op == "knn":
        return _knn(s, case)
    if op == "xent":
        _, lse, loss = _xent(s)
        return {"loss": loss, "lse": lse}
    return _step(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    d = case["dim"]
    if case["op"] == "quantize":
        n, groups = case["n"], -(-d // case["group"])
        table = n * groups * (case["group"] // 2 + 2)
        # the rows in, the 4-bit form out and in again, the decoded rows out
        return {"bytes": n * d * ((4 if case["dtype"] == "f32" else 2) + 4) + 2 * table + 4 * n, "flops": 4.0 * n * d}
    if case["op"] in ("dots", "knn"):
        n, B, groups = case["n"], case["B"], -(-d // case["group"])
        table = n * groups * (case["group"] // 2 + 2)
        out = 4 * B * n if case["op"] == "dots" else 12 * B * case["k"] + 4 * n
        return {"bytes": table + 4 * B * d + out, "flops": 2.0 * B * n * d}
    T, V, e = case["T"], case["V"], 4 if case["dtype"] == "f32" else 2
    if case["op"] == "xent":
        return {"bytes": e * (T + V) * d + 12 * T, "flops": 2.0 * T * V * d}
    return {"bytes": 2 * e * (T + V) * d + 16 * T, "flops": 6.0 * T * V * d}


# ---- 64 bits -------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d, op = case["dim"], case["op"]
    if op == "quantize":
        rows, norms = [], []
        for x in s["x"].split(200_000):
            x = torch.nn.functional.pad(x.double(), (0, -d % case["group"])).unflatten(1, (-1, case["group"]))
            top = x.abs().max(2, keepdim=True).values
            step = (top / 7).float().bfloat16().double() * (top >= 2.0 ** -60)
            # the code is defined by the 32-bit product with the 32-bit reciprocal: the 64-bit product is exact, then rounded
            code = (x * (1 / step).float().double()).float().double().round().clamp(-7, 7)
            x = torch.where(step > 0, code * step, 0.0).flatten(1)[:, :d]
            rows.append(x)
            norms.append(x.pow(2).sum(1))
        return {"rows": torch.cat(rows), "sqnorms": torch.cat(norms)}
    if op in ("dots", "knn"):
        q, dots, norms = s["q"].double(), [], []
        for codes, scales in zip(s["codes"].split(500_000), s["scales"].split(500_000)):
            low, high = codes.to(torch.int16) % 16, codes.to(torch.int16).div(16, rounding_mode="floor")
            c = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device="cuda")
            c[:, 0::2], c[:, 1::2] = low - 16 * (low > 7), high - 16 * (high > 7)
            x = (c.unflatten(1, (scales.shape[1], -1)) * scales.double().unsqueeze(2)).flatten(1)[:, :d].contiguous()
            dots.append(q @ x.T)
            norms.append(x.pow(2).sum(1))
        dots, norms, qq = torch.cat(dots, 1), torch.cat(norms), q.pow(2).sum(1, keepdim=True)
        if op == "dots":
            return dots
        if case["metric"] == "L2":
            dots = dots.mul_(-2).add_(norms).add_(qq)
        elif case["metric"] == "Cosine":
            dots = dots.div_((qq * norms).sqrt()).neg_().add_(1)
        else:
            dots = dots.neg_().add_(1)
        return {"ids": None, "dist": dots.topk(case["k"], dim=1, largest=False).values}
    q, y = s["q"].double(), s["y"].long()
    some = y >= 0
    lse, hit = torch.full((case["T"],), -math.inf, dtype=torch.float64, device="cuda"), (q * s["w"][y.clamp(min=0)].double()).sum(1) * s["scale"]
    for w in s["w"].split(100_000):
        lse = torch.logaddexp(lse, (s["scale"] * (q @ w.double().T)).logsumexp(1))
    loss = torch.where(some, lse - hit, 0.0)
    if op == "xent":
        return {"loss": loss, "lse": lse}
    weight = (s["dloss"].double() * some * s["scale"]).unsqueeze(1)
    dq, dw = -weight * s["w"][y.clamp(min=0)].double(), []
    for w in s["w"].split(100_000):
        p = (s["scale"] * (q @ w.double().T) - lse.unsqueeze(1)).exp() * weight
        dq += p @ w.double()
        dw.append(p.T @ q)
    dw = torch.cat(dw)
    dw.index_add_(0, y[some], (-weight * q)[some])
    return {"loss": loss, "dq": dq, "dw": dw}
