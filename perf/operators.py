"""What is measured of the retrieval operators: products of queries with 4-bit rows behind a top-k search, pooled embedding
lookups with scaling, and the lookups' gradient by sorted tokens.

`run` computes a pass either in its plain form (elementary torch operations) or, where `own` is set, through coderag_hip's entry
points.  `exact` says the same from the definitions in float64."""
import math

import torch

own = False

GROUP = 32                                   # elements that share a scale
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # magnitudes of the 4-bit codes
EXP_MIN, EXP_MAX = -125, 125                 # exponents of the group scales


# ---- the cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one question against a small workspace: a few thousand chunks, the editor waits for the answer
        {"name": "search_1q_8k_x384", "op": "search", "rows": 8000, "dim": 384, "queries": 1, "top_k": 10, "metric": "l2"},
        # one question against a large workspace
        {"name": "search_1q_4m_x384", "op": "search", "rows": 4000000, "dim": 384, "queries": 1, "top_k": 10, "metric": "l2"},
        # a handful of questions at once, rows that end inside a tile, a dimension that is no multiple of the group
        {"name": "search_7q_1m_x500", "op": "search", "rows": 1000003, "dim": 500, "queries": 7, "top_k": 25, "metric": "ip"},
        # an agent's or an evaluation's batch of questions
        {"name": "search_256q_1m_x768", "op": "search", "rows": 1000000, "dim": 768, "queries": 256, "top_k": 10, "metric": "l2"},
        # an offline run over a log of questions, many results each
        {"name": "search_1024q_300k_x1024", "op": "search", "rows": 300007, "dim": 1024, "queries": 1024, "top_k": 100, "metric": "l2"},
        # one question for each of 64 workspaces in one call
        {"name": "multi_64x20k_x384", "op": "multi", "rows": 20001, "dim": 384, "queries": 64, "top_k": 10, "metric": "l2"},
        # the vector of one question: a short text's n-grams
        {"name": "embed_1x120", "op": "embed", "bags": 1, "mean_len": 120, "dim": 384, "vocab": 262144, "dtype": "f32", "mode": "mean", "normalize": True},
        # one step of an ingest: 100 chunks of code, their n-grams
        {"name": "embed_100x2000", "op": "embed", "bags": 100, "mean_len": 2000, "dim": 384, "vocab": 262144, "dtype": "f32", "mode": "mean", "normalize": True},
        # a large ingest with a word-piece vocabulary, bf16 table and vectors
        {"name": "embed_8192x300_bf16", "op": "embed", "bags": 8192, "mean_len": 300, "dim": 768, "vocab": 32768, "dtype": "bf16", "mode": "sqrt", "normalize": True},
        # the smallest training step: a few question/chunk pairs
        {"name": "train_32x100", "op": "train", "bags": 32, "mean_len": 100, "dim": 384, "vocab": 32768, "dtype": "f32", "mode": "mean", "normalize": True},
        # an ordinary training step over n-grams, a token that makes up a twentieth of all
        {"name": "train_1024x1000", "op": "train", "bags": 1024, "mean_len": 1000, "dim": 384, "vocab": 262144, "dtype": "f32", "mode": "mean", "normalize": True},
        # a bf16 table, sums that are not normalised, an odd number of bags and of dimensions
        {"name": "train_2047x333_bf16", "op": "train", "bags": 2047, "mean_len": 333, "dim": 516, "vocab": 50001, "dtype": "bf16", "mode": "sum", "normalize": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["search", "search", "multi", "embed", "train"])
    if op in ("search", "multi"):
        dim = rng.choice([_log(rng, 64, 1024), 384, 768])
        if op == "multi":
            queries, rows = rng.randint(2, 64), _log(rng, 300, 20000)
        else:
            queries = _log(rng, 1, 1024)
            # no more work than the largest listed one
            rows = _log(rng, 1000, min(4000000, 300000 * 1024 * 1024 // (max(queries, 64) * dim)))
        return {"op": op, "rows": rows, "dim": dim, "queries": queries, "top_k": _log(rng, 1, 100), "metric": rng.choice(["l2", "ip"])}
    bags = _log(rng, 1, 4096)
    return {"op": op, "bags": bags, "mean_len": _log(rng, 1, min(2000, 1000000 // bags)), "dim": rng.choice([_log(rng, 32, 1024), 384, 768]),
            "vocab": _log(rng, 500, 262144), "dtype": rng.choice(["f32", "bf16"]), "mode": rng.choice(["sum", "mean", "sqrt"]),
            "normalize": rng.random() < 0.7}


def _tokens(case):
    return case["bags"] * case["mean_len"]


def work(case):
    d = case["dim"]
    if case["op"] in ("search", "multi"):
        n = case["rows"] * (case["queries"] if case["op"] == "multi" else 1)
        products = case["rows"] * case["queries"]
        out = case["queries"] * (case["top_k"] * 20 + 4)
        return {"bytes": n * d // 2 + n * -(-d // GROUP) + n + case["queries"] * d * 4 + out, "flops": 2 * products * d}
    t, v, b = _tokens(case), case["vocab"], case["bags"]
    esz = 4 if case["dtype"] == "f32" else 2
    # rows of the table that occur among t tokens drawn with p_i ~ 1 / i
    i = torch.arange(1, v + 1, dtype=torch.float64)
    p = torch.log1p(1 / i) / math.log(v + 1)
    rows = float((1 - torch.exp(t * torch.log1p(-p.clamp(max=0.999999)))).sum())
    if case["op"] == "embed":
        return {"bytes": int(t * 8 + rows * d * esz + (b + 1) * 8 + b * d * esz), "flops": 2 * t * d}
    # forward (y), the gradient of y read, the whole table's gradient and every weight's written
    return {"bytes": int(t * 12 + rows * d * esz + (b + 1) * 8 + 2 * b * d * 4 + v * d * esz), "flops": 6 * t * d}


# ---- 4-bit rows, plain ------------------------------------------------------------------------------------------------------
def _quantize(rows):
    """float32 [n, d] -> (codes uint8 [n, dp/2], exponents int8 [n, dp/32]): each group's scale is the smallest power of two that
    keeps its largest element within 7, each element the nearest code (ties to the even one)."""
    n, d = rows.shape
    dp = -(-d // GROUP) * GROUP
    x = torch.nn.functional.pad(rows, (0, dp - d)).view(n, dp // GROUP, GROUP)
    m, ex = torch.frexp(x.abs().amax(-1))
    e = (ex - 3 + (m > 0.875).int()).clamp(EXP_MIN, EXP_MAX)
    v = torch.ldexp(x, -e.unsqueeze(-1))
    neg = v < 0
    v = v.abs()
    c = (v > 0.25).to(torch.uint8)
    c += v >= 0.75
    c += v > 1.25
    c += v >= 1.75
    c += v > 2.5
    c += v >= 3.5
    c += v > 5
    c |= neg.to(torch.uint8) << 3
    c = c.view(n, dp)
    return c[:, 0::2] | (c[:, 1::2] << 4), e.to(torch.int8)


def _dequantize(codes, exps, dtype):
    n = codes.shape[0]
    lut = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=dtype, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).view(n, -1).int()
    x = lut[c].view(n, exps.shape[1], GROUP)
    return torch.ldexp(x, exps.int().unsqueeze(-1)).view(n, -1)


def _rerank(dist, ids, cls, top_k):
    """dist float32 [b, c] of candidates with ascending ids [b, c] and path classes [b, c] -> what a search returns: of the 2 * top_k
    nearest (ties to the lower id) the top_k by 1 / (1 + distance) times the path's factor, those over 0.01."""
    b = dist.shape[0]
    kc = 2 * top_k
    if dist.shape[1] < kc:
        more = kc - dist.shape[1]
        dist = torch.cat((dist, dist.new_full((b, more), math.inf)), 1)
        ids = torch.cat((ids, ids.new_full((b, more), -1)), 1)
        cls = torch.cat((cls, cls.new_zeros((b, more))), 1)
    dist, o = torch.sort(dist, dim=1, stable=True)
    dist, o = dist[:, :kc], o[:, :kc]
    ids, cls = ids.gather(1, o), cls.gather(1, o)
    factor = torch.tensor([1.0, 0.1, 1.2, 1.0], dtype=torch.float64, device=dist.device)[cls.long()]
    score = 1.0 / (1.0 + dist.double()) * factor
    kept = (score > 0.01) & (ids >= 0)
    score, o = torch.sort(torch.where(kept, score, -1.0), dim=1, descending=True, stable=True)
    score, o = score[:, :top_k], o[:, :top_k]
    kept, ids, dist = score > 0, ids.gather(1, o), dist.gather(1, o)
    return (torch.where(kept, ids, -1), torch.where(kept, score, 0.0), torch.where(kept, dist, math.inf), kept.sum(1).int())


def _nearest_plain(rows, queries, cls, case):
    """rows float32 [..., n, dp], queries float32 [..., b, dp]: float32 scores choose the candidates, their distances are computed in
    float64 (neighbours in the order differ by less than float32 products resolve)."""
    n, top_k = rows.shape[-2], case["top_k"]
    dots = queries @ rows.transpose(-1, -2)
    scores = (rows * rows).sum(-1).unsqueeze(-2) - 2 * dots if case["metric"] == "l2" else -dots
    c = min(n, 2 * top_k + 64)
    ids = torch.topk(scores, c, dim=-1, largest=False).indices.sort(-1).values      # [..., b, c]
    b = queries.shape[-2]
    if rows.dim() == 3:   # one query for each collection
        near = rows.gather(1, ids[:, 0].unsqueeze(-1).expand(-1, -1, rows.shape[-1])).double()
        q, ids, cls = queries[:, 0].double(), ids[:, 0], cls.gather(1, ids[:, 0])
    else:
        near = rows[ids.view(-1)].view(b, c, -1).double()
        q, cls = queries.double(), cls[ids]
    dist = (near - q.unsqueeze(1)).square().sum(-1) if case["metric"] == "l2" else 1 - (near * q.unsqueeze(1)).sum(-1)
    return _rerank(dist.float(), ids, cls, top_k)


# ---- embedding lookups, plain -------------------------------------------------------------------------------------------------
def _bag_of(offsets, t):
    return torch.bucketize(torch.arange(t, device=offsets.device), offsets[1:], right=True)


def _pool_factor(offsets, mode):
    n = (offsets[1:] - offsets[:-1]).clamp(min=1).double()
    return {"sum": torch.ones_like(n), "mean": 1 / n, "sqrt": n.rsqrt()}[mode].unsqueeze(-1)


def _run_sums(rows, edges):
    """sums of rows[edges[i]:edges[i + 1]]: differences of running sums in float64"""
    run = rows.t().contiguous().double().cumsum(1)
    run = torch.nn.functional.pad(run, (1, 0))
    return (run[:, edges[1:]] - run[:, edges[:-1]]).t()


def _embed_plain(case, table, ids, weights, offsets):
    rows = table[ids.long()].float() * weights.unsqueeze(-1)
    factor = case["scale"] * _pool_factor(offsets, case["mode"])
    p = _run_sums(rows, offsets) * factor
    norm = p.square().sum(-1, keepdim=True).sqrt() if case["normalize"] else torch.ones_like(factor)
    return torch.where(norm > 0, p / norm, 0.0), factor, norm


def _train_plain(case, table, ids, weights, offsets, grad):
    y, factor, norm = _embed_plain(case, table, ids, weights, offsets)
    g = grad.double()
    if case["normalize"]:
        g = torch.where(norm > 0, (g - y * (g * y).sum(-1, keepdim=True)) / norm, 0.0)
    each = (g * factor).float()[_bag_of(offsets, ids.numel())]
    d_weights = (each * table[ids.long()].float()).sum(-1)
    order = torch.sort(ids, stable=True).indices
    edges = torch.nn.functional.pad(torch.bincount(ids, minlength=case["vocab"]).cumsum(0), (1, 0))
    d_table = _run_sums((each * weights.unsqueeze(-1))[order], edges)
    return y, d_table, d_weights


# ---- state and pass -----------------------------------------------------------------------------------------------------------
def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _rows(n, d, g):
    """unit vectors around some hundred centres, as an embedder's are"""
    centres = torch.randn((256, d), generator=g, device="cuda")
    at = torch.randint(0, 256, (n,), generator=g, device="cuda")
    x = torch.randn((n, d), generator=g, device="cuda").add_(centres[at], alpha=0.5)
    return x.div_(x.norm(dim=-1, keepdim=True))


def _framework():
    import sys
    if "code-rag_amd" not in sys.path:
        sys.path.insert(0, "code-rag_amd")
    import coderag_hip
    return coderag_hip


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("search", "multi"):
        cols = case["queries"] if case["op"] == "multi" else 1
        n, d = case["rows"], case["dim"]
        rows = _rows(cols * n, d, g)
        # path classes: 0 neutral, 1 tests and declarations, 2 sources
        cls = torch.randint(0, 3, (cols * n,), generator=g, device="cuda", dtype=torch.uint8)
        # a question lies near some chunk
        at = torch.randint(0, n, (case["queries"],), generator=g, device="cuda")
        if cols > 1:
            at += n * torch.arange(cols, device="cuda")
        queries = _unit(rows[at] + torch.randn((case["queries"], d), generator=g, device="cuda") * (0.7 / math.sqrt(d)))
        state = {"case": case, "queries": queries}
        if own:
            ch = _framework()
            state["cols"] = []
            for k in range(cols):
                col = ch.GpuCollection(d, "fp4", case["metric"])
                col.add_device(rows[k * n:(k + 1) * n], path_class=cls[k * n:(k + 1) * n])
                col.finalize()
                state["cols"].append(col)
        else:
            state["codes"], state["exps"] = _quantize(rows)
            state["cls"] = cls
        return state
    case = dict(case, scale=1.0 if case["normalize"] else 0.25)
    b, d, v = case["bags"], case["dim"], case["vocab"]
    dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    # lengths of texts scatter around the mean; a long run of them holds some empty ones
    lens = torch.exp(0.4 * torch.randn((b,), generator=g, device="cuda", dtype=torch.float64))
    if b >= 64:
        lens[torch.randint(0, b, (b // 64,), generator=g, device="cuda")] = 0
    t = b * case["mean_len"]
    offsets = torch.zeros((b + 1,), dtype=torch.int64, device="cuda")
    offsets[1:] = (lens.cumsum(0) / lens.sum() * t).round().long()
    offsets[b] = t
    # tokens with p_i ~ 1 / i, spread over the table as hashed n-grams are
    u = torch.rand((t,), generator=g, device="cuda", dtype=torch.float64)
    rank = torch.exp(u * math.log(v + 1)).long().sub_(1).clamp_(0, v - 1)
    ids = ((rank * 7919 + seed) % v).int()
    # frequent tokens weigh less; hashed ones carry a sign
    weights = torch.where(torch.rand((t,), generator=g, device="cuda") < 0.5, -1.0, 1.0) / (1.0 + 4.0 / (1.0 + rank.float()))
    table = torch.randn((v, d), generator=g, device="cuda").to(dt)
    state = {"case": case, "table": table, "ids": ids, "weights": weights, "offsets": offsets}
    if case["op"] == "train":
        state["table"].requires_grad_(True)
        state["weights"].requires_grad_(True)
        state["grad"] = torch.randn((b, d), generator=g, device="cuda") / math.sqrt(d)
    return state


def run(state):
    case = state["case"]
    if own:
        ch = _framework()
        if case["op"] == "search":
            return state["cols"][0].search_device(state["queries"], top_k=case["top_k"])
        if case["op"] == "multi":
            return ch.search_multi_device(state["cols"], state["queries"], top_k=case["top_k"])
        how = {"mode": case["mode"], "scale": case["scale"], "normalize": case["normalize"]}
        if case["op"] == "embed":
            return ch.embed_bags(state["table"], state["ids"], state["offsets"], state["weights"], out_dtype=state["table"].dtype, **how)
        y = ch.embed_bags(state["table"], state["ids"], state["offsets"], state["weights"], **how)
        return (y.detach(),) + torch.autograd.grad(y, (state["table"], state["weights"]), state["grad"])
    if case["op"] in ("search", "multi"):
        rows = _dequantize(state["codes"], state["exps"], torch.float32)
        q = torch.nn.functional.pad(state["queries"], (0, rows.shape[-1] - case["dim"]))
        if case["op"] == "multi":
            return _nearest_plain(rows.view(case["queries"], case["rows"], -1), q.unsqueeze(1), state["cls"].view(case["queries"], -1), case)
        return _nearest_plain(rows, q, state["cls"], case)
    with torch.no_grad():
        if case["op"] == "embed":
            return _embed_plain(case, state["table"], state["ids"], state["weights"], state["offsets"])[0].to(state["table"].dtype)
        y, d_table, d_weights = _train_plain(case, state["table"], state["ids"], state["weights"], state["offsets"], state["grad"])
        return y.float(), d_table.to(state["table"].dtype), d_weights


# ---- the definitions in float64 -------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    if case["op"] in ("search", "multi"):
        return _exact_search(case, s)
    return _exact_lookup(s)


def _exact_search(case, s):
    d, k, n = case["dim"], case["top_k"], case["rows"]
    step = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    out = {"ids": [], "score": [], "dist": [], "count": []}
    factor = {0: 1.0, 1: 0.1, 2: 1.2}

    def values(lo, hi):
        packed = s["codes"][lo:hi].long()
        x = torch.empty((hi - lo, packed.shape[1] * 2), dtype=torch.float64, device="cuda")
        for half, code in ((0, packed % 16), (1, packed // 16)):
            x[:, half::2] = step[code % 8] * (1 - 2 * (code // 8).double())
        scale = torch.pow(2.0, s["exps"][lo:hi].double()).repeat_interleave(GROUP, dim=1)
        return (x * scale)[:, :d]

    queries = s["queries"].double()
    for first in range(0, len(queries), 64 if case["op"] == "search" else 1):
        q = queries[first:first + (64 if case["op"] == "search" else 1)]
        base = first * n if case["op"] == "multi" else 0
        kept_d, kept_i = None, None
        for lo in range(0, n, 500000):
            hi = min(n, lo + 500000)
            x = values(base + lo, base + hi)
            if case["metric"] == "l2":   # |x|^2 - 2 <x, q> + |q|^2 loses at most a few 1e-16 of values near 1
                dist = x.square().sum(1).unsqueeze(0) - 2 * (q @ x.T) + q.square().sum(1, keepdim=True)
            else:
                dist = 1 - q @ x.T
            near, at = dist.topk(min(hi - lo, 2 * k + 64), dim=1, largest=False)
            kept_d = near if kept_d is None else torch.cat((kept_d, near), 1)
            kept_i = at + lo if kept_i is None else torch.cat((kept_i, at + lo), 1)
        for row in range(len(q)):
            pairs = sorted(zip(kept_d[row].float().tolist(), kept_i[row].tolist()))[:2 * k]
            cls = s["cls"][base + torch.tensor([i for _, i in pairs], device="cuda")].tolist()
            scored = [(1.0 / (1.0 + dv) * factor[c], dv, i) for (dv, i), c in zip(pairs, cls)]
            best = sorted((x for x in scored if x[0] > 0.01), key=lambda x: -x[0])[:k]
            pad = k - len(best)
            out["score"].append([x[0] for x in best] + [0.0] * pad)
            out["dist"].append([x[1] for x in best] + [math.inf] * pad)
            out["ids"].append([x[2] for x in best] + [-1] * pad)
            out["count"].append(len(best))
    as_tensor = lambda v, t: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    return (as_tensor(out["ids"], torch.int64), as_tensor(out["score"], torch.float64), as_tensor(out["dist"], torch.float64),
            as_tensor(out["count"], torch.int32))


def _exact_lookup(s):
    """by sorted tokens and running sums' differences nowhere: plain products with selection matrices, a slice of columns at a time"""
    case = s["case"]
    t, b, v, d = s["ids"].numel(), case["bags"], case["vocab"], case["dim"]
    ids, w = s["ids"].long(), s["weights"].detach().double()
    starts = s["offsets"].tolist()
    table = s["table"].detach()
    lens = torch.tensor([e - a for a, e in zip(starts, starts[1:])], device="cuda")
    bag = torch.arange(b, device="cuda").repeat_interleave(lens)
    pick = torch.sparse_coo_tensor(torch.stack((bag, torch.arange(t, device="cuda"))), w, (b, t)).coalesce()
    p = torch.empty((b, d), dtype=torch.float64, device="cuda")
    for c in range(0, d, 64):
        p[:, c:c + 64] = torch.sparse.mm(pick, table[:, c:c + 64].double()[ids])
    count = lens.clamp(min=1).double().unsqueeze(1)
    factor = case["scale"] / {"sum": torch.ones_like(count), "mean": count, "sqrt": count.sqrt()}[case["mode"]]
    p *= factor
    length = p.norm(dim=1, keepdim=True)
    y = torch.where(length > 0, p / length.clamp(min=1e-300), torch.zeros_like(p)) if case["normalize"] else p
    if case["op"] == "embed":
        return y
    g = s["grad"].double()
    if case["normalize"]:
        g = torch.where(length > 0, (g - (g * y).sum(1, keepdim=True) * y) / length.clamp(min=1e-300), torch.zeros_like(g))
    g = g * factor
    put = torch.sparse_coo_tensor(torch.stack((ids, torch.arange(t, device="cuda"))), w, (v, t)).coalesce()
    d_table = torch.empty((v, d), dtype=torch.float64, device="cuda")
    d_weights = torch.zeros((t,), dtype=torch.float64, device="cuda")
    for c in range(0, d, 64):
        part = g[:, c:c + 64][bag]
        d_table[:, c:c + 64] = torch.sparse.mm(put, part)
        d_weights += (part * table[:, c:c + 64].double()[ids]).sum(1)
    return y, d_table, d_weights
