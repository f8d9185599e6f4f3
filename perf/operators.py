"""The work on which vfsx's probability and 8-bit score operators are measured.

Two operators over a resident store of n rows (a table of embeddings, or a model's output table):

  log_probs   log probabilities of given rows under softmax(sim(q, rows) / temperature + bias), the log of the sum, the
              entropy, and the k most probable rows
  scores      the product of queries and rows, both in 8-bit floating point (e4m3) with a power-of-two scale for each
              block of 128 elements

`own = False` computes them from elementary torch operations, `own = True` calls vfs_amd.  Rows come as f32 ("f32"), as
int8 with one scale ("i8"), or as f32 that is read through its 8-bit floating point copy ("f8").
"""
import math

import torch

own = False

I8_SCALE = 127.0  # what a quantizing store uses
BLOCK = 128       # elements that share one scale in the 8-bit floating point copy
E4M3_MAX = 448.0


def _lp(name, store, n, d, nq, given, k, sim, bias="none"):
    return {"name": name, "op": "log_probs", "store": store, "n": n, "d": d, "nq": nq, "given": given, "k": k, "sim": sim,
            "bias": bias, "temperature": _temperature(store, d, sim)}


def _sc(name, n, d, nq, sim, out):
    return {"name": name, "op": "scores", "store": "f8", "n": n, "d": d, "nq": nq, "sim": sim, "out": out}


def _temperature(store, d, sim):
    """Logits of rows that have nothing to do with the query get a spread of about 2 (queries have a spread of 2 an element)."""
    if sim == "cosine":
        return round(0.5 / math.sqrt(d), 5)
    return round(0.577 * math.sqrt(d), 4) if store == "i8" else 1.0


def listed():
    return [
        # a small store behind the HTTP server, one query with its five best rows: latency alone counts
        _lp("lp sample store", "f32", 2153, 16, 1, 1, 5, "cosine"),
        # one query against 100k short rows
        _lp("lp one 100k x 128", "f32", 100_000, 128, 1, 1, 10, "dot"),
        # one query of the default benchmark's store: bound by reading it
        _lp("lp one 1M x 768", "f32", 1_000_000, 768, 1, 1, 10, "cosine"),
        # one query of the benchmark's large int8 store
        _lp("lp one i8 10M x 128", "i8", 10_000_000, 128, 1, 1, 10, "dot"),
        # sizes that fill no tile, a few queries with several given rows and a mask
        _lp("lp ragged, masked", "f32", 32_749, 777, 37, 4, 20, "dot", "some"),
        # a batch as large as the batch benchmark's (4096 queries): the log probability of one row for each
        _lp("lp batch 4096", "f32", 100_000, 768, 4096, 1, 10, "dot"),
        # an int8 store and a batch of the server's size
        _lp("lp i8 batch 64", "i8", 100_000, 128, 64, 1, 10, "cosine"),
        # one query through the 8-bit floating point copy: a quarter of the bytes
        _lp("lp one f8 1M x 768", "f8", 1_000_000, 768, 1, 1, 10, "dot"),
        # a batch through that copy
        _lp("lp f8 batch 512", "f8", 200_000, 1024, 512, 1, 10, "cosine"),
        # every score of one query
        _sc("sc one 100k x 128", 100_000, 128, 1, "dot", "f32"),
        # sizes that fill no tile
        _sc("sc ragged", 32_749, 777, 37, "cosine", "f32"),
        # a large product with 16-bit results
        _sc("sc batch 4096", 131_072, 1024, 4096, "dot", "bf16"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        n, d, nq = log_int(1, 400_000), log_int(8, 2048), log_int(1, 4096)
        if n * d <= 1 << 28 and n * nq <= 400_000_000 and n * d * nq <= 300_000_000_000:
            break
    sim = rng.choice(("dot", "cosine"))
    if rng.random() < 0.3:
        c = _sc("", n, d, nq, sim, rng.choice(("f32", "bf16")))
    else:
        c = _lp("", rng.choice(("f32", "i8", "f8")), n, d, nq, rng.choice((0, 1, 1, 2, 7)),
                rng.choice((0, 1, 5, 10, 20, 64)), sim, rng.choice(("none", "none", "some", "some", "lowest")))
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _inputs(case, seed):
    """rows (f32, or int8 for an int8 store), queries, given rows and bias, on the GPU.  Half of the queries are near a
    stored row (the first given one): its logit reaches up to about log n, where its probability becomes noticeable."""
    g = torch.Generator("cuda").manual_seed(seed)
    n, d, nq = case["n"], case["d"], case["nq"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", generator=g)

    if case["store"] == "i8":
        rows = torch.randint(-127, 128, (n, d), device="cuda", generator=g, dtype=torch.int8)
    else:
        rows = normal(n, d).mul_(1.0 / math.sqrt(d)).mul_(torch.exp(0.3 * normal(n, 1)))
    twice = n // 50  # a store holds some rows more than once
    if twice:
        rows[n - twice:] = rows[whole(0, n - twice, twice)]
    near = whole(0, n, nq)
    x = rows[near].float()
    pull = torch.rand(nq, 1, device="cuda", generator=g) * math.log(n + 1.0)
    pull[1::2] = 0.0
    q = 2.0 * normal(nq, d) + pull * x / x.norm(dim=1, keepdim=True).clamp_min(1e-6)
    got = {"rows": rows, "q": q.contiguous()}
    if case["op"] == "log_probs":
        given = whole(0, n, nq, case["given"])
        if case["given"]:
            given[:, 0] = near
        if case["given"] > 2:
            given[::3, 2] = -1  # a place that is not filled
        got["given"] = given
        got["bias"] = None
        if case["bias"] != "none":
            out = torch.rand(n, device="cuda", generator=g) < 0.1
            bias = 0.5 * normal(n)
            low = torch.finfo(torch.float32).min if case["bias"] == "lowest" else -math.inf
            got["bias"] = torch.where(out, low, bias)
    return got


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    n, d, nq = case["n"], case["d"], case["nq"]
    if own:
        import vfs_amd

        rows = s.pop("rows")
        c = vfs_amd.Corpus(d, quantize=case["store"] == "i8", capacity_rows=n)
        c.append(rows.cpu().numpy())
        if case["store"] == "f8":
            c.enable_f8()
        s["corpus"] = c
        if case["op"] == "log_probs":
            k, given = case["k"], case["given"]
            c.reserve_log_probs(nq, source=_source(case))
            s["lp"] = torch.empty(nq, given, device="cuda")
            s["lse"] = torch.empty(nq, device="cuda")
            s["entropy"] = torch.empty(nq, device="cuda")
            s["top"] = torch.empty(nq, k, 24, device="cuda", dtype=torch.uint8)
            s["out"] = {"lp": s["lp"], "lse": s["lse"], "entropy": s["entropy"], "top_row": s["top"].view(torch.int64)[..., 1],
                        "top_lp": s["top"].view(torch.float32)[..., 0]}
        else:
            c.reserve_scores_f8(nq)
            s["out"] = torch.empty(nq, n, device="cuda", dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16)
        return s
    if case["sim"] == "cosine":  # a store keeps the norms of its rows
        s["norm"] = _norms(s["rows"])
    if case["store"] == "f8":
        s["rows8"], s["exp"] = _quantize(s.pop("rows"))
    return s


def _norms(rows):
    return torch.cat([r.double().norm(dim=1) for r in rows.split(1 << 18)])


def _source(case):
    return "f8" if case["store"] == "f8" else "rows"


# ---- one pass ---------------------------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if own:
        return _own_log_probs(s, case) if case["op"] == "log_probs" else _own_scores(s, case)
    return _plain_log_probs(s, case) if case["op"] == "log_probs" else _plain_scores(s, case)


def _own_log_probs(s, case):
    s["corpus"].log_probs_device(
        s["q"].data_ptr(), case["nq"], d_rows=s["given"].data_ptr() if case["given"] else 0, given=case["given"], k=case["k"],
        similarity=case["sim"], temperature=case["temperature"], d_bias=0 if s["bias"] is None else s["bias"].data_ptr(),
        source=_source(case), d_log_probs=s["lp"].data_ptr() if case["given"] else 0, d_lse=s["lse"].data_ptr(),
        d_entropy=s["entropy"].data_ptr(), d_top=s["top"].data_ptr() if case["k"] else 0,
        stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_scores(s, case):
    s["corpus"].scores_f8_device(s["q"].data_ptr(), case["nq"], s["out"].data_ptr(), dtype=case["out"], similarity=case["sim"],
                                 stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _quantize(x):
    """e4m3 values and one exponent for each block of 128 elements: the least with max|x| <= 448 * 2^e."""
    blocks = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
    top = blocks.abs().amax(-1)
    f, e = torch.frexp(top)  # top = f * 2^e with f in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(top > 0, (e - 9 + (f > 0.875)).clamp(-127, 127), 0)
    return torch.ldexp(blocks, -e.unsqueeze(-1)).to(torch.float8_e4m3fn), e


def _values(x8, e):
    return torch.ldexp(x8.float(), e.unsqueeze(-1)).flatten(1)  # (padded with zeros to whole blocks)


def _plain_operands(s, case):
    """Queries and rows as f32 matrices whose product the scores are."""
    q = s["q"]
    if case["store"] == "f8":
        return _values(*_quantize(q)), _values(s["rows8"], s["exp"])
    return q, s["rows"].float()


def _plain_scores(s, case):
    q, x = _plain_operands(s, case)
    y = q @ x.T
    if case["sim"] == "cosine":
        y = y / (s["q"].norm(dim=1, keepdim=True) * s["norm"].float())
    return y.to(torch.float32 if case["out"] == "f32" else torch.bfloat16)


def _plain_log_probs(s, case):
    k, t = case["k"], case["temperature"]
    q, x = _plain_operands(s, case)
    logit = q @ x.T
    if case["sim"] == "cosine":
        logit = logit / (s["q"].norm(dim=1, keepdim=True) * (s["norm"].float() * t))
    else:
        logit = logit / (t * I8_SCALE if case["store"] == "i8" else t)
    if s["bias"] is not None:
        logit = logit + s["bias"]
    high = logit.amax(1, keepdim=True)
    high = torch.where(high == -math.inf, 0.0, high)
    rel = logit - high
    w = torch.exp(rel)
    total = w.sum(1)
    lse = high[:, 0] + torch.log(total)
    entropy = torch.where(total > 0, torch.log(total) - torch.where(w > 0, w * rel, 0.0).sum(1) / total, 0.0)
    out = {"lse": lse, "entropy": entropy}
    given = s["given"]
    inside = (given >= 0) & (given < case["n"])
    lp = logit.gather(1, given.clamp(0, case["n"] - 1))
    out["lp"] = torch.where(inside & (lp > -math.inf), lp - lse[:, None], -math.inf)
    out["top_row"], out["top_lp"] = _plain_top(s, case, q, x, logit, lse, k)
    return out


def _plain_top(s, case, q, x, logit, lse, k):
    """The k largest logits, ties to the lowest row.  Logits that are near one another are computed in 64 bits to be ordered."""
    nq, n = logit.shape
    rows = torch.full((nq, k), -1, device=logit.device, dtype=torch.int64)
    lps = torch.full((nq, k), -math.inf, device=logit.device)
    if k == 0:
        return rows, lps
    kth = torch.topk(logit, min(k, n), dim=1).values[:, -1:]
    kth = torch.where(kth == -math.inf, torch.finfo(torch.float32).min, kth)
    margin = 2e-5 * (1.0 + kth.abs().clamp_max(1e4))
    at_q, at_row = torch.nonzero(logit >= kth - margin, as_tuple=True)
    exact = torch.cat([_dot64(q, x, a, b) for a, b in zip(at_q.split(1 << 16), at_row.split(1 << 16))]) if len(at_q) else at_q.double()
    if case["sim"] == "cosine":
        exact = exact / (s["q"].double().norm(dim=1)[at_q] * s["norm"][at_row] * case["temperature"])
    else:
        exact = exact / (case["temperature"] * (I8_SCALE if case["store"] == "i8" else 1.0))
    if s["bias"] is not None:
        exact = exact + s["bias"].double()[at_row]
    order = torch.sort(exact, stable=True, descending=True).indices
    order = order[torch.sort(at_q[order], stable=True).indices]
    at_q, at_row, exact = at_q[order], at_row[order], exact[order]
    place = torch.arange(len(at_q), device=at_q.device) - torch.searchsorted(at_q, at_q)
    keep = place < k
    at_q, at_row, exact, place = at_q[keep], at_row[keep], exact[keep], place[keep]
    rows[at_q, place] = at_row
    lps[at_q, place] = (exact - lse.double()[at_q]).float()
    return rows, lps


def _dot64(q, x, at_q, at_row):
    return (q[at_q].double() * x[at_row].double()).sum(1)


# ---- the cost, and the definition in 64 bits ------------------------------------------------------------------------------


def work(case):
    n, d, nq = case["n"], case["d"], case["nq"]
    element = {"f32": 4.0, "i8": 1.0, "f8": 1.0 + 1.0 / BLOCK}[case["store"]]
    moved = n * d * element + 4 * nq * d
    if case["op"] == "scores":
        moved += nq * n * (4 if case["out"] == "f32" else 2)
    else:
        moved += (4 * n if case["bias"] != "none" else 0) + nq * (12 * case["given"] + 8 + 24 * case["k"])
    return {"bytes": moved, "flops": 2.0 * n * d * nq}


def _e4m3_grid(x):
    """The values that an 8-bit copy of x (f64) stands for, by the definition: to nearest, ties to even, three bits after the
    leading one and steps of 2^-9 at least, under a scale for each block of 128."""
    b = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)).clamp(-127, 127))
    unit = torch.where(top > E4M3_MAX * unit, 2 * unit, unit)
    unit = torch.where(top <= E4M3_MAX * unit / 2, unit / 2, unit)
    unit = torch.where(top > 0, unit, 1.0)
    v = b / unit
    step = torch.exp2((torch.frexp(v).exponent - 4).clamp_min(-9).double())
    return (torch.round(v / step) * step * unit).flatten(1)[:, :x.shape[1]]


def exact(case, seed):
    a = _inputs(case, seed)
    n, nq = case["n"], case["nq"]
    q = a["q"].double()
    q_norm = q.square().sum(1).sqrt()
    if case["store"] == "f8":
        q = _e4m3_grid(q)
    per = max(1, (1 << 28) // case["d"])

    def part(at, scale):
        """Rows [at, at + per) as they are stored, in 64 bits, and what their product with a query is divided by."""
        x = a["rows"][at:at + per].double()
        by = x.square().sum(1).sqrt() if case["sim"] == "cosine" else torch.full((len(x),), I8_SCALE if case["store"] == "i8" else 1.0,
                                                                                 device="cuda", dtype=torch.float64)
        return (_e4m3_grid(x) if case["store"] == "f8" else x), by * scale

    if case["op"] == "scores":
        out = torch.empty(nq, n, device="cuda", dtype=torch.float64)
        for at in range(0, n, per):
            x, by = part(at, 1.0)
            out[:, at:at + per] = (q @ x.T) / by
        return out / q_norm[:, None] if case["sim"] == "cosine" else out

    k, given = case["k"], a["given"]
    got = {"lp": torch.full(given.shape, -math.inf, device="cuda", dtype=torch.float64),
           "lse": torch.empty(nq, device="cuda", dtype=torch.float64), "entropy": torch.empty(nq, device="cuda", dtype=torch.float64),
           "top_row": torch.full((nq, k), -1, device="cuda", dtype=torch.int64),
           "top_lp": torch.full((nq, k), -math.inf, device="cuda", dtype=torch.float64)}
    few = max(1, (1 << 27) // n)
    for first in range(0, nq, few):
        sl = slice(first, min(nq, first + few))
        z = torch.empty(sl.stop - first, n, device="cuda", dtype=torch.float64)
        for at in range(0, n, per):
            x, by = part(at, case["temperature"])
            z[:, at:at + per] = (q[sl] @ x.T) / by
        if case["sim"] == "cosine":
            z /= q_norm[sl, None]
        if a["bias"] is not None:
            z += a["bias"].double()
        lse = torch.logsumexp(z, 1)
        logp = z - torch.where(lse == -math.inf, 0.0, lse)[:, None]
        got["lse"][sl] = lse
        got["entropy"][sl] = -torch.special.xlogy(logp.exp(), logp.exp()).sum(1)
        at = given[sl]
        inside = (at >= 0) & (at < n)
        got["lp"][sl] = torch.where(inside, logp.gather(1, at.clamp(0, n - 1)), -math.inf)
        if k:
            # equal rows are to have equal logits, whatever place of the product they came from: 2^-40 of a logit is no difference
            m = min(n, k + 200)
            v, r = torch.topk(logp, m, dim=1)
            v = torch.where(v == -math.inf, v, torch.round(v * 2.0**36) / 2.0**36)
            o = torch.sort(r, dim=1).indices
            v, r = v.gather(1, o), r.gather(1, o)
            o = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]
            v, r = v.gather(1, o), r.gather(1, o)
            got["top_lp"][sl, :min(n, k)] = v
            got["top_row"][sl, :min(n, k)] = torch.where(v > -math.inf, r, -1)
    return got
