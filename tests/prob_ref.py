"""64-bit definitions of the operators over a store that tests/test_gpu_prob.py and tests/test_gpu_f8.py compare with."""
import numpy as np


def e4m3_values(x):
    """What the 8-bit floating point copy of x ([n, d] f32) stands for, in f64: blocks of 128 share the least scale
    2^e, e >= -127, with max|x| <= 448 * 2^e; values to nearest even with three bits after the leading one, in
    steps of 2^-9 at least.  Blocks with a NaN or an infinity are NaN."""
    x = np.asarray(x, np.float64)
    n, d = x.shape
    out = np.empty((n, d))
    for at in range(0, d, 128):
        b = x[:, at:at + 128]
        with np.errstate(invalid="ignore"):
            top = np.abs(b).max(axis=1)
        bad = ~np.isfinite(b).all(axis=1)
        top = np.where(bad, 0.0, top)
        m, e = np.frexp(np.where(top > 0, top, 1.0))  # top = m 2^e, m in [0.5, 1);  448 = 0.875 * 2^9
        e = np.maximum(e - 9 + (m > 0.875), -127)
        e = np.where(top > 0, e, 0)
        v = np.ldexp(np.where(bad[:, None], 0.0, b), -e[:, None])
        step = np.ldexp(1.0, np.maximum(np.frexp(v)[1] - 4, -9))
        q = np.rint(v / step) * step
        out[:, at:at + 128] = np.where(bad[:, None], np.nan, np.ldexp(q, e[:, None]))
    return out


def there(rows, q, bias, cosine):
    """[nq, n]: which rows take part."""
    n, nq = len(rows), len(q)
    ok = np.ones((nq, n), bool)
    if bias is not None:
        ok &= ~np.isneginf(bias)[None, :]
    if cosine:
        with np.errstate(over="ignore", under="ignore", invalid="ignore"):
            ok &= ((rows.astype(np.float64) ** 2).sum(1).astype(np.float32) != 0)[None, :]
            ok &= ((q.astype(np.float64) ** 2).sum(1).astype(np.float32) != 0)[:, None]
    return ok


def logits(rows, q, *, cosine=False, temperature=1.0, bias=None, f8=False, scale=None):
    """[nq, n] f64; rows f32, or int8 with `scale`.  Rows that take no part are -inf."""
    x = rows.astype(np.float64) if scale is None else rows.astype(np.float64) / scale
    qd = q.astype(np.float64)
    a, b = (e4m3_values(q), e4m3_values(rows)) if f8 else (qd, x)
    with np.errstate(all="ignore"):
        l = a @ b.T
        if cosine:
            l = l / (np.linalg.norm(qd, axis=1)[:, None] * np.linalg.norm(x, axis=1)[None, :])
        l = l / temperature
        if bias is not None:
            l = l + bias.astype(np.float64)[None, :]
    return np.where(there(rows, q, bias, cosine), l, -np.inf)


def softmax_of(l, rows=None, k=0):
    """lse, entropy, log probabilities of `rows` [nq, t] (local, outside -> -inf), top rows and their log probabilities,
    and how many there are."""
    nq, n = l.shape
    m = l.max(axis=1, initial=-np.inf)
    with np.errstate(all="ignore"):
        z = l - np.where(np.isneginf(m), 0, m)[:, None]
        s = np.exp(z).sum(1)
        lse = np.where(np.isneginf(m), 0, m) + np.log(s)
        lp = l - np.where(np.isneginf(lse), 0, lse)[:, None]
        entropy = -np.where(np.isneginf(lp), 0, np.exp(lp) * lp).sum(1)
    out = {"lse": lse, "entropy": entropy}
    if rows is not None:
        r = np.asarray(rows, np.int64)
        inside = (r >= 0) & (r < n)
        got = np.full(r.shape, -np.inf)
        if n:
            got = np.where(inside, np.take_along_axis(lp, np.clip(r, 0, n - 1), axis=1), -np.inf)
        out["log_probs"] = got
    if k:
        # equal rows have to have equal logits here: 2^-36 is no difference
        order = np.argsort(-np.where(np.isneginf(l), -np.inf, np.rint(l * 2.0**36)), axis=1, kind="stable")[:, :k]
        top_l = np.take_along_axis(l, order, axis=1)
        out["top_rows"] = np.where(np.isneginf(top_l), -1, order)
        out["top_log_probs"] = np.take_along_axis(lp, order, axis=1)
        out["top_count"] = (~np.isneginf(top_l)).sum(1)
    return out


def logit_bound(rows, q, *, cosine=False, temperature=1.0, bias=None, scale=None, f8=False):
    """[nq]: how far an f32-grade logit may be from its value.  A product of d terms from operands that are exact to 2^-22,
    accumulated in f32 in any order, is within (d + 64) 2^-24 |q||x|; three more roundings of the logit itself."""
    x = rows.astype(np.float64) / (1.0 if scale is None else scale)
    d = rows.shape[1]
    qn = np.linalg.norm(q.astype(np.float64), axis=1)
    xn = np.linalg.norm(x, axis=1).max(initial=0.0)
    part = np.ones(len(q)) if cosine else qn * xn
    e = (d + 64) * 2.0**-24 * part / temperature * (1.25 if f8 else 1.0)
    top = part / temperature
    if bias is not None:
        b = np.abs(bias[np.isfinite(bias) & (np.abs(bias) < 1e30)])
        top = top + (b.max() if b.size else 0.0)
    return e + 3 * 2.0**-24 * top


def compare(got, want, l, bound):
    """got: a vfs_amd.LogProbs.  The sums: 128 f32 terms and f64 beyond (128 * 2^-24), exponentials good to 2^-20."""
    sums = 2.0**-17 + 2.0**-20
    tol = bound + sums
    for name in ("lse",):
        g, w = getattr(got, name).astype(np.float64), want[name]
        fin = np.isfinite(w)
        assert np.array_equal(g[~fin], w[~fin]), (name, g[~fin], w[~fin])
        err = np.abs(np.where(fin, g, 0) - np.where(fin, w, 0)) - (tol + 2.0**-24 * np.abs(np.where(fin, w, 0)))
        assert (err <= 0).all(), (name, err.max())
    h = want["entropy"]
    err = np.abs(got.entropy - h) - (2 * h * bound + 2 * sums * (1 + h))
    assert (err <= 0).all(), ("entropy", err.max(), got.entropy, h)
    for name in ("log_probs", "top_log_probs"):
        if name not in want:
            continue
        g, w = getattr(got, name).astype(np.float64), want[name]
        if name == "top_log_probs":  # places that are not filled
            pad = g.shape[1] - w.shape[1]
            assert np.isneginf(g[:, w.shape[1]:]).all() and pad >= 0
            g = g[:, :w.shape[1]]
        fin = np.isfinite(w)
        assert np.array_equal(g[~fin], w[~fin]), name
        err = np.abs(np.where(fin, g, 0) - np.where(fin, w, 0)) - (tol[:, None] + 2.0**-24 * np.abs(np.where(fin, w, 0)))
        assert (err <= 0).all(), (name, err.max())
    if "top_rows" in want:
        w = want["top_rows"]
        assert np.array_equal(got.top_rows.astype(np.int64)[:, :w.shape[1]], w), (got.top_rows.astype(np.int64)[:, :w.shape[1]], w)
        assert (got.top_rows[:, w.shape[1]:] == np.uint64(2**64 - 1)).all()
        assert np.array_equal(got.top_count, want["top_count"])


def refused(call):
    """The code of the VfsxError that call() raises, or None.  The exception is not kept: its traceback would keep the caller's stores and
    graphs until a garbage collection, wherever that comes."""
    import vfs_amd
    try:
        call()
    except vfs_amd.VfsxError as e:
        return e.code
    return None


def no_collection():
    """For tests that capture graphs: garbage of earlier tests goes first, and none is collected in between.  (A graph that is destroyed
    inside a capture synchronizes the device, which the capture forbids: torch's destructor then ends the process.)"""
    import gc
    gc.collect()
    gc.disable()
    yield
    gc.enable()
