"""GPU: log probabilities, entropy and most probable rows over a store, against their definition in 64 bits."""
import numpy as np
import pytest

import vfs_amd
from vfs_amd import _lib
from tests import prob_ref as ref

pytestmark = pytest.mark.gpu
no_collection = pytest.fixture(ref.no_collection)


def make(store, n, d, rng, spread=1.0):
    if store == "i8":
        return rng.integers(-128, 128, (n, d)).astype(np.int8)
    x = rng.standard_normal((n, d)) * spread / np.sqrt(d) * np.exp(0.3 * rng.standard_normal((n, 1)))
    return x.astype(np.float32)


def corpus_of(store, rows, **kw):
    c = vfs_amd.Corpus(rows.shape[1], quantize=store == "i8", **kw)
    if len(rows):
        c.append(rows)
    if store == "f8":
        c.enable_f8()
    return c


def check(c, store, rows, q, *, given=None, k=0, cosine=False, temperature=1.0, bias=None):
    kw = dict(cosine=cosine, temperature=temperature, bias=bias, scale=127.0 if store == "i8" else None, f8=store == "f8")
    l = ref.logits(rows, q, **kw)
    got = c.log_probs(q, given, k, similarity="cosine" if cosine else "dot", temperature=temperature, bias=bias,
                      source="f8" if store == "f8" else "rows")
    ref.compare(got, ref.softmax_of(l, given, k), l, ref.logit_bound(rows, q, **kw))
    return got


def masked(n, rng, kind):
    if kind == "none":
        return None
    b = (0.5 * rng.standard_normal(n)).astype(np.float32)
    b[rng.random(n) < 0.2] = -np.inf if kind == "some" else np.finfo(np.float32).min
    if kind == "all":
        b[:] = -np.inf
    return b


SIZES = [  # n, d, nq, given, k
    (1, 1, 1, 1, 1), (2, 3, 3, 2, 5), (15, 4, 1, 0, 1), (16, 5, 2, 1, 16), (17, 8, 5, 1, 3), (63, 16, 1, 1, 64), (64, 33, 4, 3, 10),
    (65, 12, 33, 1, 128), (127, 100, 2, 1, 7), (128, 128, 9, 2, 10), (129, 129, 17, 1, 10), (255, 40, 64, 1, 1), (257, 260, 65, 2, 20),
    (1000, 31, 3, 5, 128), (2153, 16, 1, 1, 5), (5003, 200, 8, 1, 10), (5003, 200, 130, 0, 10), (4096, 64, 300, 1, 0), (20011, 72, 31, 1, 33),
    (3001, 777, 5, 7, 20), (70000, 20, 2, 1, 10), (1500, 2050, 40, 1, 10),
]


@pytest.mark.parametrize("store", ["f32", "i8", "f8"])
@pytest.mark.parametrize("cosine", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_against_definition(store, cosine, size):
    n, d, nq, t, k = size
    rng = np.random.default_rng(n * 7 + d)
    rows = make(store, n, d, rng)
    if n > 40:
        rows[-n // 20:] = rows[:n // 20 + (n % 20 > 0)][:len(rows[-n // 20:])]  # some rows twice: ties go to the lowest
    q = (2.0 * rng.standard_normal((nq, d))).astype(np.float32)
    near = rng.integers(0, n, nq)
    q[::2] += (3.0 * rows[near] / np.maximum(np.linalg.norm(rows[near].astype(np.float64), axis=1, keepdims=True), 1e-6)).astype(np.float32)[::2]
    given = rng.integers(-1, n + 2, (nq, t))
    if t:
        given[:, 0] = near
    temperature = 0.5 / np.sqrt(d) if cosine else (0.577 * np.sqrt(d) if store == "i8" else 1.0)
    bias = masked(n, rng, ("none", "some", "lowest")[(n + d) % 3])
    check(corpus_of(store, rows), store, rows, q, given=given, k=k, cosine=cosine, temperature=temperature, bias=bias)


LARGE = [  # n, d, nq: enough tiles for the large workgroups, more than one for some of them; queries too long for the first pass of a few
    (9001, 777, 513), (30011, 72, 700), (16384, 128, 257), (66000, 130, 33), (200003, 20, 64), (300, 2100, 8), (200, 20000, 1), (70, 40001, 3),
]


@pytest.mark.parametrize("store", ["f32", "i8", "f8"])
@pytest.mark.parametrize("size", LARGE, ids=lambda s: "x".join(map(str, s)))
def test_many_tiles_and_long_rows(store, size):
    n, d, nq = size
    rng = np.random.default_rng(n + d)
    rows = make(store, n, d, rng)
    q = (2.0 * rng.standard_normal((nq, d))).astype(np.float32)
    cosine = bool(nq % 2)
    temperature = 0.5 / np.sqrt(d) if cosine else (0.577 * np.sqrt(d) if store == "i8" else 1.0)
    check(corpus_of(store, rows), store, rows, q, given=rng.integers(0, n, (nq, 2)), k=7, cosine=cosine, temperature=temperature,
          bias=masked(n, rng, ("none", "some", "lowest")[d % 3]))


@pytest.mark.parametrize("store", ["f32", "i8", "f8"])
@pytest.mark.parametrize("nq", [1, 40])
def test_every_row_at_the_lowest_bias(store, nq):
    """Logits round to the lowest f32 alike: a uniform distribution, not an empty one."""
    rng = np.random.default_rng(21)
    rows, q = make(store, 300, 24, rng), rng.standard_normal((nq, 24)).astype(np.float32)
    b = np.full(300, np.finfo(np.float32).min)
    got = corpus_of(store, rows).log_probs(q, np.array([[5, -1, 299]] * nq), 3, bias=b, source="f8" if store == "f8" else "rows")
    assert (got.lse == b[0]).all()
    # (f32 sums of 64 equal terms and f64 beyond are exact; what is left is the rounding of a logarithm of 300, and of what is taken from it)
    assert np.abs(got.entropy - np.log(300)).max() <= 2.0**-17 + 2.0**-20
    assert np.isneginf(got.log_probs[:, 1]).all() and got.top_rows.shape == (nq, 3) and (got.top_rows >= 0).all()


@pytest.mark.parametrize("store", ["f32", "i8", "f8"])
def test_nothing_there(store):
    rng = np.random.default_rng(1)
    rows, q = make(store, 300, 24, rng), rng.standard_normal((3, 24)).astype(np.float32)
    c = corpus_of(store, rows)
    got = check(c, store, rows, q, given=np.zeros((3, 1), int), k=4, bias=masked(300, rng, "all"))
    assert np.isneginf(got.lse).all() and (got.entropy == 0).all() and np.isneginf(got.log_probs).all()
    assert (got.top_count == 0).all() and (got.top_ids == np.uint64(2**64 - 1)).all() and np.isneginf(got.top_log_probs).all()
    # one row left of all
    b = masked(300, rng, "all")
    b[211] = -3.0
    got = check(c, store, rows, q, given=np.full((3, 1), 211), k=4, bias=b)
    assert (got.top_rows[:, 0] == 211).all() and (got.top_count == 1).all() and (got.entropy == 0).all() and (got.log_probs == 0).all()
    empty = corpus_of(store, rows[:0])
    got = empty.log_probs(q, np.zeros((3, 2), int), 2, source="f8" if store == "f8" else "rows")
    assert np.isneginf(got.lse).all() and (got.entropy == 0).all() and np.isneginf(got.log_probs).all() and (got.top_count == 0).all()


def test_masked_rows_may_hold_anything():
    rng = np.random.default_rng(2)
    for store in ("f32", "f8"):
        rows, q = make(store, 700, 130, rng), rng.standard_normal((40, 130)).astype(np.float32)
        clean = rows.copy()
        rows[5, 3], rows[130, 129], rows[400] = np.nan, np.inf, -np.inf
        b = (0.1 * rng.standard_normal(700)).astype(np.float32)
        b[[5, 130, 400]] = -np.inf
        for nq in (1, 40):
            for cosine in (False, True):
                t = 0.05 if cosine else 1.0
                kw = dict(cosine=cosine, temperature=t, bias=b, f8=store == "f8")
                l = ref.logits(clean, q[:nq], **kw)
                got = corpus_of(store, rows).log_probs(q[:nq], np.array([[5, 130, 6]] * nq), 10, similarity="cosine" if cosine else "dot",
                                                       temperature=t, bias=b, source="f8" if store == "f8" else "rows")
                ref.compare(got, ref.softmax_of(l, np.array([[5, 130, 6]] * nq), 10), l, ref.logit_bound(clean, q[:nq], **kw))


@pytest.mark.parametrize("nq", [1, 5, 70])
@pytest.mark.parametrize("what", ["nan row", "inf row", "-inf row", "nan query", "inf query", "nan bias", "inf bias", "overflow"])
def test_a_logit_that_is_not_finite_spoils_its_queries(what, nq):
    rng = np.random.default_rng(3)
    n, d = 500, 36
    rows, q = make("f32", n, d, rng), rng.standard_normal((nq, d)).astype(np.float32)
    b = np.zeros(n, np.float32)
    bad = np.ones(nq, bool)
    if what == "nan row":
        rows[77, 35] = np.nan
    elif what.endswith("inf row"):
        rows[499, 0] = float(what.split()[0])
    elif what.endswith("query"):
        q[0, 7] = float(what.split()[0])
        bad = np.arange(nq) == 0
    elif what.endswith("bias"):
        b[3] = float(what.split()[0])
    else:
        rows[10], q[:] = 1e30, 1e30
    got = corpus_of("f32", rows).log_probs(q, np.array([1, 2]), 5, bias=b)
    for a in (got.lse, got.entropy, got.log_probs, got.top_log_probs):
        assert np.isnan(a[bad]).all() and np.isfinite(a[~bad]).all(), (what, a)
    assert (got.top_count[bad] == 0).all() and (got.top_count[~bad] == 5).all()


def test_rows_and_queries_without_a_cosine():
    rng = np.random.default_rng(4)
    for store in ("f32", "i8", "f8"):
        rows, q = make(store, 300, 20, rng), rng.standard_normal((6, 20)).astype(np.float32)
        rows[[0, 17, 299]] = 0
        if store != "i8":
            rows[18] = 1e-30  # its square is 0 in f32
        q[2] = 0
        got = check(corpus_of(store, rows), store, rows, q, given=np.array([[0, 17, 1, 299]] * 6), k=12, cosine=True, temperature=0.1)
        assert np.isneginf(got.lse[2]) and got.top_count[2] == 0 and np.isneginf(got.log_probs[:, [0, 1, 3]]).all()


def test_wide_ranges_of_values():
    """Rows and queries from 2^-40 to 2^40 in one store: every logit is good relative to its own row and query."""
    rng = np.random.default_rng(5)
    n, d, nq = 600, 96, 48
    rows = (make("f32", n, d, rng) * 2.0 ** rng.integers(-40, 40, (n, 1))).astype(np.float32)
    q = (rng.standard_normal((nq, d)) * 2.0 ** rng.integers(-40, 40, (nq, 1))).astype(np.float32)
    for m in (1, 3, nq):
        check(corpus_of("f32", rows), "f32", rows, q[:m], given=rng.integers(0, n, (m, 2)), k=10, cosine=True, temperature=0.05)
    rows = make("f32", n, d, rng)
    rows[:, :3] *= 1000.0  # a few large elements, many small ones
    check(corpus_of("f32", rows), "f32", rows, q[:, :] / np.linalg.norm(q, axis=1, keepdims=True) * 0.1, given=rng.integers(0, n, (nq, 2)), k=10)


@pytest.mark.parametrize("store", ["f32", "i8", "f8"])
@pytest.mark.parametrize("nq", [1, 40])
def test_one_vector_stored_very_often(store, nq):
    """More ties than the second pass keeps at once: the lowest rows, in order."""
    rng = np.random.default_rng(6)
    rows = np.repeat(make(store, 2, 24, rng), [3, 6000], axis=0)
    q = rng.standard_normal((nq, 24)).astype(np.float32)
    check(corpus_of(store, rows), store, rows, q, given=np.zeros((nq, 1), int), k=128, temperature=20.0 if store == "i8" else 1.0)
    rows[1000:] = rows[1000:] // 2 if store == "i8" else rows[1000:] * np.float32(0.5)
    check(corpus_of(store, rows), store, rows, q, given=np.zeros((nq, 1), int), k=20, temperature=20.0 if store == "i8" else 1.0)


def test_order_is_that_of_64_bits():
    """Logits that differ by less than an f32 step: the first pass cannot tell them apart."""
    rng = np.random.default_rng(7)
    d = 64
    base = rng.standard_normal(d).astype(np.float32)
    rows = np.tile(base, (900, 1))
    rows[:, 5] = np.nextafter(base[5], np.float32(9), dtype=np.float32)
    hit = rng.permutation(900)[:30]
    rows[hit, 5] = base[5] + np.arange(2, 32).astype(np.float32) * np.spacing(base[5])
    q = np.tile(rng.standard_normal(d).astype(np.float32), (40, 1))
    q[:, 5] = np.abs(q[:, 5])
    rest = np.setdiff1d(np.arange(900), hit)
    up = rows.copy()
    up[hit, 5] = base[5] + np.arange(2, 32).astype(np.float32) * np.abs(np.spacing(base[5]))
    for nq in (1, 40):
        # base[5] < 0, so its spacing is too: the others are the larger ones, all equal
        got = check(corpus_of("f32", rows), "f32", rows, q[:nq], given=np.zeros((nq, 1), int), k=30)
        assert base[5] < 0 and got.top_rows[0].tolist() == rest[:30].tolist()
        got = check(corpus_of("f32", up), "f32", up, q[:nq], given=np.zeros((nq, 1), int), k=30)
        assert got.top_rows[0].tolist() == hit[::-1].tolist()


def test_row_base_and_ids():
    rng = np.random.default_rng(8)
    rows, q = make("f32", 200, 16, rng), rng.standard_normal((4, 16)).astype(np.float32)
    c = vfs_amd.Corpus(16)
    c.append(rows, ids=np.arange(200) * 10 + 7)
    c.set_row_base(1 << 40)
    got = c.log_probs(q, np.array([[1 << 40, (1 << 40) + 199, 0, (1 << 40) + 200, -1]] * 4), 3)
    l = ref.logits(rows, q)
    want = ref.softmax_of(l, np.array([[0, 199, -1, -1, -1]] * 4), 3)
    assert np.allclose(got.log_probs, want["log_probs"], atol=1e-5)
    assert np.array_equal(got.top_rows.astype(np.int64) - (1 << 40), want["top_rows"])
    assert np.array_equal(got.top_ids.astype(np.int64), want["top_rows"] * 10 + 7)


@pytest.mark.parametrize("store", ["f32", "i8", "f8"])
def test_appended_rows_take_part(store):
    rng = np.random.default_rng(9)
    rows, q = make(store, 1000, 48, rng), rng.standard_normal((7, 48)).astype(np.float32)
    c = corpus_of(store, rows[:130])
    c.set_insert_batch(64)
    at = 130
    for more in (1, 3, 126, 500, 5, 235):
        check(c, store, rows[:at], q, given=np.full((7, 1), at - 1), k=9, temperature=25.0 if store == "i8" else 1.0)
        c.append(rows[at:at + more])
        at += more
    check(c, store, rows[:at], q, given=np.full((7, 1), at - 1), k=9, temperature=25.0 if store == "i8" else 1.0)


def test_searches_and_probabilities_on_one_store():
    """As the server uses them: the hits of a search are the most probable rows of the cosine softmax, and log p follows from the
    distance; the 8-bit scores are near the distances."""
    rng = np.random.default_rng(10)
    rows, q = make("f32", 3000, 96, rng), rng.standard_normal((5, 96)).astype(np.float32)
    c = corpus_of("f8", rows)
    ids, dist, _ = c.search_batch(q, 10, int(vfs_amd.DistanceMethod.Cosine))
    got = c.log_probs(q, ids.astype(np.int64) - 1, 10, similarity="cosine", temperature=0.05)
    assert np.array_equal(got.top_ids, ids)
    # cosine: both within 2^-18 of exact at d = 96; log p = (1 - dist) / T - lse
    assert np.abs(got.log_probs - ((1 - dist) / 0.05 - got.lse[:, None])).max() < 2 * 2.0**-18 / 0.05
    assert np.array_equal(got.log_probs, got.top_log_probs)
    s = c.scores_f8(q, "cosine")
    # e4m3 on both sides: at most (1 + 2^-4)^2 - 1 of sum |q||x| <= |q||x|
    assert np.abs(np.take_along_axis(s, ids.astype(np.int64) - 1, 1) - (1 - dist)).max() < (1 + 2.0**-4) ** 2 - 1
    ids2, dist2, _ = c.search_batch(q, 10, int(vfs_amd.DistanceMethod.Cosine))
    assert np.array_equal(ids, ids2) and np.array_equal(dist, dist2)


def test_refusals():
    rng = np.random.default_rng(11)
    rows, q = make("f32", 50, 8, rng), rng.standard_normal((2, 8)).astype(np.float32)
    c = corpus_of("f32", rows)
    for kw in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
               dict(temperature=1e-300), dict(k=129), dict(k=-1), dict(similarity="euclid"), dict(source="f8"), dict(source="x"),
               dict(bias=np.zeros(49, np.float32)), dict(rows=np.zeros((2, 1))), dict(rows=np.zeros((3, 1), int)), dict(rows=5)):
        assert ref.refused(lambda: c.log_probs(q, **kw)) == _lib.ERR_INVALID_VECTOR, kw
    with pytest.raises(vfs_amd.VfsxError):
        c.log_probs(q[:, :7])
    lib = c._lib
    f = np.zeros(64, np.float32)
    p = f.ctypes.data
    u = np.zeros(64, np.uint64).ctypes.data
    bad = _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_log_probs(c.handle, None, 2, 0, 1.0, 0, None, None, 0, 0, None, p, p, None) == bad       # no queries
    assert lib.vfsx_log_probs(c.handle, p, 2, 0, 1.0, 0, None, None, 1, 0, p, p, p, None) == bad             # no rows
    assert lib.vfsx_log_probs(c.handle, p, 2, 0, 1.0, 0, None, u, 1, 0, None, p, p, None) == bad             # nowhere to put them
    assert lib.vfsx_log_probs(c.handle, p, 2, 0, 1.0, 0, None, None, 0, 3, None, p, p, None) == bad          # no top
    assert lib.vfsx_log_probs(c.handle, p, 2, 0, 1.0, 0, None, None, 0, 0, None, None, None, None) == bad    # nothing asked for
    assert lib.vfsx_log_probs(c.handle, p, 2, 2, 1.0, 0, None, None, 0, 0, None, p, p, None) == bad
    assert lib.vfsx_log_probs(c.handle, None, 0, 0, 1.0, 0, None, None, 0, 0, None, None, None, None) == 0   # no queries at all: nothing to do
    zero = vfs_amd.Corpus(8, quantize=True, scale=0.0)
    with pytest.raises(vfs_amd.VfsxError):
        zero.log_probs(q)
    only = c.log_probs(q, k=3)  # the store still works
    assert only.log_probs.shape == (2, 0) and (only.top_count == 3).all()


# ---- device buffers: streams, graphs, several rounds ----------------------------------------------------------------------------


def device_call(c, torch, q, given, k, out, bias=None, stream=None, **kw):
    c.log_probs_device(q.data_ptr(), q.shape[0], d_rows=given.data_ptr() if given is not None else 0,
                       given=given.shape[1] if given is not None else 0, k=k, d_bias=0 if bias is None else bias.data_ptr(),
                       d_log_probs=out["lp"].data_ptr() if given is not None else 0, d_lse=out["lse"].data_ptr(),
                       d_entropy=out["entropy"].data_ptr(), d_top=out["top"].data_ptr() if k else 0,
                       stream=(stream or torch.cuda.current_stream()).cuda_stream, **kw)


def buffers(torch, nq, t, k):
    return {"lp": torch.full((nq, t), 7.0, device="cuda"), "lse": torch.full((nq,), 7.0, device="cuda"),
            "entropy": torch.full((nq,), 7.0, device="cuda"), "top": torch.full((nq, k, 24), 7, device="cuda", dtype=torch.uint8)}


@pytest.mark.parametrize("store", ["f32", "i8", "f8"])
@pytest.mark.parametrize("nq", [1, 3, 33, 200])
def test_device_equals_host_and_leaves_the_rest(store, nq):
    import torch
    rng = np.random.default_rng(12)
    rows, qh = make(store, 4001, 100, rng), rng.standard_normal((nq, 100)).astype(np.float32)
    c = corpus_of(store, rows)
    kw = dict(temperature=20.0 if store == "i8" else 0.7, source="f8" if store == "f8" else "rows")
    given = rng.integers(0, 4001, (nq, 2))
    want = c.log_probs(qh, given, 6, **kw)
    q, g = torch.from_numpy(qh).cuda(), torch.from_numpy(given).cuda()
    out = buffers(torch, nq + 1, 2, 6)  # one place more than the call fills
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side, side, torch.cuda.current_stream()):
        for o in out.values():
            o.fill_(7)
        stream.wait_stream(torch.cuda.current_stream())
        device_call(c, torch, q, g, 6, out, stream=stream, **kw)
        torch.cuda.synchronize()
        assert np.array_equal(out["lp"][:nq].cpu().numpy(), want.log_probs) and np.array_equal(out["lse"][:nq].cpu().numpy(), want.lse)
        assert np.array_equal(out["entropy"][:nq].cpu().numpy(), want.entropy)
        top = np.ascontiguousarray(out["top"].cpu().numpy()).view(np.dtype([("d", "f4"), ("f", "u4"), ("row", "u8"), ("id", "u8")]))[..., 0]
        assert np.array_equal(top["row"][:nq], want.top_rows) and np.array_equal(top["d"][:nq], want.top_log_probs)
        assert all((o[nq] == 7).all() for o in out.values())


@pytest.mark.parametrize("store", ["f32", "f8"])
def test_captured_graphs(store, no_collection):
    """Two graphs on one store, replayed among eager calls and after a larger call has replaced the workspace."""
    import torch
    rng = np.random.default_rng(13)
    rows = make(store, 3000, 64, rng)
    c = corpus_of(store, rows)
    kw = dict(source="f8" if store == "f8" else "rows")
    qs = [torch.from_numpy(rng.standard_normal((n, 64)).astype(np.float32)).cuda() for n in (2, 40)]
    given = [torch.from_numpy(rng.integers(0, 3000, (n, 1))).cuda() for n in (2, 40)]
    outs = [buffers(torch, n, 1, 5) for n in (2, 40)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.reserve_log_probs(2, **kw)
    graphs = []
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            device_call(c, torch, qs[0], given[0], 5, outs[0], **kw)
        graphs.append(g)
        g = torch.cuda.CUDAGraph()
        big = torch.zeros(2000, 64, device="cuda")
        with torch.cuda.graph(g, stream=side):  # not reserved for this many
            code = ref.refused(lambda: c.log_probs_device(big.data_ptr(), 2000, d_lse=outs[1]["lse"].data_ptr(), stream=side.cuda_stream, **kw))
        assert code == _lib.ERR_MEMTABLE
        del g
        c.reserve_log_probs(40, **kw)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            device_call(c, torch, qs[1], given[1], 5, outs[1], **kw)
        graphs.append(g)
    torch.cuda.synchronize()
    for turn in range(4):
        for i in (0, 1):
            qs[i].copy_(torch.from_numpy(rng.standard_normal(tuple(qs[i].shape)).astype(np.float32)))
            torch.cuda.synchronize()
            for o in outs[i].values():
                o.zero_()
            torch.cuda.synchronize()
            graphs[i].replay()
            torch.cuda.synchronize()
            want = c.log_probs(qs[i].cpu().numpy(), given[i].cpu().numpy(), 5, **kw)
            assert np.array_equal(outs[i]["lp"].cpu().numpy(), want.log_probs)
            assert np.array_equal(outs[i]["lse"].cpu().numpy(), want.lse)
            rows_got = outs[i]["top"].cpu().numpy().view(np.uint64)[..., 1]
            assert np.array_equal(rows_got, want.top_rows)
        if turn == 1:  # a larger call: another workspace, the graphs keep theirs
            c.log_probs(rng.standard_normal((3000, 64)).astype(np.float32), k=1, **kw)
    # rows added: a capture says so instead of leaving them out
    c.append(rows[:3])
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            code = ref.refused(lambda: device_call(c, torch, qs[0], given[0], 5, outs[0], **kw))
        assert code == _lib.ERR_MEMTABLE


def test_current_device_is_left_alone():
    import torch
    c = corpus_of("f32", np.ones((3, 4), np.float32))
    before = torch.cuda.current_device()
    c.log_probs(np.ones((1, 4), np.float32), k=1)
    assert torch.cuda.current_device() == before


def test_several_rounds_of_queries():
    """Queries whose statistics do not fit one round: 512 MiB hold 128 of them here."""
    rng = np.random.default_rng(14)
    n, nq = 5_000_000, 300
    c = vfs_amd.Corpus(4, capacity_rows=n)
    rows = rng.standard_normal((n, 4)).astype(np.float32)
    c.append(rows)
    q = rng.standard_normal((nq, 4)).astype(np.float32)
    got = c.log_probs(q, np.arange(nq)[:, None], 3)
    for i in (0, 1, 127, 128, 129, 255, 256, 257, 299):
        l = ref.logits(rows, q[i:i + 1])
        one = type(got)(*(a[i:i + 1] for a in got))
        ref.compare(one, ref.softmax_of(l, np.array([[i]]), 3), l, ref.logit_bound(rows, q[i:i + 1]))


def test_server_search_with_temperature(tmp_path):
    import json
    from vfs_amd.server import App
    app = App(state_dir=str(tmp_path / "state"), data_dir=str(tmp_path / "data"))
    assert app.handle("POST", "/init", json.dumps({"vector_dimension": 3, "truncate_data": True, "quantize": False}))[0] == 200
    vs = [[1.0, 0.0, 0.0], [0.8, 0.6, 0.0], [0.0, 1.0, 0.0], [-1.0, 0.0, 0.2]]
    for v in vs:
        assert app.handle("POST", "/vectors", json.dumps({"values": v, "name": "v", "tags": []}))[0] == 201
    ask = {"values": [1.0, 0.1, 0.0], "top_k": 5, "ef_search": 2, "search_type": "exact", "distance_method": "cosine"}
    plain = json.loads(app.handle("POST", "/search", json.dumps(ask))[1])
    status, body = app.handle("POST", "/search", json.dumps(dict(ask, temperature=0.5)))
    body = json.loads(body)
    assert status == 200 and "entropy" not in plain and all("log_prob" not in r for r in plain["results"])
    x = np.array(vs, np.float32)
    want = ref.softmax_of(ref.logits(x, np.array([ask["values"]], np.float32), cosine=True, temperature=0.5), [[0, 1]])
    assert [r["id"] for r in body["results"]] == [1, 2] == [r["id"] for r in plain["results"]]
    assert np.allclose([r["log_prob"] for r in body["results"]], want["log_probs"][0], atol=1e-5)
    assert abs(body["entropy"] - want["entropy"][0]) < 1e-5
    for t in (0, -1, "1", True, 1e40):
        assert app.handle("POST", "/search", json.dumps(dict(ask, temperature=t)))[0] == 400, t
    assert app.handle("POST", "/search", json.dumps(dict(ask, temperature=1.0, distance_method="euclidean")))[0] == 400
