"""CPU: the 64-bit definitions behind the probability and 8-bit tests, and what the entry points refuse before any device work."""
import numpy as np
import pytest

import vfs_amd
from vfs_amd import _lib
from tests import prob_ref as ref


def test_e4m3_grid_against_torch():
    import torch
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((40, 300)) * 2.0 ** rng.integers(-30, 30, (40, 1))).astype(np.float32)
    x[3] = 0
    x[4, :128] = 448.0            # exactly the largest value: e = 0
    x[5, :128] = np.nextafter(np.float32(448.0), np.float32(1e9))
    x[6, 7] = 2.0**-140           # a subnormal among zeros
    x[6, :7] = x[6, 8:128] = 0
    want = ref.e4m3_values(x)
    t = torch.from_numpy(np.pad(x, ((0, 0), (0, 84)))).unflatten(1, (3, 128)).double()
    top = t.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -127.0)
    for k in range(-127, 120):    # by the definition: the least e >= -127 that holds the maximum
        e = torch.where(top > 448.0 * 2.0**k, float(k + 1), e)
    e = torch.where(top > 0, e, 0.0)
    got = ((t / 2.0**e).float().to(torch.float8_e4m3fn).double() * 2.0**e).flatten(1)[:, :300].numpy()
    assert np.array_equal(got, want)


def test_softmax_definition():
    l = np.array([[0.0, np.log(3.0), -np.inf], [-np.inf, -np.inf, -np.inf]])
    w = ref.softmax_of(l, rows=[[1, 2, 7], [0, 1, -1]], k=3)
    assert np.allclose(w["lse"], [np.log(4.0), -np.inf])
    assert np.allclose(w["entropy"], [0.25 * np.log(4) + 0.75 * np.log(4 / 3), 0])
    assert np.allclose(w["log_probs"], [[np.log(0.75), -np.inf, -np.inf], [-np.inf] * 3])
    assert w["top_rows"].tolist() == [[1, 0, -1], [-1, -1, -1]] and w["top_count"].tolist() == [2, 0]


def test_null_handle_is_refused():
    lib = vfs_amd.load()
    assert lib.vfsx_log_probs(None, None, 1, 0, 1.0, 0, None, None, 0, 0, None, None, None, None) == _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_log_probs_device(None, None, 1, 0, 1.0, 0, None, None, 0, 0, None, None, None, None, None) == _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_reserve_log_probs(None, 1, 0) == _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_corpus_enable_f8(None, 1) == _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_corpus_get_rows_f8(None, None, 0, None) == _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_scores_f8(None, None, 1, 0, 0, None, 0) == _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_scores_f8_device(None, None, 1, 0, 0, None, 0, None) == _lib.ERR_INVALID_VECTOR
    assert lib.vfsx_reserve_scores_f8(None, 1) == _lib.ERR_INVALID_VECTOR
    assert b"null corpus" in lib.vfsx_last_error()


@pytest.mark.parametrize("table,value", [(_lib.SIMILARITY, "euclid"), (_lib.SOURCE, "f16"), (_lib.SCORES_DTYPE, None)])
def test_unknown_choices_are_named(table, value):
    with pytest.raises(vfs_amd.VfsxError) as e:
        vfs_amd.Corpus._choice(table, value, "it")
    assert e.value.code == _lib.ERR_INVALID_VECTOR and "must be one of" in str(e.value)
