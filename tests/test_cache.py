"""The attention cache without a GPU: its oracle, sizes, and every refusal of its entry points."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import cache_oracle as O
import maivs_b200 as M
from maivs_b200 import _lib

P = 4096  # an address that is aligned for every type; no call here gets as far as using it


@pytest.fixture()
def cache():
    return M.AttentionCache(3, 100, 2, 80, device=None)


def test_sizes(cache):
    st = cache.stats()
    assert st["row_bytes"] == 144.0 and st["capacity"] == 100.0 and st["device"] == -1.0
    # 128 rows (capacity rounded up to 32) of 3 sequences and 2 heads
    assert st["device_bytes"] == 3 * 2 * 128 * 144 + 256
    one = cache.attend_workspace(3, 4)
    assert cache.attend_workspace(3, 4, weights=True) > one
    assert cache.attend_found_workspace(3, 4, 10) > 0
    assert cache.evict_workspace() >= 2 * 4 * 3 * 100
    # dimensions are padded to 64, 128, 256 and 384
    for dim, row in ((1, 72), (64, 72), (65, 144), (128, 144), (129, 288), (256, 288), (257, 432), (384, 432)):
        assert M.AttentionCache(1, 1, 1, dim, device=None).stats()["row_bytes"] == row


@pytest.mark.parametrize("args", [(0, 8, 1, 64), (65536, 8, 1, 64), (1, 0, 1, 64), (1, 2**27 + 1, 1, 64),
                                  (1, 8, 0, 64), (1, 8, 1025, 64), (1, 8, 1, 0), (1, 8, 1, 385), (-1, 8, 1, 64),
                                  (65535, 2**27, 1024, 64)])
def test_new_refuses(args):
    with pytest.raises(ValueError):
        M.AttentionCache(*args, device=None)


def test_null_handles_and_outputs():
    L = _lib.lib()
    n = C.c_size_t(0)
    assert L.maivs_cache_new(1, 1, 1, 64, -1, None) == _lib.BAD_ARG
    assert L.maivs_cache_evict_workspace(None, C.byref(n)) == _lib.BAD_ARG
    assert L.maivs_cache_append(None, P, P, 0, 1, 0, 0, P, P, None, None, None, None) == _lib.BAD_ARG
    L.maivs_cache_free(None)
    h = C.c_void_p()
    assert L.maivs_cache_new(1, 1, 1, 64, -1, C.byref(h)) == _lib.OK
    assert L.maivs_cache_evict_workspace(h, None) == _lib.BAD_ARG
    assert L.maivs_cache_flags(h, None, None) == _lib.BAD_ARG
    v = C.c_double(0)
    assert L.maivs_cache_stat(h, b"nothing", C.byref(v)) == _lib.NOT_FOUND
    L.maivs_cache_free(h)


def good_append(c, **kw):
    a = dict(d_keys=P, d_values=P, n_tokens=4, d_offsets=P, d_lengths=P)
    a.update(kw)
    c.append(**a)


def good_attend(c, **kw):
    a = dict(d_queries=P, n_tokens=4, n_query_heads=4, d_offsets=P, d_lengths=P, d_out=P, d_workspace=P,
             workspace_bytes=1 << 30)
    a.update(kw)
    c.attend(**a)


def good_found(c, **kw):
    a = dict(d_queries=P, n_tokens=4, n_query_heads=4, d_offsets=P, d_lengths=P, d_rows=P, k=10, d_out=P,
             d_workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    c.attend_found(**a)


def good_evict(c, **kw):
    a = dict(d_lengths=P, keep=5, d_weights_in=P, d_weights_out=P, d_new_lengths=2 * P, d_ids_in=P, d_ids_out=P,
             d_workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    c.evict(**a)


@pytest.mark.parametrize("call", [good_append, good_attend, good_found, good_evict])
def test_good_arguments_reach_the_device_check(cache, call):
    with pytest.raises(M.MaivsError, match="no storage"):
        call(cache)


def test_read_and_flags_reach_the_device_check(cache):
    with pytest.raises(M.MaivsError, match="no storage"):
        cache.read(P, P, 4, P, P)
    with pytest.raises(M.MaivsError, match="no storage"):
        cache.flags()


@pytest.mark.parametrize("kw", [dict(dtype="f64"), dict(n_tokens=-1), dict(n_tokens=2**27 + 1), dict(d_offsets=0),
                                dict(d_lengths=0), dict(d_offsets=P + 2), dict(d_keys=0), dict(d_values=P + 1),
                                dict(key_stride=159), dict(value_stride=1), dict(d_ids=P), dict(d_token_ids=P),
                                dict(d_weights=P + 2), dict(d_ids=P + 4, d_token_ids=P)])
def test_append_refuses(cache, kw):
    with pytest.raises(ValueError):
        good_append(cache, **kw)


@pytest.mark.parametrize("kw", [dict(n_query_heads=3), dict(n_query_heads=0), dict(d_queries=0), dict(d_out=0),
                                dict(d_out=P + 1), dict(dtype="int4"), dict(query_stride=319), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(scale=-1.3e30), dict(decay=float("nan")), dict(d_weights_in=P),
                                dict(d_weights_out=P), dict(d_lse=P + 1), dict(d_offsets=0), dict(n_tokens=-4),
                                dict(d_workspace=P + 8, d_weights_in=P, d_weights_out=P),
                                dict(d_weights_in=P, d_weights_out=P, workspace_bytes=8),
                                dict(d_weights_in=P, d_weights_out=P, d_workspace=0), dict(max_rows=-1)])
def test_attend_refuses(cache, kw):
    with pytest.raises(ValueError):
        good_attend(cache, **kw)


@pytest.mark.parametrize("kw", [dict(k=0), dict(k=-1), dict(d_rows=0), dict(d_rows=P + 4), dict(n_query_heads=5),
                                dict(d_weights=P, workspace_bytes=16), dict(k=2**27 + 1)])
def test_attend_found_refuses(cache, kw):
    with pytest.raises(ValueError):
        good_found(cache, **kw)


@pytest.mark.parametrize("kw", [dict(d_lengths=0), dict(d_weights_in=0), dict(d_weights_out=0), dict(d_new_lengths=0),
                                dict(d_new_lengths=P), dict(d_ids_in=0), dict(d_ids_out=0), dict(keep=-1),
                                dict(d_ids_in=0, d_ids_out=0, d_evicted=P), dict(d_workspace=0),
                                dict(d_ids_in=0, d_ids_out=0, d_protect_from=P), dict(workspace_bytes=100),
                                dict(d_evicted=P + 4)])
def test_evict_refuses(cache, kw):
    with pytest.raises(ValueError):
        good_evict(cache, **kw)


def test_workspace_refuses(cache):
    with pytest.raises(ValueError):
        cache.attend_workspace(4, 3)
    with pytest.raises(ValueError):
        cache.attend_found_workspace(4, 4, 0)
    with pytest.raises(ValueError, match="2\\^30"):
        cache.attend_workspace(2**20, 2048)
    with pytest.raises(ValueError, match="2\\^38"):
        cache.attend_found_workspace(2**20, 2, 2**20)
    # a grid of more than 2^31 blocks
    big = M.AttentionCache(65535, 16, 1024, 64, device=None)
    with pytest.raises(ValueError, match="blocks"):
        big.attend_workspace(1 << 17, 1024 * 8, max_tokens=1 << 17)


def test_without_a_gpu_a_cache_fails_loudly():
    from conftest import has_gpu

    if has_gpu():
        pytest.skip("a GPU is present")
    with pytest.raises(M.MaivsError, match="no CUDA device"):
        M.AttentionCache(1, 8, 1, 64)


# ---- the oracle itself ----------------------------------------------------------------------------
def test_oracle_levels():
    x = np.array([[0.0, 1.0, 7.4, 7.5, 8.5, 15.0, 3.0, 14.5]], np.float32)
    v, low, step = O.quantise(x)
    # step 1, low 0: the nearest whole number, ties to the even one
    assert v.tolist() == [[0.0, 1.0, 7.0, 8.0, 8.0, 15.0, 3.0, 14.0]]
    assert (low == 0).all() and (step == 1).all()
    v, _, step = O.quantise(np.full((1, 70), 0.3, np.float32))
    assert (step == 0).all() and np.allclose(v, float(O.bf16(np.float32([0.3]))[0]))
    assert np.isnan(O.quantise(np.array([[1.0, np.inf]], np.float32))[0]).all()


def test_oracle_attend_and_evict():
    rng = np.random.default_rng(1)
    r = O.Rows(rng.standard_normal((9, 70)).astype(np.float32), rng.standard_normal((9, 70)).astype(np.float32))
    q = rng.standard_normal(70)
    out, lse, p, err, _, _ = O.attend_head(q, r, [2, 5, 5], 0.1, "f32")
    z = 0.1 * (r.k[[2, 5, 5]] @ q)
    assert np.allclose(p, np.exp(z) / np.exp(z).sum()) and np.allclose(out, p @ r.v[[2, 5, 5]])
    assert np.isclose(lse, np.log(np.exp(z).sum())) and (err > 0).all()
    m, src, gone = O.evict(6, 3, [0.1, 0.5, 0.1, 0.5, 0.5, 0.5])
    assert (m, src, gone) == (3, [3, 1, 4], [0, 2, 5])
