"""Decode and verify over int8 pools on the GPU within what that path's own roundings allow (tests/int8_attention_lib.py): a dropped
remainder of the probabilities, a lost limb of the query or a coarser step is outside it."""
import numpy as np
import pytest
import torch

from oracle import paged_attention_oracle as O
from tests.int8_attention_lib import attention_and_tolerance, orthogonal_rows
from tests.int8_kv_lib import assert_within, bf16, context, dev, int8_pool, quantise_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pa():
    import nkipy_amd
    from nkipy_amd import _lib
    _lib.load()
    return nkipy_amd


@pytest.fixture
def debug_switch():
    from nkipy_amd import _lib
    lib = _lib.load()
    yield lambda key, value: lib.pa_debug_set(key, value)
    lib.pa_debug_set(0, 0)
    lib.pa_debug_set(5, 0)


def _refill(pool, name, b, rows, bs):
    """The first rows of sequence b's K or V, [n, Hkv, D] float64, quantised into the pool."""
    codes, scale = quantise_rows(O.round_to_bf16(rows.astype(np.float32)))
    for t in range(len(rows)):
        blk = pool["tables"][b, t // bs]
        pool[name][blk, t % bs], pool[name + "s"][blk, :, t % bs] = codes[t], scale[t]


def _run(pa, pool, q, ctxs, bs, scale, qlens=None, window=0, sinks=None, **kw):
    args = (dev(pool["k"]), dev(pool["v"]), dev(pool["tables"]), dev(np.asarray(ctxs, np.int32)))
    kw.update(k_scale=dev(pool["ks"]), v_scale=dev(pool["vs"]), sliding_window=window or None, sinks=None if sinks is None else dev(sinks))
    if qlens is None:
        got, qlens = pa.decode(bf16(q[:, 0]), *args, scale, **kw)[:, None], [1] * len(ctxs)
    else:
        got = pa.verify(bf16(q), *args, dev(np.asarray(qlens, np.int32)), scale, **kw)
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b, c in enumerate(ctxs):
        n = min(qlens[b], c)
        if n:
            want[b, :n], tol[b, :n] = attention_and_tolerance(q[b, :n], context(pool, "k", b, c, bs), context(pool, "v", b, c, bs), scale,
                                                              c - n, window, sinks)
    assert_within(got, want, tol)


def _queries(rng, kind, shape):
    q = O.round_to_bf16(rng.standard_normal(shape).astype(np.float32))
    if kind == "outlier":           # one channel 8 to 2 000 times the others
        q[..., 7] = O.round_to_bf16((1.7 * 2.0 ** rng.integers(3, 11, shape[:-1])).astype(np.float32))
    return q


@pytest.mark.parametrize("impl", [0, 2, 3])
@pytest.mark.parametrize("kind", ["ordinary", "outlier"])
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(32, 8, 128, 32), (8, 8, 64, 16), (7, 1, 64, 64), (6, 3, 128, 128)])
def test_decode(pa, rng, debug_switch, Hq, Hkv, D, bs, kind, impl):
    debug_switch(0, impl)
    ctxs = [1, 0, 2, 31, 33, 700, 16, 1500]
    pool = int8_pool(rng, ctxs, bs, Hkv, D, spread=0.5)
    q = _queries(rng, kind, (len(ctxs), 1, Hq, D))
    if kind == "outlier":
        for b, c in enumerate(ctxs):
            k = context(pool, "k", b, c, bs)
            k[..., 7] *= 2.0 ** -6
            _refill(pool, "k", b, k, bs)
    _run(pa, pool, q, ctxs, bs, 1.0 / np.sqrt(D))


@pytest.mark.parametrize("impl", [0, 2, 3])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_that_cancel(pa, rng, debug_switch, D, impl):
    """Keys nearly orthogonal to the query under a large scale: the scores are small, what a rounded query adds to them is not."""
    debug_switch(0, impl)
    H, bs, ctxs = 8, 16, [5, 40, 300]
    pool = int8_pool(rng, ctxs, bs, H, D, spread=0.5)
    q = _queries(rng, "ordinary", (len(ctxs), 1, H, D))
    q = O.round_to_bf16((np.sign(q) * rng.uniform(0.06, 1.9, q.shape)).astype(np.float32))
    for b, c in enumerate(ctxs):
        _refill(pool, "k", b, orthogonal_rows(rng, q[b, 0], c), bs)
    _run(pa, pool, q, ctxs, bs, 6.0)


@pytest.mark.parametrize("rows", [0, 16, 32])
@pytest.mark.parametrize("kind", ["ordinary", "outlier"])
@pytest.mark.parametrize("Hq,Hkv,D,T,bound", [(32, 8, 128, 4, None), (64, 8, 64, 3, 1024), (8, 1, 128, 8, 1024), (8, 2, 64, 33, None)])
def test_verify(pa, rng, debug_switch, Hq, Hkv, D, T, bound, kind, rows):
    debug_switch(5, rows)
    ctxs = [T, 500, 40, 1000, T + 31]
    pool = int8_pool(rng, ctxs, 32, Hkv, D, spread=0.5)
    q = _queries(rng, kind, (len(ctxs), T, Hq, D))
    _run(pa, pool, q, ctxs, 32, 1.0 / np.sqrt(D), qlens=[T, 1, 0, min(T, 2), T], max_seq_len=bound)


@pytest.mark.parametrize("impl", [0, 2, 3])
@pytest.mark.parametrize("window", [1, 7, 100])
def test_window_and_sinks(pa, rng, debug_switch, window, impl):
    debug_switch(0, impl)
    Hq, Hkv, D, bs, ctxs = 16, 4, 128, 16, [1, 99, 101, 600, 0]
    pool = int8_pool(rng, ctxs, bs, Hkv, D, spread=0.5)
    _run(pa, pool, _queries(rng, "ordinary", (len(ctxs), 1, Hq, D)), ctxs, bs, 1.0 / np.sqrt(D), window=window,
         sinks=rng.standard_normal(Hq).astype(np.float32))


def test_a_long_context(pa, rng):
    Hq, Hkv, D, bs, ctxs = 8, 2, 128, 64, [9000]
    pool = int8_pool(rng, ctxs, bs, Hkv, D, spread=0.5)
    _run(pa, pool, _queries(rng, "outlier", (1, 1, Hq, D)), ctxs, bs, 1.0 / np.sqrt(D))
