"""Packed prompts whose values hold infinities and NaN: they reach the queries that see them, in their columns, and no others."""
import numpy as np
import pytest
import torch

from oracle import paged_attention_oracle as O
from tests.int8_kv_lib import attention64, attention_tolerance, bf16, dev, to_np
from tests.test_gpu_packed_prefill import _starts, debug_switch, pa  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu
BAD = [np.inf, -np.inf, np.nan]


def _check(pa, rng, qn, kn, Hq, Hkv, D, n_bad, window=None, with_sinks=False, whole=False, **kw):  # noqa: F811
    cu_q, cu_k = _starts(qn), _starts(kn)
    q, k, v = (O.round_to_bf16(rng.standard_normal((int(c[-1]), h, D)).astype(np.float32)) for c, h in ((cu_q, Hq), (cu_k, Hkv), (cu_k, Hkv)))
    bad = np.zeros(v.shape, bool)
    value = np.zeros(v.shape, np.float32)
    for _ in range(n_bad):
        at = int(rng.integers(0, len(v))), int(rng.integers(0, Hkv)), slice(None) if whole else int(rng.integers(0, D))
        bad[at], value[at] = True, BAD[int(rng.integers(0, 3))]
    sinks = rng.standard_normal(Hq).astype(np.float32) if with_sinks else None
    scale = 1.0 / np.sqrt(D)
    dv = bf16(v)
    dv[dev(bad)] = dev(value)[dev(bad)].to(torch.bfloat16)
    got = to_np(pa.packed_prefill(bf16(q), bf16(k), dv, dev(cu_q), scale, cu_seqlens_k=dev(cu_k), sliding_window=window,
                                  sinks=None if sinks is None else dev(sinks), **kw))
    v[bad] = 0
    spoilt = 0
    for i in range(len(qn)):
        rows, keys = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
        first = kn[i] - qn[i]
        want, mag, reach = attention64(q[rows].astype(np.float64), k[keys].astype(np.float64), v[keys].astype(np.float64), scale, first, window or 0, sinks)
        pos, key = first + np.arange(qn[i])[:, None], np.arange(kn[i])[None]
        sees = (key <= pos) & (key > pos - (window or 1 << 30))
        hit = np.einsum("tc,chd->thd", sees.astype(np.int64), bad[keys].astype(np.int64)).repeat(Hq // Hkv, 1) > 0
        assert np.array_equal(~np.isfinite(got[rows]), hit), f"sequence {i}"
        over = np.abs(got[rows] - want) - attention_tolerance(want, mag, reach, D)
        assert (over[~hit] <= 0).all(), f"sequence {i}: {over[~hit].max()}"
        spoilt += int(hit.sum())
    return spoilt


HEADS = [(8, 2, 128), (4, 4, 128), (12, 2, 64), (6, 3, 64), (5, 1, 64), (8, 1, 64)]


@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("impl", [0, 4, 6, 7, 8])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_a_value_that_is_no_number_reaches_who_sees_it(pa, rng, debug_switch, Hq, Hkv, D, impl, window):  # noqa: F811
    """Every tile form: whole prompts, prefixes, sequences with fewer keys than queries, whose first rows see nothing."""
    if impl == 8 and window:
        impl = 0
    debug_switch(3, impl)
    debug_switch(6, 0)
    assert _check(pa, rng, [1, 64, 129, 300, 33], [1, 64, 129, 300, 33], Hq, Hkv, D, 12, window) > 0
    assert _check(pa, rng, [60, 64, 129, 300, 5], [200, 3, 100, 700, 65], Hq, Hkv, D, 12, window, with_sinks=True) > 0
    _check(pa, rng, [150, 40], [150, 240], Hq, Hkv, D, 3, window, whole=True)


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("split", [2, 5])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_the_same_with_the_keys_split(pa, rng, debug_switch, Hq, Hkv, D, split, window):  # noqa: F811
    debug_switch(6, split)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    _check(pa, rng, [60, 64, 129, 30, 5], [700, 3, 100, 900, 65], Hq, Hkv, D, 14, window, with_sinks=True, workspace=ws)
    _check(pa, rng, [40, 100], [400, 620], Hq, Hkv, D, 3, window, whole=True, workspace=ws)


@pytest.mark.parametrize("D", [64, 128])
def test_values_that_are_none_at_all(pa, rng, D):  # noqa: F811
    """A prompt all of whose values are NaN, beside one that is sound."""
    Hq, Hkv, n = 8, 2, [900, 130]
    q, k, v = (bf16(rng.standard_normal((sum(n), h, D))) for h in (Hq, Hkv, Hkv))
    cu = dev(_starts(n))
    want = pa.packed_prefill(q, k, v, cu, 0.1)
    v[:900] = float("nan")
    got = pa.packed_prefill(q, k, v, cu, 0.1)
    assert bool(torch.isnan(got[:900]).all()) and torch.equal(got[900:], want[900:])


def test_a_chunk_over_an_int8_cache(pa):  # noqa: F811
    """A token whose K and V hold an infinity: the queries in front of it in its chunk are those of a chunk that ends there."""
    from tests.test_gpu_int8_engine import _engine, _rows
    D, Hq, Hkv, T, at = 64, 8, 2, 150, 100
    g = torch.Generator(device="cuda").manual_seed(9)
    (_, layer), (_, short) = (_engine(D, 16, Hq, Hkv, 2, rope=False) for _ in range(2))
    xq, xk, xv = _rows(g, 2, T, Hq, Hkv, D)
    xk[0, at, 0, 3], xv[0, at, 1, 5] = float("inf"), float("nan")
    got = layer.step(xq, xk, xv, [T, 90])
    want = short.step(*(t[:, :at].contiguous() for t in (xq, xk, xv)), [at, 90])
    # (twice the kernel's own roundings: that of the probabilities and that of the result, 2^-8 of max |v| each)
    assert bool(torch.isfinite(got[0, :at]).all()) and torch.isfinite(got[1]).all()
    assert (got[0, :at].float() - want[0].float()).abs().max() <= 4 * 2.0 ** -8 * xv[0, :at].float().abs().max()
    assert bool(torch.isnan(got[0, at:, :4]).all()) and bool(torch.isnan(got[0, at:, 4:]).all())


@pytest.mark.parametrize("D", [64, 128])
def test_sinks_that_leave_the_keys_nothing(pa, rng, D):  # noqa: F811
    """A sink whose share of the sum is past float32's range: zeros, also for a row whose tile hides a NaN from it."""
    Hq, Hkv, n = 4, 2, 100
    q, k, v = (bf16(rng.standard_normal((n, h, D))) for h in (Hq, Hkv, Hkv))
    v[70] = float("nan")
    got = pa.packed_prefill(q, k, v, dev(_starts([n])), 0.1, sinks=torch.full((Hq,), 300.0, device="cuda"))
    assert bool((got[:70] == 0).all()) and bool(torch.isnan(got[70:]).all())
