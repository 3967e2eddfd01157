"""Packed prompt attention on the GPU against float64, element by element within what the roundings allow."""
import numpy as np
import pytest
import torch

from oracle import paged_attention_oracle as O
from tests.int8_kv_lib import assert_within, attention64, attention_tolerance, bf16, dev

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
    lib.pa_debug_set(3, 0)
    lib.pa_debug_set(6, 1)


def _starts(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def _want(q, k, v, cu_q, cu_k, scale, window, sinks, qlens=None, klens=None):
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(len(cu_q) - 1):
        n = cu_q[i + 1] - cu_q[i] if qlens is None else min(qlens[i], cu_q[i + 1] - cu_q[i])
        c = cu_k[i + 1] - cu_k[i] if klens is None else min(klens[i], cu_k[i + 1] - cu_k[i])
        rows = slice(cu_q[i], cu_q[i] + n)
        o, mag, reach = attention64(q[rows].astype(np.float64), k[cu_k[i]:cu_k[i] + c].astype(np.float64),
                                    v[cu_k[i]:cu_k[i] + c].astype(np.float64), scale, c - n, window or 0, sinks)
        out[rows], tol[rows] = o, attention_tolerance(o, mag, reach, q.shape[2])
    return out, tol


def _run(pa, rng, qn, Hq, Hkv, D, kn=None, window=None, with_sinks=False, strided=False, tail=0, **kw):
    cu_q = _starts(qn)
    cu_k = cu_q if kn is None else _starts(kn)
    nq, nk = int(cu_q[-1]) + tail, int(cu_k[-1]) + tail
    q, k, v = (O.round_to_bf16(rng.standard_normal((n, h, D)).astype(np.float32)) for n, h in ((nq, Hq), (nk, Hkv), (nk, Hkv)))
    scale = 1.0 / np.sqrt(D)
    sinks = rng.standard_normal(Hq).astype(np.float32) if with_sinks else None
    if strided:
        wide = torch.full((nq, Hq + 2 * Hkv + 1, D), float("nan"), dtype=torch.bfloat16, device="cuda")
        dq, dk, dv = wide[:, :Hq], wide[:, Hq:Hq + Hkv], wide[:, Hq + Hkv + 1:]
        dq.copy_(bf16(q)), dk.copy_(bf16(k)), dv.copy_(bf16(v))
    else:
        dq, dk, dv = bf16(q), bf16(k), bf16(v)
    if tail:
        dk[-tail:] = float("nan")
        dv[-tail:] = float("nan")
    out = torch.full((nq, Hq, D), 3.0, dtype=torch.bfloat16, device="cuda")
    got = pa.packed_prefill(dq, dk, dv, dev(cu_q), scale, cu_seqlens_k=None if kn is None else dev(cu_k), sliding_window=window,
                            sinks=None if sinks is None else dev(sinks), out=out, **kw)
    want, tol = _want(q, k, v, cu_q, cu_k, scale, window, sinks)
    if tail:
        assert (got[-tail:] == 3.0).all()
        got, want, tol = got[:-tail], want[:-tail], tol[:-tail]
    assert_within(got, want, tol)
    return dq, dk, dv, got


HEADS = [(8, 2, 128), (4, 4, 128), (6, 1, 128), (5, 5, 128), (12, 2, 64), (8, 4, 64), (6, 3, 64), (5, 1, 64), (8, 1, 64), (2, 2, 64),
         (1, 1, 64), (20, 10, 128)]


@pytest.mark.parametrize("impl", [0, 8])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_ragged_prompts(pa, rng, debug_switch, Hq, Hkv, D, impl):
    debug_switch(3, impl)
    _run(pa, rng, [1, 64, 0, 63, 129, 300, 2, 65, 33, 0], Hq, Hkv, D, tail=5)


@pytest.mark.parametrize("form", [4, 6, 7])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_tile_forms(pa, rng, debug_switch, Hq, Hkv, D, form):
    """64-key tiles, those with one q head per wave, 32-key tiles: whole prompts, prefixes, fewer keys than queries, a
    window with sinks, whatever the sizes would choose."""
    debug_switch(3, form)
    debug_switch(6, 0)
    _run(pa, rng, [1, 64, 0, 63, 129, 300, 2, 65, 33, 0], Hq, Hkv, D, tail=5)
    _run(pa, rng, [40, 1, 130, 3, 70, 20], Hq, Hkv, D, kn=[400, 777, 130, 0, 5, 65], tail=3)
    for window in (1, 40, 200):
        _run(pa, rng, [150, 1, 300, 31], Hq, Hkv, D, kn=[150, 260, 700, 31], window=window, with_sinks=True)


@pytest.mark.parametrize("n", [1, 20, 90])
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 64), (6, 2, 64), (16, 4, 128)])
def test_forms_the_sizes_choose(pa, rng, Hq, Hkv, D, n):
    """Calls of a few and of many workgroups, short and long."""
    _run(pa, rng, [int(x) for x in rng.integers(100, 300, n)], Hq, Hkv, D)
    _run(pa, rng, [int(x) for x in rng.integers(1, 60, 2 * n)] + [1500], Hq, Hkv, D)


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (64, 8, 64), (16, 2, 128), (16, 16, 64)])
def test_strided_rows(pa, rng, Hq, Hkv, D):
    _run(pa, rng, [100, 1, 200, 17], Hq, Hkv, D, strided=True)


@pytest.mark.parametrize("impl,split", [(0, 1), (0, 0), (0, 2), (0, 5), (0, 16), (8, 0)])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 2, 64), (3, 1, 64), (3, 3, 128)])
def test_more_keys_than_queries_and_fewer(pa, rng, debug_switch, Hq, Hkv, D, split, impl):
    """Cached prefixes, sequences with fewer keys than queries (their first rows see nothing), and with none at all."""
    debug_switch(3, impl)
    debug_switch(6, split)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    _run(pa, rng, [40, 1, 130, 3, 70, 20], Hq, Hkv, D, kn=[400, 777, 130, 0, 5, 65], tail=3, workspace=ws)


@pytest.mark.parametrize("split", [1, 3])
@pytest.mark.parametrize("window", [1, 30, 64, 200, 5000])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 4, 64), (6, 3, 64)])
def test_window_and_sinks(pa, rng, debug_switch, Hq, Hkv, D, window, split):
    debug_switch(6, split)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    _run(pa, rng, [150, 1, 300, 31], Hq, Hkv, D, kn=[150, 260, 700, 31], window=window, with_sinks=True, workspace=ws)


@pytest.mark.parametrize("split", [1, 2])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 2, 64)])
def test_rows_with_room_to_spare(pa, rng, debug_switch, Hq, Hkv, D, split):
    """query_lens / seq_lens: padding query rows are zero, key rows past the length (NaN here) are never used, gaps too."""
    debug_switch(6, split)
    cu_q, cu_k = _starts([64, 64, 64, 64, 200]), _starts([300, 300, 300, 300, 300])
    qlens, klens = [64, 1, 0, 30, 150], [300, 17, 200, 20, 260]
    q = O.round_to_bf16(rng.standard_normal((int(cu_q[-1]), Hq, D)).astype(np.float32))
    k, v = (O.round_to_bf16(rng.standard_normal((int(cu_k[-1]), Hkv, D)).astype(np.float32)) for _ in range(2))
    dk, dv = bf16(k), bf16(v)
    for i, c in enumerate(klens):
        dk[cu_k[i] + c:cu_k[i + 1]] = float("nan")
        dv[cu_k[i] + c:cu_k[i + 1]] = float("inf")
    i32 = lambda x: dev(np.asarray(x, np.int32))               # noqa: E731
    got = pa.packed_prefill(bf16(q), dk, dv, dev(cu_q), 0.1, cu_seqlens_k=dev(cu_k), query_lens=i32(qlens), seq_lens=i32(klens),
                            workspace=torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    want, tol = _want(q, k, v, cu_q, cu_k, 0.1, None, None, qlens, klens)
    assert_within(got, want, tol)


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (16, 4, 64)])
def test_against_the_paged_kernel(pa, rng, Hq, Hkv, D):
    """The same prompt through a paged bfloat16 pool, written packed."""
    n, bs = 700, 32
    q, k, v = (bf16(rng.standard_normal((n, h, D))) for h in (Hq, Hkv, Hkv))
    cu = dev(np.asarray([0, n], np.int32))
    got = pa.packed_prefill(q, k, v, cu, 0.1)
    blocks = (n + bs - 1) // bs
    kc, vc = (torch.zeros((blocks, bs, Hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    tables = dev(rng.permutation(blocks).astype(np.int32)[None])
    ln = dev(np.asarray([n], np.int32))
    pa.kv_write(k, v, kc, vc, tables, ln, ln, cu_seqlens=cu)
    ref = pa.prefill(q[None], kc, vc, tables, ln, ln, 0.1)[0]
    assert (got.float() - ref.float()).abs().max() <= 2e-2
    k2, v2 = pa.read_kv(kc, vc, tables, ln, cu, n)
    assert torch.equal(k2, k) and torch.equal(v2, v)


def test_large_scores_move_the_reference(pa, rng):
    """Scores that grow along the keys by far more than float32's exponent range allows for a fixed reference."""
    n, D = 400, 128
    q, k, v = (O.round_to_bf16(rng.standard_normal((n, 2, D)).astype(np.float32)) for _ in range(3))
    q[:] = 1.0
    k *= 0.05
    k += O.round_to_bf16(np.linspace(-40, 60, n).astype(np.float32))[:, None, None]
    k = O.round_to_bf16(k)
    got = pa.packed_prefill(bf16(q), bf16(k), bf16(v), dev(np.asarray([0, n], np.int32)), 0.125)
    want, tol = _want(q, k, v, [0, n], [0, n], 0.125, None, None)
    assert_within(got, want, tol)


@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_other_scales(pa, rng, scale):
    n, D = 150, 64
    q, k, v = (O.round_to_bf16(rng.standard_normal((n, 2, D)).astype(np.float32)) for _ in range(3))
    got = pa.packed_prefill(bf16(q), bf16(k), bf16(v), dev(np.asarray([0, n], np.int32)), scale)
    want, tol = _want(q, k, v, [0, n], [0, n], scale, None, None)
    assert_within(got, want, tol)


def test_boundaries_that_lie(pa, rng):
    """Boundaries outside the tensors count as their ends: nothing outside is read or written."""
    n, D = 130, 128
    q, k, v = (bf16(rng.standard_normal((n, 2, D))) for _ in range(3))
    for cu in ([0, 1 << 30], [-5, 2 ** 31 - 1], [50, 10], [0, 100, 20, 130], [-2 ** 31, 2 ** 31 - 1], [200, 300]):
        out = pa.packed_prefill(q, k, v, dev(np.asarray(cu, np.int32)), 0.1, out=torch.zeros_like(q))
        assert torch.isfinite(out).all()
    full = pa.packed_prefill(q, k, v, dev(np.asarray([-5, 2 ** 31 - 1], np.int32)), 0.1)
    assert torch.equal(full, pa.packed_prefill(q, k, v, dev(np.asarray([0, n], np.int32)), 0.1))


def test_graph_replays_with_other_lengths(pa, rng):
    D, Hq, Hkv, n = 128, 8, 2, 512
    q, k, v = (torch.zeros((n, h, D), dtype=torch.bfloat16, device="cuda") for h in (Hq, Hkv, Hkv))
    cu = dev(_starts([200, 312]))
    run = lambda: pa.packed_prefill(q, k, v, cu, 0.1)          # noqa: E731
    for x in (q, k, v):
        x.copy_(bf16(rng.standard_normal(x.shape)))
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for lens in ([200, 312], [1, 511], [512, 0], [256, 100]):
        cu.copy_(dev(_starts(lens)))
        for x in (q, k, v):
            x.copy_(bf16(rng.standard_normal(x.shape)))
        g.replay()
        torch.cuda.synchronize()
        a = out[:sum(lens)].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            b = run()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert torch.equal(a, b[:sum(lens)])


@pytest.mark.parametrize("S", [100, 300, 600])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 128), (2, 2, 64)])
def test_many_sequences(pa, rng, S, Hq, Hkv, D):
    """More sequences than a wave has lanes, and than the ranking holds (their own order then); prefixes of any length."""
    qn = [int(x) for x in rng.integers(0, 40, S)]
    _run(pa, rng, qn, Hq, Hkv, D, kn=[n + int(x) for n, x in zip(qn, rng.integers(0, 90, S))])


def test_keys_and_values_of_different_strides(pa, rng):
    n, Hq, Hkv, D = 200, 8, 2, 128
    q, k, v = (O.round_to_bf16(rng.standard_normal((n, h, D)).astype(np.float32)) for h in (Hq, Hkv, Hkv))
    wide = torch.zeros((n, Hkv + 3, D), dtype=torch.bfloat16, device="cuda")
    dk = wide[:, 1:1 + Hkv]
    dk.copy_(bf16(k))
    cu = dev(np.asarray([0, 70, n], np.int32))
    got = pa.packed_prefill(bf16(q), dk, bf16(v), cu, 0.1)
    assert torch.equal(got, pa.packed_prefill(bf16(q), bf16(k), bf16(v), cu, 0.1))
    rev = torch.zeros((n, Hkv, D + 8), dtype=torch.bfloat16, device="cuda")[:, :, :D]      # heads that are not adjacent
    with pytest.raises(ValueError):
        pa.packed_prefill(bf16(q), rev, bf16(v), cu, 0.1)
    with pytest.raises(ValueError):
        pa.packed_prefill(bf16(q), bf16(k)[:1].expand(n, Hkv, D), bf16(v), cu, 0.1)


@pytest.mark.parametrize("D", [64, 128])
def test_a_row_that_is_no_number_stays_alone(pa, rng, D):
    """An infinity or a NaN in one query makes that row's result no number and leaves the others as they were; so does one in
    another sequence's keys and values."""
    n, Hq, Hkv = 150, 4, 2
    q, k, v = (bf16(rng.standard_normal((n, h, D))) for h in (Hq, Hkv, Hkv))
    cu = dev(np.asarray([0, 90, n], np.int32))
    want = pa.packed_prefill(q, k, v, cu, 0.1)
    q2 = q.clone()
    q2[40, 1, 3] = float("nan")
    q2[70, 2, 5] = float("inf")
    got = pa.packed_prefill(q2, k, v, cu, 0.1)
    assert torch.isnan(got[40, 1]).all() and torch.isnan(got[70, 2]).all()
    got[40, 1], got[70, 2] = want[40, 1], want[70, 2]
    assert torch.equal(got, want)
    k[100], v[110] = float("inf"), float("nan")
    assert torch.equal(pa.packed_prefill(q, k, v, cu, 0.1)[:90], want[:90])


def test_many_boundaries_that_lie(pa, rng):
    """The same past the number of sequences that the ranking holds: a first boundary behind the first row, and one far out."""
    n, S, D = 900, 700, 64
    q, k, v = (bf16(rng.standard_normal((n, 2, D))) for _ in range(3))
    cu = np.sort(rng.integers(300, n, S + 1)).astype(np.int32)
    want = pa.packed_prefill(q, k, v, dev(cu), 0.1, out=torch.full_like(q, 3.0))
    assert (want[:cu[0]] == 3).all() and (want[cu[-1]:] == 3).all()
    for i in range(0, S, 97):
        a, z = int(cu[i]), int(cu[i + 1])
        one = pa.packed_prefill(q[a:z], k[a:z], v[a:z], dev(np.asarray([0, z - a], np.int32)), 0.1) if z > a else q[a:z]
        assert torch.equal(want[a:z], one)
    cu[[0, 350, 600]] = [-7, 2 ** 31 - 1, -2 ** 31]
    assert torch.isfinite(pa.packed_prefill(q, k, v, dev(cu), 0.1, out=torch.zeros_like(q))).all()


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 128), (4, 2, 64)])
def test_rows_past_32_bits(pa, rng, Hq, Hkv, D):
    """Rows of a tensor of 5 GB, on both sides of 2^31 elements and bytes, against the same rows packed closely."""
    stride, n = 1 << 16, 40000
    wide = torch.empty((n, stride), dtype=torch.bfloat16, device="cuda")
    dq, dk, dv = (wide[:, a:a + h * D].view(n, h, D) for a, h in ((0, Hq), (8192, Hkv), (16384, Hkv)))
    q, k, v = (torch.randn((n, h, D), device="cuda").to(torch.bfloat16) for h in (Hq, Hkv, Hkv))
    dq.copy_(q), dk.copy_(k), dv.copy_(v)
    cu = dev(np.asarray([0, 100, 16300, 16500, 32700, 32900, 39800, n], np.int32))
    lens = dev(np.asarray([100, 150, 200, 150, 200, 150, 200], np.int32))
    for kw in ({}, {"sliding_window": 64}):
        got = pa.packed_prefill(dq, dk, dv, cu, 0.1, query_lens=lens, seq_lens=lens, **kw)
        assert torch.equal(got, pa.packed_prefill(q, k, v, cu, 0.1, query_lens=lens, seq_lens=lens, **kw))


def test_empty_calls(pa):
    e = lambda n, h: torch.empty((n, h, 64), dtype=torch.bfloat16, device="cuda")      # noqa: E731
    i32 = lambda x: dev(np.asarray(x, np.int32))                                       # noqa: E731
    assert pa.packed_prefill(e(0, 4), e(0, 2), e(0, 2), i32([0]), 0.1).shape == (0, 4, 64)
    assert pa.packed_prefill(e(0, 4), e(0, 2), e(0, 2), i32([0, 0, 0]), 0.1).shape == (0, 4, 64)
    out = torch.full((5, 4, 64), 2.0, dtype=torch.bfloat16, device="cuda")
    assert (pa.packed_prefill(torch.ones_like(out), e(0, 2), e(0, 2), i32([0, 3]), 0.1, cu_seqlens_k=i32([0, 0]), out=out)[:3] == 0).all()
    assert (out[3:] == 2).all()
    out.fill_(2.0)
    assert (pa.packed_prefill(torch.ones_like(out), e(5, 2), e(5, 2), i32([3]), 0.1, out=out) == 2).all()


def test_refusals(pa):
    t = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device="cuda")          # noqa: E731
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    ok = (t(8, 4, 64), t(8, 2, 64), t(8, 2, 64), cu, 0.1)
    pa.packed_prefill(*ok)
    for bad in [(t(8, 4, 64, dt=torch.float32),) + ok[1:], (t(8, 3, 64),) + ok[1:], (t(8, 4, 96), t(8, 2, 96), t(8, 2, 96), cu, 0.1),
                (ok[0], t(8, 2, 128), t(8, 2, 128), cu, 0.1), (ok[0], t(9, 2, 64), t(9, 2, 64), cu, 0.1), ok[:3] + (cu.long(), 0.1),
                ok[:3] + (cu[None], 0.1), (ok[0], ok[1], t(8, 1, 64), cu, 0.1), (t(8, 4 * 64),) + ok[1:]]:
        with pytest.raises(ValueError):
            pa.packed_prefill(*bad)
    for kw in [{"cu_seqlens_k": cu[:1]}, {"query_lens": cu}, {"seq_lens": cu.long()[:1]}, {"max_seq_len": 0}, {"sliding_window": 0},
               {"sinks": t(3, dt=torch.float32)}, {"out": t(8, 4, 64, dt=torch.float32)}, {"out": t(9, 4, 64)}]:
        with pytest.raises(ValueError):
            pa.packed_prefill(*ok, **kw)
    with pytest.raises(NotImplementedError):
        pa.packed_prefill(ok[0], ok[1].cpu(), ok[2], cu, 0.1)
    odd = torch.zeros(8 * 4 * 64 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(8, 4, 64)
    with pytest.raises(ValueError):
        pa.packed_prefill(odd, *ok[1:])
