"""int8 paged cache on the GPU: quantising write (bit for bit), read-back (bit for bit), decode and verify (float64)."""
import numpy as np
import pytest
import torch

from oracle import paged_attention_oracle as O
from tests.int8_kv_lib import (assert_within, attention64, attention_tolerance, bf16, context, dev, int8_pool, quantise_rows,
                               random_tables)

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


def _rows(rng, *shape):
    return O.round_to_bf16((rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1] + (1,)))).astype(np.float32))


def _expect_write(pool, xk, xv, tables, seqs, qlens, bs, row_of):
    """NumPy write: row_of(b, t) -> index into the rows of xk / xv."""
    for x, c, s in ((xk, "k", "ks"), (xv, "v", "vs")):
        for b in range(len(seqs)):
            for t in range(int(qlens[b])):
                pos = int(seqs[b]) - int(qlens[b]) + t
                blk = tables[b, pos // bs] if pos >= 0 else -1
                if pos < 0 or int(seqs[b]) < int(qlens[b]) or not 0 <= blk < pool["blocks"]:
                    continue
                codes, sc = quantise_rows(x[row_of(b, t)])
                pool[c][blk, pos % bs] = codes
                pool[s][blk, :, pos % bs] = sc


def _stale(rng, blocks, bs, Hkv, D):
    return {"blocks": blocks, "k": rng.integers(-128, 128, (blocks, bs, Hkv, D)).astype(np.int8),
            "v": rng.integers(-128, 128, (blocks, bs, Hkv, D)).astype(np.int8),
            "ks": rng.random((blocks, Hkv, bs)).astype(np.float32), "vs": rng.random((blocks, Hkv, bs)).astype(np.float32)}


def _same(pool, d):
    for n in ("k", "v", "ks", "vs"):
        assert np.array_equal(d[n].cpu().numpy(), pool[n], equal_nan=n.endswith("s")), n


@pytest.mark.parametrize("D,bs,Hkv,T", [(128, 32, 8, 70), (64, 16, 8, 33), (128, 16, 1, 1), (64, 64, 3, 1), (32, 16, 5, 17),
                                        (256, 48, 2, 9), (128, 128, 20, 2)])
def test_write_bit_exact(pa, rng, D, bs, Hkv, T):
    B = 5
    qlens = np.asarray([T, max(T - 1, 0), 0, T, 1], np.int32)
    seqs = np.asarray([T, T + 2 * bs - 1, 40, T + 5, 1], np.int32)
    tables, blocks = random_tables(rng, seqs, bs)
    tables[3, 0] = blocks + 7                                  # a bad entry writes nothing
    pool = _stale(rng, blocks, bs, Hkv, D)
    xk, xv = _rows(rng, B, T, Hkv, D), _rows(rng, B, T, Hkv, D)
    xk[0, 0] = 0
    d = {n: dev(pool[n]) for n in ("k", "v", "ks", "vs")}
    pa.kv_write(bf16(xk), bf16(xv), d["k"], d["v"], dev(tables), dev(seqs), dev(qlens), k_scale=d["ks"], v_scale=d["vs"])
    _expect_write(pool, xk, xv, tables, seqs, qlens, bs, lambda b, t: (b, t))
    _same(pool, d)


@pytest.mark.parametrize("D,bs,Hkv", [(128, 32, 8), (64, 16, 5), (32, 16, 1), (256, 64, 2)])
@pytest.mark.parametrize("int8", [True, False])
def test_packed_write_of_strided_rows(pa, rng, D, bs, Hkv, int8):
    """Sequences of 0 .. 100 new rows, packed; k and v slices of one wide tensor; rows behind the last sequence unused."""
    qlens = np.asarray([37, 0, 1, 100, 16, 5], np.int32)
    cu = np.concatenate([[0], np.cumsum(qlens)]).astype(np.int32)
    seqs = qlens + np.asarray([0, 3, 64, 7, 200, 11], np.int32)
    used = qlens.copy()
    used[3] = 60                                               # fewer new tokens than the sequence has rows
    seqs[3] -= 40
    tables, blocks = random_tables(rng, seqs, bs)
    n = int(cu[-1]) + 9
    wide = _rows(rng, n, 2 * Hkv + 3, D)
    w = bf16(wide)
    k_new, v_new = w[:, 1:1 + Hkv], w[:, 2 + Hkv:2 + 2 * Hkv]
    xk, xv = wide[:, 1:1 + Hkv], wide[:, 2 + Hkv:2 + 2 * Hkv]
    pool = _stale(rng, blocks, bs, Hkv, D)
    row_of = lambda b, t: int(cu[b]) + t                       # noqa: E731
    args = (dev(tables), dev(seqs), dev(used))
    if int8:
        d = {m: dev(pool[m]) for m in ("k", "v", "ks", "vs")}
        pa.kv_write(k_new, v_new, d["k"], d["v"], *args, k_scale=d["ks"], v_scale=d["vs"], cu_seqlens=dev(cu))
        _expect_write(pool, xk, xv, tables, seqs, used, bs, row_of)
        _same(pool, d)
        return
    kc, vc = torch.zeros((blocks, bs, Hkv, D), dtype=torch.bfloat16, device="cuda"), torch.ones((blocks, bs, Hkv, D), dtype=torch.bfloat16, device="cuda")
    want_k, want_v = kc.clone(), vc.clone()
    pa.kv_write(k_new, v_new, kc, vc, *args, cu_seqlens=dev(cu))
    for b in range(len(seqs)):
        for t in range(int(used[b])):
            pos = int(seqs[b] - used[b]) + t
            want_k[tables[b, pos // bs], pos % bs] = k_new[cu[b] + t]
            want_v[tables[b, pos // bs], pos % bs] = v_new[cu[b] + t]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_write_of_extreme_rows(pa, rng):
    """Subnormal rows, the largest finite values, ties, infinities and NaN; the scales next to the reciprocal form's edges."""
    D, bs, Hkv = 128, 16, 1
    rows = [np.full(D, 0.0), np.full(D, 2.0 ** -133), np.full(D, 3.3e38), np.linspace(-127, 127, D),
            np.where(np.arange(D) % 2, 63.5, 127.0), np.r_[np.inf, np.ones(D - 1)], np.r_[np.ones(D - 1), np.nan],
            np.r_[-np.inf, np.nan, np.zeros(D - 2)], np.full(D, -0.0), np.r_[1e-38, np.full(D - 1, 1e-41)],
            127 * 2.0 ** -40 * np.linspace(-1, 1, D), 127 * 2.0 ** 40 * np.linspace(-1, 1, D)]
    x = O.round_to_bf16(np.asarray(rows, np.float32)).reshape(1, len(rows), Hkv, D)
    n = len(rows)
    tables, blocks = random_tables(rng, [n], bs)
    pool = _stale(rng, blocks, bs, Hkv, D)
    d = {m: dev(pool[m]) for m in ("k", "v", "ks", "vs")}
    one = np.asarray([n], np.int32)
    xb = torch.from_numpy(O.f32_to_bf16_bits(x).view(np.int16).copy()).cuda().view(torch.bfloat16)
    pa.kv_write(xb, xb.flip(1).contiguous(), d["k"], d["v"], dev(tables), dev(one), dev(one), k_scale=d["ks"], v_scale=d["vs"])
    _expect_write(pool, x, x[:, ::-1], tables, one, one, bs, lambda b, t: (b, t))
    _same(pool, d)
    k, v = pa.read_kv(d["k"], d["v"], dev(tables), dev(one), dev(np.asarray([0, n], np.int32)), n, k_scale=d["ks"], v_scale=d["vs"])
    bad = ~np.isfinite(x[0, :, 0]).all(-1)
    assert torch.isnan(k[:, 0]).all(-1).cpu().numpy().tolist() == bad.tolist()
    assert torch.isnan(v[:, 0]).all(-1).cpu().numpy().tolist() == bad[::-1].tolist()


@pytest.mark.parametrize("D,norm", [(64, True), (128, True), (256, False)])
def test_fused_norm_rope_write(pa, rng, D, norm):
    """The transforming write into an int8 pool holds the codes of what it writes into a bf16 pool."""
    B, T, Hq, Hkv, bs = 3, 21, 6, 3, 16
    qlens, seqs = np.asarray([21, 4, 0], np.int32), np.asarray([40, 4, 9], np.int32)
    tables, blocks = random_tables(rng, seqs, bs)
    xq, xk, xv = (bf16(_rows(rng, B, T, h, D)) for h in (Hq, Hkv, Hkv))
    cos, sin = pa.rope_tables(D, 64, 1e4)
    w = bf16(rng.random(D) + 0.5) if norm else None
    kc = torch.zeros((blocks, bs, Hkv, D), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    args = (dev(tables), dev(seqs), dev(qlens), cos, sin)
    q_ref = pa.qk_norm_rope_kv_write(xq, xk, xv, kc, vc, *args, q_norm_weight=w, k_norm_weight=w)
    k8, v8 = torch.zeros(kc.shape, dtype=torch.int8, device="cuda"), torch.zeros(kc.shape, dtype=torch.int8, device="cuda")
    ks, vs = torch.zeros((blocks, Hkv, bs), device="cuda"), torch.zeros((blocks, Hkv, bs), device="cuda")
    q = pa.qk_norm_rope_kv_write(xq, xk, xv, k8, v8, *args, q_norm_weight=w, k_norm_weight=w, k_scale=ks, v_scale=vs)
    assert torch.equal(q, q_ref)
    for c16, c8, s in ((kc, k8, ks), (vc, v8, vs)):
        codes, scale = quantise_rows(c16.float().cpu().numpy())
        live = np.zeros((blocks, bs), bool)
        for b in range(B):
            for pos in range(int(seqs[b] - qlens[b]), int(seqs[b])):
                live[tables[b, pos // bs], pos % bs] = True
        assert np.array_equal(c8.cpu().numpy()[live], codes[live])
        assert np.array_equal(s.cpu().numpy().transpose(0, 2, 1)[live], scale[live])


@pytest.mark.parametrize("kind", ["int8", "fp8", "bf16"])
@pytest.mark.parametrize("D,bs,Hkv", [(128, 32, 8), (64, 16, 3), (8, 5, 1), (96, 48, 7)])
def test_read_back_bit_exact(pa, rng, kind, D, bs, Hkv):
    """Gaps between the sequences' rows, a sequence with more tokens than rows, empty ones, a bad table entry, rows behind
    the last sequence: what no token falls on stays as it was."""
    seqs = np.asarray([70, 0, 1, 33, 130, 17], np.int32)
    room = [70, 4, 5, 20, 130, 17]
    cu = np.concatenate([[0], np.cumsum(room)]).astype(np.int32)
    tables, blocks = random_tables(rng, seqs, bs)
    tables[5, 0] = -3
    n = int(cu[-1]) + 21
    if kind == "bf16":
        pools = [bf16(rng.standard_normal((blocks, bs, Hkv, D))) for _ in range(2)]
        vals, kw = [p.float().cpu().numpy() for p in pools], {}
    else:
        raw = [rng.integers(0, 256, (blocks, bs, Hkv, D)).astype(np.uint8) for _ in range(2)]
        shape = (blocks, Hkv) if kind == "fp8" else (blocks, Hkv, bs)
        scales = [rng.random(shape).astype(np.float32) for _ in range(2)]
        if kind == "fp8":
            for r in raw:
                r[(r & 0x7f) == 0x7f] = 0x31
            pools = [dev(r).view(torch.float8_e4m3fn) for r in raw]
            vals = [p.float().cpu().numpy() * s[:, None, :, None] for p, s in zip(pools, scales)]
        else:
            pools = [dev(r.view(np.int8)) for r in raw]
            vals = [r.view(np.int8).astype(np.float32) * s.transpose(0, 2, 1)[..., None] for r, s in zip(raw, scales)]
        kw = {"k_scale": dev(scales[0]), "v_scale": dev(scales[1])}
    out = tuple(torch.full((n, Hkv, D), x, dtype=torch.bfloat16, device="cuda") for x in (7.0, -7.0))
    want = [o.clone() for o in out]
    got = pa.read_kv(*pools, dev(tables), dev(seqs), dev(cu), out=out, **kw)
    assert got[0].data_ptr() == out[0].data_ptr()
    for w, val in zip(want, vals):
        for b in range(len(seqs)):
            for t in range(min(int(seqs[b]), room[b])):
                blk = tables[b, t // bs]
                row = val[blk, t % bs] if 0 <= blk < blocks else np.zeros((Hkv, D), np.float32)
                w[cu[b] + t] = torch.from_numpy(row).to(torch.bfloat16)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    fresh = pa.read_kv(*pools, dev(tables), dev(seqs), dev(cu), n, **kw)
    for b in range(len(seqs)):
        a, z = int(cu[b]), int(cu[b]) + min(int(seqs[b]), room[b])
        assert torch.equal(fresh[0][a:z], want[0][a:z]) and torch.equal(fresh[1][a:z], want[1][a:z])


def _decode_case(pa, rng, ctxs, Hq, Hkv, D, bs, T=1, qlens=None, window=None, with_sinks=False, bound=None, size=1.0, **kw):
    pool = int8_pool(rng, ctxs, bs, Hkv, D, spread=0.5)
    B = len(ctxs)
    q = O.round_to_bf16(rng.standard_normal((B, T, Hq, D)).astype(np.float32)) * np.float32(size)
    pool["ks"] /= np.float32(size)
    scale = 1.0 / np.sqrt(D)
    sinks = rng.standard_normal(Hq).astype(np.float32) if with_sinks else None
    args = (dev(pool["k"]), dev(pool["v"]), dev(pool["tables"]), dev(np.asarray(ctxs, np.int32)))
    kw.update(k_scale=dev(pool["ks"]), v_scale=dev(pool["vs"]), max_seq_len=bound, sinks=None if sinks is None else dev(sinks),
              sliding_window=window)
    if qlens is None:
        got = pa.decode(bf16(q[:, 0]), *args, scale, **kw)[:, None]
        qlens = [1] * B
    else:
        got = pa.verify(bf16(q), *args, dev(np.asarray(qlens, np.int32)), scale, **kw)
    want, tol = np.zeros((B, T, Hq, D)), np.zeros((B, T, Hq, D))
    for b, c in enumerate(ctxs):
        n = min(qlens[b], c)
        if n == 0:
            continue
        o, mag, reach = attention64(q[b, :n].astype(np.float64), context(pool, "k", b, c, bs), context(pool, "v", b, c, bs), scale,
                                    c - n, window or 0, sinks)
        want[b, :n], tol[b, :n] = o, attention_tolerance(o, mag, reach, D)
        if size < 2.0 ** -105:
            # A row's step is its largest element / 32 512, but not below 2^-120 (the step's reciprocal has to have one
            # itself): every element may be off by 2^-121, a score by that times sum |k| scale, and a probability and the sum
            # it is divided by by twice the score's error, relatively.
            off = 2.0 ** -121 * np.abs(context(pool, "k", b, c, bs)).sum(-1).max() * scale
            tol[b, :n] += np.expm1(2 * off) * mag
    assert_within(got, want, tol)
    return got


@pytest.mark.parametrize("bound", [64, 700, 1024, 2500])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (16, 4, 64), (12, 1, 128)])
def test_decode_with_a_bound(pa, rng, Hq, Hkv, D, bound):
    """The kernels a length bound chooses: one partition on eight waves, several, the balanced schedule."""
    _decode_case(pa, rng, [1, 0, 31, bound, bound // 2 + 1, 33], Hq, Hkv, D, 64, bound=bound)


def test_refusals(pa):
    t = lambda *s, dt=torch.int8: torch.zeros(s, dtype=dt, device="cuda")              # noqa: E731
    kc, sc = t(4, 16, 2, 64), t(4, 2, 16, dt=torch.float32)
    tb, ln = t(1, 4, dt=torch.int32), t(1, dt=torch.int32)
    q, x = t(1, 4, 64, dt=torch.bfloat16), t(1, 3, 2, 64, dt=torch.bfloat16)
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    fp8_scale = t(4, 2, dt=torch.float32)
    pa.decode(q, kc, kc, tb, ln, 0.1, k_scale=sc, v_scale=sc)
    for kw in [{}, {"k_scale": sc}, {"k_scale": fp8_scale, "v_scale": fp8_scale}, {"k_scale": sc.double(), "v_scale": sc.double()}]:
        for call in (lambda **k: pa.decode(q, kc, kc, tb, ln, 0.1, **k), lambda **k: pa.kv_write(x, x, kc, kc, tb, ln, ln, **k),
                     lambda **k: pa.read_kv(kc, kc, tb, ln, cu, 3, **k), lambda **k: pa.verify(x.repeat(1, 1, 2, 1), kc, kc, tb, ln, ln, 0.1, **k)):
            with pytest.raises(ValueError):
                call(**kw)
    s = {"k_scale": sc, "v_scale": sc}
    long = t(1, 65, 4, 64, dt=torch.bfloat16)
    odd = t(4, 24, 2, 64)
    odd_s = t(4, 2, 24, dt=torch.float32)
    for call in (lambda: pa.prefill(long, kc, kc, tb, ln, ln, 0.1, **s), lambda: pa.prefill(long[:, :4].contiguous(), kc, kc, tb, ln, ln, 0.1, route="tiled", **s),
                 lambda: pa.decode(q, odd, odd, tb, ln, 0.1, k_scale=odd_s, v_scale=odd_s), lambda: pa.decode(q.float(), kc, kc, tb, ln, 0.1, **s),
                 lambda: pa.read_kv(kc, kc, tb, ln, cu, **s), lambda: pa.read_kv(kc, kc, tb, ln, cu, -1, **s), lambda: pa.read_kv(kc, kc, tb, ln, cu.long(), 3, **s),
                 lambda: pa.read_kv(kc, kc, tb, ln, cu, 3, out=(x[0], x[0].float()), **s), lambda: pa.read_kv(kc, kc, tb, ln, cu, 4, out=(x[0], x[0]), **s),
                 lambda: pa.read_kv(kc.float(), kc.float(), tb, ln, cu, 3), lambda: pa.kv_write(x, x, kc, kc, tb, ln, ln, cu_seqlens=cu, **s),
                 lambda: pa.kv_write(x[0], x[0], kc, kc, tb, ln, ln, cu_seqlens=cu[:1], **s),
                 lambda: pa.kv_write(x[0], x[0], kc.view(torch.float8_e4m3fn), kc.view(torch.float8_e4m3fn), tb, ln, ln, cu_seqlens=cu, k_scale=fp8_scale, v_scale=fp8_scale)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("impl", [0, 2, 3])
@pytest.mark.parametrize("Hq,Hkv,D,bs", [(32, 8, 128, 32), (8, 8, 64, 16), (40, 2, 128, 16), (7, 1, 64, 64), (6, 3, 128, 128)])
def test_decode(pa, rng, debug_switch, Hq, Hkv, D, bs, impl):
    debug_switch(0, impl)
    _decode_case(pa, rng, [1, 0, 31, 32, 33, 700, 16, 1500], Hq, Hkv, D, bs)


@pytest.mark.parametrize("impl", [0, 2, 3])
@pytest.mark.parametrize("window", [1, 7, 100])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_window_and_sinks(pa, rng, debug_switch, impl, window, D):
    debug_switch(0, impl)
    _decode_case(pa, rng, [1, 99, 101, 600, 0], 16, 4, D, 16, window=window, with_sinks=True)


@pytest.mark.parametrize("bound", [None, 1024])
@pytest.mark.parametrize("Hq,Hkv,D,T", [(32, 8, 128, 4), (64, 8, 64, 3), (8, 1, 128, 8), (8, 2, 64, 33), (16, 1, 128, 5)])
def test_verify(pa, rng, Hq, Hkv, D, T, bound):
    qlens = [T, 1, 0, min(T, 2), T]
    _decode_case(pa, rng, [T, 500, 40, 1000, T + 31], Hq, Hkv, D, 32, T=T, qlens=qlens, bound=bound)


@pytest.mark.parametrize("size", [2.0 ** -118, 2.0 ** -110, 2.0 ** -103, 2.0 ** -60, 2.0 ** 60, 2.0 ** 114])
def test_queries_of_any_size(pa, rng, size):
    """A query's size cancels against the keys': sizes near either end of the type's range take the same way."""
    _decode_case(pa, rng, [1, 33, 700], 8, 2, 128, 16, size=size)


def test_the_largest_queries(pa, rng):
    """An element near the type's largest number, on a channel where all keys are zero: all scores are zero."""
    D, bs, c = 128, 16, 300
    pool = int8_pool(rng, [c], bs, 2, D)
    pool["k"][..., 5] = 0
    q = np.zeros((1, 8, D), np.float32)
    q[..., 5] = O.round_to_bf16(np.float32(3.3e38) * rng.uniform(0.26, 1.0, (1, 8)).astype(np.float32))
    got = pa.decode(bf16(q), dev(pool["k"]), dev(pool["v"]), dev(pool["tables"]), dev(np.asarray([c], np.int32)), 0.1,
                    k_scale=dev(pool["ks"]), v_scale=dev(pool["vs"]))
    o, mag, reach = attention64(q.astype(np.float64), context(pool, "k", 0, c, bs), context(pool, "v", 0, c, bs), 0.1, c - 1)
    assert reach == 0.0
    assert_within(got, o, attention_tolerance(o, mag, reach, D))


@pytest.mark.parametrize("rows", [16, 32])
def test_verify_rows_per_wave(pa, rng, debug_switch, rows):
    debug_switch(5, rows)
    try:
        _decode_case(pa, rng, [300, 1000, 64], 32, 4, 128, 32, T=4, qlens=[4, 3, 4], window=200, with_sinks=True)
        _decode_case(pa, rng, [300, 1000, 64], 32, 4, 64, 32, T=4, qlens=[4, 3, 4])
    finally:
        debug_switch(5, 0)


@pytest.mark.parametrize("Hq,Hkv,D,T,B", [(64, 8, 64, 4, 8), (64, 8, 64, 1, 16), (32, 8, 128, 8, 16), (32, 2, 128, 16, 16), (40, 4, 64, 3, 24), (9, 3, 64, 8, 32), (16, 1, 128, 8, 16)])
def test_slots_that_share_lines(pa, rng, debug_switch, Hq, Hkv, D, T, B):
    """Where the head slots that read the same lines go to one XCD (calls of at least 128 workgroups), the results are those
    of the other grid order bit for bit, for every pool type."""
    ctxs = [1024] + [int(c) for c in rng.integers(T, 1024, B - 1)]
    pool = int8_pool(rng, ctxs, 32, Hkv, D)
    q = bf16(rng.standard_normal((B, T, Hq, D)))
    tables, lens, qlens = dev(pool["tables"]), dev(np.asarray(ctxs, np.int32)), dev(np.asarray([T - (i % 2) * (T > 1) for i in range(B)], np.int32))
    codes = [dev(pool[n]) for n in "kv"]
    pools = [(codes, {"k_scale": dev(pool["ks"]), "v_scale": dev(pool["vs"])}), ([c.to(torch.bfloat16) for c in codes], {}),
             ([c.view(torch.uint8).bitwise_and(0x77).view(torch.float8_e4m3fn) for c in codes],
              {n: torch.full((pool["blocks"], Hkv), 0.02, device="cuda") for n in ("k_scale", "v_scale")})]
    for kv, scales in pools:
        got = []
        for order in (1, 0):
            debug_switch(2, order)
            try:
                got.append(pa.decode(q[:, 0].contiguous(), *kv, tables, lens, 0.05, max_seq_len=1024, **scales) if T == 1 else
                           pa.verify(q, *kv, tables, lens, qlens, 0.05, max_seq_len=1024, **scales))
            finally:
                debug_switch(2, 1)
        assert torch.isfinite(got[0]).all() and torch.equal(*got)


def test_a_masked_token_of_any_scale_leaves_no_trace(pa, rng):
    """Tokens that a window hides may have NaN scales (a row that held an infinity): they must not reach the result."""
    D, bs, Hkv, Hq, c = 128, 16, 2, 8, 300
    pool = int8_pool(rng, [c], bs, Hkv, D)
    for pos in range(0, c - 40):
        pool["ks"][pool["tables"][0, pos // bs], :, pos % bs] = np.nan
        pool["vs"][pool["tables"][0, pos // bs], :, pos % bs] = np.inf
    q = O.round_to_bf16(rng.standard_normal((1, Hq, D)).astype(np.float32))
    got = pa.decode(bf16(q), dev(pool["k"]), dev(pool["v"]), dev(pool["tables"]), dev(np.asarray([c], np.int32)), 0.1,
                    k_scale=dev(pool["ks"]), v_scale=dev(pool["vs"]), sliding_window=40)
    k, v = context(pool, "k", 0, c, bs)[-40:], context(pool, "v", 0, c, bs)[-40:]
    o, mag, reach = attention64(q.astype(np.float64), k, v, 0.1, 39)
    assert_within(got, o, attention_tolerance(o, mag, reach, D))


def test_many_sequences_and_bad_tables(pa, rng):
    """More than 512 sequences (their own launch for the tile sums); table entries outside the pool are clamped, not followed."""
    ctxs = [int(x) for x in rng.integers(0, 60, 700)]
    _decode_case(pa, rng, ctxs, 8, 2, 64, 16)
    pool = int8_pool(rng, [100], 16, 2, 128)
    tables = pool["tables"].copy()
    tables[0, :4] = [-5, 1 << 30, 2 ** 31 - 1, -2 ** 31]
    out = pa.decode(bf16(rng.standard_normal((1, 8, 128))), dev(pool["k"]), dev(pool["v"]), dev(tables), dev(np.asarray([100], np.int32)), 0.1,
                    k_scale=dev(np.nan_to_num(pool["ks"])), v_scale=dev(np.nan_to_num(pool["vs"])))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("D", [64, 128])
def test_steps_equal_the_separate_calls(pa, rng, T, D):
    """decode_step / verify_step over an int8 pool, with the transform and the projection, against the three calls."""
    B, Hq, Hkv, bs, N = 4, 8, 2, 16, 128
    seqs = np.asarray([T, 200, 33 + T, 700], np.int32)
    qlens = np.asarray([T, T, 0, 1], np.int32)
    pool = int8_pool(rng, [int(s) for s in seqs], bs, Hkv, D)
    cos, sin = pa.rope_tables(D, 1024, 1e4)
    w = bf16(rng.random(D) + 0.5)
    qt = pa.QTransform(cos, sin, w)
    xq, xk, xv = (bf16(_rows(rng, B, T, h, D)) for h in (Hq, Hkv, Hkv))
    ow, ob = bf16(rng.standard_normal((Hq * D, N)) * 0.05), bf16(rng.standard_normal(N))
    res = []
    for one in (True, False):
        kc, vc, ks, vs = (dev(pool[n]) for n in ("k", "v", "ks", "vs"))
        tail = (dev(pool["tables"]), dev(seqs), dev(qlens))
        kw = dict(k_scale=ks, v_scale=vs)
        if one and T == 1:
            out = pa.decode_step(xq[:, 0].contiguous(), xk[:, 0].contiguous(), xv[:, 0].contiguous(), kc, vc, *tail, 0.1, q_transform=qt,
                                 k_norm_weight=w, o_weight=ow, o_bias=ob, max_seq_len=704, **kw)
        elif one:
            out = pa.verify_step(xq, xk, xv, kc, vc, *tail, 0.1, q_transform=qt, k_norm_weight=w, o_weight=ow, o_bias=ob, max_seq_len=704, **kw)
        else:
            pa.qk_norm_rope_kv_write(None, xk, xv, kc, vc, *tail, cos, sin, k_norm_weight=w, **kw)
            if T == 1:
                a = pa.decode(xq[:, 0].contiguous(), kc, vc, tail[0], tail[1], 0.1, q_transform=qt, max_seq_len=704, **kw)
            else:
                a = pa.verify(xq, kc, vc, *tail, 0.1, q_transform=qt, max_seq_len=704, **kw)
            out = pa.o_proj(a, ow, ob)
        res.append((out, kc, vc, ks.nan_to_num(nan=-1.0), vs.nan_to_num(nan=-1.0)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_graph_replays_and_other_streams(pa, rng):
    """Write, decode and read-back captured into a graph and replayed with other rows, eager work and waits in between;
    the same calls on a stream that is not the current one's default."""
    D, bs, Hkv, Hq, B = 128, 16, 4, 16, 3
    seqs = np.asarray([50, 400, 17], np.int32)
    pool = int8_pool(rng, [int(s) for s in seqs], bs, Hkv, D)
    kc, vc, ks, vs = (dev(pool[n]) for n in ("k", "v", "ks", "vs"))
    tables, sl, ql = dev(pool["tables"]), dev(seqs), dev(np.ones(B, np.int32))
    cu = dev(np.concatenate([[0], np.cumsum(seqs)]).astype(np.int32))
    n = int(seqs.sum())
    q, xk, xv = (torch.zeros((B, h, D), dtype=torch.bfloat16, device="cuda") for h in (Hq, Hkv, Hkv))
    kw = dict(k_scale=ks, v_scale=vs)

    def step():
        pa.kv_write(xk[:, None], xv[:, None], kc, vc, tables, sl, ql, **kw)
        return pa.decode(q, kc, vc, tables, sl, 0.1, **kw), pa.read_kv(kc, vc, tables, sl, cu, n, **kw)

    for x in (q, xk, xv):
        x.copy_(bf16(_rows(rng, *x.shape)))
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, (k, v) = step()
    for i in range(4):
        for x in (q, xk, xv):
            x.copy_(bf16(_rows(rng, *x.shape)))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, k, v)]
        if i % 2:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                o2, (k2, v2) = step()
            torch.cuda.current_stream().wait_stream(s)
        else:
            o2, (k2, v2) = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], o2) and torch.equal(got[1], k2) and torch.equal(got[2], v2)


def test_offsets_past_32_bits(pa, rng):
    """A pool of more than 2^31 bytes: writes to, reads from and decodes over its last blocks."""
    D, bs, Hkv, Hq = 128, 64, 8, 32
    blocks = (2 ** 32) // (bs * Hkv * D) + 40
    kc = torch.zeros((blocks, bs, Hkv, D), dtype=torch.int8, device="cuda")
    vc = torch.zeros_like(kc)
    ks, vs = (torch.full((blocks, Hkv, bs), float("nan"), device="cuda") for _ in range(2))
    n = 150
    tables = np.asarray([[blocks - 1, blocks - 7, 3, -1]], np.int32)
    one = dev(np.asarray([n], np.int32))
    xk, xv = _rows(rng, 1, n, Hkv, D), _rows(rng, 1, n, Hkv, D)
    pa.kv_write(bf16(xk), bf16(xv), kc, vc, dev(tables), one, one, k_scale=ks, v_scale=vs)
    (ck, sk), (cv, sv) = quantise_rows(xk[0]), quantise_rows(xv[0])
    k, v = pa.read_kv(kc, vc, dev(tables), one, dev(np.asarray([0, n], np.int32)), n, k_scale=ks, v_scale=vs)
    want = [torch.from_numpy(c.astype(np.float32) * s[..., None]).to(torch.bfloat16) for c, s in ((ck, sk), (cv, sv))]
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])
    q = O.round_to_bf16(rng.standard_normal((1, Hq, D)).astype(np.float32))
    got = pa.decode(bf16(q), kc, vc, dev(tables), one, 0.09, k_scale=ks, v_scale=vs)
    o, mag, reach = attention64(q.astype(np.float64), ck.astype(np.float64) * sk[..., None].astype(np.float64),
                                cv.astype(np.float64) * sv[..., None].astype(np.float64), 0.09, n - 1)
    assert_within(got, o, attention_tolerance(o, mag, reach, D))
