"""The engine over an int8 cache: prompts in chunks, verify and decode steps, forks, graphs; the new operators through the
dispatcher and under the name-keyed convention; a serving run of them together against float64."""
import numpy as np
import pytest
import torch

from tests.int8_kv_lib import assert_within, attention64, attention_tolerance, bf16, dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pa():
    import nkipy_amd
    from nkipy_amd import _lib
    _lib.load()
    return nkipy_amd


def _engine(D, bs, Hq, Hkv, slots, dtype=torch.int8, rope=True, norm=True, seed=3, **kw):
    from nkipy_amd.engine import PagedAttention, PagedKVCache
    cache = PagedKVCache(200, bs, Hkv, D, max_seqs=slots, max_blocks_per_seq=40, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = lambda n: (torch.rand(n, generator=g, device="cuda") + 0.5).to(torch.bfloat16)         # noqa: E731
    layer = PagedAttention(cache, Hq, rope_base=1e4 if rope else None, max_positions=40 * bs if rope else 0,
                           q_norm_weight=w(D) if rope and norm else None, k_norm_weight=w(D) if rope and norm else None, **kw)
    return cache, layer


def _rows(g, slots, T, Hq, Hkv, D):
    return tuple(torch.randn((slots, T, h, D), generator=g, device="cuda").to(torch.bfloat16) for h in (Hq, Hkv, Hkv))


STEPS = [(150, [150, 0, 90]), (130, [130, 70, 0]), (100, [0, 100, 64]), (3, [3, 3, 1]), (1, [1, 1, 1]), (1, [0, 1, 1])]


@pytest.mark.parametrize("D,bs,Hq,Hkv", [(128, 32, 16, 4), (64, 16, 16, 4), (128, 16, 8, 8)])
@pytest.mark.parametrize("variant", [{}, {"sinks": True, "sliding_window": 70}])
def test_steps_against_a_bfloat16_cache(pa, D, bs, Hq, Hkv, variant):
    """Chunks (written, read back, attended to packed), verify and decode steps; a bfloat16 cache given the same rows differs by
    what the codes differ: at most half a step of absmax / 127, 0.4 % of a row's largest value."""
    variant = dict(variant)
    if variant.pop("sinks", None):
        variant["sinks"] = torch.linspace(-1, 1, Hq, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(11)
    both = [_engine(D, bs, Hq, Hkv, 3, dtype=dt, **variant) for dt in (torch.int8, torch.bfloat16)]
    for T, lens in STEPS:
        xq, xk, xv = _rows(g, 3, T, Hq, Hkv, D)
        outs = [layer.step(xq.clone(), xk.clone(), xv.clone(), lens).clone() for _, layer in both]
        for b, n in enumerate(lens):
            assert torch.isfinite(outs[0][b, :n]).all()
            d = (outs[0][b, :n].float() - outs[1][b, :n].float()).abs().max() if n else 0.0
            assert d <= 5e-2, (T, b, float(d))
            if T > 1:
                assert (outs[0][b, n:] == 0).all()


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 8, 2)])
def test_a_serving_run_against_float64(pa, rng, D, Hq, Hkv):
    """Prompt without a prefix (packed, its rows written packed), a chunk behind it through the read-back, verify, decode: each
    against float64 on the values that the cache stands for."""
    bs, scale = 16, 1.0 / np.sqrt(D)
    total = [60, 33]
    blocks = 40
    perm = rng.permutation(blocks).astype(np.int32)
    tables = dev(np.stack([perm[:12], perm[12:24]]))
    kc, vc = (torch.zeros((blocks, bs, Hkv, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((blocks, Hkv, bs), float("nan"), device="cuda") for _ in range(2))
    sc = dict(k_scale=ks, v_scale=vs)
    i32 = lambda x: dev(np.asarray(x, np.int32))               # noqa: E731
    cum = lambda x: i32(np.concatenate([[0], np.cumsum(x)]))   # noqa: E731

    def held(lens):
        """float64 rows of the two contexts as the cache holds them (codes x scales)."""
        out = []
        for b, c in enumerate(lens):
            ids = tables[b, :(c + bs - 1) // bs].long()
            out.append([(x[ids].double() * s[ids].double().transpose(1, 2)[..., None]).flatten(0, 1)[:c].cpu().numpy() for x, s in ((kc, ks), (vc, vs))])
        return out

    # the prompts: attention on the rows themselves, and the write
    q, k, v = (bf16(rng.standard_normal((sum(total), h, D))) for h in (Hq, Hkv, Hkv))
    cu = cum(total)
    got = pa.packed_prefill(q, k, v, cu, scale)
    pa.kv_write(k, v, kc, vc, tables, i32(total), i32(total), cu_seqlens=cu, **sc)
    at = 0
    for b, n in enumerate(total):
        o, mag, reach = attention64(*(x[at:at + n].double().cpu().numpy() for x in (q, k, v)), scale, 0)
        assert_within(got[at:at + n], o, attention_tolerance(o, mag, reach, D))
        at += n
    # a chunk of new tokens behind them
    new = [70, 40]
    lens = [a + b for a, b in zip(total, new)]
    q, k, v = (bf16(rng.standard_normal((sum(new), h, D))) for h in (Hq, Hkv, Hkv))
    pa.kv_write(k, v, kc, vc, tables, i32(lens), i32(new), cu_seqlens=cum(new), **sc)
    k2, v2 = pa.read_kv(kc, vc, tables, i32(lens), cum(lens), sum(lens), **sc)
    got = pa.packed_prefill(q, k2, v2, cum(new), scale, cu_seqlens_k=cum(lens), max_seq_len=max(lens))
    at = 0
    for b, (kk, vv) in enumerate(held(lens)):
        o, mag, reach = attention64(q[at:at + new[b]].double().cpu().numpy(), kk, vv, scale, total[b])
        # the rows read back are rounded once (half a bf16 step of every k and v)
        tol = attention_tolerance(o, mag, reach, D) + (2.0 ** -8 + np.expm1(2 * 2.0 ** -8 * reach)) * mag
        assert_within(got[at:at + new[b]], o, tol)
        at += new[b]
    # verify of two tokens, then a decode step
    for T in (2, 1):
        lens = [c + T for c in lens]
        q, k, v = (bf16(rng.standard_normal((2, T, h, D))) for h in (Hq, Hkv, Hkv))
        if T == 2:
            got = pa.verify_step(q, k, v, kc, vc, tables, i32(lens), i32([T, T]), scale, **sc)
        else:
            got = pa.decode_step(q[:, 0].contiguous(), k[:, 0].contiguous(), v[:, 0].contiguous(), kc, vc, tables, i32(lens), i32([1, 1]), scale, **sc)[:, None]
        for b, (kk, vv) in enumerate(held(lens)):
            o, mag, reach = attention64(q[b].double().cpu().numpy(), kk, vv, scale, lens[b] - T)
            assert_within(got[b], o, attention_tolerance(o, mag, reach, D))


def test_projection_fork_and_release(pa):
    D, bs, Hq, Hkv = 128, 16, 8, 2
    w = bf16(np.random.default_rng(0).standard_normal((Hq * D, 64)) * 0.05)
    cache, layer = _engine(D, bs, Hq, Hkv, 2, o_weight=w)
    g = torch.Generator(device="cuda").manual_seed(1)
    assert layer.step(*_rows(g, 2, 90, Hq, Hkv, D), [90, 0]).shape == (2, 90, 64)
    cache.fork(0, 1)
    x = _rows(g, 2, 1, Hq, Hkv, D)
    x = tuple(t[:1].expand_as(t).contiguous() for t in x)
    out = layer.step(*x, [1, 1])
    assert torch.equal(out[0], out[1])                          # the fork holds the same codes and scales
    assert layer.step(*_rows(g, 2, 100, Hq, Hkv, D), [100, 0])[0].isfinite().all()
    cache.release(0)
    assert layer.step(*_rows(g, 2, 1, Hq, Hkv, D), [0, 1])[1].isfinite().all()


def test_a_captured_chunk_replays_on_other_lengths(pa):
    """A chunk over an int8 cache captured once and replayed for chunks of other lengths behind other prefixes."""
    D, bs, Hq, Hkv, T = 64, 16, 8, 2, 100
    g = torch.Generator(device="cuda").manual_seed(2)
    (cache, layer), (c2, l2) = (_engine(D, bs, Hq, Hkv, 3) for _ in range(2))
    x = _rows(g, 3, T, Hq, Hkv, D)
    lens = [100, 30, 0]
    cache.begin_step(lens, T)
    c2.begin_step(lens, T)
    layer.attend(*x, max_seq_len=400)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.attend(*x, max_seq_len=400)
    for lens in ([100, 30, 0], [50, 0, 100], [100, 100, 1], [0, 99, 77]):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(torch.bfloat16))
        if lens != [100, 30, 0]:
            cache.begin_step(lens, T)
            c2.begin_step(lens, T)
        graph.replay()
        want = l2.attend(*(t.clone() for t in x), max_seq_len=400)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_dispatcher_and_named_kernels(pa, rng):
    import nkipy_amd.torch_ops  # noqa: F401
    from nkipy_amd.runtime import DeviceKernel, DeviceTensor
    D, bs, Hq, Hkv = 64, 16, 4, 2
    n = [40, 21]
    q, k, v = (bf16(rng.standard_normal((sum(n), h, D))) for h in (Hq, Hkv, Hkv))
    cu = dev(np.asarray([0, 40, 61], np.int32))
    want = pa.packed_prefill(q, k, v, cu, 0.1, sliding_window=9)
    out = torch.empty_like(q)
    torch.ops.nkipy_amd.packed_prefill(q, k, v, cu, 0.1, out, sliding_window=9)
    assert torch.equal(out, want)
    kern = DeviceKernel.compile_and_load("packed_prefill", q=q, k=k, v=v, cu_seqlens=cu, scale=0.1, sliding_window=9)
    got = kern(inputs={"q": DeviceTensor(q), "k": DeviceTensor(k), "v": DeviceTensor(v), "cu_seqlens": DeviceTensor(cu)})
    assert torch.equal(got.tensor, want)
    tables, lens = dev(np.asarray([[0, 1, 2], [3, 4, 5]], np.int32)), dev(np.asarray(n, np.int32))
    kc, vc = (torch.zeros((6, bs, Hkv, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((6, Hkv, bs), device="cuda") for _ in range(2))
    torch.ops.nkipy_amd.paged_kv_write_int8(k, v, kc, vc, ks, vs, tables, lens, lens, cu)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    torch.ops.nkipy_amd.read_kv(kc, vc, tables, lens, cu, ko, vo, ks, vs)
    k2, v2 = pa.read_kv(kc, vc, tables, lens, cu, 61, k_scale=ks, v_scale=vs)
    assert torch.equal(ko, k2) and torch.equal(vo, v2)
    assert (k2.float() - k.float()).abs().max() <= k.float().abs().max() * (0.5 / 127 + 2.0 ** -8)
    dq = q[:2].contiguous()
    o = torch.empty_like(dq)
    torch.ops.nkipy_amd.paged_decode(dq, kc, vc, tables, lens, 0.1, o, ks, vs)
    assert torch.equal(o, pa.decode(dq, kc, vc, tables, lens, 0.1, k_scale=ks, v_scale=vs))
