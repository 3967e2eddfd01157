"""Refusals of the int8 cache and packed operators, found on the host: no GPU needed."""
import ctypes
import os

import numpy as np
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nkipy_amd import _lib, build
    if not os.path.exists(build.LIB_PATH):
        build.build()
    return _lib.load()


Z = ctypes.c_void_p(0)
P = ctypes.c_void_p(4096)          # an aligned address that nothing dereferences: the calls below are refused before a launch
INT8 = 4


def _err(lib, rc, text):
    assert rc == -1 and text in lib.pa_last_error(), (rc, lib.pa_last_error())


def test_packed_prefill_arguments(lib):
    def call(**kw):
        a = dict(q=P, k=P, v=P, qs=512, ks=256, vs=256, cuq=P, cuk=P, out=P, ws=Z, wsb=0, S=2, nq=10, nk=10, Hq=4, Hkv=2, D=128, bound=10,
                 dtype=1, win=0)
        a.update(kw)
        return lib.pa_packed_prefill(a["q"], a["k"], a["v"], a["qs"], a["ks"], a["vs"], a["cuq"], a["cuk"], Z, Z, a["out"], a["ws"], a["wsb"],
                                     a["S"], a["nq"], a["nk"], a["Hq"], a["Hkv"], a["D"], a["bound"], 0.1, a["dtype"], Z, a["win"], Z)
    _err(lib, call(Hkv=3), b"multiple")
    _err(lib, call(D=96, qs=384, ks=192, vs=192), b"64 or 128")
    _err(lib, call(dtype=0), b"bf16")
    _err(lib, call(win=-1), b"sliding_window")
    _err(lib, call(bound=-1), b"max_seq_len")
    _err(lib, call(qs=504), b"strides")
    _err(lib, call(ks=257), b"strides")
    _err(lib, call(vs=248), b"strides")
    _err(lib, call(ks=1 << 29), b"2^28")
    _err(lib, call(nq=1 << 30), b"2^31")
    _err(lib, call(nq=-1), b"sizes")
    _err(lib, call(q=Z), b"null")
    _err(lib, call(cuk=Z), b"null")
    _err(lib, call(out=ctypes.c_void_p(4104)), b"aligned")
    _err(lib, call(ws=ctypes.c_void_p(4104), wsb=64), b"workspace")
    assert call(S=0) == 0 and call(nq=0) == 0
    assert lib.pa_packed_prefill_workspace_bytes(1, 256, 32256, 32, 8, 128, 32256) > 0        # few queries, many keys
    assert lib.pa_packed_prefill_workspace_bytes(1, 1024, 1024, 32, 8, 128, 1024) == 0       # a prompt
    assert lib.pa_packed_prefill_workspace_bytes(0, 256, 32256, 32, 8, 128, 32256) == 0
    assert lib.pa_packed_prefill_workspace_bytes(1, 256, 32256, 32, 8, 96, 32256) == 0


def test_read_kv_arguments(lib):
    def call(**kw):
        a = dict(k=P, v=P, ks=P, vs=P, bt=P, sl=P, cu=P, ko=P, vo=P, n=10, B=2, Hkv=2, D=128, bs=16, mb=4, nb=8, kd=INT8)
        a.update(kw)
        return lib.pa_read_kv(a["k"], a["v"], a["ks"], a["vs"], a["bt"], a["sl"], a["cu"], a["ko"], a["vo"], a["n"], a["B"], a["Hkv"], a["D"],
                              a["bs"], a["mb"], a["nb"], a["kd"], Z)
    _err(lib, call(kd=0), b"kv_dtype")
    _err(lib, call(kd=3), b"kv_dtype")
    _err(lib, call(D=100), b"multiple of 8")
    _err(lib, call(bs=0), b"paging")
    _err(lib, call(ks=Z), b"k_scale")
    _err(lib, call(cu=Z), b"null")
    _err(lib, call(vo=ctypes.c_void_p(4100)), b"aligned")
    _err(lib, call(n=-1), b"sizes")
    _err(lib, call(mb=1 << 30), b"capacity")
    assert call(B=0) == 0 and call(n=0) == 0


def test_writes_and_decode_of_int8_pools(lib):
    def kvw(**kw):
        a = dict(ks=P, vs=P, B=2, T=4, Hkv=2, D=128)
        a.update(kw)
        return lib.pa_kv_write(P, P, P, P, a["ks"], a["vs"], P, P, P, a["B"], a["T"], a["Hkv"], a["D"], 16, 4, 8, INT8, Z)
    _err(lib, kvw(ks=Z), b"k_scale")
    _err(lib, kvw(D=96), b"32, 64, 128 or 256")
    _err(lib, kvw(vs=ctypes.c_void_p(4100)), b"16-byte")

    def packed(**kw):
        a = dict(k=P, kst=256, vst=256, cu=P, n=10, ks=P, vs=P, D=128, kd=INT8, B=2)
        a.update(kw)
        return lib.pa_kv_write_packed(a["k"], P, a["kst"], a["vst"], a["cu"], a["n"], P, P, a["ks"], a["vs"], P, P, P, a["B"], 2, a["D"], 16, 4, 8,
                                      a["kd"], Z)
    _err(lib, packed(kd=2), b"fp8")
    _err(lib, packed(kst=250), b"strides")
    _err(lib, packed(vst=128), b"strides")
    _err(lib, packed(D=80), b"32, 64, 128 or 256")
    _err(lib, packed(cu=Z), b"null")
    _err(lib, packed(ks=Z), b"k_scale")
    assert packed(n=0) == 0 and packed(B=0) == 0

    def dec(D=128, bs=16, ks=P, **kw):
        return lib.pa_decode(P, P, P, ks, P, P, P, P, Z, 0, 2, 8, 2, D, bs, 4, 8, 0, 1.0, 512, kw.get("qd", 1), INT8, Z, 0, Z, Z)
    _err(lib, dec(D=256), b"int8")
    _err(lib, dec(bs=24), b"int8")
    _err(lib, dec(ks=Z), b"k_scale")
    _err(lib, dec(qd=0), b"dtype")
    rc = lib.pa_prefill(P, P, P, P, P, P, P, P, P, 1, 4, 4, 4, 128, 16, 4, 8, 0, 1.0, 1, INT8, Z, 0, Z, 0, Z, Z)
    _err(lib, rc, b"pa_read_kv")


def test_python_refusals_without_a_gpu():
    import nkipy_amd as pa
    host = np.zeros((3, 2, 64), np.float32)
    with pytest.raises(NotImplementedError):
        pa.packed_prefill(host, host, host, np.zeros(2, np.int32), 0.1)
    with pytest.raises(NotImplementedError):
        pa.packed_prefill(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(2, dtype=torch.int32), 0.1)
    pool = torch.zeros((2, 16, 2, 64), dtype=torch.int8)
    with pytest.raises(NotImplementedError):
        pa.read_kv(pool, pool, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 4)


def test_int8_cache_bookkeeping():
    from nkipy_amd.engine import PagedKVCache
    with pytest.raises(ValueError):
        PagedKVCache(8, 16, 2, 96, max_seqs=2, max_blocks_per_seq=4, dtype=torch.int8, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(8, 24, 2, 64, max_seqs=2, max_blocks_per_seq=4, dtype=torch.int8, device="cpu")
    c = PagedKVCache(8, 16, 2, 64, max_seqs=3, max_blocks_per_seq=4, dtype=torch.int8, device="cpu")
    assert c.k_scale.shape == (8, 2, 16) and c.k_cache.dtype == torch.int8
    c.begin_step([20, 0, 7], 20)
    assert c.row_starts.tolist() == [0, 20, 20, 27]
    c.begin_step([0, 5, 3], 5)
    assert c.row_starts.tolist() == [0, 0, 5, 15] and c.seq_lens.tolist() == [20, 5, 10]
    c.release(1)
    assert c.seq_lens.tolist()[1] == 0
    assert PagedKVCache(8, 16, 2, 64, max_seqs=3, max_blocks_per_seq=4, device="cpu").row_starts is None


FLOAT_DIV = [1, 2, 3, 5, 7, 8, 10, 12, 127, 255, 256, 1000, 4095, 65535, 1 << 20, (1 << 30) + 1, (1 << 31) - 1]


@pytest.mark.parametrize("d", FLOAT_DIV)
def test_division_by_a_known_number(d):
    """The multiply-and-shift division of the packed kernels, restated: floor(x / d) for all 32-bit x (edges and random)."""
    s = 0
    while (1 << s) < d:
        s += 1
    m = (((1 << 32) * ((1 << s) - d)) // d + 1) & 0xffffffff
    s1, s2 = min(s, 1), max(s - 1, 0)
    rng = np.random.default_rng(d)
    xs = [0, 1, d - 1, d, d + 1, 2 * d - 1, 2 * d, (1 << 31) - 1, (1 << 32) - 1] + [int(x) for x in rng.integers(0, 1 << 32, 2000, dtype=np.uint64)]
    for x in xs:
        x &= 0xffffffff
        t = (m * x) >> 32
        assert (t + ((x - t) >> s1)) >> s2 == x // d, x


def test_tile_numbers_cover_every_tile_once():
    """The numbering that packed work is dealt by, restated: every (sequence, tile) has one number, all below total + n."""
    rng = np.random.default_rng(1)
    for shift, mult in ((4, 1), (7, 4), (7, 3), (6, 1)):
        for _ in range(50):
            lens = rng.integers(0, 300, rng.integers(1, 20))
            cu = np.concatenate([[0], np.cumsum(lens)])
            seen = set()
            for i, n in enumerate(lens):
                for t in range(-(-int(n) * mult >> shift) if n == 0 else (int(n) * mult + (1 << shift) - 1) >> shift):
                    x = (mult * int(cu[i]) >> shift) + i + t
                    assert x not in seen
                    seen.add(x)
                    lo = max(j for j in range(len(lens)) if (mult * int(cu[j]) >> shift) + j <= x)
                    assert lo == i and x < (mult * int(cu[-1]) >> shift) + len(lens)
