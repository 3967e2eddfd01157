"""The chunk path of an int8 cache under the name-keyed convention and through the dispatcher."""
import numpy as np
import pytest
import torch


def _i32(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def test_read_kv_names_without_gpu():
    """Two results by position, their rows known from total_tokens; refusals before a device is touched."""
    from nkipy_amd.runtime import DeviceKernel
    pool, sc = torch.zeros(6, 16, 2, 64, dtype=torch.int8), torch.zeros(6, 2, 16)
    ins = dict(k_cache=pool, v_cache=pool, block_tables=_i32([[0, 1], [2, 3]]), seq_lens=_i32([20, 9]), cu_seqlens=_i32([0, 20, 29]),
               k_scale=sc, v_scale=sc)
    k = DeviceKernel.compile_and_load("read_kv", total_tokens=29, **ins)
    assert k.output_names == ["output0", "output1"] and k.static_kwargs == {"total_tokens": 29} and set(k.input_names) == set(ins)
    room = torch.zeros(29, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        k(inputs=ins, outputs={"output0": room, "output1": room[:28]})
    with pytest.raises(AssertionError):
        k(inputs=ins, outputs={"output0": room.float(), "output1": room})
    with pytest.raises(ValueError):
        k(inputs=ins, outputs={"output2": room})
    with pytest.raises(NotImplementedError):
        k(inputs=ins, outputs={"output0": room, "output1": room.clone()})
    with pytest.raises(ValueError):
        DeviceKernel.compile_and_load("read_kv", **ins)


@pytest.mark.gpu
def test_a_chunk_by_names():
    """Write (packed), read back, attend: three kernels that pass their tensors by name, against the calls themselves."""
    import nkipy_amd as pa
    from nkipy_amd.runtime import DeviceKernel, DeviceTensor
    g = torch.Generator(device="cuda").manual_seed(3)
    Hq, Hkv, D, bs = 4, 2, 64, 16
    past, new = [30, 0], [21, 40]
    ctx = [a + b for a, b in zip(past, new)]
    q, k, v = (torch.randn((61, h, D), generator=g, device="cuda").to(torch.bfloat16) for h in (Hq, Hkv, Hkv))
    old = torch.randn((30, Hkv, D), generator=g, device="cuda").to(torch.bfloat16)
    kc, vc = (torch.zeros((8, bs, Hkv, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((8, Hkv, bs), device="cuda") for _ in range(2))
    tables, cu, cu_ctx = _i32([[0, 1, 2, 3], [4, 5, 6, 7]], "cuda"), _i32([0, 21, 61], "cuda"), _i32([0, 51, 91], "cuda")
    sc = dict(k_scale=ks, v_scale=vs)
    pa.kv_write(old, old, kc, vc, tables, _i32(past, "cuda"), _i32(past, "cuda"), cu_seqlens=_i32([0, 30, 30], "cuda"), **sc)
    k8, v8, s8, t8 = kc.clone(), vc.clone(), ks.clone(), vs.clone()
    lens, qlens = _i32(ctx, "cuda"), _i32(new, "cuda")
    write = DeviceKernel.compile_and_load("kv_write", k_new=k, v_new=v, k_cache=kc, v_cache=vc, block_tables=tables, seq_lens=lens,
                                          query_lens=qlens, cu_seqlens=cu, **sc)
    write(inputs={"k_new": k, "v_new": v, "k_cache.must_alias_input": kc, "v_cache.must_alias_input": vc, "k_scale.must_alias_input": ks,
                  "v_scale.must_alias_input": vs, "block_tables": tables, "seq_lens": lens, "query_lens": qlens, "cu_seqlens": cu})
    pa.kv_write(k, v, k8, v8, tables, lens, qlens, k_scale=s8, v_scale=t8, cu_seqlens=cu)
    assert torch.equal(kc, k8) and torch.equal(vs, t8)
    ins = {"k_cache": kc, "v_cache": vc, "block_tables": tables, "seq_lens": lens, "cu_seqlens": cu_ctx, **sc}
    read = DeviceKernel.compile_and_load("read_kv", total_tokens=91, **ins)
    k2, v2 = read(inputs={n: DeviceTensor(t) for n, t in ins.items()})
    want = pa.read_kv(kc, vc, tables, lens, cu_ctx, 91, **sc)
    assert torch.equal(k2.torch(), want[0]) and torch.equal(v2.torch(), want[1])
    room = [torch.zeros_like(want[0]) for _ in range(2)]
    assert read(inputs=ins, outputs={"output0": room[0], "output1": DeviceTensor(room[1])}) is None
    assert torch.equal(room[0], want[0]) and torch.equal(room[1], want[1])
    only = torch.zeros_like(want[0])
    read(inputs=ins, outputs={"output1": only})
    assert torch.equal(only, want[1])
    att = {"q": q, "k": k2, "v": v2, "cu_seqlens": cu, "cu_seqlens_k": cu_ctx}
    out = DeviceKernel.compile_and_load("packed_prefill", scale=0.125, max_seq_len=51, **att)(inputs=att)
    assert torch.equal(out.torch(), pa.packed_prefill(q, *want, cu, 0.125, cu_seqlens_k=cu_ctx, max_seq_len=51))


def test_packed_writes_are_in_the_dispatcher():
    import nkipy_amd.torch_ops  # noqa: F401
    for name in ("paged_kv_write", "paged_kv_write_int8"):
        assert "Tensor? cu_seqlens=None" in str(getattr(torch.ops.nkipy_amd, name).default._schema)


@pytest.mark.gpu
def test_a_packed_write_through_the_dispatcher():
    """bfloat16 pools: packed rows, slices of a wider tensor, as the Python call writes them."""
    import nkipy_amd as pa
    import nkipy_amd.torch_ops  # noqa: F401
    rng = np.random.default_rng(4)
    Hkv, D, bs, n = 2, 128, 32, [37, 0, 50]
    wide = torch.from_numpy(rng.standard_normal((87, 3 * Hkv, D)).astype(np.float32)).cuda().to(torch.bfloat16)
    k, v = wide[:, :Hkv], wide[:, 2 * Hkv:]
    tables, lens, cu = _i32([[0, 1], [2, 3], [4, 5]], "cuda"), _i32([40, 3, 50], "cuda"), _i32([0, 37, 37, 87], "cuda")
    pools = [torch.zeros((6, bs, Hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    torch.ops.nkipy_amd.paged_kv_write(k, v, pools[0], pools[1], tables, lens, _i32(n, "cuda"), cu)
    pa.kv_write(k, v, pools[2], pools[3], tables, lens, _i32(n, "cuda"), cu_seqlens=cu)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3]) and bool((pools[0] != 0).any())
    k2, v2 = pa.read_kv(pools[0], pools[1], tables, _i32([40, 0, 50], "cuda"), _i32([0, 40, 40, 90], "cuda"), 90)
    assert torch.equal(k2[3:40], k[:37]) and torch.equal(v2[40:], v[37:])
