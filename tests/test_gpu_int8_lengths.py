"""The row-wise cache write (int8 pools, packed rows) under lengths that name no row."""
import numpy as np
import pytest
import torch

from tests.int8_kv_lib import bf16, dev

pytestmark = pytest.mark.gpu

LO = -2 ** 31
SEQS = [LO, LO + 1, LO + 3, -1, 0, 2, 1]
QLENS = [1, 5, 4, 1, 1, 3, LO]


CASES = [("int8", D, packed) for D in (32, 64, 128) for packed in (False, True)] + [("bf16", D, True) for D in (32, 64, 128)] + \
        [("fused", D, False) for D in (64, 128)]


@pytest.mark.parametrize("kind,D,packed", CASES)
def test_lengths_that_name_no_row_write_nothing(rng, kind, D, packed):
    """A context below its query length, down to the smallest integer, and query lengths below zero: the pool keeps its bits."""
    import nkipy_amd as pa
    B, T, Hkv, bs = len(SEQS), 5, 2, 16
    x = bf16(rng.standard_normal((B, T, Hkv, D)))
    dt = torch.bfloat16 if kind == "bf16" else torch.int8
    pools = [torch.full((4, bs, Hkv, D), 3, dtype=dt, device="cuda") for _ in range(2)]
    scales = [torch.full((4, Hkv, bs), 0.5, device="cuda") for _ in range(2)]
    kw = {} if kind == "bf16" else {"k_scale": scales[0], "v_scale": scales[1]}
    tables = torch.arange(4, dtype=torch.int32, device="cuda").repeat(B, 1)
    args = (*pools, tables, dev(np.asarray(SEQS, np.int32)), dev(np.asarray(QLENS, np.int32)))
    if kind == "fused":
        pa.qk_norm_rope_kv_write(x, x, x, *args, *pa.rope_tables(D, 64), **kw)
    elif packed:
        rows = x.view(B * T, Hkv, D)
        pa.kv_write(rows, rows, *args, cu_seqlens=dev(np.arange(0, B * T + 1, T).astype(np.int32)), **kw)
    else:
        pa.kv_write(x, x, *args, **kw)
    assert all(bool((p == 3).all()) for p in pools) and all(bool((s == 0.5).all()) for s in scales)
