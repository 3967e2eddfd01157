"""Packed prompts under windows at the ends of their range, and in front of prefixes."""
import numpy as np
import pytest
import torch

from oracle import paged_attention_oracle as O
from tests.int8_kv_lib import bf16, dev
from tests.test_gpu_packed_prefill import _run, _starts, debug_switch, pa  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 140])
@pytest.mark.parametrize("split", [0, 1, 3])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 4, 64), (3, 1, 64)])
def test_the_longest_windows(pa, rng, debug_switch, Hq, Hkv, D, split, window):  # noqa: F811
    """A window longer than any context is none, for sequences with fewer keys than queries too: the reach of their first
    queries lies before the first key, and a window's length behind it is past the smallest integer."""
    debug_switch(6, split)
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    _run(pa, rng, [40, 1, 130, 300, 70, 20], Hq, Hkv, D, kn=[400, 777, 127, 3, 5, 65], tail=3, window=window, workspace=ws)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 2, 64)])
def test_a_window_of_all_rows_is_none(pa, rng, Hq, Hkv, D):  # noqa: F811
    n = [90, 33, 200]
    q, k, v = (bf16(O.round_to_bf16(rng.standard_normal((sum(n), h, D)).astype(np.float32))) for h in (Hq, Hkv, Hkv))
    cu = dev(_starts(n))
    want = pa.packed_prefill(q, k, v, cu, 0.1)
    for window in (sum(n), sum(n) + 1, 2 ** 31 - 1):
        assert torch.equal(pa.packed_prefill(q, k, v, cu, 0.1, sliding_window=window), want)


@pytest.mark.parametrize("window", [50, 600, 1500, None])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (8, 2, 64), (3, 1, 64)])
def test_chunks_behind_long_prefixes_in_the_shares_the_rule_gives(pa, rng, Hq, Hkv, D, window):  # noqa: F811
    """The call's own scratch, and scratch of exactly the size asked for."""
    qn, kn = [30, 1, 77, 100], [2100, 1500, 1300, 2600]
    need = pa.packed_prefill_workspace_bytes(4, sum(qn), sum(kn), Hq, Hkv, D, max(kn), window)
    assert need > 0 if window is None else window > 50 or need == 0
    _, _, _, got = _run(pa, rng, qn, Hq, Hkv, D, kn=kn, window=window, max_seq_len=max(kn))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    _run(pa, rng, qn, Hq, Hkv, D, kn=kn, window=window, max_seq_len=max(kn), workspace=ws)
    if need:
        with pytest.raises(ValueError):
            _run(pa, rng, qn, Hq, Hkv, D, kn=kn, window=window, max_seq_len=max(kn), workspace=ws[:need - 16])


def test_a_window_past_32_bits_is_none(pa, rng):  # noqa: F811
    """Every call that takes a window, over contexts longer than what is left of it in 32 bits.  Either result is off by the
    rounding of its probabilities and its own, 2^-8 of max |v| each."""
    Hq, Hkv, D, bs, n = 8, 2, 128, 32, 150
    q, k, v = (bf16(O.round_to_bf16(rng.standard_normal((n, h, D)).astype(np.float32))) for h in (Hq, Hkv, Hkv))
    cu, ln = dev(np.asarray([0, n], np.int32)), dev(np.asarray([n], np.int32))
    tables = dev(rng.permutation(5).astype(np.int32)[None])
    kc, vc = (torch.zeros((5, bs, Hkv, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pa.kv_write(k, v, kc, vc, tables, ln, ln, cu_seqlens=cu)
    four = dev(np.asarray([4], np.int32))
    for call in (lambda w: pa.packed_prefill(q, k, v, cu, 0.1, sliding_window=w), lambda w: pa.decode(q[-1:], kc, vc, tables, ln, 0.1, sliding_window=w),
                 lambda w: pa.prefill(q[None], kc, vc, tables, ln, ln, 0.1, sliding_window=w),
                 lambda w: pa.verify(q[None, -4:].contiguous(), kc, vc, tables, ln, four, 0.1, sliding_window=w)):
        assert (call(2 ** 32 + 5).float() - call(None).float()).abs().max() <= 4 * 2.0 ** -8 * v.float().abs().max()
