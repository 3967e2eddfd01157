"""What the packed operators refuse and how they size themselves, on the host: no GPU needed."""
import ctypes
import os

import pytest


@pytest.fixture(scope="module")
def lib():
    from nkipy_amd import _lib, build
    if not os.path.exists(build.LIB_PATH):
        build.build()
    return _lib.load()


Z = ctypes.c_void_p(0)
P = ctypes.c_void_p(4096)          # an aligned address that nothing dereferences: the calls below are refused before a launch


def test_rows_beyond_the_positions_of_32_bits(lib):
    def call(nq, nk):
        return lib.pa_packed_prefill(P, P, P, 128, 128, 128, P, P, Z, Z, P, Z, 0, 2, nq, nk, 1, 1, 128, 0, 0.1, 1, Z, 0, Z)
    assert call((1 << 31) - (1 << 17), 1 << 17) == -1 and b"2^31 together" in lib.pa_last_error()
    assert call(0, 1 << 17) == 0


# Without a device the library counts 256 compute units.
def _shares(lib, S, nq, nk, Hq, Hkv, D, bound, window=0):
    """Shares of a query tile's keys that a call asks scratch for (1: none)."""
    n = lib.pa_packed_prefill_workspace_bytes_for(S, nq, nk, Hq, Hkv, D, bound, window)
    per = nq * Hq * (D + 2) * 4
    assert n % per == 0 and n // per != 1
    return max(n // per, 1)


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (64, 8, 64)])
def test_shares_under_a_window_are_those_of_its_keys(lib, Hq, Hkv, D):
    """Four chunks of 100 tokens behind some 3 000 keys: many keys in front split a tile, the few of a narrow window do not;
    a window over all of them changes nothing."""
    args = (4, 400, 12600, Hq, Hkv, D, 3200)
    assert _shares(lib, *args) >= 4
    for window in (1, 50, 128, 500):
        assert _shares(lib, *args, window) == 1
    assert _shares(lib, *args, 2000) <= 4
    assert _shares(lib, *args, 12600) == _shares(lib, *args, 2 ** 31 - 1) == _shares(lib, *args)
    assert lib.pa_packed_prefill_workspace_bytes(*args) == lib.pa_packed_prefill_workspace_bytes_for(*args, 0)
    assert lib.pa_packed_prefill_workspace_bytes_for(*args, -1) == 0


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (16, 2, 128), (7, 1, 128), (64, 8, 64), (8, 2, 64), (7, 1, 64)])
def test_shares_of_a_call_without_a_bound(lib, Hq, Hkv, D):
    """No bound on the contexts is not one context of all the batch's rows: prompts without a prefix stay whole, a few tokens
    behind long contexts are split as with the bound."""
    assert _shares(lib, 8, 2400, 2400, Hq, Hkv, D, 0) == 1
    assert _shares(lib, 64, 64 * 64, 64 * 64, Hq, Hkv, D, 0) == 1
    assert _shares(lib, 1, 1024, 1024, Hq, Hkv, D, 0) == 1
    assert _shares(lib, 1, 64, 8192, Hq, Hkv, D, 0) == _shares(lib, 1, 64, 8192, Hq, Hkv, D, 8192) >= 8
    assert _shares(lib, 2, 64, 16384, Hq, Hkv, D, 0) >= 4


def test_shares_at_head_dim_64_are_more_workgroups_than_none(lib):
    """A split wave takes two q heads where a whole one of a small call takes one: two shares are as many workgroups as none."""
    for Hq, Hkv in ((64, 8), (8, 2), (16, 4), (32, 8), (2, 1)):
        for S, T, ctx in ((4, 100, 3200), (8, 64, 1064), (8, 64, 1564), (2, 256, 2304), (1, 512, 2048), (1, 512, 4608), (4, 300, 3300), (1, 64, 8192)):
            for window in (0, 700, 1500):
                assert _shares(lib, S, S * T, S * ctx, Hq, Hkv, 64, ctx, window) != 2
    assert _shares(lib, 8, 512, 8512, 8, 2, 64, 1064) == 1
    assert _shares(lib, 2, 512, 4608, 64, 8, 64, 2304) == 1
    assert _shares(lib, 1, 512, 4608, 64, 8, 64, 4608) == 4
    assert _shares(lib, 1, 256, 33024, 64, 8, 64, 33024) == 8
    assert _shares(lib, 4, 64, 2464, 7, 1, 64, 1232) == 2             # one q head per wave either way


def test_a_window_past_32_bits_is_no_short_one():
    from nkipy_amd import paged_attn
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40):
        assert paged_attn._check_variant(None, window, 4, None) == (None, 2 ** 31 - 1)
    assert paged_attn._check_variant(None, 5, 4, None) == (None, 5) and paged_attn._check_variant(None, None, 4, None) == (None, 0)
    with pytest.raises(ValueError):
        paged_attn._check_variant(None, -5, 4, None)
    assert paged_attn.packed_prefill_workspace_bytes(4, 400, 12600, 32, 8, 128, 3200, 2 ** 32 + 5) == \
        paged_attn.packed_prefill_workspace_bytes(4, 400, 12600, 32, 8, 128, 3200)


def test_one_long_context_among_empty_ones_is_split_without_a_bound(lib):
    """256 queries behind 32 K keys, alone and as one sequence of 64 whose others are empty: the mean says nothing there."""
    for Hq, Hkv, D in ((32, 8, 128), (8, 2, 64)):
        alone = _shares(lib, 1, 256, 33024, Hq, Hkv, D, 0)
        assert alone == _shares(lib, 1, 256, 33024, Hq, Hkv, D, 33024) >= 8
        assert _shares(lib, 64, 256, 33024, Hq, Hkv, D, 0) == _shares(lib, 64, 256, 33024, Hq, Hkv, D, 33024) >= 2


def test_shares_under_the_longest_window_that_is_one(lib):
    """A window a little shorter than 2^31 keys reaches as far as they do: the sum that says so is not of 32 bits."""
    k = (1 << 31) - 1000
    assert _shares(lib, 1, 64, k, 32, 8, 128, k, k - 1) == _shares(lib, 1, 64, k, 32, 8, 128, k) == 16
