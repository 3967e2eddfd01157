"""The tolerance of attention over int8 pools on the CPU: the path's arithmetic is inside it, that arithmetic with a mistake in it
is not."""
import numpy as np
import pytest

from oracle import paged_attention_oracle as O
from tests.int8_attention_lib import attention_and_tolerance, int8_model, orthogonal_rows, query_step
from tests.int8_kv_lib import quantise_rows


def _case(kind, seed, C=40, Hq=4, D=128):
    rng = np.random.default_rng(seed)
    q = O.round_to_bf16(rng.standard_normal((Hq, D)).astype(np.float32))
    scale = D ** -0.5
    k = rng.standard_normal((C, Hq, D)) * np.exp(0.5 * rng.standard_normal((C, Hq, 1)))
    if kind == "outlier":                       # one channel far above the others, in the query and (small there) in the keys
        q[:, 7] = O.round_to_bf16((2.0 ** rng.integers(3, 11, Hq)).astype(np.float32) * 1.7)
        k[..., 7] *= 2.0 ** -6
    if kind == "cancel":
        q = O.round_to_bf16((np.sign(q) * rng.uniform(0.06, 1.9, q.shape)).astype(np.float32))
        k, scale = orthogonal_rows(rng, q, C), 6.0
    if kind == "one key":
        k = k[:1]
    v = rng.standard_normal(k.shape) * np.exp(0.5 * rng.standard_normal(k.shape[:2] + (1,)))
    (kc, ks), (vc, vs) = (quantise_rows(O.round_to_bf16(x.astype(np.float32))) for x in (k, v))
    want, tol = attention_and_tolerance(q[None], kc * ks[..., None].astype(np.float64), vc * vs[..., None].astype(np.float64), scale, len(k) - 1)
    return (q, kc, ks, vc, vs, scale), want[0], tol[0]


def _worst(kind, seeds=range(6), C=40, **kw):
    worst = 0.0
    for seed in seeds:
        args, want, tol = _case(kind, seed, C)
        worst = max(worst, float((np.abs(int8_model(*args, **({k: f(args[0]) if callable(f) else f for k, f in kw.items()})) - want) / tol).max()))
    return worst


@pytest.mark.parametrize("kind", ["ordinary", "outlier", "cancel", "one key"])
def test_the_arithmetic_is_inside(kind):
    assert _worst(kind) <= 1.0


def test_a_mistake_is_not():
    assert _worst("ordinary", C=8, terms=1) > 1.0              # the probabilities' second term
    assert _worst("one key", terms=1) > 1.0
    assert _worst("ordinary", limbs=1) > 1.0                   # the query's low limb
    assert _worst("cancel", limbs=1) > 1.0
    # a step that is no power of two (the largest element / 32 512) rounds nearly every element
    assert _worst("cancel", step=lambda q: np.abs(q).max(-1, keepdims=True).astype(np.float64) / 32512) > 1.0


def test_the_step_takes_every_element_it_should():
    """Every largest element: within the limbs; elements of at least 2^-6 of it are whole numbers of steps, the others off by
    at most half a step, 2^-15 of it (256 / 255 of that at the significand that takes the next power)."""
    rng = np.random.default_rng(0)
    f = lambda bits: (np.asarray(bits, np.uint32) << 16).view(np.float32).astype(np.float64)       # noqa: E731
    tops = np.arange(1, 0x7f80)
    step = query_step(f(tops)[:, None])[:, 0]
    whole = np.rint(f(tops) / step)
    assert whole.max() <= 127 * 256 + 127 and ((whole.astype(int) + 128) >> 8).max() <= 127
    for t in rng.integers(22 << 7, 0x7f80, 500):
        x, m, st = f(rng.integers(0, t + 1, 300)), f([t])[0], query_step(f([t]))[0]
        err = np.abs(np.rint(x / st) * st - x)
        assert (err[x >= m * 2.0 ** -6] == 0).all() and err.max() <= m * 2.0 ** -15 * 256 / 255
