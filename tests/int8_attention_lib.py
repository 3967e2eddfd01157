"""Attention over an int8 pool: float64 with a tolerance counted from that path's own roundings, and the path's arithmetic
restated in NumPy."""
import numpy as np

from oracle import paged_attention_oracle as O
from tests.int8_kv_lib import H


def query_step(q):
    """The step of each row's fixed-point form, [..., 1]: 2^-14 of the power of two below the row's largest element (the one
    significand that rounds past the limbs takes the next power), not below 2^-120."""
    top = O.f32_to_bf16_bits(np.abs(np.asarray(q, np.float32)).max(-1)).astype(np.int64)
    return np.exp2(np.maximum((top + 1) >> 7, 21) - 141.0)[..., None]


def attention_and_tolerance(q, k, v, scale, first, window=0, sinks=None):
    """float64 attention of bf16 rows q [T, Hq, D] at positions first + i over k / v [C, Hkv, D] (codes x scales), and what the
    kernels may be off by, element by element.

    * A query element that is no whole number of steps is rounded to one: |error| <= half a step.  That moves the score of
      key j by e_j = scale * sum over such elements of step / 2 * |k_j|.
    * The product with the codes is exact.  What follows is a handful of float32 roundings of the score (the integer's, the
      product of the two scales, the product with it, log2 e, the difference to the maximum) and exp2's own: 16 half steps of
      2^-24, of the largest |score| the row sees.
    * A score's error changes a probability by as much, relatively, and the sum it is divided by by at most the largest one.
    * Probability times the value's scale goes in as two bf16 terms: H^2 of it is lost.
    * n keys are summed in float32, here and in the denominator, and partitions are merged: 2 (n + 64) 2^-24.
    * The result is rounded once: H of itself."""
    T, Hq, D = q.shape
    C, Hkv = k.shape[:2]
    r = Hq // Hkv
    q = np.asarray(q, np.float64)
    out, tol = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    if C == 0:
        return out, tol
    step = query_step(q)
    lost = np.where(np.rint(q / step) * step == q, 0.0, step / 2)
    pos, key = first + np.arange(T)[:, None], np.arange(C)[None]
    live = key <= pos
    if window:
        live &= key > pos - window
    for h in range(Hq):
        kk, vv = k[:, h // r], v[:, h // r]
        s = np.where(live, (q[:, h] @ kk.T) * scale, -np.inf)
        m = s.max(1, keepdims=True)
        if sinks is not None:
            m = np.maximum(m, float(sinks[h]))
        m = np.where(np.isinf(m), 0.0, m)
        p = np.exp(s - m)
        den = p.sum(1, keepdims=True)
        if sinks is not None:
            den = np.where(den > 0, den + np.exp(float(sinks[h]) - m), den)
        p = p / np.where(den > 0, den, 1.0)
        e = np.where(live, (lost[:, h] @ np.abs(kk).T) * abs(scale), 0.0)
        e = e + 16 * 2.0 ** -24 * np.where(live, np.abs(s), 0.0).max(1, keepdims=True) + 16 * 2.0 ** -24
        rel = np.expm1(np.minimum(e + e.max(1, keepdims=True), 1.0)) + H * H + 2 * (live.sum(1, keepdims=True) + 64) * 2.0 ** -24
        out[:, h] = p @ vv
        part = (p * rel) @ np.abs(vv)
        tol[:, h] = part + H * (np.abs(out[:, h]) + part) + 1e-30
    return out, tol


def int8_model(q, kc, ks, vc, vs, scale, *, step=None, limbs=2, terms=2):
    """The kernels' arithmetic for one decode row: q [Hq, D] bf16 values, codes [C, Hkv, D], scales [C, Hkv].  step, limbs
    and terms plant mistakes: another step for the query, its high limb alone, the probabilities as one bf16 term."""
    Hq, r = q.shape[0], q.shape[0] // kc.shape[1]
    bf = O.round_to_bf16
    out = np.zeros(q.shape)
    step = query_step(q) if step is None else step
    ints = np.rint(np.asarray(q, np.float64) / step).astype(np.int64)
    if limbs == 1:
        ints = (ints + 128) // 256 * 256
    for h in range(Hq):
        g = h // r
        dots = (ints[h] @ kc[:, g].astype(np.int64).T).astype(np.float32)
        per = np.float32(np.float32(scale * np.log2(np.e)) * np.float32(step[h, 0]))
        s = dots * (per * ks[:, g])
        p = np.exp2(s - s.max()).astype(np.float32)
        pr = p * vs[:, g]
        hi = bf(pr)
        w = hi.astype(np.float64) + (bf(pr - hi) if terms == 2 else 0.0)
        out[h] = bf((w @ vc[:, g].astype(np.float64) / p.astype(np.float64).sum()).astype(np.float32))
    return out


def orthogonal_rows(rng, q, n):
    """n rows [n, Hkv, D] that are nearly orthogonal to every q row of their group ([Hq, D], as many groups as q heads): scores
    that cancel, which leave a query's own rounding nothing to hide behind."""
    x = rng.standard_normal((n, q.shape[0], q.shape[1]))
    u = q / np.linalg.norm(q, axis=-1, keepdims=True)
    return x - (x * u).sum(-1, keepdims=True) * u
