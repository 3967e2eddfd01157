"""Plain forms for the int8 paged cache and packed prompt attention: NumPy for what is exact, float64 for the rest."""
import numpy as np
import torch

from oracle import paged_attention_oracle as O

H = 2.0 ** -8          # half a bf16 step, relative


def quantise_rows(x):
    """float32 rows [..., D] (bf16 values) -> (int8 codes, float32 scales): absmax / 127, 1 for zeros, nearest even;
    a row with an infinity or a NaN: scale NaN, codes 0."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    y = np.where(bad[..., None], np.float32(0), x)
    s = np.abs(y).max(-1) / np.float32(127)
    s = np.where(s == 0, np.float32(1), s).astype(np.float32)
    codes = np.clip(np.rint(y / s[..., None]), -127, 127).astype(np.int8)
    return codes, np.where(bad, np.float32(np.nan), s)


def random_tables(rng, ctxs, bs, extra=3, pad=2):
    n = [(c + bs - 1) // bs for c in ctxs]
    blocks = sum(n) + extra
    ids = rng.permutation(blocks).astype(np.int32)
    tables = np.full((len(ctxs), max(max(n), 1) + pad), -1, np.int32)
    at = 0
    for b, k in enumerate(n):
        tables[b, :k] = ids[at:at + k]
        at += k
    return tables, blocks


def int8_pool(rng, ctxs, bs, Hkv, D, spread=1.0):
    """Pool of random rows for the given contexts; every row no token stands on has garbage codes and a NaN scale."""
    tables, blocks = random_tables(rng, ctxs, bs)
    out = {"tables": tables, "blocks": blocks}
    for name in "kv":
        codes = rng.integers(-128, 128, (blocks, bs, Hkv, D)).astype(np.int8)
        scale = np.full((blocks, Hkv, bs), np.nan, np.float32)
        for b, c in enumerate(ctxs):
            for j in range((c + bs - 1) // bs):
                n = min(bs, c - j * bs)
                x = rng.standard_normal((n, Hkv, D)) * np.exp(spread * rng.standard_normal((n, Hkv, 1)))
                q, s = quantise_rows(O.round_to_bf16(x.astype(np.float32)))
                codes[tables[b, j], :n] = q
                scale[tables[b, j], :, :n] = s.T
        out[name], out[name + "s"] = codes, scale
    return out


def context(pool, which, b, c, bs):
    """float64 values of the first c tokens of sequence b, [c, Hkv, D]."""
    ids = pool["tables"][b, :(c + bs - 1) // bs]
    val = pool[which][ids].astype(np.float64) * pool[which + "s"][ids].transpose(0, 2, 1)[..., None].astype(np.float64)
    return val.reshape(-1, *val.shape[2:])[:c]


def attention64(q, k, v, scale, first, window=0, sinks=None):
    """float64 attention of rows q [T, Hq, D] at positions first + i over k / v [C, Hkv, D]: (out, sum of p |v|, largest
    sum of |q| |k| scale over visible keys)."""
    T, Hq, D = q.shape
    C, Hkv = k.shape[:2]
    r = Hq // Hkv
    out, mag = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    reach = 0.0
    if C == 0:
        return out, mag, reach
    pos = first + np.arange(T)[:, None]
    key = np.arange(C)[None]
    live = key <= pos
    if window:
        live &= key > pos - window
    for h in range(Hq):
        kk, vv = k[:, h // r], v[:, h // r]
        s = np.where(live, (q[:, h] @ kk.T) * scale, -np.inf)
        absd = np.where(live, (np.abs(q[:, h]) @ np.abs(kk).T) * abs(scale), 0.0)
        reach = max(reach, float(absd.max(initial=0.0)))
        m = s.max(1, keepdims=True)
        if sinks is not None:
            m = np.maximum(m, float(sinks[h]))
        m = np.where(np.isinf(m), 0.0, m)
        p = np.exp(s - m)
        den = p.sum(1, keepdims=True)
        if sinks is not None:
            den = np.where(den > 0, den + np.exp(float(sinks[h]) - m), den)
        p = p / np.where(den > 0, den, 1.0)
        out[:, h] = p @ vv
        mag[:, h] = p @ np.abs(vv)
    return out, mag, reach


def attention_tolerance(out, mag, reach, D):
    """What the kernels may be off by, element by element.  The probabilities (times the value's scale) are rounded to bf16
    once, at most H relative each: H * sum p |v|.  The result is rounded once: H |out|.  Scores are float32 sums of D
    products (and of the scale and the reference): an absolute error of at most (D + 8) 2^-24 reach, which moves a
    probability and the sum it is divided by by twice that, relatively; exp2 itself and the sums over the keys stay
    within 2^-18.  (Over an int8 pool the probabilities are rounded to 16 bits and the query's elements to 2^-16 of the
    row's largest, which is below what the 8 bits of the other kernels allow: 2^-16 q_max sum |k| scale <= 2^-8 of the
    room H * sum p |v| leaves as long as the scores stay below a few hundred.)"""
    score = (D + 8) * 2.0 ** -24 * reach
    grow = np.expm1(min(2 * score, 1.0))
    return (H + grow + 2.0 ** -18) * mag * (1 + H) + H * np.abs(out) + 1e-30


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def bf16(a):
    return dev(np.asarray(a, np.float32)).to(torch.bfloat16)


def to_np(t):
    return t.detach().double().cpu().numpy()


def assert_within(got, want, tol):
    got = to_np(got) if isinstance(got, torch.Tensor) else got
    assert np.isfinite(got).all(), "non-finite values in the result"
    over = np.abs(got - want) - tol
    at = np.unravel_index(int(np.argmax(over)), over.shape) if over.size else ()
    assert over.size == 0 or over.max() <= 0, f"at {at}: got {got[at]:.6e}, want {want[at]:.6e}, tolerance {tol[at]:.3e}"
