"""The 8-bit key/value cache and its attention in 64 bits: what
include/trit_cuda.h says the cache holds, written in numpy."""
import numpy as np


def held(x, page):
    """What the cache holds of a sequence's rows x [t][kv][hd]: (values as f32, codes of the full pages)."""
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.asarray(x, np.float64)
        x = np.where(np.isnan(x), 0.0, np.clip(x, -65504.0, 65504.0)).astype(np.float16)
    t = x.shape[0] // page * page
    out = x.astype(np.float32)
    if t:
        b = x[:t].astype(np.float64).reshape(-1, page, *x.shape[1:])
        scale = (np.abs(b).max(axis=(1, 3), keepdims=True) / 127.0).astype(np.float32)
        code = np.rint(np.divide(b, scale.astype(np.float64), out=np.zeros_like(b), where=np.broadcast_to(scale > 0, b.shape)))
        out[:t] = (code.astype(np.float32) * scale).reshape(t, *x.shape[1:])
    return out


def attend(q, k, v, scale, causal):
    """(out, tolerance of the f32 kernel) of rows q [m][heads][hd] against k, v [t][kv][hd] (values that the cache holds).

    The tolerance: with S = scale * max_j sum_d |q_d k_jd|, a score is off by at most 2^-22 S from the split query, 8 steps
    of sums at 2^-23 S, and 2^-22 (S + 1) from the exponent's argument, so a weight by a factor within 2^-19 (S + 1); numerator and
    denominator each carry that, the weights' 22-bit form, and f32 sums over t positions (t / 16 additions a lane at
    2^-24, doubled for the joins). Everything is relative to max |v|."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    m, heads, hd = q.shape
    t, kv = k.shape[0], k.shape[1]
    out = np.zeros_like(q)
    tol = np.zeros_like(q)
    for h in range(heads if t else 0):
        kk, vv = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        s = scale * q[:, h] @ kk.T
        if causal:
            s = np.where(np.arange(t)[None] <= np.arange(t - m, t)[:, None], s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = p @ vv / p.sum(-1, keepdims=True)
        big = abs(scale) * (np.abs(q[:, h]) @ np.abs(kk).T).max(-1, keepdims=True)
        tol[:, h] = np.abs(vv).max() * (2 * 2.0**-19 * (big + 1) + 2.0**-21 + (t / 8 + 8) * 2.0**-24)
    return out, tol
