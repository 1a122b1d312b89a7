"""Attention of many rows over the 8-bit cache (trit_cuda_kv_attend) where a
row's running maximum rises inside a step of 128 positions, which makes the
kernel take back and rescale what it has written of that step."""
import math

import numpy as np
import pytest

from tests.kv_oracle import held
from trit_b200 import KvCache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
HD, HEADS = 64, 32


def attention(s, v, dtype, causal=False):
    """(out, tolerance) for scores s [rows][t] against values v [t][hd] in 64 bits.

    With S the row's largest |score|, a weight is off by a factor within 2^-19 (S + 1) (as derived in kv_oracle.attend), in
    the numerator and in the denominator; 16-bit rows round each weight of the numerator to 2^-11. Both are relative to
    sum p |v| / sum p. Besides, a weight's last place: 2^-25 where the row's largest weight is at least 2^7 (f16
    subnormals), and f32 sums over t positions, relative to max |v|."""
    m, t = s.shape
    if causal:
        s = np.where(np.arange(t)[None] <= np.arange(t - m, t)[:, None], s, -np.inf)
    big = np.abs(np.where(np.isfinite(s), s, 0.0)).max(-1, keepdims=True)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    out, size = p @ v, p @ np.abs(v)
    tol = size * (2 * 2.0**-19 * (big + 1) + (2.0**-11 if dtype != "f32" else 0.0) + t / 8 * 2.0**-24)
    return out, tol + HALF_STEP[dtype] * np.abs(out) + np.abs(v).max() * t * 2.0**-32


def run(key, sizes, v, dtype, page, causal=False):
    """Rows q = sizes[r] e_0 of every head against keys key[j] e_0, so that a score is sizes[r] key[j] in units of log 2:
    (outputs [rows][heads][hd], the scores that the cache's keys give, its values)."""
    t, m = len(key), len(sizes)
    k = np.zeros((t, 1, HD), np.float32)
    k[:, 0, 0] = key
    v = v.astype(np.float16).astype(np.float32).reshape(t, 1, HD)
    q = np.zeros((m, HEADS, HD), np.float32)
    q[:, :, 0] = np.asarray(sizes)[:, None]
    scale = np.float32(math.log(2))
    dq = torch.from_numpy(q).to(TYPES[dtype]).cuda()
    out = torch.full_like(dq, float("nan"))
    dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    with KvCache(kv_heads=1, pages=t // page + 1, head_dim=HD, page_tokens=page, sequences=1, max_tokens=t) as kv:
        s = kv.open(1)
        kv.extend(s, [t])
        torch.cuda.synchronize()
        kv.append(0, s, [t], dk.data_ptr(), dv.data_ptr())
        kv.attend(0, s, [m], dq.data_ptr(), out.data_ptr(), heads=HEADS, scale=float(scale), dtype=dtype, causal=causal)
        torch.cuda.synchronize()
    scores = dq[:, 0, 0].double().cpu().numpy()[:, None] * held(k, page)[None, :, 0, 0].astype(np.float64) * np.float64(scale)
    return out.double().cpu().numpy(), scores, held(v, page)[:, 0].astype(np.float64)


def check(key, sizes, v, dtype, page, causal=False):
    got, scores, values = run(key, sizes, v, dtype, page, causal)
    want, tol = attention(scores, values, dtype, causal)
    assert np.isfinite(got).all()
    bad = np.abs(got - want[:, None]) > tol[:, None]
    assert not bad.any(), f"{bad.sum()} values off, worst {np.abs(got - want[:, None]).max()} (tolerance {tol.max()})"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rise", [15.0, 21.5])
def test_the_maximum_rises_in_every_block(dtype, causal, rise):
    """Scores that climb by more than a raise every 32 positions, over several steps, for most rows of a warp; others fall
    or stay."""
    t, m = 400, 256
    rng = np.random.default_rng(3)
    sizes = rng.choice([1.0, 1.0, 1.0, 0.75, 0.5, -1.0, 0.0], m)
    check(rise * (np.arange(t) // 32), sizes, rng.standard_normal((t, HD)), dtype, 128, causal)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [24.5, 25.0, 26.0, 28.0])
def test_a_late_maximum_far_above(dtype, top):
    """One step: low scores, many just below what raises the maximum, then one 18 to 21 powers of two above those. The
    output is the many's share alone, 2e-4 and less, which one f16 factor between the two maxima cannot hold."""
    t, m = 127, 256
    key = np.zeros(t)
    key[32:96] = 6.9
    key[96] = top
    v = np.zeros((t, HD))
    v[:96] = 1.0
    v[:, HD // 2:] *= np.linspace(0.5, 1.5, t)[:, None]
    sizes = np.ones(m)
    sizes[1::3] = 0.97
    check(key, sizes, v, dtype, 128)
