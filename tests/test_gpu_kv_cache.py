"""The key/value cache held in 8 bits (trit_cuda_kv_*): what it holds, the
attention over it, and its page operations, against 64-bit numpy."""
import math

import numpy as np
import pytest

from tests.kv_oracle import attend, held
from trit_b200 import KvCache, TritError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def rows(seed, *shape, dtype="f32"):
    """Rows as the type holds them: (device tensor, f64)."""
    x = torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32)).to(TYPES[dtype]).cuda()
    return x, x.double().cpu().numpy()


def fill(kv, layer, seqs, parts, dtype="f32", extend=True):
    """Appends parts[i] = (k, v) device rows to seqs[i]."""
    counts = [k.shape[0] for k, _ in parts]
    if extend:
        kv.extend(seqs, counts)
    k, v = torch.cat([k for k, _ in parts]), torch.cat([v for _, v in parts])
    torch.cuda.synchronize()
    kv.append(layer, seqs, counts, k.data_ptr(), v.data_ptr(), dtype=dtype)
    torch.cuda.synchronize()


def contents(kv, layer, seq, kv_heads, hd, count=None, first=0):
    n = kv.length(seq) - first if count is None else count
    k = torch.full((n, kv_heads, hd), float("nan"), device="cuda")
    v = torch.full((n, kv_heads, hd), float("nan"), device="cuda")
    kv.read(layer, [seq], [first], [n], k.data_ptr() if n else None, v.data_ptr() if n else None)
    torch.cuda.synchronize()
    return k.cpu().numpy(), v.cpu().numpy()


def run_attend(kv, layer, seqs, q, counts, heads, scale, dtype, causal=True, stream=None):
    out = torch.full_like(q, float("nan"))
    torch.cuda.synchronize()
    kv.attend(layer, seqs, counts, q.data_ptr(), out.data_ptr(), heads=heads, scale=scale, dtype=dtype, causal=causal,
              stream=stream)
    torch.cuda.synchronize()
    return out


def check_attend(out, q64, ks, vs, counts, scale, dtype, causal=True):
    at = 0
    for k, v, m in zip(ks, vs, counts):
        want, tol = attend(q64[at:at + m], k, v, scale, causal)
        # Rows of 16-bit types: the weights are one f16 (2^-11 each, numerator only), and the output is rounded.
        if dtype != "f32" and len(v):
            tol = tol + 2.0**-10 * np.abs(v).max() + HALF_STEP[dtype] * np.abs(want)
        got = out[at:at + m].double().cpu().numpy()
        assert np.isfinite(got).all()
        bad = np.abs(got - want) > tol
        assert not bad.any(), f"{bad.sum()} values off, worst {np.abs(got - want).max()} (tolerance {tol.max()})"
        at += m


@pytest.mark.parametrize("page, hd", [(16, 64), (32, 128), (64, 128), (64, 64), (128, 128)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_holds_what_the_definition_says(page, hd, dtype):
    """Lengths around a page's borders, two layers, values equal to the bit."""
    lens = [1, 2, page - 1, page, page + 1, 2 * page + 3, 3 * page]
    with KvCache(kv_heads=3, pages=16, layers=2, head_dim=hd, page_tokens=page, sequences=8, max_tokens=512) as kv:
        seqs = kv.open(len(lens))
        kv.extend(seqs, lens)
        for layer in range(2):
            data = [(rows(100 * layer + i, n, 3, hd, dtype=dtype), rows(100 * layer + 50 + i, n, 3, hd, dtype=dtype))
                    for i, n in enumerate(lens)]
            fill(kv, layer, seqs, [(k[0], v[0]) for k, v in data], dtype, extend=False)
            for s, (k, v) in zip(seqs, data):
                gk, gv = contents(kv, layer, s, 3, hd)
                assert np.array_equal(gk, held(k[1], page)) and np.array_equal(gv, held(v[1], page))


@pytest.mark.parametrize("pieces", [[1] * 40, [5, 30, 5], [17, 1, 1, 21], [16, 16, 8], [3, 37]])
def test_pieces_do_not_change_the_codes(pieces):
    (k, k64), (v, v64) = rows(1, 40, 2, 64), rows(2, 40, 2, 64)
    with KvCache(kv_heads=2, pages=4, head_dim=64, page_tokens=16, sequences=2, max_tokens=64) as kv:
        s = kv.open(1)
        at = 0
        for n in pieces:
            fill(kv, 0, s, [(k[at:at + n], v[at:at + n])])
            at += n
            gk, gv = contents(kv, 0, s[0], 2, 64)
            assert np.array_equal(gk, held(k64[:at], 16)) and np.array_equal(gv, held(v64[:at], 16))


def test_odd_values():
    """Zero pages, ties between codes, infinities and NaN, subnormal and huge values."""
    page, hd = 16, 64
    x = np.zeros((5 * page, 1, hd), np.float32)
    x[page:2 * page] = np.arange(page * hd).reshape(page, 1, hd) % 255 / 2 - 63.5  # halves: ties, with the next line
    x[page, 0, 0] = 127.0
    x[2 * page, 0, :4] = [np.inf, -np.inf, np.nan, 1e30]
    x[3 * page:4 * page] = 6e-8
    x[4 * page:] = np.random.default_rng(0).standard_normal((page, 1, hd)) * 6e4
    d = torch.from_numpy(x).cuda()
    with KvCache(kv_heads=1, pages=8, head_dim=hd, page_tokens=page, sequences=2, max_tokens=128) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(d, -d)])
        gk, gv = contents(kv, 0, s[0], 1, hd)
        assert np.array_equal(gk, held(x, page)) and np.array_equal(gv, held(-x, page))


def test_codes_beside_every_border():
    """Pages whose values are the f16 numbers next to (n + 1/2) scale, at scales of many sizes: the code is the nearest,
    exactly, wherever the page's scale puts the border."""
    page, hd, pages = 16, 64, 200
    rng = np.random.default_rng(3)
    tops = np.concatenate([[65504.0, 127.0, 63.5, 1.0, 6e-8, 1.2e-7], np.exp(rng.uniform(np.log(1e-6), np.log(6e4), pages - 6))])
    tops = tops.astype(np.float16).astype(np.float64)
    scale = (tops / 127).astype(np.float32).astype(np.float64)
    n = rng.integers(-127, 127, (pages, page * hd))
    x = ((n + 0.5) * scale[:, None]).astype(np.float16)
    step = rng.integers(-1, 2, x.shape)
    x = np.where(step < 0, np.nextafter(x, np.float16(-np.inf)), np.where(step > 0, np.nextafter(x, np.float16(np.inf)), x))
    x = np.clip(x.astype(np.float64), -tops[:, None], tops[:, None])
    x[:, 0] = tops
    x = x.astype(np.float32).reshape(pages * page, 1, hd)
    with KvCache(kv_heads=1, pages=pages, head_dim=hd, page_tokens=page, sequences=1, max_tokens=pages * page) as kv:
        s = kv.open(1)
        d = torch.from_numpy(x).cuda()
        fill(kv, 0, s, [(d, -d)])
        gk, gv = contents(kv, 0, s[0], 1, hd)
        assert np.array_equal(gk, held(x, page)) and np.array_equal(gv, held(-x, page))


@pytest.mark.parametrize("kv_heads, group", [(1, 1), (2, 2), (1, 3), (2, 4), (1, 5), (1, 8), (1, 20)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_next_token(kv_heads, group, dtype):
    """One row a sequence over lengths of one position to many pages."""
    hd, page = 128, 32
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 64, 257, 600]
    heads = kv_heads * group
    with KvCache(kv_heads=kv_heads, pages=64, head_dim=hd, page_tokens=page, sequences=16, max_tokens=1024) as kv:
        seqs = kv.open(len(lens))
        data = [(rows(i, n, kv_heads, hd, dtype=dtype), rows(50 + i, n, kv_heads, hd, dtype=dtype)) for i, n in enumerate(lens)]
        fill(kv, 0, seqs, [(k[0], v[0]) for k, v in data], dtype)
        q, q64 = rows(99, len(lens), heads, hd, dtype=dtype)
        out = run_attend(kv, 0, seqs, q, [1] * len(lens), heads, 1 / math.sqrt(hd), dtype)
        check_attend(out, q64, [held(k[1], page) for k, _ in data], [held(v[1], page) for _, v in data], [1] * len(lens),
                     1 / math.sqrt(hd), dtype)


@pytest.mark.parametrize("hd, page, heads, kv_heads", [(128, 64, 8, 2), (64, 16, 6, 2), (128, 128, 5, 1), (64, 64, 4, 4)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_behind_a_context(hd, page, heads, kv_heads, dtype, causal):
    """Prompt pieces (causal) and rows that see every position, ragged; sequences without rows, and, without causal
    order, without positions, among them."""
    lens, counts = [300, 1, 65, 128, 200, 40], [130, 1, 65, 0, 3, 17]
    if not causal:
        lens, counts = lens + [0, 1], counts + [5, 70]
    scale = 0.17
    with KvCache(kv_heads=kv_heads, pages=128, head_dim=hd, page_tokens=page, sequences=8, max_tokens=512) as kv:
        seqs = kv.open(len(lens))
        data = [(rows(i, n, kv_heads, hd, dtype=dtype), rows(50 + i, n, kv_heads, hd, dtype=dtype)) for i, n in enumerate(lens)]
        fill(kv, 0, seqs, [(k[0], v[0]) for k, v in data], dtype)
        q, q64 = rows(99, sum(counts), heads, hd, dtype=dtype)
        out = run_attend(kv, 0, seqs, q, counts, heads, scale, dtype, causal)
        check_attend(out, q64, [held(k[1], page) for k, _ in data], [held(v[1], page) for _, v in data], counts, scale, dtype, causal)


def test_many_runs_and_repeated_sequences():
    """More sequences than one launch takes, some named several times."""
    hd, page, n = 64, 16, 150
    with KvCache(kv_heads=1, pages=400, head_dim=hd, page_tokens=page, sequences=n, max_tokens=64) as kv:
        seqs = kv.open(n)
        lens = [1 + i % 37 for i in range(n)]
        data = [(rows(i, t, 1, hd), rows(1000 + i, t, 1, hd)) for i, t in enumerate(lens)]
        fill(kv, 0, seqs, [(k[0], v[0]) for k, v in data])
        who = list(range(n)) + [3, 3, 149, 0]
        q, q64 = rows(5, len(who), 2, hd)
        out = run_attend(kv, 0, [seqs[i] for i in who], q, [1] * len(who), 2, 0.125, "f32")
        check_attend(out, q64, [held(data[i][0][1], page) for i in who], [held(data[i][1][1], page) for i in who], [1] * len(who),
                     0.125, "f32")


@pytest.mark.parametrize("size", [1.0, 40.0, 1e-6, 3e4])
def test_scores_and_values_of_any_size(size):
    """Sharp and flat softmaxes; a page of zero values and one of large ones beside small ones. The tolerance grows with
    the scores as derived."""
    hd, page, t = 128, 16, 90
    (q, q64), (k, k64), (v, v64) = rows(1, 3, 4, hd), rows(2, t, 1, hd), rows(3, t, 1, hd)
    q, q64 = q * size, q64.astype(np.float32) * np.float32(size)
    v[16:32] = 0
    v64[16:32] = 0
    v[32:48] *= 128
    v64[32:48] *= 128
    with KvCache(kv_heads=1, pages=16, head_dim=hd, page_tokens=page, sequences=1, max_tokens=128) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(k, v)])
        out = run_attend(kv, 0, s, q, [3], 4, 0.09, "f32")
        check_attend(out, q64, [held(k64, page)], [held(v64, page)], [3], 0.09, "f32")


def test_strides_and_unaligned_rows():
    """Keys, values and queries as columns of one wider tensor, at odd offsets, and an output with its own stride whose
    other places stay as they were."""
    hd, page, heads, kv_heads, t = 64, 16, 4, 2, 37
    for off in (0, 1, 3):
        wide, wide64 = rows(off, t, (heads + 2 * kv_heads) * hd + 5)
        a, b = off + heads * hd, off + (heads + kv_heads) * hd
        with KvCache(kv_heads=kv_heads, pages=8, head_dim=hd, page_tokens=page, sequences=1, max_tokens=64) as kv:
            s = kv.open(1)
            kv.extend(s, [t])
            kv.append(0, s, [t], wide.data_ptr() + 4 * a, wide.data_ptr() + 4 * b, k_stride=wide.shape[1], v_stride=wide.shape[1])
            out = torch.full((t + 2, heads * hd + 3), 7.0, device="cuda")
            kv.attend(0, s, [t], wide.data_ptr() + 4 * off, out.data_ptr() + 4, heads=heads, scale=0.125, q_stride=wide.shape[1],
                      out_stride=out.shape[1])
            torch.cuda.synchronize()
            k = held(wide64[:, a:a + kv_heads * hd].reshape(t, kv_heads, hd), page)
            v = held(wide64[:, b:b + kv_heads * hd].reshape(t, kv_heads, hd), page)
            got = out[:t, 1:1 + heads * hd].reshape(t, heads, hd)
            check_attend(got, wide64[:, off:off + heads * hd].reshape(t, heads, hd), [k], [v], [t], 0.125, "f32")
            rest = out.clone()
            rest[:t, 1:1 + heads * hd] = 7.0
            assert bool((rest == 7.0).all())


def test_output_may_be_the_query():
    hd, page = 128, 64
    (k, k64), (v, v64), (q, q64) = rows(1, 700, 2, hd), rows(2, 700, 2, hd), rows(3, 2, 4, hd)
    with KvCache(kv_heads=2, pages=16, head_dim=hd, page_tokens=page, sequences=1, max_tokens=1024) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(k, v)])
        kv.attend(0, s, [2], q.data_ptr(), q.data_ptr(), heads=4, scale=0.1)
        torch.cuda.synchronize()
        check_attend(q, q64, [held(k64, page)], [held(v64, page)], [2], 0.1, "f32")


def test_what_a_sequence_left_does_not_reach_the_next():
    """A sequence full of infinities and NaN goes; a shorter one takes its place."""
    hd, page = 64, 32
    bad = torch.full((50, 1, hd), float("inf"), device="cuda")
    bad[::2] = float("nan")
    with KvCache(kv_heads=1, pages=2, head_dim=hd, page_tokens=page, sequences=1, max_tokens=64) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(bad, bad)])
        kv.release(s)
        for t in (1, 5, 33):
            s = kv.open(1)
            (k, k64), (v, v64), (q, q64) = rows(t, t, 1, hd), rows(t + 1, t, 1, hd), rows(t + 2, 1, 2, hd)
            fill(kv, 0, s, [(k, v)])
            out = run_attend(kv, 0, s, q, [1], 2, 0.125, "f32")
            check_attend(out, q64, [held(k64, page)], [held(v64, page)], [1], 0.125, "f32")
            kv.release(s)


@pytest.mark.parametrize("cut", [0, 1, 15, 16, 17, 32, 40, 41])
def test_fork(cut):
    """A branch at any position: shared full pages, its own open page; parent and branch then grow apart."""
    hd, page, t = 64, 16, 41
    (k, k64), (v, v64) = rows(1, t, 2, hd), rows(2, t, 2, hd)
    with KvCache(kv_heads=2, pages=8, layers=2, head_dim=hd, page_tokens=page, sequences=4, max_tokens=96) as kv:
        s = kv.open(1)
        kv.extend(s, [t])
        for layer in range(2):
            fill(kv, layer, s, [(k, v)], extend=False)
        used = kv.pages()[0]
        a, b = kv.fork([s[0], s[0]], [cut, t])
        assert kv.pages()[0] == used and kv.length(a) == cut and kv.length(b) == t
        hk, hv = held(k64, page), held(v64, page)
        # A cut inside a full page keeps that page's values, in f16.
        ck, cv = hk[:cut].copy(), hv[:cut].copy()
        ck[cut // page * page:] = ck[cut // page * page:].astype(np.float16)
        cv[cut // page * page:] = cv[cut // page * page:].astype(np.float16)
        (k2, k264), (v2, v264) = rows(3, 20, 2, hd), rows(4, 20, 2, hd)
        kv.extend([a, b, s[0]], [20, 3, 1])
        for layer in range(2):
            gk, gv = contents(kv, layer, s[0], 2, hd, t - t % page)
            assert np.array_equal(gk, hk[:t - t % page]) and np.array_equal(gv, hv[:t - t % page])
            fill(kv, layer, [a, b, s[0]], [(k2, v2), (k2[:3], v2[:3]), (k2[5:6], v2[5:6])], extend=False)
            for q, old, new in ((a, (ck, cv), (k264, v264)), (b, (k64, v64), (k264[:3], v264[:3])),
                                (s[0], (k64, v64), (k264[5:6], v264[5:6]))):
                gk, gv = contents(kv, layer, q, 2, hd)
                for got, o, w in ((gk, old[0], new[0]), (gv, old[1], new[1])):
                    whole = o.shape[0] // page * page
                    want = np.concatenate([held(o, page)[:whole] if o.dtype == np.float64 else o[:whole],
                                           held(np.concatenate([o[whole:], w]), page)])
                    assert np.array_equal(got, want)
        kv.release([s[0]])
        gk, _ = contents(kv, 1, b, 2, hd, 32)
        assert np.array_equal(gk, hk[:32])
        kv.release([a, b])
        assert kv.pages()[0] == 0


def test_copy_compact_release():
    """Copies on pages of their own; gaps close; every sequence keeps what it holds, shared pages too."""
    hd, page, n = 64, 16, 9
    with KvCache(kv_heads=2, pages=64, layers=3, head_dim=hd, page_tokens=page, sequences=32, max_tokens=128) as kv:
        lens = [5, 16, 33, 48, 100, 17, 64, 1, 80]
        seqs = kv.open(n)
        kv.extend(seqs, lens)
        want = {}
        for layer in range(3):
            data = [(rows(layer * 100 + i, t, 2, hd), rows(layer * 100 + 50 + i, t, 2, hd)) for i, t in enumerate(lens)]
            fill(kv, layer, seqs, [(k[0], v[0]) for k, v in data], extend=False)
            for s, (k, v) in zip(seqs, data):
                want[layer, s] = held(k[1], page), held(v[1], page)
        full = sum(t // page for t in lens)
        copies, forks = kv.copy(seqs), kv.fork(seqs[2:5])
        assert kv.pages() == (2 * full, 64)
        kv.release(seqs[0::2] + copies[1::3])
        same = {q: s for q, s in list(zip(copies, seqs)) + list(zip(forks, seqs[2:5])) + list(zip(seqs, seqs))}
        alive = [q for q in same if q not in seqs[0::2] + copies[1::3]]
        used = kv.pages()[0]
        moved = kv.compact()
        assert moved > 0 and kv.pages()[0] == used and kv.compact() == 0
        for q in alive:
            for layer in range(3):
                gk, gv = contents(kv, layer, q, 2, hd)
                assert np.array_equal(gk, want[layer, same[q]][0]) and np.array_equal(gv, want[layer, same[q]][1])
        kv.release(alive)
        assert kv.pages()[0] == 0


def test_pages_far_into_the_pool():
    """A page whose codes lie beyond 2^32 bytes."""
    hd, page, kv_heads = 128, 64, 8
    skip = 33000  # 131072 bytes a page and layer
    with KvCache(kv_heads=kv_heads, pages=skip + 8, head_dim=hd, page_tokens=page, sequences=3, max_tokens=skip * page) as kv:
        kv.extend(kv.open(1), [skip * page])
        s = kv.open(1)
        (k, k64), (v, v64), (q, q64) = rows(1, 150, kv_heads, hd), rows(2, 150, kv_heads, hd), rows(3, 1, kv_heads, hd)
        fill(kv, 0, s, [(k, v)])
        gk, gv = contents(kv, 0, s[0], kv_heads, hd)
        assert np.array_equal(gk, held(k64, page)) and np.array_equal(gv, held(v64, page))
        out = run_attend(kv, 0, s, q, [1], kv_heads, 0.1, "f32")
        check_attend(out, q64, [held(k64, page)], [held(v64, page)], [1], 0.1, "f32")
        c = kv.copy(s)
        assert np.array_equal(contents(kv, 0, c[0], kv_heads, hd)[0], held(k64, page))


# Enough rows and heads for the kernel of many rows (8192 columns in a call, 64 in a run).
@pytest.mark.parametrize("hd, page, heads, kv_heads", [(128, 64, 16, 4), (64, 16, 20, 4), (128, 128, 15, 5), (64, 32, 16, 16)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(hd, page, heads, kv_heads, dtype, causal):
    lens, counts = [300, 700, 129, 257, 31], [300, 200, 128, 1, 31]
    if not causal:
        lens, counts = lens + [0, 1], counts + [70, 70]
    with KvCache(kv_heads=kv_heads, pages=128, head_dim=hd, page_tokens=page, sequences=8, max_tokens=1024) as kv:
        seqs = kv.open(len(lens))
        data = [(rows(i, n, kv_heads, hd, dtype=dtype), rows(50 + i, n, kv_heads, hd, dtype=dtype)) for i, n in enumerate(lens)]
        fill(kv, 0, seqs, [(k[0], v[0]) for k, v in data], dtype)
        q, q64 = rows(99, sum(counts), heads, hd, dtype=dtype)
        scale = 0.1 if causal else -0.1
        out = run_attend(kv, 0, seqs, q, counts, heads, scale, dtype, causal)
        check_attend(out, q64, [held(k[1], page) for k, _ in data], [held(v[1], page) for _, v in data], counts, scale, dtype, causal)


@pytest.mark.parametrize("size", [1.0, 40.0, 1e-6])
def test_prompts_of_any_scores(size):
    """Sharp and flat softmaxes whose largest score comes late, over pages of values of very different size."""
    hd, page, t, heads = 128, 16, 400, 32
    (q, q64), (k, k64), (v, v64) = rows(1, t, heads, hd), rows(2, t, 1, hd), rows(3, t, 1, hd)
    ramp = torch.linspace(0.01, 1.0, t, device="cuda")[:, None, None] * size
    q, k = q * size, k * ramp
    v[160:176] = 0
    v[176:192] *= 1000
    q64, k64, v64 = (x.double().cpu().numpy() for x in (q, k, v))
    with KvCache(kv_heads=1, pages=32, head_dim=hd, page_tokens=page, sequences=1, max_tokens=512) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(k, v)])
        out = run_attend(kv, 0, s, q, [t], heads, 0.09, "f32")
        check_attend(out, q64, [held(k64, page)], [held(v64, page)], [t], 0.09, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_rows_behind_a_long_context(dtype, hd):
    """Few tiles of many rows, so that their positions are shared out and the shares joined; the output may be the query."""
    page, t, m, heads = 32, 6000, 300, 32
    (k, k64), (v, v64), (q, q64) = rows(1, t, 1, hd, dtype=dtype), rows(2, t, 1, hd, dtype=dtype), rows(3, m, heads, hd, dtype=dtype)
    with KvCache(kv_heads=1, pages=200, head_dim=hd, page_tokens=page, sequences=2, max_tokens=8192) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(k, v)], dtype)
        for causal in (True, False):
            out = q.clone()
            torch.cuda.synchronize()
            kv.attend(0, s, [m], out.data_ptr(), out.data_ptr(), heads=heads, scale=0.11, dtype=dtype, causal=causal)
            torch.cuda.synchronize()
            check_attend(out, q64, [held(k64, page)], [held(v64, page)], [m], 0.11, dtype, causal=causal)


def test_many_rows_of_long_sequences_unshared():
    """So many tiles that none is shared out: every warp walks all of its positions in one go."""
    hd, page, t, n = 128, 64, 1500, 600
    (k, k64), (v, v64), (q, q64) = rows(1, t, 4, hd), rows(2, t, 4, hd), rows(3, n, 4, hd)
    with KvCache(kv_heads=4, pages=32, head_dim=hd, page_tokens=page, sequences=1, max_tokens=2048) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(k, v)])
        out = run_attend(kv, 0, s * n, q, [1] * n, 4, 0.09, "f32", causal=False)
        want, tol = attend(q64, held(k64, page), held(v64, page), 0.09, False)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


def test_calls_from_two_threads():
    """Two host threads on two streams, each with its sequences: calls take turns, results are each one's own."""
    import threading

    hd, page, t = 64, 16, 50
    errors = []
    with KvCache(kv_heads=2, pages=64, head_dim=hd, page_tokens=page, sequences=8, max_tokens=64) as kv:
        def work(seed):
            try:
                stream = torch.cuda.Stream()
                for i in range(20):
                    s = kv.open(1)
                    (k, k64), (v, v64), (q, q64) = (rows(seed + 3 * i + j, t, 2, hd) for j in range(3))
                    out = torch.empty_like(q)
                    torch.cuda.synchronize()
                    kv.extend(s, [t], stream=stream.cuda_stream)
                    kv.append(0, s, [t], k.data_ptr(), v.data_ptr(), stream=stream.cuda_stream)
                    kv.attend(0, s, [t], q.data_ptr(), out.data_ptr(), heads=2, scale=0.125, stream=stream.cuda_stream)
                    stream.synchronize()
                    check_attend(out, q64, [held(k64, page)], [held(v64, page)], [t], 0.125, "f32")
                    kv.release(s)
            except BaseException as e:  # noqa: BLE001
                errors.append(e)

        threads = [threading.Thread(target=work, args=(1000 * i,)) for i in range(2)]
        for x in threads:
            x.start()
        for x in threads:
            x.join()
    assert not errors, errors


def test_steps_as_a_decoder_makes_them():
    """Everything together: prompts, steps that append and attend, a branch, a gap that closes; on two streams in turn
    without a wait between the calls."""
    hd, page, heads, kv_heads, layers = 64, 16, 4, 2, 2
    rng = np.random.default_rng(5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    with KvCache(kv_heads=kv_heads, pages=64, layers=layers, head_dim=hd, page_tokens=page, sequences=8, max_tokens=128) as kv:
        seqs = kv.open(3)
        past = {s: [[np.zeros((0, kv_heads, hd)), np.zeros((0, kv_heads, hd))] for _ in range(layers)] for s in seqs}
        checks, keep = [], []
        for step in range(24):
            stream = streams[step % 2].cuda_stream
            if step == 10:
                f = kv.fork([seqs[1]], stream=stream)[0]
                past[f] = [[a.copy(), b.copy()] for a, b in past[seqs[1]]]
                kv.release([seqs[0]])
                seqs = [seqs[1], seqs[2], f]
                kv.compact(stream=stream)
            counts = [int(c) for c in rng.integers(10, 30, 3)] if step == 0 else [1, 2, 1]
            kv.extend(seqs, counts, stream=stream)
            for layer in range(layers):
                with torch.cuda.stream(streams[step % 2]):
                    k, v, q = (torch.from_numpy(rng.standard_normal((sum(counts), h, hd)).astype(np.float32)).cuda()
                               for h in (kv_heads, kv_heads, heads))
                    out = torch.empty_like(q)
                    keep += [k, v, q, out]
                kv.append(layer, seqs, counts, k.data_ptr(), v.data_ptr(), stream=stream)
                kv.attend(layer, seqs, counts, q.data_ptr(), out.data_ptr(), heads=heads, scale=0.125, stream=stream)
                at = 0
                for s, c in zip(seqs, counts):
                    for i, x in enumerate((k, v)):
                        past[s][layer][i] = np.concatenate([past[s][layer][i], x[at:at + c].double().cpu().numpy()])
                    at += c
                checks.append((out, q, [past[s][layer][0] for s in seqs], [past[s][layer][1] for s in seqs], counts))
        torch.cuda.synchronize()
        for out, q, ks, vs, counts in checks:
            check_attend(out, q.double().cpu().numpy(), [held(k, page) for k in ks], [held(v, page) for v in vs], counts, 0.125, "f32")


def test_captured_attention():
    """Two graphs of one cache replayed at once, split over the positions, give what the calls give."""
    hd, page, t = 128, 64, 5000
    (k, _), (v, _) = rows(1, t, 2, hd), rows(2, t, 2, hd)
    with KvCache(kv_heads=2, pages=100, head_dim=hd, page_tokens=page, sequences=2, max_tokens=8192) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(k, v)])
        qs = [rows(i, 1, 8, hd)[0] for i in (3, 4)]
        want = [run_attend(kv, 0, s, q, [1], 8, 0.1, "f32") for q in qs]
        outs, graphs, streams = [torch.zeros_like(q) for q in qs], [], [torch.cuda.Stream() for _ in qs]
        for q, out, stream in zip(qs, outs, streams):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                for _ in range(4):
                    kv.attend(0, s, [1], q.data_ptr(), out.data_ptr(), heads=8, scale=0.1, stream=stream.cuda_stream)
            graphs.append(g)
        torch.cuda.synchronize()
        for _ in range(3):
            for g, out, stream in zip(graphs, outs, streams):
                out.zero_()
                torch.cuda.synchronize()
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))
        # What would write positions is not recorded.
        side = torch.cuda.Stream()
        kv.extend(s, [1])
        g = torch.cuda.CUDAGraph()
        x = torch.zeros(1, 2, hd, device="cuda")
        with torch.cuda.graph(g, stream=side):
            for call in (lambda: kv.append(0, s, [1], x.data_ptr(), x.data_ptr(), stream=side.cuda_stream),
                         lambda: kv.copy([], stream=side.cuda_stream) or kv.extend(s, [page], stream=side.cuda_stream)):
                with pytest.raises(TritError, match="being captured"):
                    call()
            x.add_(1)
        assert kv.length(s[0]) == t + 1
        kv.append(0, s, [1], x.data_ptr(), x.data_ptr())
        torch.cuda.synchronize()


def test_captured_prompt():
    """The kernel of many rows, with what it puts aside and shares out, in two graphs replayed at once."""
    hd, page, t, m, heads = 128, 64, 3000, 300, 32
    (k, _), (v, _) = rows(1, t, 1, hd), rows(2, t, 1, hd)
    with KvCache(kv_heads=1, pages=64, head_dim=hd, page_tokens=page, sequences=1, max_tokens=4096) as kv:
        s = kv.open(1)
        fill(kv, 0, s, [(k, v)])
        qs = [rows(i, m, heads, hd)[0] for i in (3, 4)]
        want = [run_attend(kv, 0, s, q, [m], heads, 0.1, "f32") for q in qs]
        outs, graphs, streams = [torch.zeros_like(q) for q in qs], [], [torch.cuda.Stream() for _ in qs]
        for q, out, stream in zip(qs, outs, streams):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                kv.attend(0, s, [m], q.data_ptr(), out.data_ptr(), heads=heads, scale=0.1, stream=stream.cuda_stream)
            graphs.append(g)
        torch.cuda.synchronize()
        for _ in range(3):
            for out in outs:
                out.zero_()
            torch.cuda.synchronize()
            for g, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_refusals():
    hd = 64
    with KvCache(kv_heads=2, pages=4, layers=2, head_dim=hd, page_tokens=16, sequences=3, max_tokens=60) as kv:
        a, b = kv.open(2)
        x = torch.zeros(64, 4, hd, device="cuda")
        p = x.data_ptr()
        host = np.zeros(64 * 4 * hd, np.float32)

        def no(text, f):
            with pytest.raises(TritError, match=text):
                f()

        no("2 sequences asked, 1 of 3", lambda: kv.open(2))
        no("not open", lambda: kv.extend([2], [1]))
        no("not open", lambda: kv.release([-1]))
        no("not open", lambda: kv.attend(0, [3], [1], p, p, heads=2, scale=1.0))
        no("named twice", lambda: kv.extend([a, a], [1, 1]))
        no("negative", lambda: kv.extend([a], [-1]))
        no("exceed max_tokens 60", lambda: kv.extend([a], [61]))
        no("counts for", lambda: kv.extend([a], [1, 2]))
        no("pages asked", lambda: kv.extend([a, b], [48, 32]))
        assert kv.length(a) == 0 and kv.pages() == (0, 4)
        kv.extend([a], [20])
        no("layer 2", lambda: kv.append(2, [a], [20], p, p))
        no("dtype", lambda: kv.append(0, [a], [20], p, p, dtype="f64"))
        no("k is NULL", lambda: kv.append(0, [a], [20], None, p))
        no("v is NULL", lambda: kv.append(0, [a], [20], p, None))
        no("aligned", lambda: kv.append(0, [a], [20], p + 2, p))
        no("not device memory", lambda: kv.append(0, [a], [20], host.ctypes.data, p))
        no("shorter than a row", lambda: kv.append(0, [a], [20], p, p, k_stride=2 * hd - 1))
        no("extend first", lambda: kv.append(0, [a], [19], p, p))
        no("a count of 21", lambda: kv.append(0, [a], [21], p, p))
        no("named twice", lambda: kv.append(0, [a, a], [20, 0], p, p))
        no("not appended yet", lambda: kv.attend(0, [a], [1], p, p, heads=2, scale=1.0))
        no("with 0 in layer 0", lambda: kv.read(0, [a], [0], [1], p, p))
        kv.append(0, [a], [20], p, p)
        no("append every position once", lambda: kv.append(0, [a], [20], p, p))
        no("not appended yet", lambda: kv.fork([a]))
        no("not appended yet", lambda: kv.copy([a]))
        kv.append(1, [a], [20], p, p)
        no("21 causal rows", lambda: kv.attend(0, [a], [21], p, p, heads=2, scale=1.0))
        no("do not share", lambda: kv.attend(0, [a], [1], p, p, heads=3, scale=1.0))
        no("do not share", lambda: kv.attend(0, [a], [1], p, p, heads=0, scale=1.0))
        no("out is NULL", lambda: kv.attend(0, [a], [1], p, None, heads=2, scale=1.0))
        no("not device memory", lambda: kv.attend(0, [a], [1], host.ctypes.data, p, heads=2, scale=1.0))
        no("a fork at 21", lambda: kv.fork([a], [21]))
        no("a fork at -1", lambda: kv.fork([a], [-1]))
        no("positions 5", lambda: kv.read(0, [a], [5], [16], p, p))
        kv.extend([b], [40])
        for layer in range(2):
            kv.append(layer, [b], [40], p, p)
        no("pages asked", lambda: kv.copy([b]))
        no("released twice", lambda: kv.release([b, b]))
        c = kv.fork([b])
        no("sequences asked", lambda: kv.fork([a]))
        kv.release([b] + c)
        # Calls of nothing.
        kv.extend([], [])
        kv.append(0, [a], [0], None, None)
        kv.attend(0, [a], [0], None, None, heads=2, scale=1.0)
        kv.read(0, [a], [20], [0], None, None)
        assert kv.fork([]) == [] and kv.copy([]) == []
        torch.cuda.synchronize()
