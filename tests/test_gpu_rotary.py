"""Rotary positions (trit_cuda_rotary_*) against 64 bits."""
import numpy as np
import pytest

from trit_b200 import Rotary, TritError
from tests import rows_oracle

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check(got, x, positions, rotary, interleaved):
    """cos and sin are off by at most 2^-23 (half a step from the angle's rounding, up to 2 steps of the function, the
    factor's product), so a value by 2^-22 (|a| + |b|) with the products' own roundings, and half a step of its type."""
    f, factor = rotary.frequencies()
    x = x.double().cpu().numpy()
    want = rows_oracle.turned(x, positions.cpu().numpy(), f, factor, interleaved)
    n, eps = len(f), torch.finfo(got.dtype).eps
    size = np.zeros_like(x)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    tiny = torch.finfo(got.dtype).smallest_normal * eps
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= size * factor * 2.0**-22 + np.abs(want) * eps / 2 * 1.01 + tiny).all(), off.max()
    assert np.array_equal(got.double().cpu().numpy()[..., 2 * n:], x[..., 2 * n:])


def call(rotary, positions, q, k, dtype, q_out=None, k_out=None, stream=None):
    rotary.apply(positions.data_ptr(), q.shape[0], q.data_ptr(), q.shape[1], k.data_ptr() if k is not None else None,
                 k.shape[1] if k is not None else 0, dtype=dtype, q_stride=q.stride(0), k_stride=k.stride(0) if k is not None else 0,
                 q_out_ptr=q_out.data_ptr() if q_out is not None else None, k_out_ptr=k_out.data_ptr() if k_out is not None else None,
                 q_out_stride=q_out.stride(0) if q_out is not None else 0, k_out_stride=k_out.stride(0) if k_out is not None else 0,
                 stream=stream)
    torch.cuda.synchronize()


def make(rows, heads, kv, hd, dtype, far=100000, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + rows)
    q = torch.randn(rows, heads, hd, generator=g, device="cuda").to(TYPES[dtype])
    k = torch.randn(rows, kv, hd, generator=g, device="cuda").to(TYPES[dtype])
    return q, k, torch.randint(-3, far, (rows,), generator=g, device="cuda")


@pytest.mark.parametrize("hd, rd", [(2, 2), (4, 2), (18, 6), (64, 64), (64, 32), (80, 36), (96, 96), (128, 128), (128, 64), (128, 126),
                                    (130, 128), (256, 256), (512, 512)])
@pytest.mark.parametrize("layout", ["halves", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_heads(hd, rd, layout, dtype):
    rotary = Rotary(hd, rotary_dim=rd, layout=layout, theta=1e4)
    for rows, heads, kv in [(1, 1, 1), (3, 8, 2), (70, 5, 1)]:
        q, k, at = make(rows, heads, kv, hd, dtype)
        qo, ko = torch.full((rows + 1, heads, hd), 3.0, dtype=q.dtype, device="cuda"), torch.full((rows + 1, kv, hd), 3.0, dtype=q.dtype,
                                                                                               device="cuda")
        call(rotary, at, q, k, dtype, qo, ko)
        check(qo[:-1], q, at, rotary, layout == "interleaved")
        check(ko[:-1], k, at, rotary, layout == "interleaved")
        assert bool((qo[-1] == 3).all() and (ko[-1] == 3).all())
        p, r = q.clone(), k.clone()
        call(rotary, at, p, r, dtype)
        assert torch.equal(p, qo[:-1]) and torch.equal(r, ko[:-1])


def test_most_heads():
    """As many heads as a call takes, one value a turn: each head as a call of few heads turns it."""
    rotary = Rotary(512)
    flat = torch.randn(2 * 65535 * 512 + 1, device="cuda").to(torch.bfloat16)
    want, at = flat.clone(), torch.tensor([77], device="cuda")
    q, k = flat[1:].view(2, 1, 65535, 512)
    call(rotary, at, q, k, "bf16")
    for i in range(0, 65535 * 2, 6555):
        part = want[1 + i * 512:1 + min(i + 6555, 65535 * 2) * 512]
        call(rotary, at, part.view(1, -1, 512), None, "bf16")
    assert torch.equal(flat, want)


@pytest.mark.parametrize("rows, heads, kv", [(1, 32, 8), (2, 64, 1), (64, 32, 8), (500, 16, 16), (4001, 8, 1)])
@pytest.mark.parametrize("layout", ["halves", "interleaved"])
def test_rows(rows, heads, kv, layout):
    """Out of fused rows of q | k | v, in place: the values stay."""
    rotary = Rotary(128, layout=layout, scaling="bands", factor=8.0, trained=8192, theta=5e5)
    g = torch.Generator("cuda").manual_seed(rows)
    qkv = torch.randn(rows, heads + 2 * kv, 128, generator=g, device="cuda").to(torch.bfloat16)
    at = torch.randint(0, 60000, (rows,), generator=g, device="cuda")
    x = qkv.clone()
    call(rotary, at, x[:, :heads], x[:, heads:heads + kv], "bf16")
    check(x[:, :heads], qkv[:, :heads], at, rotary, layout == "interleaved")
    check(x[:, heads:heads + kv], qkv[:, heads:heads + kv], at, rotary, layout == "interleaved")
    assert torch.equal(x[:, heads + kv:], qkv[:, heads + kv:])


def test_unaligned():
    """Heads and addresses that no wide load fits."""
    for layout in ("halves", "interleaved"):
        rotary = Rotary(64, layout=layout)
        flat = torch.randn(9 * 261 + 1, device="cuda").to(torch.float16)
        for first in (0, 1):
            q = flat[first:first + 9 * 261].view(9, 261)[:, :256].unflatten(1, (4, 64))
            at = torch.arange(9, device="cuda") * 1000
            out = torch.empty(9, 4, 64, dtype=q.dtype, device="cuda")
            call(rotary, at, q, None, "f16", out)
            check(out, q, at, rotary, layout == "interleaved")


def test_far_positions_and_back():
    """Positions far behind 32 bits, and the way back by negative ones."""
    rotary = Rotary(64, theta=1e4)
    q, k, _ = make(6, 4, 2, 64, "f32")
    at = torch.tensor([0, 1, 2**24 + 1, 2**31 + 5, -(2**33), 2**40 + 7], device="cuda")
    x = q.clone()
    call(rotary, at[:4], x[:4], None, "f32")
    check(x[:4], q[:4], at[:4], rotary, False)
    # The way back has the same angle: what is left is the two rotations' roundings.
    x, back = q.clone(), -at
    call(rotary, at, x, None, "f32")
    call(rotary, back, x, None, "f32")
    assert float((x - q).abs().max()) <= float(q.abs().max()) * 2.0**-19


def test_copied_values_stay_as_they_are():
    """Infinities and NaN behind the part that turns, and in one pair: nothing else sees them."""
    for layout in ("halves", "interleaved"):
        rotary = Rotary(64, rotary_dim=20, layout=layout)
        q, _, at = make(5, 3, 1, 64, "f32")
        q[:, :, 20:] = torch.tensor([float("inf"), float("nan"), -0.0, 1.0], device="cuda").repeat(11)
        out = torch.empty_like(q)
        call(rotary, at, q, None, "f32", out)
        assert torch.equal(out.view(torch.int32)[:, :, 20:], q.view(torch.int32)[:, :, 20:])
        assert bool(out[:, :, :20].isfinite().all())


def test_streams_and_replay():
    rotary = Rotary(128)
    q, k, at = make(200, 8, 2, 128, "bf16")
    outs = [(torch.empty_like(q), torch.empty_like(k)) for _ in range(3)]
    s1, s2, g = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    def one(i, s):
        rotary.apply(at.data_ptr(), 200, q.data_ptr(), 8, k.data_ptr(), 2, dtype="bf16", q_out_ptr=outs[i][0].data_ptr(),
                     k_out_ptr=outs[i][1].data_ptr(), stream=s.cuda_stream)
    torch.cuda.synchronize()
    for _ in range(10):
        one(0, s1)
        one(1, s2)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s2):
        one(2, s2)
    at.add_(11)
    g.replay()
    torch.cuda.synchronize()
    check(outs[2][0], q, at, rotary, False)
    at.sub_(11)
    for i in (0, 1):
        check(outs[i][0], q, at, rotary, False)
        check(outs[i][1], k, at, rotary, False)


def test_refused_pointers():
    rotary = Rotary(64)
    q, at, host = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, 2, 64)
    for args, words in [((at.data_ptr(), 4, host.data_ptr(), 2), "q is not device memory"), ((None, 4, q.data_ptr(), 2), "positions is NULL"),
                        ((at.data_ptr() + 4, 4, q.data_ptr(), 2), "positions is not aligned"),
                        ((at.data_ptr(), 4, q.data_ptr() + 1, 2), "q is not aligned"), ((at.data_ptr(), 4, None, 2), "q is NULL")]:
        with pytest.raises(TritError, match=words):
            rotary.apply(*args)
