"""Products with 4-bit weights (trit_dense_q4_0) against 64 bits."""
import numpy as np
import pytest

from trit_b200 import Dense

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def layer(n, k, seed):
    """Q4_0 blocks, and the weights they stand for."""
    rng = np.random.default_rng(seed)
    d = (rng.standard_normal((n, k // 32)) * 0.01).astype(np.float16)
    c = rng.integers(0, 16, (n, k // 32, 32))
    packed = (c[..., :16] | (c[..., 16:] << 4)).astype(np.uint8)
    blocks = np.concatenate([d[..., None].view(np.uint8).reshape(n, k // 32, 2), packed], axis=2)
    return blocks, (d.astype(np.float64)[..., None] * (c - 8)).reshape(n, k)


def rounded(x):
    """Rows as the layer's int8 activations stand for them (the quantizer of a Q8_0 layer, in its f32 steps)."""
    g = x.reshape(x.shape[0], -1, 32)
    top = np.abs(g).max(-1, keepdims=True)
    scale = np.where(top > 0, top / np.float32(127), np.float32(1)).astype(np.float32)
    code = np.clip(np.rint(g * (np.float32(1) / scale)), -127, 127)
    return (code.astype(np.float64) * scale.astype(np.float16).astype(np.float64)).reshape(x.shape)


def check(got, x, w):
    """Off by at most: 2^-22 of the row's largest a value from the two f16 of x, and f32 sums (2 steps a group, k / 32
    groups over 8 warps, 8 joins; 2^-23 each, as sums on the tensor cores need not round to nearest)."""
    want = x @ w.T
    k = x.shape[1]
    size = np.abs(x) @ np.abs(w).T
    tol = 2.0**-22 * np.abs(x).max(1, keepdims=True) * np.abs(w).sum(1)[None] + size * (k / 128 + 12) * 2.0**-23
    assert got.shape == want.shape and np.isfinite(got).all()
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} off, worst {np.abs(got - want).max()} of {tol.max()}"


@pytest.mark.parametrize("n, k", [(1, 32), (16, 64), (33, 96), (500, 1024), (4097, 2080), (96, 12320)])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 9, 16, 17, 40])
@pytest.mark.parametrize("table", [False, True])
def test_product(n, k, rows, table):
    blocks, w = layer(n, k, n + k)
    x = np.random.default_rng(rows).standard_normal((rows, k)).astype(np.float32)
    x[:, ::7] *= 30
    got = Dense.q4_0(blocks, n, k, table=table).forward(x)
    check(got, x.astype(np.float64) if table else rounded(x), w)


@pytest.mark.parametrize("rows", [32, 33, 100])
def test_many_rows_on_the_tensor_cores(rows):
    """n a multiple of 32 and k of 128: from 33 rows on the int8 product, with the same codes. Its f32 chain runs over the
    groups in order (k / 32 steps)."""
    n, k = 256, 1024
    blocks, w = layer(n, k, 5)
    dense = Dense.q4_0(blocks, n, k)
    for seed in (1, 2):
        x = np.random.default_rng(seed).standard_normal((rows, k)).astype(np.float32)
        got = dense.forward(x)
        want, size = rounded(x) @ w.T, np.abs(rounded(x)) @ np.abs(w).T
        assert (np.abs(got - want) <= size * (k / 32 + 4) * 2.0**-23 + 2.0**-22 * np.abs(x).max() * np.abs(w).sum(1)).all()
        assert np.array_equal(dense.forward(x[:3]), Dense.q4_0(blocks, n, k).forward(x[:3]))


def test_odd_rows():
    """Zero rows, very large and very small ones, and rows that are not numbers, each apart from the others."""
    n, k = 64, 256
    blocks, w = layer(n, k, 3)
    x = np.random.default_rng(1).standard_normal((6, k)).astype(np.float32)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, 5] = np.inf
    x[4, 7] = np.nan
    got = Dense.q4_0(blocks, n, k, table=True).forward(x)
    assert not np.isfinite(got[3:5]).any()
    for r in (0, 1, 2, 5):
        check(got[r:r + 1], x[r:r + 1].astype(np.float64), w)
    got = Dense.q4_0(blocks, n, k).forward(x[[0, 2, 5]])
    check(got, rounded(x[[0, 2, 5]]), w)


def test_device_calls_overlap_and_replay():
    """Calls on two streams at once, and a captured one, on the caller's tensors; places behind the output stay."""
    n, k = 1000, 512
    blocks, w = layer(n, k, 9)
    dense = Dense.q4_0(blocks, n, k, table=True)
    xs = [torch.randn(r, k, device="cuda") for r in (1, 7)]
    outs = [torch.full((x.shape[0] + 1, n), 5.0, device="cuda") for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, out, s in zip(xs, outs, streams):
            dense.forward_device(x.data_ptr(), x.shape[0], out.data_ptr(), s.cuda_stream)
    torch.cuda.synchronize()
    for x, out in zip(xs, outs):
        check(out[:-1].cpu().numpy(), x.double().cpu().numpy(), w)
        assert bool((out[-1] == 5.0).all())
    want, g = outs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[0]):
        dense.forward_device(xs[0].data_ptr(), 1, outs[0].data_ptr(), streams[0].cuda_stream)
    outs[0].fill_(5.0)
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
