"""RMSNorm with the residual's addition and 8-bit rows (trit_cuda_rms_norm) against its definition."""
import numpy as np
import pytest

from trit_b200 import TritError, rms_norm
from tests import rows_oracle

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def run(x, w, residual=None, eps=1e-6, values=True, codes=True, stream=None, **more):
    """(sum, out, codes, scales) of one call, out of place, between guards that have to stay."""
    m, d = x.shape
    kind = {v: k for k, v in TYPES.items()}
    def guarded(shape, dtype):
        return torch.full((shape[0] + 2, *shape[1:]), 7, dtype=dtype, device="cuda")
    h = guarded((m, d), x.dtype) if residual is not None else None
    y = guarded((m, d), x.dtype) if values else None
    q = guarded((m, d), torch.uint8) if codes else None
    s = guarded((m, (d + 127) // 128), torch.float32) if codes else None
    at = [t[1:].data_ptr() if t is not None else None for t in (h, y, q, s)]
    rms_norm(x.data_ptr(), w.data_ptr(), m, d, dtype=kind[x.dtype], weight_dtype=kind[w.dtype], eps=eps, sum_ptr=at[0],
             out_ptr=at[1], codes_ptr=at[2], scales_ptr=at[3], residual_ptr=residual.data_ptr() if residual is not None else None,
             x_stride=x.stride(0), residual_stride=residual.stride(0) if residual is not None else 0, stream=stream, **more)
    torch.cuda.synchronize()
    for t in (h, y, q, s):
        assert t is None or bool((t[0] == 7).all() and (t[-1] == 7).all())
    return [t[1:-1] if t is not None else None for t in (h, y, q, s)]


def check(x, w, residual, eps, got):
    """The sum is exact but for its rounding to the type, and the codes follow from it in the defined f32 steps. Values
    are off by the type's rounding and three f32 ones (of s, s w and the product)."""
    total, out, codes, scales = got
    if residual is not None:
        x = (x.float() + residual.float()).to(x.dtype)
        assert torch.equal(total, x)
    h, w = x.float().cpu().numpy(), w.float().cpu().numpy()
    if out is not None:
        h64 = h.astype(np.float64)
        want = h64 / np.sqrt((h64**2).mean(-1, keepdims=True) + eps) * w
        tiny = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
        tol = np.abs(want) * (torch.finfo(out.dtype).eps / 2 + 3.1 * 2.0**-24) + tiny
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()
    if codes is not None:
        c, s = rows_oracle.rows_of(rows_oracle.norm_f32(h, w, eps))
        assert np.array_equal(scales.cpu().numpy(), s)
        assert np.array_equal(codes.view(torch.float8_e4m3fn).double().cpu().numpy(), c)


def make(m, d, dtype, weight, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(m, d, generator=g, device="cuda") * (0.5 + 30 * (torch.rand(1, d, generator=g, device="cuda") > 0.98))
    r = torch.randn(m, d, generator=g, device="cuda") * 3
    w = 1 + 0.4 * torch.randn(d, generator=g, device="cuda")
    return x.to(TYPES[dtype]), r.to(TYPES[dtype]), w.to(TYPES[weight])


WIDTHS = [1, 2, 7, 8, 16, 120, 127, 128, 129, 136, 255, 256, 257, 264, 1000, 1001, 1024, 1032, 2048, 2056, 4096, 4099, 5120, 8192, 8200,
          8201, 16384, 20000, 33333]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_widths(width, dtype):
    for rows in (1, 3, 19):
        x, r, w = make(rows, width, dtype, "f32" if rows == 3 else dtype, width + rows)
        check(x, w, r, 1e-6, run(x, w, r))
        check(x, w, None, 1e-5, run(x, w, None, eps=1e-5))


@pytest.mark.parametrize("rows, width", [(1, 2048), (64, 4096), (700, 1024), (3000, 128), (1500, 2048), (300, 8192), (2001, 1000)])
@pytest.mark.parametrize("values, codes", [(True, False), (False, True), (True, True)])
def test_outputs(rows, width, values, codes):
    x, r, w = make(rows, width, "bf16", "bf16", rows)
    got = run(x, w, r, values=values, codes=codes)
    check(x, w, r, 1e-6, got)
    assert (got[1] is None) != values and (got[2] is None) != codes


@pytest.mark.parametrize("width", [96, 1024, 3001, 10000])
def test_strides_and_places(width):
    """Rows of wider tensors, in place of x and of the residual, and unaligned addresses."""
    x, r, w = make(13, width + 24, "bf16", "f32", 5)
    for first in (0, 8, 3):
        a, b = x[:, first:first + width], r[:, first:first + width]
        check(a, w[:width], b, 1e-6, run(a, w[:width].clone(), b))
    a, b, ww = x[:, :width].contiguous(), r[:, :width].contiguous(), w[:width].clone()
    want = run(a, ww, b)
    p, q = a.clone(), b.clone()
    rms_norm(p.data_ptr(), ww.data_ptr(), 13, width, dtype="bf16", residual_ptr=q.data_ptr(), out_ptr=p.data_ptr())
    assert torch.equal(q, want[0]) and torch.equal(p, want[1])
    p, q = a.clone(), b.clone()
    rms_norm(p.data_ptr(), ww.data_ptr(), 13, width, dtype="bf16", residual_ptr=q.data_ptr(), sum_ptr=p.data_ptr(), out_ptr=a.data_ptr())
    assert torch.equal(p, want[0]) and torch.equal(a, want[1]) and torch.equal(q, b)
    p = b.clone()
    rms_norm(p.data_ptr(), ww.data_ptr(), 13, width, dtype="bf16", residual_ptr=p.data_ptr(), out_ptr=a.data_ptr())
    assert torch.equal(p, b + b)


@pytest.mark.parametrize("width", [200, 2048, 9000])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_odd_values(width, dtype):
    """Zero rows, rows of the type's largest and smallest values, and rows that are not numbers, each apart from the others."""
    x, _, w = make(8, width, dtype, "f32", 3)
    top = torch.finfo(TYPES[dtype])
    x[0] = 0
    x[1] = x[1].float().sign().to(x.dtype) * top.max
    x[2] = x[2].float().sign().to(x.dtype) * top.tiny
    x[3, 130] = float("nan")
    x[4, 5] = float("inf")
    x[6, 128:] = 0
    _, out, codes, scales = run(x, w)
    good = [0, 1, 2, 5, 6, 7]
    check(x[good], w, None, 1e-6, [None, out[good], codes[good], scales[good]])
    assert bool((codes[0].view(torch.float8_e4m3fn).float() == 0).all() and (scales[0] == 1).all())
    assert bool(out[3].isnan().all() and scales[3].isnan().all())
    # An infinity: its own place is 0 * inf, every other value is 0.
    assert bool(out[4, 5].isnan() and (out[4].nan_to_num(0) == 0).all() and scales[4, 0].isnan() and (scales[4, 1:] == 1).all())


def test_smallest_scales():
    """Values whose scale would be so small that its inverse is infinite keep the floor's."""
    x = torch.zeros(2, 256, device="cuda")
    x[0, :128] = torch.linspace(-1e-36, 1e-36, 128, device="cuda")
    x[1, 7] = 1e-44
    w = torch.ones(256, device="cuda")
    got = run(x, w, eps=1.0)
    check(x, w, None, 1.0, got)
    assert bool((got[3] >= 2.0**-126).all())


def test_tiny_rows_without_eps():
    x, w = torch.full((3, 300), 1e-42, device="cuda"), torch.linspace(0.5, 2, 300, device="cuda")
    x[1] *= -1e4
    x[2, 100:] = 0
    check(x, w, None, 0.0, run(x, w, eps=0.0))


def test_zero_row_without_eps():
    x, w = torch.zeros(1, 160, device="cuda"), torch.ones(160, device="cuda")
    _, out, _, scales = run(x, w, eps=0.0)
    assert bool(out.isnan().all() and scales.isnan().all())


def test_streams_and_replay():
    """Calls on two streams at once; a captured one reads what lies in its tensors when it is replayed."""
    x, r, w = make(100, 1536, "f16", "f16", 1)
    want = run(x, w, r)
    s1, s2, g = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    outs = [torch.empty_like(x) for _ in range(3)]
    sums = [torch.empty_like(x) for _ in range(3)]
    def call(i, s):
        rms_norm(x.data_ptr(), w.data_ptr(), 100, 1536, dtype="f16", weight_dtype="f16", residual_ptr=r.data_ptr(),
                 sum_ptr=sums[i].data_ptr(), out_ptr=outs[i].data_ptr(), stream=s.cuda_stream)
    torch.cuda.synchronize()
    for _ in range(10):
        call(0, s1)
        call(1, s2)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s1):
        call(2, s1)
    x0 = x.clone()
    x.copy_(x.flip(0))
    g.replay()
    torch.cuda.synchronize()
    check(x, w, r, 1e-6, [sums[2], outs[2], None, None])
    x.copy_(x0)
    for i in (0, 1):
        assert torch.equal(sums[i], want[0]) and torch.equal(outs[i], want[1])


def test_refused_pointers():
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(64, device="cuda")
    host = torch.zeros(4, 64)
    for args, words in [(dict(x_ptr=host.data_ptr()), "x is not device memory"), (dict(x_ptr=x.data_ptr() + 2), "x is not aligned"),
                        (dict(weight_ptr=host.data_ptr()), "weight is not device memory"), (dict(x_ptr=None), "x is NULL"),
                        (dict(out_ptr=host.data_ptr()), "out is not device memory")]:
        call = dict(x_ptr=x.data_ptr(), weight_ptr=w.data_ptr(), rows=4, width=64, out_ptr=x.data_ptr())
        call.update(args)
        with pytest.raises(TritError, match=words):
            rms_norm(**call)
