"""A decoder layer of a caller's own from the library's operators: norm, q | k | v product, rotary positions, 8-bit cache and
its attention, output product, norm, gate and up, down, over a prompt and single steps of two sequences."""
import numpy as np
import pytest

from tests import kv_oracle, rows_oracle
from tests.test_gpu_dense_fp8 import check as check_product
from tests.test_gpu_dense_fp8 import layer
from tests.test_gpu_rotary import check as check_rotary
from trit_b200 import KvCache, Rotary, rms_norm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D, HEADS, KV, HD, FFN, PAGE = 512, 8, 2, 64, 640, 16


class Layer:
    def __init__(self):
        self.qkv, self.wqkv = layer((HEADS + 2 * KV) * HD, D, 1)
        self.o, self.wo = layer(D, HEADS * HD, 2)
        self.up, self.wup = layer(2 * FFN, D, 3)
        self.down, self.wdown = layer(D, FFN, 4)
        g = torch.Generator("cuda").manual_seed(5)
        self.n1, self.n2 = (1 + 0.2 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
        self.rotary = Rotary(HD, theta=1e4, scaling="bands", factor=4.0, trained=64)
        self.cache = KvCache(kv_heads=KV, pages=16, head_dim=HD, page_tokens=PAGE, sequences=2, max_tokens=128)
        self.seqs = self.cache.open(2)

    def step(self, h, delta, counts, positions, stream, sync=lambda: None):
        """One pass: the residual h (updated) and what the layer adds to it; every intermediate tensor by name."""
        m, s, t = h.shape[0], stream.cuda_stream, {}
        def new(name, *shape, dtype=torch.bfloat16):
            t[name] = torch.empty(*shape, dtype=dtype, device="cuda")
            return t[name].data_ptr()
        def norm(name, weight, delta):
            rms_norm(delta.data_ptr(), weight.data_ptr(), m, D, dtype="bf16", residual_ptr=h.data_ptr(), stream=s,
                     codes_ptr=new(name, m, D, dtype=torch.uint8), scales_ptr=new(name + "_scales", m, D // 128, dtype=torch.float32))
            t[name + "_h"] = h.clone()
            sync()
        norm("a", self.n1, delta)
        self.qkv.forward_codes(t["a"].data_ptr(), t["a_scales"].data_ptr(), m, new("qkv", m, (HEADS + 2 * KV) * HD), dtype="bf16", stream=s)
        sync()
        t["raw"] = t["qkv"].clone()
        wide, q = (HEADS + 2 * KV) * HD, t["qkv"].data_ptr()
        self.rotary.apply(positions.data_ptr(), m, q, HEADS, q + 2 * HEADS * HD, KV, dtype="bf16", q_stride=wide, k_stride=wide, stream=s)
        sync()
        self.cache.extend(self.seqs, counts, stream=s)
        self.cache.append(0, self.seqs, counts, q + 2 * HEADS * HD, q + 2 * (HEADS + KV) * HD, dtype="bf16", k_stride=wide, v_stride=wide,
                          stream=s)
        sync()
        self.cache.attend(0, self.seqs, counts, q, new("att", m, HEADS * HD), heads=HEADS, dtype="bf16", scale=HD**-0.5, q_stride=wide,
                          stream=s)
        sync()
        self.o.forward_rows(t["att"].data_ptr(), m, new("o", m, D), dtype="bf16", stream=s)
        sync()
        norm("b", self.n2, t["o"])
        self.up.forward_codes(t["b"].data_ptr(), t["b_scales"].data_ptr(), m, new("up", m, 2 * FFN), dtype="bf16", stream=s)
        sync()
        t["act"] = torch.nn.functional.silu(t["up"][:, :FFN].float()) * t["up"][:, FFN:].float()
        self.down.forward_rows(t["act"].data_ptr(), m, new("down", m, D, dtype=torch.float32), dtype="f32", stream=s)
        sync()
        return t["down"].to(torch.bfloat16), t


def passes():
    """Two prompts of 37 and 19 tokens, then single tokens of both."""
    return [[37, 19]] + [[1, 1]] * 6


def inputs(seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return [torch.randn(sum(c), D, generator=g, device="cuda").to(torch.bfloat16) for c in passes()]


def test_every_step_follows_from_the_one_before():
    lay, stream, lens = Layer(), torch.cuda.current_stream(), [0, 0]
    held = [[torch.zeros(0, KV, HD, device="cuda"), torch.zeros(0, KV, HD, device="cuda")] for _ in range(2)]
    for h, counts in zip(inputs(1), passes()):
        at = torch.cat([torch.arange(n, n + c) for n, c in zip(lens, counts)]).cuda()
        h0 = h.clone()
        _, t = lay.step(h, torch.zeros_like(h), counts, at, stream)
        torch.cuda.synchronize()
        m = h.shape[0]
        for name, weight, before, add in (("a", lay.n1, h0, torch.zeros_like(h0)), ("b", lay.n2, h0, t["o"])):
            want = (before.float() + add.float()).to(torch.bfloat16)
            assert torch.equal(t[name + "_h"], want)
            c, s = rows_oracle.rows_of(rows_oracle.norm_f32(want.float().cpu().numpy(), weight.cpu().numpy(), 1e-6))
            assert np.array_equal(t[name + "_scales"].cpu().numpy(), s)
            assert np.array_equal(t[name].view(torch.float8_e4m3fn).double().cpu().numpy(), c)
        def values(codes, scales):
            return torch.from_numpy(rows_oracle.values_of(codes.view(torch.float8_e4m3fn).double().cpu().numpy(), scales.cpu().numpy())).cuda()
        def rounded(x):
            return torch.from_numpy(rows_oracle.values_of(*rows_oracle.rows_of(x.float().cpu().numpy()))).cuda()
        check_product(t["raw"], values(t["a"], t["a_scales"]), lay.wqkv)
        check_product(t["up"], values(t["b"], t["b_scales"]), lay.wup)
        check_product(t["o"], rounded(t["att"]), lay.wo)
        check_product(t["down"], rounded(t["act"]), lay.wdown)
        raw, turned = (x.view(m, HEADS + 2 * KV, HD) for x in (t["raw"], t["qkv"]))
        check_rotary(turned[:, :HEADS + KV], raw[:, :HEADS + KV], at, lay.rotary, False)
        assert torch.equal(turned[:, HEADS + KV:], raw[:, HEADS + KV:])
        row = 0
        for i, c in enumerate(counts):
            mine = turned[row:row + c].float()
            held[i] = [torch.cat([held[i][0], mine[:, HEADS:HEADS + KV]]), torch.cat([held[i][1], mine[:, HEADS + KV:]])]
            k, v = (kv_oracle.held(x.cpu().numpy(), PAGE) for x in held[i])
            want, tol = kv_oracle.attend(mine[:, :HEADS].cpu().numpy(), k, v, HD**-0.5, True)
            got = t["att"][row:row + c].double().cpu().numpy().reshape(want.shape)
            # (bf16 rows: the weights hold 11 bits, the output 8.)
            assert (np.abs(got - want) <= tol + np.abs(v).max() * 2.0**-11 + np.abs(want) * 2.0**-8).all()
            row += c
            lens[i] += c


def test_calls_without_a_wait_between():
    """The same passes with a wait behind every call and with none at all, on a stream of their own: to the bit the same.
    Kernels that start before the one in front has ended must not read what it writes too early, nor write too early."""
    results = []
    for waits in (True, False):
        lay, stream, lens, outs = Layer(), torch.cuda.Stream(), [0, 0], []
        xs = inputs(2)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for h, counts in zip(xs, passes()):
                at = torch.cat([torch.arange(n, n + c) for n, c in zip(lens, counts)]).cuda()
                delta, _ = lay.step(h, torch.zeros_like(h), counts, at, stream, torch.cuda.synchronize if waits else lambda: None)
                outs += [h, delta]
                lens = [n + c for n, c in zip(lens, counts)]
        torch.cuda.synchronize()
        results.append(outs)
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_chained_calls_many_times():
    """A hundred norms, products and rotations in a row, each on the last one's output, with no wait and no other kernel
    between, against the same with waits."""
    n = k = 256
    dense, _ = layer(n, k, 9)
    rotary, w = Rotary(64), torch.ones(n, device="cuda")
    for m in (1, 40, 300):
        at = torch.arange(m, device="cuda")
        results = []
        for waits in (True, False):
            g = torch.Generator("cuda").manual_seed(m)
            x = torch.randn(m, n, generator=g, device="cuda").to(torch.bfloat16)
            h = torch.randn(m, n, generator=g, device="cuda").to(torch.bfloat16)
            codes, scales = torch.empty(m, n, dtype=torch.uint8, device="cuda"), torch.empty(m, n // 128, device="cuda")
            torch.cuda.synchronize()
            for _ in range(100):
                rms_norm(x.data_ptr(), w.data_ptr(), m, n, dtype="bf16", residual_ptr=h.data_ptr(), codes_ptr=codes.data_ptr(),
                         scales_ptr=scales.data_ptr())
                if waits:
                    torch.cuda.synchronize()
                dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, x.data_ptr(), dtype="bf16")
                if waits:
                    torch.cuda.synchronize()
                rotary.apply(at.data_ptr(), m, x.data_ptr(), n // 64, dtype="bf16")
                if waits:
                    torch.cuda.synchronize()
                dense.forward_rows(x.data_ptr(), m, x.data_ptr(), dtype="bf16")
                if waits:
                    torch.cuda.synchronize()
            torch.cuda.synchronize()
            results.append((x.clone(), h.clone(), codes.clone(), scales.clone()))
        for a, b in zip(*results):
            assert torch.equal(a, b)
        assert bool(results[0][0].isfinite().all())
