"""Cases and plain forms of the operators that a decoder layer has between its
cache calls when its products run in 8-bit floating point: the norm that feeds
them, the products, and the rotary positions of queries and keys.

Rows of 8-bit numbers. A row of `width` values is e4m3 numbers (1 sign, 4
exponent and 3 fraction bits, largest 448) with one f32 scale for each 128 of
them (the last group may be shorter):

    scale = max(f32(max |y| / 448), 2^-126), 1 where all are zero
    code  = e4m3(f32(y * f32(1 / scale)))   (nearest, ties to even)

and stands for code * scale.

Norm:     h = x + residual, rounded to the rows' type; s = f32(1 / sqrt(mean h^2 + eps)); y = h * f32(s * w), in f32; y as
          values of the rows' type, as 8-bit rows, or both.
Products: W is e4m3 with one f32 scale for each block of 128 x 128; out = x W^T for 8-bit rows x, or for rows that are
          rounded so first.
Rotary:   pair i of a head at position p turns by the angle p * f_i (pairs (i, i + d / 2), or (2 i, 2 i + 1), of the head's
          first d values) and is multiplied by a factor; the rest of the head stays. The frequencies f_i are
          theta^(-2 i / d), or those scaled for contexts longer than the trained one.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ------------------------------------------------------------------ cases

def listed():
    return [
        # Next token of one stream, in front of a product: the smallest call, bound by its latency.
        dict(name="norm_step", kind="norm", rows=1, width=2048, dtype="bf16", weight="f32", residual=True, out="codes"),
        # A step of 64 streams with the residual held in f32.
        dict(name="norm_streams", kind="norm", rows=64, width=4096, dtype="f32", weight="f32", residual=True, out="codes"),
        # The rows of a long prompt.
        dict(name="norm_prompt", kind="norm", rows=8000, width=4096, dtype="bf16", weight="bf16", residual=True, out="codes"),
        # Encoder rows of an odd width, as values for one reader and 8-bit rows for another, no residual.
        dict(name="norm_odd", kind="norm", rows=20011, width=1000, dtype="f16", weight="f16", residual=False, out="both"),
        # The gate and up product of a layer for one stream, from 8-bit rows.
        dict(name="dense_row", kind="dense", n=12288, k=2048, rows=1, dtype="bf16", form="codes"),
        # The same product of a wider layer for 64 streams, from f32 rows as the decoder makes them.
        dict(name="dense_streams", kind="dense", n=16384, k=4096, rows=64, dtype="f32", form="rows"),
        # The output table for three streams.
        dict(name="dense_table", kind="dense", n=151936, k=2048, rows=3, dtype="f32", form="codes"),
        # Pieces of prompts, sizes that no tile divides.
        dict(name="dense_odd", kind="dense", n=5001, k=2064, rows=333, dtype="f16", form="codes"),
        # A long prompt: the arithmetic counts.
        dict(name="dense_prompt", kind="dense", n=12288, k=4096, rows=8000, dtype="bf16", form="codes"),
        # Queries and keys of 64 streams' next tokens, out of fused q | k | v rows.
        dict(name="rotary_step", kind="rotary", rows=64, heads=32, kv=8, hd=128, rd=128, layout="halves", scaling="none", dtype="f32",
             far=1300, theta=1e6),
        # A long prompt of several packed sequences, with frequencies in bands for a long context.
        dict(name="rotary_prompt", kind="rotary", rows=8000, heads=32, kv=8, hd=128, rd=128, layout="halves", scaling="bands",
             dtype="bf16", far=8000, theta=5e5),
        # Neighbouring pairs over a part of an odd-sized head, far out in a stretched context.
        dict(name="rotary_part", kind="rotary", rows=1501, heads=15, kv=5, hd=80, rd=36, layout="interleaved", scaling="yarn",
             dtype="f16", far=500000, theta=1e4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "dense", "dense", "rotary"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "norm":
        width = _log(rng, 16, 16384)
        rows = min(_log(rng, 1, 20000), max(1, 16000000 // width))
        return dict(kind=kind, rows=rows, width=width, dtype=dtype, weight=rng.choice(["f32", dtype]), residual=rng.random() < 0.6,
                    out=rng.choice(["codes", "codes", "values", "both"]))
    if kind == "dense":
        k, n = 16 * _log(rng, 2, 700), _log(rng, 30, 30000)
        rows = rng.choice([1, 2, 5, _log(rng, 6, 130), _log(rng, 100, 8000)])
        while n * k * rows > 8000 * 12288 * 4096:
            rows = rows // 2
        return dict(kind=kind, n=n, k=k, rows=rows, dtype=dtype, form=rng.choice(["codes", "rows"]))
    hd = rng.choice([64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    rows = min(_log(rng, 1, 8000), max(1, 8000 * 40 * 128 // ((heads + kv) * hd)))
    return dict(kind=kind, rows=rows, heads=heads, kv=kv, hd=hd, rd=rng.choice([hd, hd, hd // 2, 2 * rng.randint(4, hd // 2)]),
                layout=rng.choice(["halves", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]), dtype=dtype,
                far=_log(rng, 100, 1000000), theta=rng.choice([1e4, 5e5, 1e6]))


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "norm":
        m, d = case["rows"], case["width"]
        rows = size * m * d
        b = rows * (3 if case["residual"] else 1) + d * SIZE[case["weight"]]
        b += rows if case["out"] != "codes" else 0
        b += m * d + 4 * m * ((d + 127) // 128) if case["out"] != "values" else 0
        return {"bytes": b, "flops": 8 * m * d}
    if case["kind"] == "dense":
        n, k, m = case["n"], case["k"], case["rows"]
        kb = (k + 127) // 128
        x = m * k + 4 * m * kb if case["form"] == "codes" else size * m * k
        return {"bytes": n * k + 4 * kb * ((n + 127) // 128) + x + size * m * n, "flops": 2 * n * k * m}
    m, heads = case["rows"], case["heads"] + case["kv"]
    return {"bytes": 2 * size * m * heads * case["hd"] + 8 * m, "flops": 3 * m * heads * case["rd"]}


# ----------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62) + 29)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _stream_rows(g, rows, width):
    """Rows as a decoder's residual stream holds them: a few channels far larger than the others."""
    x = _randn(g, rows, width)
    x *= 0.7 + 20.0 * (torch.rand(1, width, generator=g, device="cuda") > 0.995)
    return x


def _weights(g, n, k):
    """e4m3 weights [n][k] and their scales [n / 128][k / 128], from normal weights of another size a block."""
    nb, kb = (n + 127) // 128, (k + 127) // 128
    codes = torch.empty(n, k, dtype=torch.float8_e4m3fn, device="cuda")
    scales = 0.00005 + 0.0002 * torch.rand(nb, kb, generator=g, device="cuda")
    for a in range(0, n, 16384):
        codes[a:a + 16384] = (_randn(g, min(16384, n - a), k) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, scales


def _raw(case, seed):
    g = _gen(seed)
    dtype = TYPES[case["dtype"]]
    if case["kind"] == "norm":
        s = {"x": _stream_rows(g, case["rows"], case["width"]).to(dtype),
             "weight": (1.0 + 0.3 * _randn(g, case["width"])).to(TYPES[case["weight"]])}
        if case["residual"]:
            s["residual"] = (3 * _stream_rows(g, case["rows"], case["width"])).to(dtype)
        return s
    if case["kind"] == "dense":
        codes, scales = _weights(g, case["n"], case["k"])
        s = {"w": codes, "w_scales": scales}
        if case["form"] == "codes":
            x = (_randn(g, case["rows"], case["k"]) * 110).clamp(-448, 448)
            s["x"] = x.to(torch.float8_e4m3fn)
            s["x_scales"] = 0.002 + 0.02 * torch.rand(case["rows"], (case["k"] + 127) // 128, generator=g, device="cuda")
        else:
            s["x"] = _stream_rows(g, case["rows"], case["k"]).to(dtype)
        return s
    m, heads, kv, hd = case["rows"], case["heads"], case["kv"], case["hd"]
    s = {"qkv": _randn(g, m, (heads + 2 * kv) * hd).to(dtype)}
    if m > 200:  # packed sequences at consecutive positions
        piece = (m + 2) // 3
        first = torch.randint(0, max(1, case["far"] - piece + 1), (3,), generator=g, device="cuda")
        row = torch.arange(m, device="cuda")
        s["positions"] = first[row // piece] + row % piece
    else:
        s["positions"] = torch.randint(0, case["far"] + 1, (m,), generator=g, device="cuda")
    return s


def _scaling(case):
    return {"none": {}, "linear": dict(scaling="linear", factor=4.0), "ntk": dict(scaling="ntk", factor=4.0),
            "yarn": dict(scaling="yarn", factor=16.0, trained=32768),
            "bands": dict(scaling="bands", factor=8.0, trained=8192, low=1.0, high=4.0)}[case["scaling"]]


def prepare(case, seed):
    s = _raw(case, seed)
    s["case"] = case
    if own:
        import trit_b200

        s["lib"] = trit_b200
        s["stream"] = torch.cuda.current_stream().cuda_stream
        if case["kind"] == "dense":
            w, scales = s.pop("w"), s.pop("w_scales")
            s["layer"] = trit_b200.Dense.fp8(w.view(torch.uint8).cpu().numpy(), scales.cpu().numpy(), case["n"], case["k"])
        elif case["kind"] == "rotary":
            s["rotary"] = trit_b200.Rotary(case["hd"], rotary_dim=case["rd"], layout=case["layout"], theta=case["theta"],
                                           **_scaling(case))
    elif case["kind"] == "rotary":
        f, factor = _frequencies(case)
        s["frequencies"], s["factor"] = torch.tensor(f, dtype=torch.float64, device="cuda"), factor
    return s


# ------------------------------------------------------------- plain form

def _to_codes(y):
    """f32 rows as e4m3 numbers and scales of 128."""
    m, d = y.shape
    g = torch.nn.functional.pad(y, (0, -d % 128)).view(m, -1, 128)
    most = g.abs().amax(-1)
    scale = torch.where(most > 0, (most.double() / 448.0).float().clamp_min(2.0**-126), 1.0)
    codes = (g * (1.0 / scale)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(m, -1)[:, :d].contiguous(), scale


def _norm_plain(s):
    case, x = s["case"], s["x"]
    out = []
    if case["residual"]:
        x = (x.float() + s["residual"].float()).to(x.dtype)
        out.append(x)
    h = x.float()
    inv = (1.0 / torch.sqrt(h.double().square().mean(-1, keepdim=True) + EPS)).float()
    y = h * (inv * s["weight"].float())
    if case["out"] != "codes":
        out.append(y.to(x.dtype))
    if case["out"] != "values":
        out += _to_codes(y)
    return out


def _values(codes, scales):
    """What 8-bit rows stand for, f32."""
    m, d = codes.shape
    return codes.float() * scales.repeat_interleave(128, 1)[:, :d]


def _dense_plain(s):
    case, x = s["case"], s["x"]
    x, scales = (x, s["x_scales"]) if case["form"] == "codes" else _to_codes(x.float())
    w = _values(s["w"], s["w_scales"].repeat_interleave(128, 0)[:case["n"]])
    return torch.matmul(_values(x, scales), w.t()).to(TYPES[case["dtype"]])


def _frequencies(case):
    """(f_i in turns of radians a position, the factor of the rotated values)."""
    d, theta, c = case["rd"], case["theta"], _scaling(case)
    kind, by = c.get("scaling"), c.get("factor", 1.0)
    if kind == "ntk":
        theta = theta * by ** (d / (d - 2)) if d > 2 else theta
    f = [theta ** (-2.0 * i / d) for i in range(d // 2)]
    if kind == "linear":
        return [v / by for v in f], 1.0
    if kind == "yarn":
        def at(turns):  # the pair that makes so many turns over the trained context
            return d * math.log(c["trained"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        keep = [1.0 - min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(d // 2)]
        return [v / by * (1.0 - u) + v * u for v, u in zip(f, keep)], 0.1 * math.log(by) + 1.0
    if kind == "bands":
        keep = [min(max((c["trained"] * v / (2 * math.pi) - c["low"]) / (c["high"] - c["low"]), 0.0), 1.0) for v in f]
        return [v / by * (1.0 - u) + v * u for v, u in zip(f, keep)], 1.0
    return f, 1.0


def _turned(x, cos, sin, case):
    """x [m][heads][hd] in f32 with its pairs turned."""
    d = case["rd"]
    if case["layout"] == "halves":
        a, b = x[..., :d // 2], x[..., d // 2:d]
        parts = [a * cos - b * sin, b * cos + a * sin]
        return torch.cat(parts + [x[..., d:]], -1)
    a, b = x[..., 0:d:2], x[..., 1:d:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., d:]], -1)


def _rotary_plain(s):
    case, m = s["case"], s["case"]["rows"]
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    cos, sin = (torch.cos(angle) * s["factor"]).float(), (torch.sin(angle) * s["factor"]).float()
    x = s["qkv"].float().view(m, -1, case["hd"])[:, :case["heads"] + case["kv"]]
    out = _turned(x, cos, sin, case).to(s["qkv"].dtype)
    return [out[:, :case["heads"]].contiguous(), out[:, case["heads"]:].contiguous()]


# -------------------------------------------------------------- one pass

def _run_own(s):
    case, lib, x = s["case"], s["lib"], s.get("x")
    if case["kind"] == "norm":
        m, d = x.shape
        h = torch.empty_like(x) if case["residual"] else None
        y = torch.empty_like(x) if case["out"] != "codes" else None
        codes = scales = None
        if case["out"] != "values":
            codes = torch.empty(m, d, dtype=torch.float8_e4m3fn, device="cuda")
            scales = torch.empty(m, (d + 127) // 128, device="cuda")
        made = [t for t in (h, y, codes, scales) if t is not None]
        at = [t.data_ptr() if t is not None else None for t in (h, y, codes, scales)]
        lib.rms_norm(x.data_ptr(), s["weight"].data_ptr(), m, d, eps=EPS, dtype=case["dtype"], weight_dtype=case["weight"],
                     residual_ptr=s["residual"].data_ptr() if case["residual"] else None, sum_ptr=at[0], out_ptr=at[1],
                     codes_ptr=at[2], scales_ptr=at[3], stream=s["stream"])
        return made
    if case["kind"] == "dense":
        m, out = case["rows"], torch.empty(case["rows"], case["n"], dtype=TYPES[case["dtype"]], device="cuda")
        if case["form"] == "codes":
            s["layer"].forward_codes(x.data_ptr(), s["x_scales"].data_ptr(), m, out.data_ptr(), dtype=case["dtype"], stream=s["stream"])
        else:
            s["layer"].forward_rows(x.data_ptr(), m, out.data_ptr(), dtype=case["dtype"], stream=s["stream"])
        return out
    m, heads, kv, hd, qkv = case["rows"], case["heads"], case["kv"], case["hd"], s["qkv"]
    q, k = torch.empty(m, heads, hd, dtype=qkv.dtype, device="cuda"), torch.empty(m, kv, hd, dtype=qkv.dtype, device="cuda")
    wide = qkv.shape[1]
    s["rotary"].apply(s["positions"].data_ptr(), m, qkv.data_ptr(), heads, qkv.data_ptr() + heads * hd * qkv.element_size(), kv,
                      dtype=case["dtype"], q_stride=wide, k_stride=wide, q_out_ptr=q.data_ptr(), k_out_ptr=k.data_ptr(), stream=s["stream"])
    return [q, k]


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _norm_plain, "dense": _dense_plain, "rotary": _rotary_plain}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- 64 bits

def _exact_codes(y):
    """8-bit rows of f32 rows: the border between two codes is defined in f32 steps; the numbers are exact."""
    m, d = y.shape
    scales = torch.empty(m, (d + 127) // 128, dtype=torch.float64, device="cuda")
    codes = torch.empty(m, d, dtype=torch.float64, device="cuda")
    for b in range(scales.shape[1]):
        part = y[:, b * 128:b * 128 + 128]
        most = part.abs().max(1).values
        scale = (most.double() / 448).float()
        scale = torch.maximum(scale, torch.full_like(scale, 2.0**-126)).masked_fill(most == 0, 1.0)
        v = (part * torch.reciprocal(scale)[:, None]).double()
        step = torch.exp2(torch.frexp(v).exponent.clamp_min(-5).double() - 4)  # |v| in [2^(e-1), 2^e): 8 steps
        codes[:, b * 128:b * 128 + 128] = (torch.round(v / step) * step).clamp(-448, 448)
        scales[:, b] = scale.double()
    return codes, scales


def exact(case, seed):
    s = _raw(case, seed)
    if case["kind"] == "norm":
        x, w, out = s["x"], s["weight"].float(), []
        if case["residual"]:
            out.append(x.double() + s["residual"].double())
            x = (x.float() + s["residual"].float()).to(x.dtype)
        power = torch.einsum("md,md->m", x.double(), x.double()) / case["width"]
        inv = (power + EPS) ** -0.5
        if case["out"] != "codes":
            out.append(x.double() * inv[:, None] * w.double())
        if case["out"] != "values":
            out += _exact_codes(x.float() * (inv.float()[:, None] * w[None]))
        return out
    if case["kind"] == "dense":
        if case["form"] == "codes":
            x, scales = s["x"].double(), s["x_scales"].double()
        else:
            x, scales = _exact_codes(s["x"].float())
        out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for a in range(0, case["n"], 128 * 64):
            w = s["w"][a:a + 128 * 64].double()
            total = torch.zeros(case["rows"], w.shape[0], dtype=torch.float64, device="cuda")
            sw = s["w_scales"][a // 128:a // 128 + 64].double()
            for b in range(scales.shape[1]):
                at = slice(b * 128, b * 128 + 128)
                total += (x[:, at] * scales[:, b:b + 1]) @ (w[:, at] * sw[:, b].repeat_interleave(128)[:w.shape[0], None]).t()
            out[:, a:a + 128 * 64] = total
        return out
    f, factor = _frequencies(case)
    m, heads, kv, hd, d = case["rows"], case["heads"], case["kv"], case["hd"], case["rd"]
    x = s["qkv"].double().view(m, heads + 2 * kv, hd)[:, :heads + kv].clone()
    for i, v in enumerate(f):
        angle = (s["positions"].double() * v)[:, None]
        a, b = (i, i + d // 2) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.full_like(angle, factor), angle)
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
    return [x[:, :heads], x[:, heads:]]
