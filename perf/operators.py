"""Cases and plain forms of the operators that a greedy step spends its bytes
on: the key/value cache held in 8 bits (append, attention, page operations)
and products with 4-bit weights.

The 8-bit cache. A page holds `page` consecutive positions of one sequence.
Keys and values are rounded to f16 on arrival. The positions of a page that is
not full yet (the open page, one a sequence) stay f16; when the page's last
position arrives, every kv head's keys of the page, and its values, become
8-bit codes with one scale:

    scale = f32(max |x| / 127),   code = the whole number nearest x / scale
                                  (ties to even; 0 where scale is 0)

and the cache from then on holds code * scale. Attention of a query row at
position p of a sequence of T positions, head h of kv head h / (heads / kv):

    out = sum_j softmax_j(scale * q . k_j) v_j,   j <= p (causal) or j < T

and zero where a row has no key.

4-bit weights. A row of the matrix is groups of 32 values, each group an f16
scale d and 32 codes c in 0..15 that stand for d * (c - 8) (ggml Q4_0 blocks:
18 bytes, code i in the low half of byte i, code 16 + i in its high half).
out = x W^T, with x as it is ("table"), or with x rounded to 8-bit codes in
groups of 32 first: scale = f32(max |x| / 127) (1 for a zero group), code =
clamp(rint(x * f32(1 / scale)), +-127), the scale then rounded to f16.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # The next token of one stream, 16 query heads on 8 kv heads: the smallest call, bound by its latency.
        dict(name="step_one", kind="attend", seqs=1, lo=217, hi=217, rlo=1, rhi=1, heads=16, kv=8, hd=128, page=64, dtype="f32",
             causal=True),
        # A greedy step of 64 transcript streams of mixed lengths: the batch workload.
        dict(name="step_streams", kind="attend", seqs=64, lo=601, hi=1279, rlo=1, rhi=1, heads=32, kv=8, hd=128, page=64,
             dtype="f32", causal=True),
        # Long recordings: few streams, each of tens of thousands of positions, split over its length.
        dict(name="step_long", kind="attend", seqs=6, lo=40001, hi=65535, rlo=1, rhi=1, heads=32, kv=8, hd=128, page=128,
             dtype="bf16", causal=True),
        # A whole prompt in one pass, f32 rows as the decoder makes them.
        dict(name="prompt", kind="attend", seqs=1, lo=4000, hi=4000, rlo=4000, rhi=4000, heads=32, kv=8, hd=128, page=64,
             dtype="f32", causal=True),
        # Prompt pieces of several streams behind what they hold already, small pages, 64-wide heads.
        dict(name="prompt_pieces", kind="attend", seqs=7, lo=300, hi=2111, rlo=33, rhi=300, heads=16, kv=4, hd=64, page=16,
             dtype="bf16", causal=True),
        # Decoder rows that look at an encoder's states (another length, no causal order), plain multi-head; a stream
        # without any state among them.
        dict(name="cross", kind="attend", seqs=24, lo=0, hi=1500, rlo=1, rhi=9, heads=16, kv=16, hd=64, page=32, dtype="f16",
             causal=False),
        # One new position for every stream of a batch, written to branches of the streams and read back.
        dict(name="append_step", kind="append", seqs=64, lo=601, hi=1279, new=1, layers=1, kv=8, hd=128, page=64, dtype="f32"),
        # Prompts of several streams written at once, every layer, and read back as values.
        dict(name="append_prompt", kind="append", seqs=5, lo=0, hi=0, new=1301, layers=4, kv=8, hd=128, page=64, dtype="bf16"),
        # Candidates: every stream branches, each branch grows, one of each set stays, and the cache closes its gaps.
        dict(name="branch", kind="branch", seqs=4, lo=801, hi=1203, forks=4, new=70, layers=4, kv=8, hd=128, page=64, dtype="f16"),
        # Streams copied page for page, half of the copies given up, and the pages moved together.
        dict(name="copies", kind="copies", seqs=24, lo=901, hi=2047, layers=8, kv=8, hd=128, page=64, dtype="f16"),
        # The gate and up product of a decoder layer for one stream, with 8-bit activations.
        dict(name="dense_row", kind="dense", n=12288, k=2048, rows=1, table=False),
        # The output table for three streams, f32 arithmetic.
        dict(name="dense_table", kind="dense", n=151936, k=2048, rows=3, table=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "branch", "copies", "dense", "dense"])
    kv = rng.choice([1, 2, 4, 8])
    case = dict(kind=kind)
    if kind == "dense":
        table = rng.random() < 0.5
        k = 32 * _log(rng, 8, 256) if table else 128 * _log(rng, 2, 64)
        n = _log(rng, 64, 150000) if table else 32 * _log(rng, 4, 4096)
        while n * k > 151936 * 2048:
            n = n // 2 // 32 * 32 if not table else n // 2
        return dict(case, n=n, k=k, rows=rng.choice([1, 1, 1, 2, 3, 4, 7, 8, 16]), table=table)
    case.update(kv=kv, hd=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 64, 128]), dtype=rng.choice(["f32", "f16", "bf16"]))
    if kind == "attend":
        form = rng.choice(["step", "step", "prompt", "cross"])
        heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
        if form == "step":
            hi = _log(rng, 1, 60000)
            seqs = min(_log(rng, 1, 128), max(1, 400000 // hi))
            return dict(case, heads=heads, seqs=seqs, lo=max(1, hi // 2), hi=hi, rlo=1, rhi=rng.choice([1, 1, 3]) if hi > 5 else 1,
                        causal=True)
        if form == "cross":
            hi = _log(rng, 8, 3000)
            return dict(case, heads=heads, seqs=_log(rng, 1, 32), lo=0, hi=hi, rlo=1, rhi=_log(rng, 1, 40), causal=False)
        hi = _log(rng, 20, 4000)
        rhi = _log(rng, 10, hi)
        seqs = min(_log(rng, 1, 8), max(1, 4000 * 4000 * 32 // (hi * rhi * heads)))
        return dict(case, heads=heads, seqs=seqs, lo=max(rhi, hi // 3), hi=hi, rlo=max(1, rhi // 3), rhi=rhi, causal=True)
    layers = rng.choice([1, 2, 5])
    hi = _log(rng, 20, 2000)
    if kind == "append":
        step = rng.random() < 0.5
        return dict(case, layers=layers, seqs=_log(rng, 1, 64 if step else 8), lo=hi // 2 if step else 0, hi=hi if step else 0,
                    new=_log(rng, 1, 12) if step else hi)
    if kind == "branch":
        return dict(case, layers=layers, seqs=_log(rng, 1, 8), lo=hi // 2, hi=hi, forks=rng.choice([2, 3, 4]), new=_log(rng, 1, 130))
    return dict(case, layers=layers, seqs=_log(rng, 2, 24), lo=hi // 2, hi=hi)


def _spread(lo, hi, n):
    """n whole numbers over lo..hi, in a mixed order that the case alone fixes."""
    return [lo + ((i * 7919 + 3) % n if n > 1 else 0) * (hi - lo) // max(1, n - 1) for i in range(n)]


def _lens(case):
    return _spread(case["lo"], case["hi"], case["seqs"])


def _rows(case):
    rows = _spread(case["rlo"], case["rhi"], case["seqs"])
    return [min(r, t) for r, t in zip(rows, _lens(case))] if case["causal"] else rows


def work(case):
    if case["kind"] == "dense":
        n, k, r = case["n"], case["k"], case["rows"]
        return {"bytes": n * k // 32 * 18 + 4 * r * (n + k), "flops": 2 * n * k * r}
    kv, hd, page, size = case["kv"], case["hd"], case["page"], SIZE[case["dtype"]]

    def held(t):  # bytes of t positions of one layer in the cache
        return 2 * kv * ((t // page) * (page * hd + 4) + t % page * hd * 2)

    lens = _lens(case)
    if case["kind"] == "attend":
        rows, heads = _rows(case), case["heads"]
        pairs = sum(r * t - (r * (r - 1) // 2 if case["causal"] else 0) for r, t in zip(rows, lens))
        return {"bytes": sum(held(t) for t, r in zip(lens, rows) if r) + 2 * size * heads * hd * sum(rows),
                "flops": 4 * pairs * heads * hd}
    layers = case["layers"]
    if case["kind"] == "append":
        new, out = case["new"], sum(t + case["new"] - t // page * page for t in lens)
        write = sum(held(t + new) - held(t // page * page) for t in lens)
        return {"bytes": layers * (2 * kv * hd * size * (new * len(lens) + out) + 2 * write), "flops": layers * 4 * kv * hd * new * len(lens)}
    if case["kind"] == "branch":
        new, f = case["new"], case["forks"]
        grown = sum(held(t + new) - held(t // page * page) for t in lens) * f
        out = sum(t + new for t in lens)
        return {"bytes": layers * (2 * kv * hd * size * (new * f * len(lens) + out) + 2 * grown + sum(held(t + new) for t in lens)),
                "flops": layers * 4 * kv * hd * new * f * len(lens)}
    kept = lens[1::2]
    return {"bytes": layers * (2 * sum(held(t) for t in lens) + sum(held(t) for t in kept) + 2 * kv * hd * size * sum(kept)),
            "flops": layers * 2 * kv * hd * sum(kept)}


# ----------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (1 << 62) + 17)
    return g


def _keys_values(g, positions, kv, hd, dtype):
    """Keys with the few strong channels that rotary keys have, and values: [positions][kv][hd]."""
    k = torch.randn(positions, kv, hd, generator=g, device="cuda")
    k *= 0.5 + 3.5 * (torch.rand(1, kv, hd, generator=g, device="cuda") > 0.94)
    v = torch.randn(positions, kv, hd, generator=g, device="cuda")
    return k.to(dtype), v.to(dtype)


def _raw(case, seed):
    """What the program has: the streams' keys and values (packed rows, a layer after another), and the new rows or queries."""
    g = _gen(seed)
    kv, hd, dtype = case["kv"], case["hd"], TYPES[case["dtype"]]
    lens = _lens(case)
    layers = case.get("layers", 1)
    s = {"lens": lens, "kv0": [_keys_values(g, sum(lens), kv, hd, dtype) for _ in range(layers)]}
    if case["kind"] == "attend":
        s["rows"] = _rows(case)
        q = torch.randn(sum(s["rows"]), case["heads"], hd, generator=g, device="cuda")
        s["q"] = (q * 1.3).to(dtype)
        s["scale"] = 1.0 / math.sqrt(hd)
    elif case["kind"] in ("append", "branch"):
        m = case["new"] * len(lens) * case.get("forks", 1)
        s["new"] = [_keys_values(g, m, kv, hd, dtype) for _ in range(layers)]
    return s


def _blocks(case, seed):
    g = _gen(seed)
    n, k = case["n"], case["k"]
    scales = (0.002 + 0.004 * torch.rand(n, k // 32, generator=g, device="cuda")).to(torch.float16)
    scales = scales * torch.where(torch.rand(n, k // 32, generator=g, device="cuda") < 0.5, -1.0, 1.0).to(torch.float16)
    packed = torch.randint(0, 256, (n, k // 32, 16), generator=g, device="cuda", dtype=torch.uint8)
    x = torch.randn(case["rows"], k, generator=g, device="cuda") * (0.2 + 2 * torch.rand(1, k, generator=g, device="cuda"))
    return scales, packed, x


def prepare(case, seed):
    if case["kind"] == "dense":
        scales, packed, x = _blocks(case, seed)
        s = {"case": case, "x": x}
        if own:
            from trit_b200 import Dense

            blocks = torch.cat([scales.view(torch.uint8).reshape(case["n"], -1, 2), packed], dim=2)
            s["layer"] = Dense.q4_0(blocks.cpu().numpy(), case["n"], case["k"], table=case["table"])
        else:
            s.update(scales=scales, packed=packed)
        return s
    s = _raw(case, seed)
    s["case"] = case
    lens, layers = s["lens"], case.get("layers", 1)
    kv0 = s.pop("kv0")
    if own:
        from trit_b200 import KvCache

        page, new, f = case["page"], case.get("new", 0), case.get("forks", 1)
        pages = sum(t // page for t in lens)
        grown = sum((t + new) // page - t // page for t in lens) * f
        kv = KvCache(layers=layers, kv_heads=case["kv"], head_dim=case["hd"], page_tokens=page, max_tokens=max(1, max(lens) + new),
                     pages=max(1, pages * (2 if case["kind"] == "copies" else 1) + grown), sequences=len(lens) * (1 + f))
        seqs = kv.open(len(lens))
        kv.extend(seqs, lens)
        for layer, (k, v) in enumerate(kv0):
            kv.append(layer, seqs, lens, k.data_ptr(), v.data_ptr(), dtype=case["dtype"])
        torch.cuda.synchronize()
        s.update(cache=kv, seqs=seqs, stream=torch.cuda.current_stream().cuda_stream)
    else:
        s.update(_plain_cache(kv0, lens, case))
    return s


# ------------------------------------------------------------- plain form

def _quantized(x):
    """8-bit codes and scales of whole pages: x f16 [..., page, hd] -> int8, f32 [...]. The scale and the border between two
    codes are decided in 64 bits."""
    scale = (x.abs().amax(dim=(-1, -2)).double() / 127.0).float()
    s = scale[..., None, None].double()
    code = torch.where(s > 0, torch.round(x.double() / torch.where(s > 0, s, 1.0)), 0.0)
    return code.to(torch.int8), scale


def _padded(x, lens, page):
    """Packed rows [sum lens][kv][hd] as f16 pages [seq][page number][kv][page][hd], zero behind each sequence's end."""
    most = max(1, -(-max(lens) // page))
    out = torch.zeros(len(lens), most * page, *x.shape[1:], dtype=torch.float16, device=x.device)
    at = torch.cat([torch.arange(t) + i * most * page for i, t in enumerate(lens)]).to(x.device)
    out.flatten(0, 1)[at] = x.to(torch.float16)
    return out.unflatten(1, (most, page)).transpose(2, 3).contiguous()


def _plain_cache(kv0, lens, case):
    """The cache as one pool of pages for all layers, the sequences' page numbers, and their open pages."""
    page = case["page"]
    pools, scales, opened = [], [], []
    full = [t // page for t in lens]
    for pair in kv0:
        for x in pair:
            pages = _padded(x, lens, page)
            whole = torch.cat([pages[i, :f] for i, f in enumerate(full)])
            code, scale = _quantized(whole)
            pools.append(code)
            scales.append(scale)
            opened.append(torch.stack([pages[i, min(f, pages.shape[1] - 1)] for i, f in enumerate(full)]))
    first = np.cumsum([0] + full)
    most = max(1, max(full))
    table = np.zeros((len(lens), most), np.int64)
    for i, f in enumerate(full):
        table[i, :f] = np.arange(first[i], first[i] + f)
    L = case.get("layers", 1)
    dev = "cuda"
    s = {"pool": torch.stack(pools, 1).unflatten(1, (L, 2)), "scales": torch.stack(scales, 1).unflatten(1, (L, 2)),
         "open": torch.stack(opened, 1).unflatten(1, (L, 2)), "full": torch.tensor(full, device=dev),
         "len": torch.tensor(lens, device=dev), "table": torch.tensor(table, device=dev)}
    if case["kind"] == "attend":
        rows = _rows(case)
        most_rows = max(1, max(rows))
        s["at"] = torch.tensor([i * most_rows + r for i, m in enumerate(rows) for r in range(m)], device=dev, dtype=torch.int64)
        s["row_len"] = torch.tensor(rows, device=dev)
        s["most_rows"] = most_rows
    return s


def _held(s, layer, which):
    """Every position's key (which = 0) or value as f32 [seq][position][kv][hd], through the page numbers."""
    pool, scales, table, page = s["pool"], s["scales"], s["table"], s["open"].shape[-2]
    n, most = table.shape
    if pool.shape[0]:
        x = pool[:, layer, which][table].float() * scales[:, layer, which][table][..., None, None]
    else:
        x = torch.zeros(n, most, *pool.shape[3:], device=pool.device)
    x = torch.cat([x, torch.zeros_like(x[:, :1])], 1)
    x[torch.arange(n, device=x.device), s["full"]] = s["open"][:, layer, which].float()
    return x.transpose(2, 3).flatten(1, 2)


def _attend_plain(s):
    case = s["case"]
    heads, kv, hd = case["heads"], case["kv"], case["hd"]
    g = heads // kv
    k, v = _held(s, 0, 0), _held(s, 0, 1)  # [n][t][kv][hd]
    n, t = k.shape[:2]
    q = torch.zeros(n * s["most_rows"], heads, hd, device="cuda")
    q[s["at"]] = s["q"].float()
    q = q.view(n, -1, kv, g, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]  # [n][kv][rows * g][t]
    key = torch.arange(t, device="cuda")
    row = torch.arange(s["most_rows"], device="cuda")
    last = s["len"][:, None] - 1
    if case["causal"]:
        last = (s["len"] - s["row_len"])[:, None] + row[None]
    ok = key[None, None, :] <= last[:, :, None]  # [n][rows or 1][t]
    ok = ok.expand(n, s["most_rows"], t)[:, None, :, None, :].expand(n, kv, s["most_rows"], g, t).reshape(n, kv, -1, t)
    sc = torch.where(ok, sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.transpose(1, 2)) / torch.where(total > 0, total, 1.0)
    out = out.view(n, kv, -1, g, hd).permute(0, 2, 1, 3, 4).reshape(-1, heads, hd)
    return out[s["at"]].to(TYPES[case["dtype"]])


def _grown_plain(opened, new, start, page):
    """Open pages [m][kv][page][hd] with `new` [m][count][kv][hd] behind position `start` [m] of the page, as pages
    [m][pages][kv][page][hd]."""
    m, count = new.shape[:2]
    most = (page - 1 + count) // page + 1
    out = torch.zeros(m, most * page, *new.shape[2:], dtype=torch.float16, device="cuda")
    out[:, :page] = opened.transpose(1, 2)
    at = start[:, None] + torch.arange(count, device="cuda")
    out.scatter_(1, at[:, :, None, None].expand(m, count, *new.shape[2:]), new.to(torch.float16))
    return out.unflatten(1, (most, page)).transpose(2, 3)


def _values(pages, lens, dtype):
    """f16 pages [m][pages][kv][page][hd] as the cache holds lens[m] positions of them, packed rows of `dtype`."""
    m, most, _, page, _ = pages.shape
    code, scale = _quantized(pages)
    whole = (torch.arange(most, device="cuda")[None] + 1) * page <= lens[:, None]
    x = torch.where(whole[:, :, None, None, None], code.float() * scale[..., None, None], pages.float())
    x = x.transpose(2, 3).flatten(1, 2)
    return x[torch.arange(most * page, device="cuda")[None] < lens[:, None]].to(dtype)


def _append_plain(s):
    case = s["case"]
    start = s["len"] - s["full"] * case["page"]
    dtype = TYPES[case["dtype"]]
    out = []
    for layer, pair in enumerate(s["new"]):
        for which, x in enumerate(pair):
            pages = _grown_plain(s["open"][:, layer, which], x.unflatten(0, (-1, case["new"])), start, case["page"])
            out.append(_values(pages, start + case["new"], dtype))
    return out


def _branch_plain(s):
    case = s["case"]
    f, page, n = case["forks"], case["page"], case["seqs"]
    dtype = TYPES[case["dtype"]]
    kept = torch.arange(n, device="cuda") * f + torch.arange(n, device="cuda") % f
    start = (s["len"] - s["full"] * page).repeat_interleave(f)
    out = []
    for layer, pair in enumerate(s["new"]):
        for which, x in enumerate(pair):
            opened = s["open"][:, layer, which].repeat_interleave(f, 0)  # the branches' own open pages
            pages = _grown_plain(opened, x.unflatten(0, (-1, case["new"])), start, page)
            code, scale = _quantized(pages)  # every branch grows; those kept are read
            ends = (start + case["new"])[kept]
            whole = (torch.arange(pages.shape[1], device="cuda")[None] + 1) * page <= ends[:, None]
            tail = torch.where(whole[:, :, None, None, None], code[kept].float() * scale[kept][..., None, None], pages[kept].float())
            tail = tail.transpose(2, 3).flatten(1, 2)
            if s["pool"].shape[0]:
                head = s["pool"][:, layer, which][s["table"]].float() * s["scales"][:, layer, which][s["table"]][..., None, None]
            else:
                head = torch.zeros(n, 0, *tail.shape[2:], device="cuda").unflatten(1, (0, page)).transpose(2, 3)
            head = head.transpose(2, 3).flatten(1, 2)
            all_ = torch.cat([head, tail], 1)
            ok = torch.cat([torch.arange(head.shape[1], device="cuda")[None] < (s["full"] * page)[:, None],
                            torch.arange(tail.shape[1], device="cuda")[None] < ends[:, None]], 1)
            out.append(all_[ok].to(dtype))
    return out


def _copies_plain(s):
    case = s["case"]
    page, n = case["page"], case["seqs"]
    used = s["pool"].shape[0]
    pool = torch.cat([s["pool"], s["pool"]])  # every sequence's pages copied behind the pool
    scales = torch.cat([s["scales"], s["scales"]])
    opened = s["open"].clone()
    kept = torch.arange(1, n, 2, device="cuda")
    number = torch.arange(s["table"].shape[1], device="cuda")[None]
    live = number < s["full"][kept][:, None]
    old = (s["table"][kept] + used)[live]  # the pages that stay, moved together
    to = used + torch.arange(old.shape[0], device="cuda")
    pool[to] = pool[old]
    scales[to] = scales[old]
    table = torch.zeros_like(s["table"][kept])
    table[live] = to
    t = {"pool": pool, "scales": scales, "open": opened[kept], "table": table, "full": s["full"][kept]}
    out = []
    for layer in range(case["layers"]):
        for which in (0, 1):
            x = _held(t, layer, which)
            out.append(x[torch.arange(x.shape[1], device="cuda")[None] < s["len"][kept][:, None]].to(TYPES[case["dtype"]]))
    return out


def _dense_plain(s):
    case = s["case"]
    packed, x = s["packed"], s["x"]
    code = torch.cat([packed & 15, packed >> 4], -1).float() - 8.0  # [n][groups][32]
    w = code * s["scales"].float()[..., None]
    if not case["table"]:
        g = x.unflatten(1, (-1, 32))
        most = g.abs().amax(-1, keepdim=True)
        scale = torch.where(most > 0, (most.double() / 127.0).float(), 1.0)
        q = torch.clamp(torch.round(g * (1.0 / scale)), -127, 127)
        x = (q * scale.to(torch.float16).float()).flatten(1)
    return torch.matmul(x, w.flatten(1).t())


# -------------------------------------------------------------- one pass

def _empty(rows, case):
    return torch.empty(rows, case["kv"], case["hd"], dtype=TYPES[case["dtype"]], device="cuda")


def _read(s, seqs, firsts, counts):
    case, out = s["case"], []
    for layer in range(case["layers"]):
        k, v = _empty(sum(counts), case), _empty(sum(counts), case)
        s["cache"].read(layer, seqs, firsts, counts, k.data_ptr(), v.data_ptr(), dtype=case["dtype"], stream=s["stream"])
        out += [k, v]
    return out


def _grow(s, seqs):
    case, kv = s["case"], s["cache"]
    counts = [case["new"]] * len(seqs)
    kv.extend(seqs, counts, stream=s["stream"])
    for layer, (k, v) in enumerate(s["new"]):
        kv.append(layer, seqs, counts, k.data_ptr(), v.data_ptr(), dtype=case["dtype"], stream=s["stream"])


def _run_own(s):
    case = s["case"]
    if case["kind"] == "dense":
        out = torch.empty(case["rows"], case["n"], device="cuda")
        s["layer"].forward_device(s["x"].data_ptr(), case["rows"], out.data_ptr(), torch.cuda.current_stream().cuda_stream or 1)
        return out
    kv, stream, lens = s["cache"], s["stream"], s["lens"]
    if case["kind"] == "attend":
        out = torch.empty_like(s["q"])
        kv.attend(0, s["seqs"], s["rows"], s["q"].data_ptr(), out.data_ptr(), heads=case["heads"], dtype=case["dtype"],
                  scale=s["scale"], causal=case["causal"], stream=stream)
        return out
    if case["kind"] == "append":
        branches = kv.fork(s["seqs"], stream=stream)
        _grow(s, branches)
        firsts = [t // case["page"] * case["page"] for t in lens]
        out = _read(s, branches, firsts, [t + case["new"] - a for t, a in zip(lens, firsts)])
        kv.release(branches)
        return out
    if case["kind"] == "branch":
        f = case["forks"]
        branches = kv.fork([q for q in s["seqs"] for _ in range(f)], stream=stream)
        _grow(s, branches)
        kept = [branches[i * f + i % f] for i in range(len(lens))]
        stay = set(kept)
        kv.release([b for b in branches if b not in stay])
        kv.compact(stream=stream)
        out = _read(s, kept, [0] * len(lens), [t + case["new"] for t in lens])
        kv.release(kept)
        return out
    copies = kv.copy(s["seqs"], stream=stream)
    kv.release(copies[0::2])
    kv.compact(stream=stream)
    out = _read(s, copies[1::2], [0] * len(lens[1::2]), lens[1::2])
    kv.release(copies[1::2])
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"attend": _attend_plain, "append": _append_plain, "branch": _branch_plain, "copies": _copies_plain,
            "dense": _dense_plain}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- 64 bits

def _exact_held(x, page):
    """What the cache holds of one sequence's rows x [t][kv][hd], in 64 bits."""
    x = x.to(torch.float16).double()
    t = x.shape[0] // page * page
    if t:
        b = x[:t].reshape(-1, page, *x.shape[1:])
        scale = (b.abs().amax(dim=(1, 3), keepdim=True) / 127.0).float().double()
        x = torch.cat([torch.where(scale > 0, torch.round(b / scale.clamp_min(1e-300)) * scale, 0.0).reshape(t, *x.shape[1:]), x[t:]])
    return x


def _parts(x, counts):
    return list(torch.split(x, counts))


def exact(case, seed):
    if case["kind"] == "dense":
        scales, packed, x = _blocks(case, seed)
        if case["table"]:
            x = x.double()
        else:
            # The rounding of the activations is defined in f32 steps; what follows is exact.
            g = x.cpu().numpy().reshape(case["rows"], -1, 32)
            most = np.abs(g).max(-1, keepdims=True)
            step = np.where(most > 0, most / np.float32(127), np.float32(1)).astype(np.float32)
            code = np.clip(np.rint(g * (np.float32(1) / step)), -127, 127)
            x = torch.from_numpy((code.astype(np.float64) * step.astype(np.float16).astype(np.float64)).reshape(case["rows"], -1)).cuda()
        out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for a in range(0, case["n"], 8192):
            c = packed[a:a + 8192].int()
            w = torch.cat([c % 16, c // 16], -1).double().sub(8).mul(scales[a:a + 8192].double()[..., None])
            out[:, a:a + 8192] = x @ w.flatten(1).t()
        return out
    s, page = _raw(case, seed), case["page"]
    lens, kv, hd = s["lens"], case["kv"], case["hd"]
    if case["kind"] == "attend":
        heads = case["heads"]
        g, out = heads // kv, []
        k0, v0 = (_parts(x, lens) for x in s["kv0"][0])
        for q, k, v in zip(_parts(s["q"], s["rows"]), k0, v0):
            q, k, v = q.double(), _exact_held(k, page), _exact_held(v, page)
            m, t = q.shape[0], k.shape[0]
            if not t or not m:
                out.append(torch.zeros_like(q))
                continue
            seen = torch.ones(m, t, dtype=torch.bool, device="cuda")
            if case["causal"]:
                seen = torch.arange(t, device="cuda")[None] <= torch.arange(t - m, t, device="cuda")[:, None]
            o = torch.empty_like(q)
            for h in range(heads):
                sc = (q[:, h] @ k[:, h // g].t() * s["scale"]).masked_fill(~seen, -math.inf)
                o[:, h] = torch.softmax(sc, -1) @ v[:, h // g]
            out.append(o)
        return torch.cat(out)
    out = []
    for layer in range(case["layers"]):
        for which in (0, 1):
            old = _parts(s["kv0"][layer][which], lens)
            if case["kind"] == "copies":
                out.append(torch.cat([_exact_held(x, page) for x in old[1::2]]))
                continue
            f = case.get("forks", 1)
            new = _parts(s["new"][layer][which], [case["new"]] * (len(lens) * f))
            rows = [_exact_held(torch.cat([x, new[i * f + i % f]]), page) for i, x in enumerate(old)]
            out.append(torch.cat(rows if f > 1 else [x[t // page * page:] for x, t in zip(rows, lens)]))
    return out
