"""Cases of the operators that serve a packed batch of sequences with a 4-bit KV cache:

  qk      norms of the query and key heads with the position rotation, QKV rows -> q, k, v
  prompt  causal attention of packed prompts with grouped heads
  store   rows of K and V into the pages of the 4-bit cache, and read back
  decode  attention of one query row per sequence over its pages

Where `own` is false `run` computes them with elementary torch operations in 32 bits (angles
in 64), where it is true through the package.

The cache: pages of 64 rows, one block of 80*hd bytes per (page, KV head). Groups of 32
consecutive values of a head are held as d*code + m (code 0..15, d and m f16). A block is
[K codes 32hd | K d 4hd | K m 4hd | V codes 32hd | V d 4hd | V m 4hd] bytes; with J =
min(hd/32, 4), plane P and group j = P*J + i:
  K codes  u32 [P][row][t 4][i J]: nibble n = element 32j + 8t + n
  V codes  u32 [P][row/16][(row%16)/8][g 8][t 4][i J], t = (row%8)/2: low half the even row,
           high half the odd row; nibble n of a half = element 32j + 8n + g
  K d, K m, V d  f16 [row][hd/32];  V m  f16 [row/2][hd/32][row%2]
"""
import importlib
import math
import random

import torch

own = False

ROWS = 64  # rows of a page
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KEPT = {}  # the package and its context


def package():
    if not KEPT:
        KEPT["rrr"] = importlib.import_module("recursive-routing-racer-rs_b200")
        KEPT["ctx"] = KEPT["rrr"].Context(torch.cuda.current_device())
    return KEPT["rrr"], KEPT["ctx"]


def listed():
    phi = {"n_heads": 24, "n_kv": 8, "hd": 128}
    return [
        # one token of the decode loop between its QKV product and its attention
        {"name": "qk_one_row", "op": "qk", "rows": 1, **phi, "rope_dim": 96, "norm": False, "halves": False,
         "factors": True, "in": "f32", "out": "f32", "far": 2048},
        # a batch of prompts of a model with per-head norms, at the far end of a long context
        {"name": "qk_prompt_norm", "op": "qk", "rows": 16000, "n_heads": 32, "n_kv": 8, "hd": 128, "rope_dim": 128,
         "norm": True, "halves": True, "factors": False, "in": "f32", "out": "bf16", "far": 131072},
        # the new row of 64 decoding sequences
        {"name": "store_64_rows", "op": "store", **phi, "n_seqs": 64, "lens": "one", "max_len": 4000, "pick": 3,
         "type": "bf16"},
        # the rows of a batch of prompts
        {"name": "store_prompts", "op": "store", **phi, "n_seqs": 9, "lens": "spread", "max_len": 3900, "pick": 4,
         "type": "f16"},
        # one short prompt: a question
        {"name": "prompt_short", "op": "prompt", **phi, "n_seqs": 1, "lens": "all", "max_len": 77, "past": 0,
         "pick": 1, "type": "bf16"},
        # packed prompts of very different lengths
        {"name": "prompt_packed", "op": "prompt", **phi, "n_seqs": 12, "lens": "spread", "max_len": 2500, "past": 0,
         "pick": 6, "type": "bf16"},
        # one long document
        {"name": "prompt_long", "op": "prompt", **phi, "n_seqs": 1, "lens": "all", "max_len": 16384, "past": 0,
         "pick": 1, "type": "bf16"},
        # continued prompts (rows before them in the cache) with narrow heads
        {"name": "prompt_continued", "op": "prompt", "n_heads": 32, "n_kv": 4, "hd": 64, "n_seqs": 5,
         "lens": "spread", "max_len": 1100, "past": 2900, "pick": 2, "type": "f16"},
        # one token of one conversation
        {"name": "decode_one", "op": "decode", **phi, "n_seqs": 1, "lens": "all", "max_len": 1023, "pick": 1,
         "type": "f32"},
        # one token over a very long context
        {"name": "decode_long", "op": "decode", **phi, "n_seqs": 1, "lens": "all", "max_len": 131000, "pick": 1,
         "type": "f32"},
        # a batch of conversations of different lengths
        {"name": "decode_batch", "op": "decode", **phi, "n_seqs": 64, "lens": "even", "max_len": 8190, "pick": 5,
         "type": "bf16"},
        # narrow heads, eight queries to a KV head
        {"name": "decode_narrow", "op": "decode", "n_heads": 64, "n_kv": 8, "hd": 64, "n_seqs": 24,
         "lens": "spread", "max_len": 6000, "pick": 7, "type": "f16"},
    ]


def draw(rng):
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["qk", "store", "prompt", "prompt", "decode", "decode"])
    hd = rng.choice([64, 128, 128, 256])
    n_kv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "n_heads": n_kv * rng.choice([1, 2, 3, 4, 8] if n_kv < 8 else [1, 2, 3, 4]), "n_kv": n_kv, "hd": hd}
    if op == "qk":
        rope_dim = rng.choice([32, 64] if hd == 64 else [64, 96, 128])
        return {**case, "rows": size(1, 12000), "rope_dim": rope_dim, "norm": rng.random() < 0.5,
                "halves": rng.random() < 0.5, "factors": rng.random() < 0.5, "in": rng.choice(["f32", "bf16", "f16"]),
                "out": rng.choice(["f32", "bf16", "f16"]), "far": size(100, 1000000)}
    case |= {"n_seqs": size(1, 60), "lens": rng.choice(["spread", "even"]), "pick": rng.randrange(1 << 30)}
    if op == "store":
        return {**case, "lens": rng.choice(["one", "spread", "even"]), "max_len": size(1, 1500), "type": rng.choice(["bf16", "f16"])}
    if op == "prompt":
        case["n_seqs"] = size(1, 16)
        most = 9000 // case["n_seqs"]
        return {**case, "max_len": size(2, most), "past": rng.choice([0, 0, size(1, most)]), "type": rng.choice(["bf16", "f16"])}
    most = min(60000, 500000 // case["n_seqs"])
    return {**case, "max_len": size(2, most), "type": rng.choice(["f32", "bf16", "f16"])}


def lengths(case):
    """The rows of each sequence: one, max_len, or spread over 1..max_len (evenly, or evenly in
    the logarithm with both ends)."""
    n, most, pick = case["n_seqs"], case["max_len"], random.Random(case["pick"])
    if case["lens"] == "one":
        return [1] * n
    if case["lens"] == "all":
        return [most] * n
    if case["lens"] == "even":
        return [pick.randint(1, most) for _ in range(n)]
    return ([most, 1] + [int(round(math.exp(pick.uniform(0, math.log(most + 0.4))))) for _ in range(n)])[:n]


def before(case):
    """The rows that each sequence has in the cache before the call."""
    pick = random.Random(case["pick"] + 1)
    if case["op"] == "prompt":
        return [pick.randrange(case["past"] + 1) if case["past"] else 0 for _ in range(case["n_seqs"])]
    if case["op"] == "store":
        return [pick.randrange(case["max_len"]) for _ in range(case["n_seqs"])]
    return [0] * case["n_seqs"]


def starts(lens):
    return [0] + [sum(lens[: i + 1]) for i in range(len(lens))]


def quantise(x):
    """Codes, d and m of x [..., hd] in groups of 32, as 32-bit values [..., hd/32, 32 or 1]."""
    x = x.float().unflatten(-1, (-1, 32))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m, d = low.half().float(), ((high - low) / 15).half().float()
    code = torch.where(d > 0, (x - m) / d, torch.zeros_like(x)).round().clamp(0, 15)
    return code, d, m


def blocks(k, v):
    """Pages of rows [pages*64, n_kv, hd] of K and V: uint8 [pages, n_kv, 80*hd]."""
    pages, n_kv, hd = k.shape[0] // ROWS, k.shape[1], k.shape[2]
    groups, j = hd // 32, min(hd // 32, 4)
    planes = groups // j
    parts = []
    for rows, is_k in ((k, True), (v, False)):
        code, d, m = quantise(rows.view(pages, ROWS, n_kv, hd).transpose(1, 2))  # [pages, n_kv, 64, groups, 32]
        code = code.to(torch.int32)
        if is_k:  # [.., row, P, i, t, nibble] -> [.., P, row, t, i, byte, 2]
            c = code.view(pages, n_kv, ROWS, planes, j, 4, 4, 2).permute(0, 1, 3, 2, 5, 4, 6, 7)
        else:  # [.., b, h, t, odd, P, i, nibble, g] -> [.., P, b, h, g, t, i, odd, byte, 2]
            c = code.view(pages, n_kv, 4, 2, 4, 2, planes, j, 2, 2, 8)
            c = c.permute(0, 1, 6, 2, 3, 10, 4, 7, 5, 8, 9)
        parts.append((c[..., 0] + 16 * c[..., 1]).to(torch.uint8).reshape(pages, n_kv, 32 * hd))
        d, m = d[..., 0].half(), m[..., 0].half()  # [pages, n_kv, 64, groups]
        if not is_k:
            m = m.view(pages, n_kv, ROWS // 2, 2, groups).transpose(3, 4)
        parts += [s.reshape(pages, n_kv, ROWS * groups).contiguous().view(torch.uint8) for s in (d, m)]
    return torch.cat(parts, -1)


def unpacked(pages, hd, wide):
    """K and V that blocks [..., n_kv, 80*hd] stand for, in the type `wide`: [..., n_kv, 64, hd]."""
    groups, j = hd // 32, min(hd // 32, 4)
    lead, planes = pages.shape[:-1], groups // j
    got = []
    for at, is_k in ((0, True), (40 * hd, False)):
        c = pages[..., at:at + 32 * hd]
        c = torch.stack((c & 15, c >> 4), -1)
        d, m = (pages[..., at + o:at + o + 4 * hd].contiguous().view(torch.float16) for o in (32 * hd, 36 * hd))
        p = len(lead)
        if is_k:
            c = c.view(*lead, planes, ROWS, 4, j, 4, 2).permute(*range(p), p + 1, p, p + 3, p + 2, p + 4, p + 5)
            m = m.view(*lead, ROWS, groups)
        else:
            c = c.view(*lead, planes, 4, 2, 8, 4, j, 2, 2, 2)
            c = c.permute(*range(p), p + 1, p + 2, p + 4, p + 6, p, p + 5, p + 7, p + 8, p + 3)
            m = m.view(*lead, ROWS // 2, groups, 2).transpose(-1, -2)
        c = c.reshape(*lead, ROWS, groups, 32).to(wide)
        d, m = d.view(*lead, ROWS, groups, 1).to(wide), m.reshape(*lead, ROWS, groups, 1).to(wide)
        got.append((c * d + m).view(*lead, ROWS, hd))
    return got


def prepare(case, seed):
    made = torch.Generator("cuda").manual_seed(seed * 1000003 + 17)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=made)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    n_heads, n_kv, hd = case["n_heads"], case["n_kv"], case["hd"]
    s = {"case": case}
    if case["op"] == "qk":
        rows, out = case["rows"], TYPES[case["out"]]
        s["qkv"] = (2 * normal(rows, (n_heads + 2 * n_kv) * hd)).to(TYPES[case["in"]])
        s["positions"] = torch.randint(0, case["far"], (rows,), device="cuda", generator=made, dtype=torch.int32)
        s["gammas"] = [torch.rand(hd, device="cuda", generator=made) + 0.5 for _ in range(2)] if case["norm"] else None
        s["factors"] = torch.rand(case["rope_dim"] // 2, device="cuda", generator=made) * 0.5 + 1 if case["factors"] else None
        s["outs"] = [torch.empty(rows, n, hd, device="cuda", dtype=out) for n in (n_heads, n_kv, n_kv)]
        return s
    # keys have a few strong channels
    strong = torch.exp(0.5 * normal(n_kv, hd))
    new, old = lengths(case), before(case)
    held = [a + b for a, b in zip(new, old)]
    s["cu_rows"], s["kv_lens"] = ints(starts(new)), ints(held)
    if case["op"] == "prompt":
        t = TYPES[case["type"]]
        s["cu_kv"] = ints(starts(held))
        s["q"] = normal(sum(new), n_heads, hd).to(t)
        s["k"] = (normal(sum(held), n_kv, hd) * strong).to(t)
        s["v"] = normal(sum(held), n_kv, hd).to(t)
        s["out"] = torch.zeros_like(s["q"])
        return s
    # pages of the sequences, in an order of their own
    per = -(-max(held) // ROWS)
    count = sum(-(-n // ROWS) for n in held)
    order = torch.randperm(count, device="cuda", generator=made).int()
    first = starts([-(-n // ROWS) for n in held])
    at = ints(first[:-1])[:, None] + torch.arange(per, device="cuda", dtype=torch.int32)
    used = torch.arange(per, device="cuda")[None] * ROWS < s["kv_lens"][:, None]
    s["page_table"] = torch.where(used, order[at.clamp(max=count - 1).long()], 0).contiguous()
    if case["op"] == "store":
        t = TYPES[case["type"]]
        s["k"] = (normal(sum(new), n_kv, hd) * strong).to(t)
        s["v"] = normal(sum(new), n_kv, hd).to(t)
        s["pages"] = torch.zeros(count, n_kv, 80 * hd, device="cuda", dtype=torch.uint8)
        s["outs"] = [torch.empty_like(s["k"]), torch.empty_like(s["v"])]
        return s
    k = normal(count * ROWS, n_kv, hd) * strong
    s["pages"] = blocks(k, normal(count * ROWS, n_kv, hd))
    s["q"] = normal(case["n_seqs"], n_heads, hd).to(TYPES[case["type"]])
    s["out"] = torch.empty_like(s["q"])
    return s


def run(state):
    op = state["case"]["op"]
    return {"qk": qk, "prompt": prompt, "store": store, "decode": decode}[op](state)


def qk(s):
    case, qkv = s["case"], s["qkv"]
    n_heads, n_kv, hd, dim = case["n_heads"], case["n_kv"], case["hd"], case["rope_dim"]
    if own:
        rrr, ctx = package()
        if "desc" not in s:
            f = s["factors"]
            s["desc"] = rrr.ffi.AttnDesc(n_heads, n_kv, hd, dim, 10000.0, 1.190238, None if f is None else f.data_ptr(),
                                         0 if f is None else f.numel(), case["far"])
        q, k, v = s["outs"]
        gq, gk = s["gammas"] or (None, None)
        rrr.qk_norm_rope(ctx, s["desc"], qkv, s["positions"], q, k, v, q_gamma=gq, k_gamma=gk, eps=1e-5, halves=case["halves"])
        return [q, k, v]
    rows, out = qkv.shape[0], TYPES[case["out"]]
    x = qkv.float().view(rows, n_heads + 2 * n_kv, hd)
    q, k, v = x[:, :n_heads], x[:, n_heads:n_heads + n_kv], x[:, n_heads + n_kv:]
    if s["gammas"]:
        q, k = ((x * g) * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) for x, g in zip((q, k), s["gammas"]))
    angle = 10000.0 ** (torch.arange(dim // 2, device="cuda", dtype=torch.float64) * (-2.0 / dim))
    angle = angle / s["factors"].double() if s["factors"] is not None else angle
    angle = s["positions"].double()[:, None, None] * angle
    cos, sin = (angle.cos() * 1.190238).float(), (angle.sin() * 1.190238).float()

    def turned(x):
        a, b = (x[..., :dim // 2], x[..., dim // 2:dim]) if case["halves"] else (x[..., :dim:2], x[..., 1:dim:2])
        a, b = a * cos - b * sin, a * sin + b * cos
        y = torch.cat((a, b), -1) if case["halves"] else torch.stack((a, b), -1).flatten(-2)
        return torch.cat((y, x[..., dim:]), -1).to(out)

    return [turned(q), turned(k), v.to(out)]


def prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        rrr, ctx = package()
        rrr.attention_packed(ctx, q, k, v, s["cu_rows"], s["cu_kv"], s["out"], causal=True)
        return s["out"]
    rows, n_heads, hd = q.shape
    n_kv = k.shape[1]
    i, j = torch.arange(rows, device="cuda"), torch.arange(k.shape[0], device="cuda")
    of_i = torch.bucketize(i, s["cu_rows"][1:], right=True)
    of_j = torch.bucketize(j, s["cu_kv"][1:], right=True)
    last = i - s["cu_rows"][of_i + 1] + s["cu_kv"][of_i + 1]  # the last row that row i sees
    seen = (of_i[:, None] == of_j) & (j <= last[:, None])
    q = q.float().view(rows, n_kv, n_heads // n_kv, hd).permute(1, 2, 0, 3)
    score = q.reshape(n_kv, -1, hd) @ k.float().permute(1, 2, 0)
    score = score.view(n_kv, n_heads // n_kv, rows, -1).mul_(1 / math.sqrt(hd)).masked_fill_(~seen, -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    o = (score.view(n_kv, -1, score.shape[-1]) @ v.float().transpose(0, 1)).view(n_kv, n_heads // n_kv, rows, hd) / total
    return o.permute(2, 0, 1, 3).reshape(rows, n_heads, hd).to(s["q"].dtype)


def store(s):
    if own:
        rrr, ctx = package()
        if "cache" not in s:
            s["cache"] = rrr.KV4Cache(ctx, s["pages"], s["page_table"], s["case"]["hd"])
        s["cache"].store(s["k"], s["v"], s["cu_rows"], s["kv_lens"])
        s["cache"].load(s["cu_rows"], s["kv_lens"], *s["outs"])
        return list(s["outs"])
    held = []
    for x in (s["k"], s["v"]):
        code, d, m = quantise(x)
        held.append((code * d + m).flatten(-2).to(x.dtype))
    return held


def decode(s):
    case = s["case"]
    if own:
        rrr, ctx = package()
        if "cache" not in s:
            s["cache"] = rrr.KV4Cache(ctx, s["pages"], s["page_table"], case["hd"])
            s["workspace"] = s["cache"].workspace(case["n_heads"])
        s["cache"].attention(s["q"], s["kv_lens"], s["out"], s["workspace"])
        return s["out"]
    n_kv, hd, n_seqs = case["n_kv"], case["hd"], case["n_seqs"]
    k, v = unpacked(s["pages"][s["page_table"].long()], hd, torch.float32)  # [n_seqs, per, n_kv, 64, hd]
    k, v = (x.transpose(1, 2).reshape(n_seqs, n_kv, -1, hd) for x in (k, v))
    q = s["q"].float().view(n_seqs, n_kv, -1, hd)
    score = q @ k.transpose(-1, -2) / math.sqrt(hd)
    unseen = torch.arange(k.shape[2], device="cuda") >= s["kv_lens"][:, None]
    score = score.masked_fill(unseen[:, None, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    o = (p @ v) / p.sum(-1, keepdim=True)
    return o.reshape(n_seqs, case["n_heads"], hd).to(s["q"].dtype)


def work(case):
    n_heads, n_kv, hd = case["n_heads"], case["n_kv"], case["hd"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "qk":
        values = case["rows"] * (n_heads + 2 * n_kv) * hd
        return {"bytes": values * (size[case["in"]] + size[case["out"]]) + 4 * case["rows"], "flops": 10 * values}
    new, held = lengths(case), [a + b for a, b in zip(lengths(case), before(case))]
    width = size[case["type"]]
    if case["op"] == "store":  # rows in, pages out; pages in, rows out
        return {"bytes": 2 * sum(new) * n_kv * (2 * hd * width + 5 * hd // 4), "flops": 16 * sum(new) * n_kv * hd}
    if case["op"] == "prompt":
        pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(new, held))
        return {"bytes": width * hd * (2 * sum(new) * n_heads + 2 * sum(held) * n_kv), "flops": 4 * hd * n_heads * pairs}
    return {"bytes": sum(held) * n_kv * (5 * hd // 4) + 2 * case["n_seqs"] * n_heads * hd * width,
            "flops": 4 * hd * n_heads * sum(held)}


def exact(case, seed):
    s = prepare(case, seed)
    n_heads, n_kv, hd = case["n_heads"], case["n_kv"], case["hd"]
    wide = torch.float64
    if case["op"] == "qk":
        dim, half = case["rope_dim"], case["rope_dim"] // 2
        x = s["qkv"].to(wide).view(case["rows"], -1, hd)
        parts = list(x.split([n_heads, n_kv, n_kv], 1))
        i = torch.arange(half, device="cuda")
        turn = torch.exp(-math.log(10000.0) * 2 * i.to(wide) / dim)
        if s["factors"] is not None:
            turn = turn / s["factors"].to(wide)
        turn = torch.polar(torch.full_like(turn, 1.190238), torch.zeros_like(turn)) * torch.exp(
            1j * (s["positions"].to(wide)[:, None] * turn))
        a, b = (i, i + half) if case["halves"] else (2 * i, 2 * i + 1)
        for n in range(2):
            y = parts[n].clone()
            if s["gammas"]:
                y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * s["gammas"][n].to(wide)
            z = torch.complex(y[..., a], y[..., b]) * turn[:, None]
            y[..., a], y[..., b] = z.real, z.imag
            parts[n] = y
        return parts
    if case["op"] == "store":
        held = []
        for x in (s["k"], s["v"]):
            x = x.to(wide)
            y = x.reshape(-1, 32)
            low, high = y.min(-1).values[:, None], y.max(-1).values[:, None]
            m, d = low.half().to(wide), ((high - low) / 15).half().to(wide)
            y = torch.where(d == 0, m, m + d * torch.round((y - m) / d.where(d != 0, 1)).clamp(0, 15))
            held.append(y.view_as(x))
        return held
    if case["op"] == "prompt":
        out = torch.zeros(s["q"].shape, dtype=wide, device="cuda")
        new, cu_q, cu_kv = lengths(case), s["cu_rows"].tolist(), s["cu_kv"].tolist()
        for n, rows in enumerate(new):
            k, v = (x[cu_kv[n]:cu_kv[n + 1]].to(wide) for x in (s["k"], s["v"]))
            held = k.shape[0]
            for h in range(n_heads):
                for at in range(0, rows, 4096):
                    q = s["q"][cu_q[n] + at:cu_q[n] + min(rows, at + 4096), h].to(wide)
                    seen = torch.ones(q.shape[0], held, device="cuda", dtype=torch.bool).tril(held - rows + at)
                    p = torch.softmax((q @ k[:, h * n_kv // n_heads].T / hd ** 0.5).where(seen, -math.inf), -1)
                    out[cu_q[n] + at:cu_q[n] + at + q.shape[0], h] = p @ v[:, h * n_kv // n_heads]
        return out
    out = torch.zeros(s["q"].shape, dtype=wide, device="cuda")
    for n, held in enumerate(lengths(case)):
        at = s["page_table"][n, :-(-held // ROWS)].long()
        k, v = unpacked(s["pages"][at], hd, wide)
        for h in range(n_heads):
            g = h * n_kv // n_heads
            p = torch.softmax(k[:, g].reshape(-1, hd)[:held] @ s["q"][n, h].to(wide) / hd ** 0.5, 0)
            out[n, h] = p @ v[:, g].reshape(-1, hd)[:held]
    return out
