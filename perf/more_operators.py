"""Cases of the operators of a speculative decoding step over the 4-bit paged KV cache:

  tree    attention of the drafted rows of every sequence (a tree given by parents) over its
          cached rows and over the drafted rows' ancestors
  verify  which drafted tokens stand, from the target's logits, given random numbers and, where
          the drafts were sampled, the draft's logits; and the token that follows them
  append  QKV rows -> rotated query rows, and K (rotated) and V into the pages of the cache; all
          rows, or the accepted ones of a drafted tree

Where `own` is false `run` computes them with elementary torch operations in 32 bits (angles,
distributions and values next to a rounding border in 64), where it is true through the package.

The rows of a sequence are its tree: row 0 its last token, whose K and V are not cached yet, the
others drafted tokens, parents[i] < i the parent's row (-1 at row 0).

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
    vocab = {"vocab": 200064}
    return [
        # one conversation with a short chain of drafts
        {"name": "tree_one", "op": "tree", **phi, "n_seqs": 1, "lens": "all", "max_len": 1023, "nodes": 6, "shape": "chain",
         "pick": 1, "type": "bf16"},
        # a batch of conversations of different lengths, a small tree each
        {"name": "tree_batch", "op": "tree", **phi, "n_seqs": 64, "lens": "even", "max_len": 8190, "nodes": 16, "shape": "tree",
         "pick": 5, "type": "bf16"},
        # a wide tree over a very long context
        {"name": "tree_long", "op": "tree", **phi, "n_seqs": 1, "lens": "all", "max_len": 131000, "nodes": 60, "shape": "tree",
         "pick": 2, "type": "bf16"},
        # narrow heads, eight queries to a KV head, trees of different sizes
        {"name": "tree_narrow", "op": "tree", "n_heads": 64, "n_kv": 8, "hd": 64, "n_seqs": 24, "lens": "spread",
         "max_len": 6000, "nodes": 33, "shape": "mixed", "pick": 7, "type": "f16"},
        # one conversation whose drafts were looked up in its text
        {"name": "verify_one", "op": "verify", **vocab, "n_seqs": 1, "nodes": 6, "shape": "chain", "draft": False,
         "greedy": 0.0, "type": "f32", "pick": 1},
        # a batch of chains drawn from a small model's logits
        {"name": "verify_chain", "op": "verify", **vocab, "n_seqs": 48, "nodes": 5, "shape": "chain", "draft": True,
         "greedy": 0.1, "type": "f32", "pick": 2},
        # a batch of trees, a quarter of the users without sampling
        {"name": "verify_tree", "op": "verify", **vocab, "n_seqs": 16, "nodes": 32, "shape": "mixed", "draft": False,
         "greedy": 0.25, "type": "bf16", "pick": 3},
        # the new row of 64 decoding sequences
        {"name": "append_64_rows", "op": "append", **phi, "rope_dim": 96, "n_seqs": 64, "lens": "one", "max_len": 4000,
         "pick": 3, "path": False, "norm": False, "halves": False, "factors": True, "in": "f32", "out": "bf16"},
        # the rows of a batch of prompts of a model with per-head norms
        {"name": "append_prompts", "op": "append", "n_heads": 32, "n_kv": 8, "hd": 128, "rope_dim": 128, "n_seqs": 9,
         "lens": "spread", "max_len": 3900, "pick": 4, "path": False, "norm": True, "halves": True, "factors": False,
         "in": "bf16", "out": "bf16"},
        # the accepted rows of 64 drafted trees
        {"name": "append_accepted", "op": "append", **phi, "rope_dim": 96, "n_seqs": 64, "lens": "even", "max_len": 16,
         "pick": 6, "path": True, "norm": False, "halves": False, "factors": True, "in": "f32", "out": "bf16"},
    ]


def draw(rng):
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["tree", "tree", "verify", "append"])
    case = {"op": op, "pick": rng.randrange(1 << 30)}
    if op == "verify":
        vocab = size(1000, 260000)
        n_seqs = size(1, 64)
        nodes = size(1, max(1, min(64, 512 // n_seqs)))
        return {**case, "vocab": vocab, "n_seqs": n_seqs, "nodes": nodes, **rng.choice(
            [{"shape": "chain", "draft": True}, {"shape": "chain", "draft": False}, {"shape": "mixed", "draft": False}]),
            "greedy": rng.choice([0.0, 0.3]), "type": rng.choice(["f32", "bf16", "f16"])}
    hd = rng.choice([64, 128, 128, 256])
    n_kv = rng.choice([1, 2, 4, 8])
    per = rng.choice([1, 2, 3, 4, 8] if n_kv < 8 else [1, 2, 3, 4])
    case |= {"n_heads": n_kv * per, "n_kv": n_kv, "hd": hd, "lens": rng.choice(["spread", "even"])}
    if op == "append":
        path = rng.random() < 0.4
        rope_dim = rng.choice([32, 64] if hd == 64 else [64, 96, 128])
        return {**case, "rope_dim": rope_dim, "n_seqs": size(1, 60), "max_len": size(1, 64 if path else 1200),
                "path": path, "norm": rng.random() < 0.5, "halves": rng.random() < 0.5, "factors": rng.random() < 0.5,
                "in": rng.choice(["f32", "bf16", "f16"]), "out": rng.choice(["bf16", "f16"])}
    n_seqs, nodes = size(1, 60), size(1, 100)
    most = min(60000, int(2.5e10 / (n_seqs * nodes * case["n_heads"] * hd * 4)) + 2, 500000 // n_seqs)
    return {**case, "n_seqs": n_seqs, "max_len": size(2, max(3, most)), "nodes": nodes,
            "shape": rng.choice(["chain", "tree", "mixed"]), "type": rng.choice(["bf16", "f16"])}


def lengths(case):
    """The rows of each sequence (append: packed ones, tree: cached ones): one, max_len, or spread
    over 1..max_len (evenly, or evenly in the logarithm with both ends)."""
    n, most, pick = case["n_seqs"], case["max_len"], random.Random(case["pick"])
    if case["lens"] == "one":
        return [1] * n
    if case["lens"] == "all":
        return [most] * n
    if case["lens"] == "even":
        return [pick.randint(1, most) for _ in range(n)]
    return ([most, 1] + [int(round(math.exp(pick.uniform(0, math.log(most + 0.4))))) for _ in range(n)])[:n]


def trees(case):
    """The parents of each sequence's rows: chains, trees of `nodes` rows that get narrower as they
    get deeper, or (mixed) trees of one row to `nodes`."""
    pick = random.Random(case["pick"] + 2)
    got = []
    for n in range(case["n_seqs"]):
        rows = case["nodes"] if case["shape"] != "mixed" or n == 0 else pick.randint(1, case["nodes"])
        if case["shape"] == "chain":
            got.append([i - 1 for i in range(rows)])
        else:  # parents in ascending order, so that a depth's rows lie together
            got.append([-1] + sorted(min(pick.randrange(i), pick.randrange(i)) for i in range(1, rows)))
            got[-1] = [min(p, i - 1) for i, p in enumerate(got[-1])]
    return got


def paths(case):
    """append: the accepted rows of each sequence, from row 0 on."""
    pick = random.Random(case["pick"] + 3)
    got = []
    for rows in lengths(case):
        deeper = sorted(pick.sample(range(1, rows), pick.randint(0, min(5, rows - 1)))) if rows > 1 else []
        got.append([0] + deeper)
    return got


def before(case):
    """append: the rows that each sequence has in the cache before the call."""
    pick = random.Random(case["pick"] + 1)
    return [pick.randrange(max(case["max_len"], 1000)) for _ in range(case["n_seqs"])]


def starts(lens):
    got = [0]
    for n in lens:
        got.append(got[-1] + n)
    return got


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
        code = code.to(torch.uint8)
        if is_k:  # [.., row, P, i, t, nibble] -> [.., P, row, t, i, byte, 2]
            c = code.view(pages, n_kv, ROWS, planes, j, 4, 4, 2).permute(0, 1, 3, 2, 5, 4, 6, 7)
        else:  # [.., b, h, t, odd, P, i, nibble, g] -> [.., P, b, h, g, t, i, odd, byte, 2]
            c = code.view(pages, n_kv, 4, 2, 4, 2, planes, j, 2, 2, 8)
            c = c.permute(0, 1, 6, 2, 3, 10, 4, 7, 5, 8, 9)
        parts.append((c[..., 0] + 16 * c[..., 1]).reshape(pages, n_kv, 32 * hd))
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
    made = torch.Generator("cuda").manual_seed(seed * 1000003 + 29)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=made)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s = {"case": case}
    if case["op"] == "verify":
        family = trees(case)
        cu = starts([len(t) for t in family])
        rows, vocab, n_seqs = cu[-1], case["vocab"], case["n_seqs"]
        s["cu_rows"] = ints(cu)
        s["parents"] = ints([p for t in family for p in t])
        up = ints([cu[n] + max(p, 0) for n, t in enumerate(family) for p in t]).long()  # the parent's packed row
        # a few dozen likely tokens over a long tail
        logits = 2.2 * normal(rows, vocab)
        strong = torch.randint(0, vocab, (rows, 24), device="cuda", generator=made)
        logits.scatter_add_(1, strong, 9 + 2.5 * normal(rows, 24))
        s["logits"] = logits.to(TYPES[case["type"]])
        # the draft knows its parent's distribution roughly
        guess = logits[up] + 0.9 * normal(rows, vocab) if case["draft"] else logits[up] + 0.4 * normal(rows, vocab)
        if case["draft"]:
            s["draft"] = guess.to(TYPES[case["type"]])
            guess = s["draft"].float()
        else:
            s["draft"] = None
        spread = torch.rand(n_seqs, device="cuda", generator=made) * 0.6 + 0.6
        greedy = torch.rand(n_seqs, device="cuda", generator=made) < case["greedy"]
        s["temperature"] = torch.where(greedy, torch.zeros_like(spread), spread)
        of = torch.repeat_interleave(torch.arange(n_seqs, device="cuda"), ints([len(t) for t in family]).long())
        heat = spread[of][:, None]
        chance = torch.rand(rows, vocab, device="cuda", generator=made).clamp_(1e-20, 1 - 1e-7)
        s["tokens"] = (guess / heat - (-chance.log()).log()).argmax(-1).int()  # drawn from the draft's distribution
        s["uniforms"] = torch.rand(rows, 2, device="cuda", generator=made)
        s["outs"] = [torch.empty(rows, device="cuda", dtype=torch.int32)] + [
            torch.empty(n_seqs, device="cuda", dtype=torch.int32) for _ in range(2)]
        return s
    n_heads, n_kv, hd = case["n_heads"], case["n_kv"], case["hd"]
    if case["op"] == "append":
        new, old = lengths(case), before(case)
        taken = [len(p) for p in paths(case)] if case["path"] else new
        held, cu = [a + b for a, b in zip(taken, old)], starts(new)
        rows = cu[-1]
        s["qkv"] = (2 * normal(rows, (n_heads + 2 * n_kv) * hd)).to(TYPES[case["in"]])
        s["gammas"] = [torch.rand(hd, device="cuda", generator=made) + 0.5 for _ in range(2)] if case["norm"] else None
        s["factors"] = torch.rand(case["rope_dim"] // 2, device="cuda", generator=made) * 0.5 + 1 if case["factors"] else None
        s["path"] = s["counts"] = s["q"] = None
        if case["path"]:
            s["path"] = ints([x for p, n in zip(paths(case), new) for x in p + [-1] * (n - len(p))])
            s["counts"] = ints(taken)
        else:
            s["q"] = torch.empty(rows, n_heads, hd, device="cuda", dtype=TYPES[case["out"]])
        s["cu_rows"], s["cu_taken"], s["kv_lens"] = ints(cu), ints(starts(taken)), ints(held)
        s["outs"] = [torch.empty(sum(taken), n_kv, hd, device="cuda", dtype=TYPES[case["out"]]) for _ in range(2)]
    else:
        held, family, t = lengths(case), trees(case), TYPES[case["type"]]
        cu = starts([len(x) for x in family])
        s["cu_rows"], s["parents"], s["kv_lens"] = ints(cu), ints([p for x in family for p in x]), ints(held)
        strong = torch.exp(0.5 * normal(n_kv, hd))  # keys have a few strong channels
        s["q"] = normal(cu[-1], n_heads, hd).to(t)
        s["k"], s["v"] = (normal(cu[-1], n_kv, hd) * strong).to(t), normal(cu[-1], n_kv, hd).to(t)
        s["out"] = torch.empty_like(s["q"])
    # pages of the sequences, in an order of their own
    per = -(-max(held) // ROWS)
    first = starts([-(-n // ROWS) for n in held])
    order = torch.randperm(first[-1], device="cuda", generator=made).int()
    at = ints(first[:-1])[:, None] + torch.arange(per, device="cuda", dtype=torch.int32)
    used = torch.arange(per, device="cuda")[None] * ROWS < s["kv_lens"][:, None]
    s["page_table"] = torch.where(used, order[at.clamp(max=first[-1] - 1).long()], 0).contiguous()
    if case["op"] == "append":
        s["pages"] = torch.zeros(first[-1], n_kv, 80 * hd, device="cuda", dtype=torch.uint8)
        return s
    k = normal(first[-1] * ROWS, n_kv, hd) * strong
    s["pages"] = blocks(k, normal(first[-1] * ROWS, n_kv, hd))
    return s


def run(state):
    return {"tree": tree, "verify": verify, "append": append}[state["case"]["op"]](state)


def rows_of(s, nodes):
    """Of packed rows: their sequence and place in it, and of places [n_seqs, nodes] the packed row and whether it is there."""
    cu = s["cu_rows"].long()
    r = torch.arange(s["rows"], device="cuda")
    of = torch.bucketize(r, cu[1:], right=True)
    there = torch.arange(nodes, device="cuda") < (cu[1:] - cu[:-1])[:, None]
    at = torch.where(there, cu[:-1, None] + torch.arange(nodes, device="cuda"), 0)
    return of, r - cu[of], at, there


def ancestors(s, at, there):
    """[n_seqs, nodes, nodes]: whether the second row is an ancestor of the first, or the row itself."""
    nodes = at.shape[1]
    up = torch.where(there, s["parents"].long()[at], -1)
    link = (up[..., None] == torch.arange(nodes, device="cuda")).float()
    one = torch.eye(nodes, device="cuda").expand_as(link)
    return torch.linalg.solve_triangular(one - link, one, upper=False) > 0.5  # 1 + link + link^2 + ..


def tree(s):
    case, q = s["case"], s["q"]
    n_heads, n_kv, hd, n_seqs = case["n_heads"], case["n_kv"], case["hd"], case["n_seqs"]
    if own:
        rrr, ctx = package()
        if "cache" not in s:
            s["cache"] = rrr.KV4Cache(ctx, s["pages"], s["page_table"], hd)
            s["workspace"] = s["cache"].tree_workspace(n_heads, q.shape[0])
        s["cache"].attention_tree(q, s["k"], s["v"], s["cu_rows"], s["parents"], s["kv_lens"], s["out"], s["workspace"])
        return s["out"]
    s["rows"], nodes = q.shape[0], case["nodes"]
    of, place, at, there = rows_of(s, nodes)
    k, v = unpacked(s["pages"][s["page_table"].long()], hd, torch.float32)  # [n_seqs, per, n_kv, 64, hd]
    k, v = (x.transpose(1, 2).reshape(n_seqs, n_kv, -1, hd) for x in (k, v))
    held = k.shape[2]
    k, v = (torch.cat((x, y.float()[at].transpose(1, 2)), 2) for x, y in ((k, s["k"]), (v, s["v"])))
    seen = torch.arange(held, device="cuda") < s["kv_lens"][:, None]
    seen = torch.cat((seen[:, None].expand(-1, nodes, -1), ancestors(s, at, there) & there[:, None]), -1)
    qs = q.float()[at].view(n_seqs, nodes, n_kv, -1, hd).permute(0, 2, 3, 1, 4)  # [n_seqs, n_kv, per head, nodes, hd]
    score = qs.reshape(n_seqs, n_kv, -1, hd) @ k.transpose(-1, -2)
    score = score.view(n_seqs, n_kv, -1, nodes, k.shape[2]).mul_(1 / math.sqrt(hd))
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    o = (score.view(n_seqs, n_kv, -1, k.shape[2]) @ v).view(n_seqs, n_kv, -1, nodes, hd) / total
    return o.permute(0, 3, 1, 2, 4).reshape(n_seqs, nodes, n_heads, hd)[of, place].to(q.dtype)


def verify(s):
    case, logits, draft = s["case"], s["logits"], s["draft"]
    path, counts, following = s["outs"]
    if own:
        rrr, ctx = package()
        if "workspace" not in s:
            s["workspace"] = rrr.verify_workspace(ctx, *logits.shape, case["n_seqs"], draft is not None)
        rrr.verify_drafts(ctx, logits, s["tokens"], s["cu_rows"], s["uniforms"], path, counts, following, s["workspace"],
                          draft=draft, parents=None if draft is not None else s["parents"], temperature=s["temperature"])
        return [path, counts, following]
    nodes, cu = case["nodes"], s["cu_rows"].long()
    s["rows"] = logits.shape[0]
    of, place, at, there = rows_of(s, nodes)
    heat = s["temperature"][of].double()[:, None]
    best = logits.float().argmax(-1)
    tokens, u = s["tokens"].long(), s["uniforms"].double()

    def chances(x, heat):
        return torch.softmax(x.double() / heat.where(heat > 0, 1), -1)

    def sampled(weights, u):
        total = weights.cumsum(-1)
        return torch.searchsorted(total, u[:, None] * total[:, -1:], right=True)[:, 0].clamp(max=weights.shape[1] - 1)

    up = (cu[of] + s["parents"].long()).clamp(min=0)  # the parent's packed row
    root = s["parents"] < 0
    if draft is None:
        chosen = torch.where(heat[:, 0] > 0, sampled(chances(logits, heat), u[:, 1]), best)
        stands = tokens == chosen[up]
        family, token = torch.where(there, s["parents"].long()[at], -2), tokens[at]
        twin = (family[:, :, None] == family[:, None]) & (token[:, :, None] == token[:, None])
        stands &= ~twin.tril(-1).any(-1)[of, place]
    else:
        p = chances(logits[up], heat).gather(1, tokens[:, None])[:, 0]
        q = chances(draft, heat).gather(1, tokens[:, None])[:, 0]
        stands = torch.where(heat[:, 0] > 0, u[:, 0] * q < p, tokens == best[up])
    stands |= root & (place == 0)
    fallen = torch.where(there, ~stands[at], True)
    kept = ~(ancestors(s, at, there) & fallen[:, None]).any(-1) & there
    count = kept.sum(-1)
    places = torch.arange(nodes, device="cuda")
    order = torch.where(kept, places, nodes).sort(-1).values
    out = torch.where(order < nodes, order, -1)
    last = cu[:-1] + torch.where(kept, places, 0).amax(-1)  # the deepest row that stands
    if draft is None:
        token = chosen[last]
    else:
        heat = s["temperature"].double()[:, None]
        p = chances(logits[last], heat)
        refused = last + 1 < cu[1:]
        rest = (p - chances(draft[torch.where(refused, last + 1, 0)], heat)).clamp(min=0)
        p = torch.where(refused[:, None] & (rest.sum(-1, keepdim=True) > 0), rest, p)
        token = torch.where(heat[:, 0] > 0, sampled(p, u[last, 1]), best[last])
    return [out[of, place].int(), count.int(), token.int()]


def append(s):
    case, qkv = s["case"], s["qkv"]
    n_heads, n_kv, hd, dim = case["n_heads"], case["n_kv"], case["hd"], case["rope_dim"]
    if own:
        rrr, ctx = package()
        if "cache" not in s:
            f = s["factors"]
            s["cache"] = rrr.KV4Cache(ctx, s["pages"], s["page_table"], hd)
            s["desc"] = rrr.ffi.AttnDesc(n_heads, n_kv, hd, dim, 10000.0, 1.190238, None if f is None else f.data_ptr(),
                                         0 if f is None else f.numel(), 131072)
        gq, gk = s["gammas"] or (None, None)
        s["cache"].append(s["desc"], qkv, s["cu_rows"], s["kv_lens"], s["q"], path=s["path"], counts=s["counts"],
                          q_gamma=gq, k_gamma=gk, eps=1e-5, halves=case["halves"])
        s["cache"].load(s["cu_taken"], s["kv_lens"], *s["outs"])
        return [s["q"], *s["outs"]] if s["q"] is not None else list(s["outs"])
    out, taken = TYPES[case["out"]], s["cu_taken"].long()
    i = torch.arange(s["outs"][0].shape[0], device="cuda")
    of = torch.bucketize(i, taken[1:], right=True)
    nth = i - taken[of]
    positions = s["kv_lens"].long()[of] - (taken[of + 1] - taken[of]) + nth
    x = qkv.view(qkv.shape[0], n_heads + 2 * n_kv, hd)
    if s["path"] is not None:
        start = s["cu_rows"].long()[of]
        x = x[start + s["path"].long()[start + nth]]
    x = x.double()
    q, k, v = x[:, :n_heads], x[:, n_heads:n_heads + n_kv], x[:, n_heads + n_kv:]
    if s["gammas"]:
        q, k = ((x * g) * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) for x, g in zip((q, k), s["gammas"]))
    angle = 10000.0 ** (torch.arange(dim // 2, device="cuda", dtype=torch.float64) * (-2.0 / dim))
    angle = angle / s["factors"].double() if s["factors"] is not None else angle
    angle = positions.double()[:, None, None] * angle
    cos, sin = angle.cos() * 1.190238, angle.sin() * 1.190238

    def turned(x):
        a, b = (x[..., :dim // 2], x[..., dim // 2:dim]) if case["halves"] else (x[..., :dim:2], x[..., 1:dim:2])
        a, b = a * cos - b * sin, a * sin + b * cos
        y = torch.cat((a, b), -1) if case["halves"] else torch.stack((a, b), -1).flatten(-2)
        return torch.cat((y, x[..., dim:]), -1)

    held = [turned(q).to(out)] if s["q"] is not None else []
    for x in (turned(k), v):
        code, d, m = quantise(x)
        held.append((code * d + m).flatten(-2).to(out))
    return held


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "verify":
        rows = sum(len(t) for t in trees(case))
        drafted = rows - case["n_seqs"] if case["draft"] else 0
        return {"bytes": (rows + drafted) * case["vocab"] * size[case["type"]] + 24 * rows,
                "flops": 4 * (rows + drafted) * case["vocab"]}
    n_heads, n_kv, hd = case["n_heads"], case["n_kv"], case["hd"]
    if case["op"] == "append":  # rows in, q and pages out; pages in, rows out
        width = size[case["out"]]
        taken = sum(len(p) for p in paths(case)) if case["path"] else sum(lengths(case))
        read = (2 * n_kv if case["path"] else n_heads + 2 * n_kv) * hd * size[case["in"]]
        written = 0 if case["path"] else n_heads * hd * width
        return {"bytes": taken * (read + written + 2 * n_kv * (2 * 5 * hd // 8 + hd * width)),
                "flops": taken * (10 * (n_heads + n_kv) + 32 * n_kv) * hd}
    held, family = lengths(case), trees(case)
    rows, width = sum(len(t) for t in family), size[case["type"]]
    pairs = 0
    for a, t in zip(held, family):
        depth = [1] * len(t)
        for i, p in enumerate(t):
            depth[i] = 1 if p < 0 else depth[p] + 1
        pairs += a * len(t) + sum(depth)
    return {"bytes": sum(held) * n_kv * (5 * hd // 4) + rows * hd * width * (2 * n_heads + 2 * n_kv),
            "flops": 4 * hd * n_heads * pairs}


def exact(case, seed):
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    n_heads, n_kv, hd = case["n_heads"], case["n_kv"], case["hd"]
    wide = torch.float64
    if case["op"] == "append":
        dim, half = case["rope_dim"], case["rope_dim"] // 2
        i = torch.arange(half, device="cuda")
        turn = torch.exp(-math.log(10000.0) * 2 * i.to(wide) / dim)
        if s["factors"] is not None:
            turn = turn / s["factors"].to(wide)
        a, b = (i, i + half) if case["halves"] else (2 * i, 2 * i + 1)
        cu, found = s["cu_rows"].tolist(), [[], [], []]
        for n, (new, old) in enumerate(zip(lengths(case), before(case))):
            rows = torch.tensor(paths(case)[n] if case["path"] else range(new), device="cuda")
            x = s["qkv"][cu[n] + rows].to(wide).view(len(rows), -1, hd)
            at = (old + torch.arange(len(rows), device="cuda", dtype=wide))[:, None] * turn
            at = 1.190238 * torch.exp(1j * at)[:, None]
            for j, y in enumerate(x.split([n_heads, n_kv, n_kv], 1)):
                y = y.clone()
                if j < 2:
                    if s["gammas"]:
                        y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * s["gammas"][j].to(wide)
                    z = torch.complex(y[..., a], y[..., b]) * at
                    y[..., a], y[..., b] = z.real, z.imag
                if j:
                    g = y.reshape(-1, 32)
                    low, high = g.min(-1).values[:, None], g.max(-1).values[:, None]
                    m, d = low.half().to(wide), ((high - low) / 15).half().to(wide)
                    y = torch.where(d == 0, m, m + d * torch.round((g - m) / d.where(d != 0, 1)).clamp(0, 15)).view_as(y)
                found[j].append(y)
        found = [torch.cat(f) for f in found]
        return found[1:] if case["path"] else found
    out = torch.zeros(s["q"].shape, dtype=wide, device="cuda")
    cu = s["cu_rows"].tolist()
    for n, (held, up) in enumerate(zip(lengths(case), trees(case))):
        at = s["page_table"][n, :-(-held // ROWS)].long()
        k, v = unpacked(s["pages"][at], hd, wide)
        rows, line = slice(cu[n], cu[n + 1]), []
        for i, p in enumerate(up):
            line.append({i} | (line[p] if p >= 0 else set()))
        seen = torch.tensor([[j in x for j in range(len(up))] for x in line], device="cuda")
        seen = torch.cat((torch.ones(len(up), held, device="cuda", dtype=torch.bool), seen), 1)
        for h in range(n_heads):
            g = h * n_kv // n_heads
            keys = torch.cat((k[:, g].reshape(-1, hd)[:held], s["k"][rows, g].to(wide)))
            values = torch.cat((v[:, g].reshape(-1, hd)[:held], s["v"][rows, g].to(wide)))
            p = torch.softmax((s["q"][rows, h].to(wide) @ keys.T / hd ** 0.5).where(seen, -math.inf), -1)
            out[rows, h] = p @ values
    return out
