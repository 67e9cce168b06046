"""What random values of one size do not show of the speculative decoding step's operators (test_speculative.py): parts of a
sequence without any row that exists, no pages at all, rows that are computed again, very many rows, drafted values of
very different sizes, tokens that both distributions mask, norms beyond 32 bits' range.

Bounds are those of test_speculative.py, with the roundings that a test's exact values do not make left out."""
import math

import numpy as np
import pytest
import torch

from test_serving import DT, U, Cache, cu_of, gen, half_step, ints, normal, ref_qk, within
from test_speculative import H16, ancestors, check_verify, compare_tree, ref_tree


# ------------------------------------------------------------------ tree
def held_rows(table, n, n_pages):
    """Which of a sequence's n rows lie on pages that exist."""
    return [r for r in range(n) if 0 <= table[r // 64] < n_pages]


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("low", [-1.0, -20.0, -110.0])
@pytest.mark.parametrize("many", [False, True])
def test_attention_tree_of_rows_behind_missing_pages(rrr, ctx, hd, kind, low, many):
    """A sequence's first pages do not exist, and the scores of all other rows are far below 0. One sequence is shared by
    CTAs block by block, of many some are a CTA's own. Keys are constant over a head, in few bits: 16-bit types, the cache
    and the operands hold them, so a score carries the sums' error alone."""
    t, g, nh, nkv, nodes = DT[kind], gen(hd), 2, 1, 3
    lens = [300, 64, 130, 520, 1] * 40 if many else [520]
    gone = [[0, 1], [0], [0, 1], [0, 1, 2, 3, 5], [0]] * 40 if many else [[0, 1, 2]]
    cache, cu = Cache(rrr, ctx, nkv, hd, lens, 3), cu_of(lens)
    n_pages = cache.pages.shape[0]
    row = torch.cat([torch.arange(n, device="cuda") for n in lens]).float()
    step = 2.0 ** math.floor(math.log2(-low)) / 32  # six bits
    level = round(low / step) * step
    k = (level + step * (row % 4))[:, None, None].expand(-1, nkv, hd).contiguous()  # scores of low .. low + 3 steps
    v = normal(g, sum(lens), nkv, hd)
    cache.c.store(k, v, cu, ints(lens))
    cache.c.load(cu, ints(lens), k, v)
    table = cache.c.page_table.cpu().numpy().copy()
    for s, pages in enumerate(gone):
        table[s, pages] = [n_pages + 5 if i % 2 else -3 for i in range(len(pages))]
    cache.c.page_table.copy_(torch.from_numpy(table))
    rows = nodes * len(lens)
    q = torch.full((rows, nh, hd), 1.0 / hd, dtype=t, device="cuda")
    kd = torch.full((rows, nkv, hd), level, dtype=t, device="cuda")
    vd = normal(g, rows, nkv, hd, dtype=t)
    out, tree = torch.empty(rows, nh, hd, dtype=t, device="cuda"), [-1, 0, 0]
    cache.c.attention_tree(q, kd, vd, cu_of([nodes] * len(lens)), ints(tree * len(lens)), ints(lens), out,
                           cache.c.tree_workspace(nh, rows), scale=1.0)
    assert ctx.device_error() == 6
    a, h = 0, half_step(t)
    for s, n in enumerate(lens):
        r, held = slice(nodes * s, nodes * (s + 1)), held_rows(table[s], n, n_pages)
        kc, vc = (x[a:a + n][held].double() for x in (k, v))
        ref, A, _ = ref_tree(q[r].double(), kd[r].double(), vd[r].double(), kc, vc, tree, 1.0)
        top = max(float(vd[r].abs().max()), float(vc.abs().max()) if held else 0.0)
        bound = (2 * torch.expm1(2 * (hd + 16) * U * A) + 2 * H16 + h + 64 * U) * top
        within(out[r], ref, ref.abs() * h * 1.01 + bound[..., None] + 2.0 ** -25)
        a += n


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kind", [(64, "bf16"), (128, "f16"), (256, "bf16")])
def test_attention_tree_computed_again_outlasts_the_waits(rrr, ctx, hd, kind):
    """Rows that are computed again take longer than a role may wait for another: every CTA has two sequences of its own, the
    first of some with an infinity, and all of the others' results are there."""
    t, g, n, limit_us = DT[kind], gen(hd), 20000, 2000
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    seqs, nodes, per = 2 * sms, 3, -(-n // 64)
    one = Cache(rrr, ctx, 1, hd, [n], 3)
    k, v = 0.2 * normal(g, n, 1, hd), normal(g, n, 1, hd)
    one.c.store(k, v, cu_of([n]), ints([n]))
    one.c.load(cu_of([n]), ints([n]), k, v)
    cache = rrr.KV4Cache(ctx, one.pages, one.c.page_table.expand(seqs, per).contiguous(), hd)  # one sequence's rows for all
    rows = seqs * nodes
    q, kd, vd = (normal(g, rows, 1, hd, dtype=t) for _ in range(3))
    bad = list(range(0, seqs, 6))
    vd[[nodes * s + 1 for s in bad], :, hd // 2] = math.inf  # of row 1: rows 0 and 2 do not see it
    out, tree = torch.full((rows, 1, hd), 7.0, dtype=t, device="cuda"), [-1, 0, 0]
    ws = cache.tree_workspace(1, rows)
    ctx.check(rrr.ffi.lib().rrr_set_wait_limit(ctx.h, limit_us * 1000))
    try:
        events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        events[0].record()
        cache.attention_tree(q, kd, vd, cu_of([nodes] * seqs), ints(tree * seqs), ints([n] * seqs), out, ws)
        events[1].record()
        torch.cuda.synchronize()
    finally:
        ctx.check(rrr.ffi.lib().rrr_set_wait_limit(ctx.h, 0))
    assert ctx.device_error() == 0
    assert events[0].elapsed_time(events[1]) * 1000 > limit_us  # (or the test shows nothing)
    for s in [*bad[:3], 1, 2, 3, seqs - 2, seqs - 1]:
        r = slice(nodes * s, nodes * (s + 1))
        if s in bad:
            assert bool(out[nodes * s + 1].isfinite().logical_not().any())
            clean, parents = [nodes * s, nodes * s + 2], [-1, 0]
        else:
            clean, parents = list(range(r.start, r.stop)), tree
        compare_tree(out[clean], q[clean], kd[clean], vd[clean], k, v, [n], [parents], kind, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 8, 1), (128, 6, 2), (256, 3, 1)])
@pytest.mark.parametrize("small,large", [(1e-6, 1.0), (1e-4, 1e4), (1e-9, 1.0), (1e-30, 1e-9), (1e-12, 1e30)])
@pytest.mark.parametrize("n", [0, 70])
def test_attention_tree_of_small_values_beside_large_ones(rrr, ctx, hd, nh, nkv, small, large, n):
    """Drafted values of bf16 rows that differ by many powers of two: a row's result owes nothing to the rows that it does not
    see. (Weights of all equal scores; cached values of zero.)"""
    t, g = torch.bfloat16, gen(hd)
    cache = Cache(rrr, ctx, nkv, hd, [max(n, 1)], 3)
    if n:
        cache.c.store(torch.zeros(n, nkv, hd, device="cuda"), torch.zeros(n, nkv, hd, device="cuda"), cu_of([n]), ints([n]))
    tree = [-1, 0, 0, 1, 2, 0]
    sizes = torch.tensor([small, small, large, small, large, small], device="cuda")[:, None, None]
    q, k = normal(g, 6, nh, hd, dtype=t), torch.zeros(6, nkv, hd, dtype=t, device="cuda")
    v = (normal(g, 6, nkv, hd) * sizes).to(t)
    v[5] = 0  # (nothing at all is no small value)
    out = torch.empty(6, nh, hd, dtype=t, device="cuda")
    cache.c.attention_tree(q, k, v, cu_of([6]), ints(tree), ints([n]), out, cache.c.tree_workspace(nh, 6))
    zero = torch.zeros(n, nkv, hd, dtype=torch.float64, device="cuda")
    ref, _, _ = ref_tree(q.double(), k.double(), v.double(), zero, zero, tree, hd ** -0.5)
    h = half_step(t)
    for i, seen in enumerate(ancestors(tree)):
        top = float(v[seen].abs().max())
        within(out[i], ref[i], ref[i].abs() * h * 1.01 + (2 * H16 + 64 * U) * top)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 4, 2), (128, 3, 1), (256, 2, 1)])
def test_attention_tree_groups_beyond_f16_among_short_sequences(rrr, ctx, hd, nh, nkv):
    """Every fourth sequence has a key that f16 does not hold and whose score counts, between sequences of drafted rows alone:
    what is noted of one segment is read before the fourth one after it takes its place."""
    g, seqs, nodes = gen(hd), 1200, 2
    lens = [70 if s % 4 == 0 else 0 for s in range(seqs)]
    cache, cu = Cache(rrr, ctx, nkv, hd, [70] * seqs, 3), cu_of(lens)
    k, v = normal(g, sum(lens), nkv, hd) * 1e-4, normal(g, sum(lens), nkv, hd)
    k[5::70, :, 3], k[5::70, :, 4] = -6e4, 2e5
    cache.c.store(k, v, cu, ints(lens))
    cache.c.load(cu, ints(lens), k, v)
    rows = seqs * nodes
    q, kd, vd = (normal(g, rows, n, hd, dtype=torch.bfloat16) * s for n, s in ((nh, 1e-4), (nkv, 1.0), (nkv, 1.0)))
    out = torch.empty(rows, nh, hd, dtype=torch.bfloat16, device="cuda")
    cache.c.attention_tree(q, kd, vd, cu_of([nodes] * seqs), None, ints(lens), out, cache.c.tree_workspace(nh, rows))
    some = [s for s in range(seqs) if s % 4 == 0 or s < 40]
    r = [nodes * s + i for s in some for i in range(nodes)]
    compare_tree(out[r], q[r], kd[r], vd[r], k, v, [lens[s] for s in some], [[-1, 0]] * len(some), "bf16", hd ** -0.5)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kind", [(64, "bf16"), (128, "f16"), (256, "bf16")])
@pytest.mark.parametrize("width", [0, 2])
def test_attention_tree_without_pages(rrr, ctx, hd, kind, width):
    """A cache that has no page at all: drafted rows see one another; lengths beside 0 are recorded."""
    t, g, nodes = DT[kind], gen(hd), [3, 0, 5]
    cache = rrr.KV4Cache(ctx, torch.empty(rrr.KV4Cache.page_shape(0, 1, hd), dtype=torch.uint8, device="cuda"),
                         torch.zeros(3, width, dtype=torch.int32, device="cuda"), hd)
    q, k, v = (normal(g, 8, n, hd, dtype=t) for n in (2, 1, 1))
    none = torch.empty(0, 1, hd, device="cuda")
    for lens in ([0, 0, 0], [0, 0, 70]):
        out = torch.empty(8, 2, hd, dtype=t, device="cuda")
        cache.attention_tree(q, k, v, cu_of(nodes), ints([-1, 0, 0, -1, 0, 1, 1, 3]), ints(lens), out, cache.tree_workspace(2, 8))
        assert ctx.device_error() == (6 if sum(lens) else 0)
        compare_tree(out, q, k, v, none, none, [0, 0, 0], [[-1, 0, 0], [], [-1, 0, 1, 1, 3]], kind, hd ** -0.5)


def shared_rows(rrr, ctx, hd, seqs, k, v):
    """One sequence's rows as those of `seqs`: their cache, and what it holds of k and v."""
    n = len(k)
    one = Cache(rrr, ctx, 1, hd, [n], 3)
    one.c.store(k, v, cu_of([n]), ints([n]))
    k, v = torch.empty_like(k), torch.empty_like(v)
    one.c.load(cu_of([n]), ints([n]), k, v)
    return rrr.KV4Cache(ctx, one.pages, one.c.page_table.expand(seqs, -1).contiguous(), hd), k, v


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh", [(64, 8), (64, 2), (128, 2), (256, 3)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_tree_sums_of_many_rows_by_one_cta(rrr, ctx, hd, nh, kind):
    """300,000 rows of one CTA's, equal weights, values of one sign in few bits: no rounding but the result's, those of sums of
    at most 128 blocks (16 cut off a block, 2 u each, in O and in the weights' sum) and of 24 such sums in 32 bits."""
    t, n, g, nodes = DT[kind], 300000, gen(hd), 2
    seqs = torch.cuda.get_device_properties(0).multi_processor_count
    v = (1 + (torch.arange(n, device="cuda") % 13).float() / 16)[:, None, None].expand(n, 1, hd).contiguous()
    cache, k, v = shared_rows(rrr, ctx, hd, seqs, torch.zeros(n, 1, hd, device="cuda"), v)
    rows = seqs * nodes
    q = normal(g, rows, nh, hd, dtype=t)
    kd, vd = torch.zeros(rows, 1, hd, dtype=t, device="cuda"), torch.ones(rows, 1, hd, dtype=t, device="cuda")
    out = torch.empty(rows, nh, hd, dtype=t, device="cuda")
    cache.attention_tree(q, kd, vd, cu_of([nodes] * seqs), None, ints([n] * seqs), out, cache.tree_workspace(nh, rows))
    total = v[:, 0, 0].double().sum()
    for i in range(nodes):
        ref = ((total + i + 1) / (n + i + 1)).expand(seqs, nh, hd)
        within(out[i::nodes], ref, ref * (half_step(t) * 1.01 + (128 * 16 * 2 + 2 * 24 + 16) * U))
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh", [(64, 8), (128, 3), (256, 2)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("more", [0, 5])
@pytest.mark.parametrize("rise", [0.25, 2.0, -0.25])
def test_attention_tree_maxima_that_grow_between_sums(rrr, ctx, hd, nh, kind, more, rise):
    """Scores that rise (or fall) over 40,000 rows of one CTA's, or of two that share them: what was summed before counts by
    the maximum that it was summed under. Keys in few bits, so that scores carry the sums' error alone."""
    t, n, g, nodes = DT[kind], 40000, gen(hd), 3
    seqs = torch.cuda.get_device_properties(0).multi_processor_count + more
    k = rise * (torch.arange(n, device="cuda") // 512).float()[:, None, None].expand(n, 1, hd)
    cache, k, v = shared_rows(rrr, ctx, hd, seqs, k.contiguous(), normal(g, n, 1, hd))
    rows = seqs * nodes
    q = torch.full((rows, nh, hd), 1.0 / hd, dtype=t, device="cuda")
    kd, vd = torch.zeros(rows, 1, hd, dtype=t, device="cuda"), normal(g, rows, 1, hd, dtype=t)
    out = torch.empty(rows, nh, hd, dtype=t, device="cuda")
    cache.attention_tree(q, kd, vd, cu_of([nodes] * seqs), None, ints([n] * seqs), out, cache.tree_workspace(nh, rows), scale=1.0)
    h = half_step(t)
    for s in (0, 1, seqs // 2, seqs - 2, seqs - 1):
        r = slice(nodes * s, nodes * (s + 1))
        ref, A, _ = ref_tree(q[r].double(), kd[r].double(), vd[r].double(), k.double(), v.double(), [-1, 0, 1], 1.0)
        top = float(max(v.abs().max(), vd[r].abs().max()))
        bound = (2 * torch.expm1(2 * (hd + 16) * U * A) + 2 * H16 + h + (128 * 16 * 2 + 2 * 3 + 16) * U) * top
        within(out[r], ref, ref.abs() * h * 1.01 + bound[..., None] + 2.0 ** -25)
    assert ctx.device_error() == 0


# ------------------------------------------------------------------ verify
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", ["inf", "nan", "lowest"])
def test_verify_drafts_of_masked_tokens(rrr, ctx, kind, mask):
    """Tokens that target and draft both mask are never drawn, and a refused draft's rest is drawn from its own tokens at u = 0
    too, wherever the distributions' sums lie."""
    t, vocab = DT[kind], 6000
    none = {"inf": -math.inf, "nan": math.nan, "lowest": torch.finfo(t).min}[mask]

    def row(at):
        x = torch.full((vocab,), none, device="cuda", dtype=torch.float32).to(t)
        for i, p in at.items():
            x[i] = p
        return x
    log = math.log
    for first in (1500, 3, 2047):  # tokens a < b < c, those before them masked by both
        a, b, c = first, 3500, 5200
        cases = [({a: log(0.4), b: log(0.6)}, {a: log(0.5), c: log(0.5)}, c),  # b alone is left
                 ({a: 0.0, b: 9.0}, {a: 1.0, c: 30.0}, c), ({a: -7.0, b: -7.0, 4999: -9.0}, {a: -5.0, c: -5.0}, c),
                 ({a: 0.0, b: 0.0}, {a: 3.0, c: 0.0}, c), ({b: 0.0}, {c: 0.0}, c), ({a: 0.0, b: 3.0}, {a: 0.0, b: 0.0}, a)]
        for p, q, token in cases:
            for u1 in (0.0, 2.0 ** -24, 0.5):
                u = torch.tensor([[0.0, u1], [1 - 2.0 ** -24, u1]], device="cuda")
                for heat in (1.0, 3.0):
                    check_verify(rrr, ctx, torch.stack([row(p), row(p)]), torch.stack([row(q), row(q)]), ints([0, token]), u,
                                 [[-1, 0]], [heat])
                check_verify(rrr, ctx, torch.stack([row(p), row(q)]), None, ints([0, token]), u, [[-1, 0]], [1.0])


@pytest.mark.gpu
def test_verify_drafts_of_faint_tokens(rrr, ctx):
    """Weights of 2^-1010 are weights: at u = 0 the first of them is drawn."""
    vocab = 6000
    x, y = (torch.full((2, vocab), -math.inf, device="cuda") for _ in range(2))
    x[:, 1200], x[:, 3000], x[:, 3001] = -700.0, 0.0, -1.0  # e^-700 = 2^-1010
    y[:, 3000], y[:, 5000] = 0.0, 1.0
    u = torch.tensor([[0.0, 0.0], [0.5, 0.0]], device="cuda")
    got = check_verify(rrr, ctx, x, y, ints([0, 5000]), u, [[-1, 0]], [1.0])
    assert got[2] == [1200]
    assert check_verify(rrr, ctx, x, None, ints([0, 5]), u, [[-1, 0]], [1.0])[2] == [1200]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_verify_drafts_of_numbers_outside_their_range(rrr, ctx, kind):
    """Numbers that no generator gives draw as the ends of the range do."""
    g, vocab = gen(2), 5000
    logits, draft = normal(g, 3, vocab).to(DT[kind]), normal(g, 3, vocab).to(DT[kind])
    logits[:, ::3] = -math.inf
    tokens = ints([0, 3, 6])  # (tokens without a chance: the first draft is refused)
    i = dict(dtype=torch.int32, device="cuda")

    def run(number, draft):
        u = torch.full((3, 2), number, device="cuda")
        path, counts, following = torch.zeros(3, **i), torch.zeros(1, **i), torch.zeros(1, **i)
        ws = rrr.verify_workspace(ctx, 3, vocab, 1, draft is not None)
        ws.fill_(0x7B)
        rrr.verify_drafts(ctx, logits, tokens, cu_of([3]), u, path, counts, following, ws, draft=draft)
        return path.tolist(), counts.tolist(), following.tolist()
    for y in (None, draft):
        first, last = run(0.0, y), run(1 - 2.0 ** -24, y)
        assert all(run(x, y) == first for x in (-1e-3, -5.0, -math.inf, math.nan))
        assert all(run(x, y)[:2] == last[:2] and run(x, y)[2][0] >= last[2][0] and run(x, y)[2][0] % 3 for x in (1.0, 7.0, math.inf))
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [700, 1023, 5001])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_verify_drafts_where_target_and_draft_are_equal(rrr, ctx, vocab, kind):
    """Equal rows leave no rest, wherever in memory they begin: a draft that cannot stand (no token of the vocabulary, a masked one)
    is followed by a token of p."""
    g = gen(vocab)
    for s in (0.5, 4.0, 20.0):
        x = s * normal(g, 3, vocab)
        x[:, 7] = -math.inf
        x = x.to(DT[kind])
        for token in (vocab, -1, 7):
            for u1 in (0.0, 0.129154, 0.5, 0.93, 1 - 2.0 ** -24):
                u = torch.full((3, 2), u1, device="cuda")
                for heat in (1.0, 0.6):
                    check_verify(rrr, ctx, x, x.roll(1, 0), ints([0, token, 3]), u, [[-1, 0, 1]], [heat])


# ------------------------------------------------------------------ append
@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv,rd,halves", [(128, 4, 2, 96, False), (128, 4, 2, 96, True), (64, 2, 2, 36, True), (256, 2, 1, 128, False)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [0.0, 1e-5])
def test_kv4_append_norms_beyond_32_bits(rrr, ctx, hd, nh, nkv, rd, halves, kind, eps):
    """Squares that 32 bits do not hold, on either side: the pages are still those of the norm in 64 bits."""
    g, n, t = gen(hd), 12, DT[kind]
    qkv = normal(g, n, (nh + 2 * nkv) * hd)
    sizes = torch.tensor([1.0, 1e20, 1e-25, 3e18, 1e-19, 1e37, 1e-30, 1.0, 1e-22, 1e19, 1e30, 1e-37], device="cuda")
    qkv[:, nh * hd:(nh + nkv) * hd] *= sizes[:, None]
    qkv = qkv.to(t)
    gammas = [torch.rand(hd, device="cuda", generator=g) + 0.5 for _ in range(2)]
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, rd, 10000.0, 1.25, None, 0, 100)
    want, got = (Cache(rrr, ctx, nkv, hd, [n], 3) for _ in range(2))
    refs, _ = ref_qk(qkv, ints(range(n)), nh, nkv, hd, rd, 10000.0, 1.25, None, gammas, float(np.float32(eps)), halves)
    want.c.store(refs[1].float().contiguous(), refs[2].float().contiguous(), cu_of([n]), ints([n]))
    got.c.append(desc, qkv, cu_of([n]), ints([n]), q_gamma=gammas[0], k_gamma=gammas[1], eps=eps, halves=halves)
    assert torch.equal(got.pages, want.pages)
    assert ctx.device_error() == 0
