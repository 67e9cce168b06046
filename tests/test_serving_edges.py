"""The packed-batch operators where a plain comparison of random values sees little: arrays that
share a buffer, streams, small values, rows of other sequences, calls of two host threads. Formulas and helpers are test_serving.py's."""
import ctypes
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

from test_serving import (DT, FINE, ROOT, U, Cache, _no_gpu, check_packed, cu_of, filled, gen, half_step, host_ctx,  # noqa: F401
                          ints, normal, np_quantise, np_values, within)


class KV4Call(ctypes.Structure):  # tests/cpp/two_threads.cpp
    _fields_ = [("ctx", ctypes.c_void_p), ("cache", ctypes.c_void_p), ("n_heads", ctypes.c_int), ("type", ctypes.c_int),
                ("q", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("kv_lens", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_int64), ("stream", ctypes.c_void_p)]


# Rows told apart. `spread`: q is zero, so that rows weigh the same, and row j has one value, in place
# j % hd: a result is (rows seen with that place) / (rows seen), of whole numbers that are summed
# exactly. `paired`: row j's key answers the queries of class j % hd alone (a score of 40, 2^-57 of the
# weight to the others), its value stands in place j / hd % hd: a key or value that is lost, read
# twice, or of another row shows in full, as one row in some (rows seen) / hd.
def told_apart(pattern, rows, n_kv, hd, t, device="cuda"):
    """Keys and values of one sequence, shifted by one row per KV head."""
    j = torch.arange(rows, device=device)[:, None] + torch.arange(n_kv, device=device)
    one = torch.eye(hd, device=device, dtype=t)
    return (one[j % hd], one[j % hd]) if pattern == "spread" else (one[j % hd], one[j // hd % hd])


def asking(pattern, rows, heads, hd, t, device="cuda"):
    if pattern == "spread":
        return torch.zeros(rows, heads, hd, device=device, dtype=t)
    i = 7 * torch.arange(rows, device=device)[:, None] + 5 * torch.arange(heads, device=device)
    return 40 * torch.eye(hd, device=device, dtype=t)[i % hd]


# ------------------------------------------------------------------ CPU
def packed_call(rrr, host_ctx, over):
    """rrr_attention_packed of 9 rows of 4 heads on 11 of 2 heads of 128, with made-up addresses."""
    a = dict(type=30, nh=4, nkv=2, hd=128, n_seqs=2, causal=1, scale=0.0, q_rows=9, kv_rows=11, q_row=512, q_head=128,
             k_row=256, k_head=128, v_row=256, v_head=128, out_row=512, out_head=128, q=1 << 20, k=2 << 20, v=4 << 20,
             out=8 << 20)
    a.update(over)
    d = rrr.ffi.PackedDesc(*(a[f] for f in ("type", "nh", "nkv", "hd", "n_seqs", "causal", "scale", "q_rows", "kv_rows",
                                            "q_row", "q_head", "k_row", "k_head", "v_row", "v_head", "out_row",
                                            "out_head")))
    return rrr.ffi.lib().rrr_attention_packed(host_ctx, ctypes.byref(d), a["q"], a["k"], a["v"], 256, 512, a["out"], None)


FAR = 1 << 38  # the longest stride


@pytest.mark.parametrize("over,code", [
    # 2^29 rows of 2^38 elements end at 2^68 bytes: out begins at one of q's rows, or between them
    (dict(q_rows=(1 << 29) + 1, q_row=FAR, out_row=FAR, out=(1 << 20) + 10 * FAR), -1),
    (dict(kv_rows=(1 << 29) + 1, k_row=FAR, out=(2 << 20) + 6 * FAR), -1),
    (dict(kv_rows=(1 << 29) + 1, v_row=FAR, out=(4 << 20) + 6 * FAR), -1),
    # rows of out that reach its next head after 2^64 elements
    (dict(q_rows=(1 << 28) + 1, out_row=FAR // 4, out_head=FAR), -3),
])
def test_attention_packed_extents_past_64_bits(rrr, host_ctx, over, code):
    _no_gpu()
    assert packed_call(rrr, host_ctx, over) == code


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [700, 3000, 9001])
def test_rows_told_apart_show_a_lost_and_a_doubled_one(hd, n):
    """The patterns against their tests' widest tolerance (bf16), with the mistake in the formula."""
    w = torch.float64
    k, v = (x[:, 0] for x in told_apart("paired", n, 1, hd, w, "cpu"))
    q = asking("paired", 1, hd, hd, w, "cpu")[0]
    s = q @ k.T
    ref, count = torch.softmax(s, -1) @ v, torch.zeros(n, dtype=w)
    for row in (0, 1, 63, 64, 127, 128, 511, 512, n // 2, n - 2, n - 1):
        for times in (0, 2):
            count.fill_(1)[row] = times
            e = s.exp() * count
            wrong = e / e.sum(-1, keepdim=True) @ v
            assert float(((wrong - ref).abs() / (ref * half_step(torch.bfloat16) * 1.01 + n * 2.0 ** -57)).max()) > 4


Q = 1 << 20


@pytest.mark.parametrize("over,code", [
    # rows of [q | out]; heads of [q | out]; the same where heads are the outer dimension
    (dict(q_row=1024, out_row=1024, out=Q + 2 * 512), FINE),
    (dict(q_row=1024, out_row=1024, out=Q + 2 * 520), -1),
    (dict(q_row=1024, out_row=1024, out=Q + 2 * 504), -1),
    (dict(q_row=1024, q_head=256, out_row=1024, out_head=256, out=Q + 2 * 128), FINE),
    (dict(q_row=1024, q_head=256, out_row=1024, out_head=256, out=Q + 2 * 120), -1),
    (dict(q_row=256, q_head=9 * 256, out_row=256, out_head=9 * 256, out=Q + 2 * 128), FINE),
    (dict(q_row=256, q_head=9 * 256, out_row=256, out_head=9 * 256, out=Q + 2 * 136), -1),
    # out's first row lies beside a later one of q, or across two of them
    (dict(q_row=1024, out_row=1024, out=Q + 2 * (3 * 1024 + 512)), FINE),
    (dict(q_row=1024, out_row=1024, out=Q + 2 * (3 * 1024 + 768)), -1),
    (dict(q_row=1024, out_row=1024, out=Q - 2 * (3 * 1024 - 512)), FINE),
    # one buffer of [q | k | v | out] rows
    (dict(q_row=1536, k_row=1536, v_row=1536, out_row=1536, k=Q + 1024, v=Q + 1536, out=Q + 2048), FINE),
    (dict(q_row=1536, k_row=1536, v_row=1536, out_row=1536, k=Q + 1024, v=Q + 1536, out=Q + 2032), -1),
    # pitches that are multiples of each other, or not; one row, whose pitch is free
    (dict(q_row=2048, out_row=1024, out=Q + 2 * 512), FINE),
    (dict(q_row=1024, out_row=2048, out=Q + 2 * 512), FINE),
    (dict(q_row=1024, out_row=1032, out=Q + 2 * 512), -1),
    (dict(q_rows=1, q_row=1032, out_row=1024, out=Q + 2 * 512), FINE),
    # what has no element overlaps nothing
    (dict(q_rows=0, out=Q), FINE),
    (dict(kv_rows=0, k=(8 << 20) + 256, v=(8 << 20) + 512), FINE),
])
def test_attention_packed_arrays_that_interleave(rrr, host_ctx, over, code):
    _no_gpu()
    assert packed_call(rrr, host_ctx, over) == code, rrr.ffi.last_error(host_ctx)


def test_python_host_runs_on_the_current_stream(rrr, monkeypatch):
    """Without `stream`, the calls go to torch's current stream of the context's GPU, where the
    tensors' other work is; `stream` overrides it. (CPU tensors and a library that notes its calls.)"""
    serving, seen = sys.modules[rrr.qk_norm_rope.__module__], []

    class Library:
        def __getattr__(self, name):
            return lambda *args: seen.append((name, args[-1])) or 0

    class Ctx:
        h, device = None, -1  # CPU tensors' device number

    monkeypatch.setattr(serving.ffi, "lib", Library)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0x5000 + device, raising=False)
    zeros, pos = torch.zeros, torch.zeros(3, dtype=torch.int32)
    q, kv, out = zeros(3, 4, 128).half(), zeros(3, 2, 128).half(), zeros(3, 4, 128).half()
    cache = rrr.KV4Cache(Ctx, zeros(4, 2, 80 * 128, dtype=torch.uint8), zeros(2, 4, dtype=torch.int32), 128)
    desc, cu, n = rrr.ffi.AttnDesc(4, 2, 128, 96, 1e4, 1.0, None, 0, 16), pos, pos[:2]

    def calls(**stream):
        rrr.qk_norm_rope(Ctx, desc, zeros(3, 8, 128), pos, q, kv, **stream)
        rrr.attention_packed(Ctx, q, kv, kv, cu, cu, out, **stream)
        cache.store(kv, kv, cu, n, **stream)
        cache.load(cu, n, kv, **stream)
        cache.attention(q[:2], n, out[:2], zeros(64, dtype=torch.uint8), **stream)

    def number(s):
        return s if isinstance(s, int) else getattr(s, "value", None)

    calls()
    assert [number(s) for _, s in seen] == [0x4fff] * 5, seen
    seen.clear()
    calls(stream=77)
    assert [number(s) for _, s in seen] == [77] * 5


# ------------------------------------------------------------------ GPU
def in_a_new_thread(call):
    """call() in a thread that has made no CUDA call before; its exception here."""
    raised = []

    def run():
        try:
            call()
        except Exception as e:
            raised.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if raised:
        raise raised[0]


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("name", ["qk_norm_rope", "attention_packed", "store", "load", "attention"])
def test_first_call_of_a_thread(rrr, ctx, hd, name):
    """A thread that has made no CUDA call yet (a worker of a server) gives the bits of the main one."""
    nh, nkv, n, t, g = 4, 2, 150, torch.bfloat16, gen(hd)
    q, k, v = (normal(g, n, h, hd, dtype=t) for h in (nh, nkv, nkv))
    cu, lens, cache = ints([0, n]), ints([n]), Cache(rrr, ctx, nkv, hd, [n], 1)
    cache.c.store(k, v, cu, lens)
    desc, ws = rrr.ffi.AttnDesc(nh, nkv, hd, 64, 1e4, 1.0, None, 0, 4096), cache.c.workspace(nh)
    x, pos = normal(g, n, (nh + 2 * nkv) * hd), torch.arange(n, dtype=torch.int32, device="cuda")
    got = []
    for where in (lambda call: call(), in_a_new_thread):
        out = [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
        if name == "store":
            cache.pages.zero_()
        torch.cuda.synchronize()
        where({"qk_norm_rope": lambda: rrr.qk_norm_rope(ctx, desc, x, pos, *out),
               "attention_packed": lambda: rrr.attention_packed(ctx, q, k, v, cu, cu, out[0]),
               "store": lambda: cache.c.store(k, v, cu, lens),
               "load": lambda: cache.c.load(cu, lens, *out[1:]),
               "attention": lambda: cache.c.attention(q[:1], lens, out[0][:1], ws)}[name])
        torch.cuda.synchronize()
        got.append([cache.pages.clone(), *out])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_continued_prompts_of_a_batch(rrr, ctx, hd):
    """New rows of several sequences over their prefixes in the cache: stored, loaded with their
    prefixes, attended as the cache holds them, and with the unrounded rows copied over theirs."""
    nh, nkv, t, g = 6, 2, torch.bfloat16, gen(hd)
    old, new = [90, 0, 200, 64, 1], [40, 17, 0, 65, 300]
    held = [a + b for a, b in zip(old, new)]
    cache = Cache(rrr, ctx, nkv, hd, held, 3)
    k, v = (normal(g, sum(old), nkv, hd, dtype=t) for _ in range(2))
    cache.c.store(k, v, cu_of(old), ints(old))
    prefix = [torch.empty_like(k) for _ in range(2)]
    cache.c.load(cu_of(old), ints(old), *prefix)
    q = normal(g, sum(new), nh, hd, dtype=t)
    rows = [normal(g, sum(new), nkv, hd, dtype=t) for _ in range(2)]
    cu_q, cu_kv, lens = cu_of(new), cu_of(held), ints(held)
    cache.c.store(*rows, cu_q, lens)
    both = [torch.empty(sum(held), nkv, hd, dtype=t, device="cuda") for _ in range(2)]
    cache.c.load(cu_kv, lens, *both)
    ends = np.cumsum(held)
    old_at = torch.tensor([e - h + i for e, h, n in zip(ends, held, old) for i in range(n)], device="cuda")
    new_at = torch.tensor([e - n + i for e, n in zip(ends, new) for i in range(n)], device="cuda")
    for whole, a, b in zip(both, prefix, rows):
        assert torch.equal(whole[old_at], a)
        assert torch.equal(whole[new_at].float().cpu(), torch.from_numpy(np_values(b.float().cpu().numpy())).to(t).float())
    out = torch.empty_like(q)
    rrr.attention_packed(ctx, q, *both, cu_q, cu_kv, out)
    check_packed(out, q, *both, new, held, True, 1 / math.sqrt(hd))
    for whole, b in zip(both, rows):
        whole[new_at] = b
    rrr.attention_packed(ctx, q, *both, cu_q, cu_kv, out)
    check_packed(out, q, *both, new, held, True, 1 / math.sqrt(hd))
    assert ctx.device_error() == 0


@pytest.mark.gpu
def test_calls_follow_the_current_stream(rrr, ctx):
    """Inputs that the current stream is still writing, and a capture of it, without `stream`."""
    nh, nkv, hd, lens, t = 4, 2, 128, [70, 300], torch.bfloat16
    g, rows, cu, n = gen(1), sum(lens), cu_of(lens), ints(lens)
    x, pos = normal(g, rows, nh + 2 * nkv, hd, dtype=t), ints([i for m in lens for i in range(m)])
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, 128, 1e4, 1.0, None, 0, 4096)
    cache = Cache(rrr, ctx, nkv, hd, lens, 1)
    ws = cache.c.workspace(nh)

    def step(qkv, q, k, v, out, kk, token):
        rrr.qk_norm_rope(ctx, desc, qkv, pos, q, k, v)
        rrr.attention_packed(ctx, q, k, v, cu, cu, out)
        cache.c.store(k, v, cu, n)
        cache.c.load(cu, n, kk)
        cache.c.attention(q[:2], n, token, ws)

    def arrays():
        return [torch.zeros_like(x)] + [torch.zeros(r, h, hd, dtype=t, device="cuda")
                                        for r, h in ((rows, nh), (rows, nkv), (rows, nkv), (rows, nh), (rows, nkv), (2, nh))]

    want, late, graphed = arrays(), arrays(), arrays()
    want[0].copy_(x)
    step(*want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # some 10 ms
        late[0].copy_(x)
        step(*late)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, late))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*graphed)
    graphed[0].copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, graphed)) and ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("theta,factors", [(10000.0, False), (500000.0, True), (1.0, False)])
@pytest.mark.parametrize("halves", [False, True])
def test_qk_norm_rope_far_positions(rrr, ctx, theta, factors, halves):
    """Angles of positions up to the last, against 80-bit floats: 2^-24 turns below 2^27 and position *
    2^-51 turns beyond, 2 u for the sine and 3 u for the rotation's own roundings. (The formula's
    frequency is theta's as a 32-bit float; its angle in 80 bits is off by position * 2^-62.)"""
    nh, nkv, hd, rd, g = 2, 1, 128, 96, gen(7)
    at = [0, 1, 2 ** 20 + 7] + [2 ** e + d for e in (24, 26, 27, 28, 30) for d in (-1, 0, 12345)] + [2 ** 31 - 2 - i for i in range(9)]
    x = normal(g, len(at), nh + 2 * nkv, hd)
    f = torch.rand(rd // 2, device="cuda", generator=g) * 3 + 1 if factors else None
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, rd, theta, 1.0, None if f is None else f.data_ptr(), 0 if f is None else f.numel(), 2 ** 31 - 1)
    outs = [torch.empty(len(at), n, hd, device="cuda") for n in (nh, nkv, nkv)]
    rrr.qk_norm_rope(ctx, desc, x.flatten(1), ints(at), *outs, halves=halves)
    wide = np.longdouble
    freq = np.power(wide(np.float32(theta)), -2 * np.arange(rd // 2, dtype=wide) / wide(rd))
    if factors:
        freq = freq / f.cpu().numpy().astype(wide)
    angle = np.array(at, wide)[:, None] * freq
    c, s = (torch.from_numpy(y.astype(np.float64)).cuda()[:, None] for y in (np.cos(angle), np.sin(angle)))
    far = torch.tensor([max(2.0 ** -24, p * 2.0 ** -51) for p in at], device="cuda", dtype=torch.float64)[:, None, None]
    e = torch.arange(rd // 2, device="cuda")
    a, b = (e, e + rd // 2) if halves else (2 * e, 2 * e + 1)
    for got, y in ((outs[0], x[:, :nh]), (outs[1], x[:, nh:nh + nkv])):
        y, want = y.double(), y.double().clone()
        want[..., a], want[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
        bound = torch.zeros_like(y)
        bound[..., a] = bound[..., b] = (y[..., a].abs() + y[..., b].abs()) * (2 * math.pi * far + 5 * U)
        within(got, want, bound)
    assert torch.equal(outs[2], x[:, nh + nkv:]) and ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["rows", "heads"])
def test_attention_packed_rows_of_inputs_and_output(rrr, ctx, order):
    """One buffer of [q | k | v | out] rows, or of heads of such rows: the bits of separate arrays, and
    nothing else written."""
    nh, nkv, hd, lens, t = 4, 2, 128, [100, 257], torch.bfloat16
    rows, heads = sum(lens), 2 * nh + 2 * nkv
    x = normal(gen(5), *((rows, heads, hd) if order == "rows" else (heads, rows, hd)), dtype=t)
    whole = x if order == "rows" else x.transpose(0, 1)
    q, k, v, out = whole.split([nh, nkv, nkv, nh], 1)
    cu, apart, before = cu_of(lens), torch.empty(rows, nh, hd, dtype=t, device="cuda"), x.clone()
    rrr.attention_packed(ctx, *(y.contiguous() for y in (q, k, v)), cu, cu, apart)
    rrr.attention_packed(ctx, q, k, v, cu, cu, out)
    assert torch.equal(out, apart) and ctx.device_error() == 0
    out.copy_((before if order == "rows" else before.transpose(0, 1))[:, -nh:])
    assert torch.equal(x, before)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("held,seqs", [(1100, 40), (2600, 1)])  # items of their own, and shared by clusters
def test_attention_packed_bits_do_not_depend_on_the_rows_behind(rrr, ctx, hd, kind, held, seqs):
    """A tile's last rows are the next sequence's queries, or rows of none: whatever those hold, and
    however their scores grow, the sequence before keeps every bit."""
    nh, nkv, t, lq = 6, 2, DT[kind], 23
    g, rows = gen(hd), lq * seqs + 40
    q, k, v = normal(g, rows, nh, hd, dtype=t), normal(g, held * seqs, nkv, hd, dtype=t), normal(g, held * seqs, nkv, hd, dtype=t)
    # keys that grow, so that larger queries' scores do too
    k *= torch.linspace(0.1, 1.5, held, device="cuda").repeat(seqs)[:, None, None].to(t)
    cu_q, cu_kv = ints([lq * i for i in range(seqs + 1)]), ints([held * i for i in range(seqs + 1)])
    outs = []
    for fill in (0.0, 25.0, math.inf, math.nan):
        x, out = q.clone(), torch.full_like(q, 3.0)
        x[lq * seqs:] = x[lq * seqs:] * fill if math.isfinite(fill) else fill
        for s in range(1, seqs, 2):  # every second sequence's queries
            x[lq * s:lq * (s + 1)] = x[lq * s:lq * (s + 1)] * fill if math.isfinite(fill) else fill
        rrr.attention_packed(ctx, x, k, v, cu_q, cu_kv, out)
        assert bool((out[lq * seqs:] == 3).all())
        outs.append(torch.stack([out[lq * s:lq * (s + 1)] for s in range(0, seqs, 2)]))
    assert bool(torch.isfinite(outs[0]).all())
    assert all(torch.equal(o, outs[0]) for o in outs[1:]) and ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 24, 8), (64, 5, 5), (128, 24, 8), (128, 4, 1), (256, 4, 2), (128, 130, 1), (64, 129, 1)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lq,lk", [
    ([1], [3000]), ([5], [9001]), ([37], [2111]), ([100], [2048]), ([3, 0, 50], [2500, 900, 2600]), ([700], [1600]),
    ([513], [513]), ([127, 1, 0, 130, 64], [127, 1, 0, 130, 64]), ([1500], [1500]), ([21] * 40, [21 + 37 * i for i in range(40)])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("pattern", ["spread", "paired"])
def test_attention_packed_every_row_counts_once(rrr, ctx, hd, nh, nkv, kind, lq, lk, causal, pattern):
    """The weights are 1 (or too small to count) and the sums whole numbers below 2^24, so all that is
    rounded is the inverse, its product and the output: half a step and 2 u, and 2^-57 times the rows
    for the others' weights."""
    t = DT[kind]
    k, v = (torch.cat(x) for x in zip(*(told_apart(pattern, n, nkv, hd, t) for n in lk)))
    q = torch.cat([asking(pattern, n, nh, hd, t) for n in lq])
    out = torch.full_like(q, 3.0)
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), out, causal=causal, scale=1.0)
    a = b = 0
    for n, m in zip(lq, lk):
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril(m - n)
        kk, vv = (x[b:b + m].double().repeat_interleave(nh // nkv, 1).transpose(0, 1) for x in (k, v))
        s = (q[a:a + n].double().transpose(0, 1) @ kk.transpose(1, 2)).masked_fill(~seen, -math.inf)
        ref = (torch.softmax(s, -1).nan_to_num(0) @ vv).transpose(0, 1)
        within(out[a:a + n], ref, ref * (half_step(t) + 2 * U) * 1.01 + m * 2.0 ** -57 + (2.0 ** -25 if t == torch.float16 else 0))
        a, b = a + n, b + m
    assert ctx.device_error() == 0


def check_packed_by_weights(out, q, k, v, scale):
    """One causal sequence within a bound that knows what a row weighs: a weight is off by
    2 ((hd + 16) A + 8) u of itself and half a step of the type (below 2^-14 of the reference f16 has
    no normal numbers: 2^-25, and the sum is at least one), the sums by (rows / 16 + 64) u."""
    t, (n, nh, hd), rows = q.dtype, q.shape, k.shape[0]
    seen = torch.ones(n, rows, dtype=torch.bool, device="cuda").tril(rows - n)
    for h in range(nh):
        x, y, z = q[:, h].double(), k[:, h * k.shape[1] // nh].double(), v[:, h * k.shape[1] // nh].double()
        A = (x.abs() @ y.abs().T * scale * seen).amax(-1, keepdim=True)
        p = torch.softmax((x @ y.T * scale).masked_fill(~seen, -math.inf), -1)
        ref, mag = p @ z, p @ z.abs()
        bound = U * (2 * ((hd + 16) * A + 8) * (mag + ref.abs()) + (rows / 16 + 64) * mag) \
            + half_step(t) * 1.01 * (mag + ref.abs())
        if t == torch.float16:
            bound = bound + 2.0 ** -25 * (1 + seen.sum(-1, keepdim=True) * float(z.abs().max()))
        within(out[:, h], ref, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n,rows", [(300, 1300), (2, 3000)])
@pytest.mark.parametrize("step", [0.0, 1.0, 7.9, 8.1, 40.0, -7.9])
def test_attention_packed_maxima_that_grow_from_block_to_block(rrr, ctx, hd, kind, n, rows, step):
    """The largest score of every 128 rows is `step` above the last ones', in powers of two: a maximum is
    taken over only when it has grown by more than 8, and weights are up to 2^8 until then."""
    t, g = DT[kind], gen(hd + n)
    q, k, v = normal(g, n, 2, hd), 0.1 * normal(g, rows, 1, hd), normal(g, rows, 1, hd, dtype=t)
    q[:, :, 0] = 1
    k[:, 0, 0] = (torch.arange(rows, device="cuda") // 128 - 5) * step * math.log(2) - 3
    k[::128, 0, 0] += 3
    q, k = q.to(t), k.to(t)
    out = torch.empty_like(q)
    rrr.attention_packed(ctx, q, k, v, cu_of([n]), cu_of([rows]), out, scale=1.0)
    check_packed_by_weights(out, q, k, v, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lq,lk,nh,nkv", [([257], [779], 8, 8), ([1121], [1121], 21, 3), ([30], [3000], 8, 8), ([90, 200, 7], [900, 1200, 2000], 5, 5)])
@pytest.mark.parametrize("scale", [0.3, 1.0, 3.0])
def test_attention_packed_warps_that_rescale_at_different_blocks(rrr, ctx, hd, kind, lq, lk, nh, nkv, scale):
    """Scores of a size at which some warps of a tile rescale their sums, and wait for the products so
    far, while others go on to the next block: no product takes weights that are not there yet."""
    t = DT[kind]
    for seed in range(3):
        g = gen(seed + hd)
        q, k, v = (normal(g, sum(n), h, hd, dtype=t) for n, h in ((lq, nh), (lk, nkv), (lk, nkv)))
        out, again, cu_q, cu_kv = torch.empty_like(q), torch.empty_like(q), cu_of(lq), cu_of(lk)
        rrr.attention_packed(ctx, q, k, v, cu_q, cu_kv, out, scale=scale)
        check_packed(out, q, k, v, lq, lk, True, scale)
        for _ in range(5):
            rrr.attention_packed(ctx, q, k, v, cu_q, cu_kv, again, scale=scale)
            assert torch.equal(out, again)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 8, 1), (64, 4, 2), (64, 5, 1), (128, 6, 2), (128, 8, 1), (128, 7, 1), (256, 4, 2), (256, 8, 1), (256, 5, 1)])
@pytest.mark.parametrize("lens", [[1, 17, 64, 0, 65, 128, 1023], [3000, 1, 130, 700], [30001], [150] * 90])
@pytest.mark.parametrize("pattern", ["spread", "paired"])
def test_attention_kv4_every_row_counts_once(rrr, ctx, hd, nh, nkv, lens, pattern):
    """As of prompts; one is held as 15 f16(1/15), and the sums of centred codes and middles may be
    off by (rows that count / 64 + 64) u of 16 d and 8 u more for weights, inverse and product."""
    cache = Cache(rrr, ctx, nkv, hd, lens, 7)
    k, v = (torch.cat(x) for x in zip(*(told_apart(pattern, n, nkv, hd, torch.float32) for n in lens)))
    cache.c.store(k, v, cu_of(lens), ints(lens))
    q = asking(pattern, len(lens), nh, hd, torch.float32)
    out = torch.empty_like(q)
    cache.c.attention(q, ints(lens), out, cache.c.workspace(nh), scale=1.0)
    one, a = 15 * float(np.float16(1 / 15)), 0
    for s, n in enumerate(lens):
        kk, vv = (x[a:a + n].double().repeat_interleave(nh // nkv, 1).transpose(0, 1) * one for x in (k, v))
        ref = (torch.softmax((kk @ q[s].double()[:, :, None])[..., 0], -1)[:, None] @ vv)[:, 0] if n else torch.zeros_like(q[s])
        count = n if pattern == "spread" else n / hd + 1
        within(out[s], ref, torch.full_like(ref, U * (count / 64 + 64 + 8) * 16 / 15 + n * 2.0 ** -57))
        a += n
    assert ctx.device_error() == 0


def check_decode_of_small_values(got, q, k, v, scale):
    """got, q [heads, hd] of one sequence with rows k, v [rows, n_kv, hd] (f32, as they are stored),
    within a bound that knows how little a row weighs: a weight is off by w = 2 (48 A + 8) u of
    itself (48 A of a score and of the maximum, the exponential and the split 8), which moves the
    result by w sum p |v - out|; a product is of d |code - 8| and m + 8 d, each rounded once or its
    sum, in (rows / 64 + 64) u of sum p (8 d + |m + 8 d|); and the rows compared with carry the
    rounding of d code + m."""
    n, n_kv, hd = v.shape
    _, d, m, _ = np_quantise(v.cpu().numpy())
    d, m = (torch.from_numpy(x.astype(np.float64)).cuda().repeat_interleave(32, -1) for x in (d, m))
    held = torch.from_numpy(np_values(v.cpu().numpy())).cuda().double()
    per = q.shape[0] // n_kv
    for h in range(q.shape[0]):
        keys = torch.from_numpy(np_values(k[:, h // per].cpu().numpy())).cuda().double()
        x = q[h].double()
        p = torch.softmax(keys @ x * scale, 0)[:, None]
        A = float((keys.abs() @ x.abs()).max()) * scale
        vv, dd, mm = held[:, h // per], d[:, h // per], m[:, h // per]
        ref = (p * vv).sum(0)
        bound = U * (2 * (48 * A + 8) * (p * (vv - ref).abs()).sum(0)
                     + (n / 64 + 64) * (p * (8 * dd + (mm + 8 * dd).abs())).sum(0) + (p * vv.abs()).sum(0))
        within(got[h], ref, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 4, 2), (64, 7, 1), (128, 6, 2), (128, 5, 1), (128, 8, 1), (256, 3, 1), (256, 7, 1)])
@pytest.mark.parametrize("size", [1e4, 1.0, 1e-2, 1e-4, 1e-6])
def test_attention_kv4_small_values_behind_a_row_that_takes_the_weight(rrr, ctx, hd, nh, nkv, size):
    """A first row of no value draws nearly all weight, as the first token of a text does: what is
    left is a sum of small weights times values of any size, and no less exact."""
    rows, g = [23, 70, 1500], gen(hd + nh)
    cache = Cache(rrr, ctx, nkv, hd, rows, 4)
    k = 0.1 * normal(g, sum(rows), nkv, hd)
    v = size * (normal(g, sum(rows), nkv, hd) + 0.3)
    q = normal(g, 3, nh, hd).sign()
    starts = [0, *np.cumsum(rows)[:-1]]
    for s, a in enumerate(starts):
        v[a] = 0
        k[a] = q[s].unflatten(0, (nkv, -1)).mean(1) * 14 / math.sqrt(hd)
    q = q + 0.05 * normal(g, 3, nh, hd)
    cache.c.store(k, v, cu_of(rows), ints(rows))
    out = torch.empty_like(q)
    cache.c.attention(q, ints(rows), out, cache.c.workspace(nh))
    for s, a in enumerate(starts):
        check_decode_of_small_values(out[s], q[s], k[a:a + rows[s]], v[a:a + rows[s]], 1 / math.sqrt(hd))
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 8, 1), (128, 3, 1), (128, 5, 1), (256, 4, 2)])
@pytest.mark.parametrize("first,last", [(1e-6, 1e4), (1e3, 1e-5), (0.0, 1e-3), (3e-3, 0.0)])
@pytest.mark.parametrize("rising", [True, False])
def test_attention_kv4_values_that_grow_or_shrink_along_a_sequence(rrr, ctx, hd, nh, nkv, first, last, rising):
    """Values from one size to another over the rows (the largest step so far sets the weights' scale),
    under scores that rise or fall along with them."""
    n, g = 5000, gen(hd)
    cache = Cache(rrr, ctx, nkv, hd, [n], 4)
    ramp = torch.linspace(0, 1, n, device="cuda")[:, None, None]
    size = (max(first, 1e-8) ** (1 - ramp)) * (max(last, 1e-8) ** ramp)
    if first == 0.0:
        size = torch.where(ramp < 0.4, 0.0, last)
    if last == 0.0:
        size = torch.where(ramp > 0.7, 0.0, first)
    v = size * normal(g, n, nkv, hd)
    k = 0.1 * normal(g, n, nkv, hd) + 1.5 * (ramp if rising else 1 - ramp) / math.sqrt(hd)
    q = 0.3 * normal(g, 1, nh, hd) + 1
    cache.c.store(k, v, ints([0, n]), ints([n]))
    out = torch.empty_like(q)
    cache.c.attention(q, ints([n]), out, cache.c.workspace(nh))
    check_decode_of_small_values(out[0], q[0], k, v, 1 / math.sqrt(hd))
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh", [(64, 3), (64, 8), (128, 4), (128, 5), (256, 2), (256, 7)])
@pytest.mark.parametrize("size", [1.0, 1e-5])
@pytest.mark.parametrize("top", [2.0 ** 18, 2.0 ** 20, 2.0 ** 23, 2.0 ** 27, 2.0 ** 31, -2.0 ** 20, -2.0 ** 26])
def test_attention_kv4_scores_whose_steps_are_coarse(rrr, ctx, hd, nh, size, top):
    """Scores of 2^18 to 2^31 that rise along the sequence in one head, beside heads of ordinary ones:
    the largest takes all, whatever the others' maxima and the values' sizes do meanwhile."""
    n, g = 3000, gen(hd)
    cache = Cache(rrr, ctx, 1, hd, [n], 4)
    k, v = normal(g, n, 1, hd), size * (normal(g, n, 1, hd) + 0.2)
    k[:, 0, 32:64] = torch.linspace(0.5, 1, n, device="cuda").flip(0 if top < 0 else ())[:, None]
    q = normal(g, 1, nh, hd)
    q[0, 0] = 0
    q[0, 0, 40] = top * math.log(2) * math.sqrt(hd)  # that head's scores, in base 2, are this times k[:, 0, 40]
    cache.c.store(k, v, ints([0, n]), ints([n]))
    out = torch.empty_like(q)
    cache.c.attention(q, ints([n]), out, cache.c.workspace(nh))
    held = torch.from_numpy(np_values(v.cpu().numpy())).cuda()[:, 0]
    keys = torch.from_numpy(np_values(k.cpu().numpy())).cuda()[:, 0, 40]
    best = (keys * top).argmax()
    # every row of a group of 32 equal keys is held exactly to f16, and 2^18 steps of 2^-11 part them
    alike = keys == keys[best]
    want = held[alike].double().mean(0)
    mag = float(held.abs().max())
    within(out[0, 0], want, torch.full_like(want, 64 * U * mag * (1 if int(alike.sum()) == 1 else 8)))
    assert bool(torch.isfinite(out).all()) and ctx.device_error() == 0
    check_decode_of_small_values(out[0, 1:], q[0, 1:], k, v, 1 / math.sqrt(hd))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_kv4_two_threads_with_a_context_each(rrr, ctx, hd, tmp_path):
    """Threads that serve models with other numbers of query heads per KV head, and so kernels with
    other amounts of shared memory, on one GPU: every launch is taken and gives its thread's bits."""
    so = str(tmp_path / "two_threads.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-pthread",
                    os.path.join(ROOT, "tests", "cpp", "two_threads.cpp"), "-o", so], check=True)
    repeat = ctypes.CDLL(so).repeat_attention_kv4
    lens, nkv = [200, 64], 2
    cache, _ = filled(rrr, ctx, nkv, hd, lens, 1)
    n, calls, keep = ints(lens), (KV4Call * 2)(), []
    for i, hpk in enumerate((4, 1)):
        q = normal(gen(hpk), len(lens), nkv * hpk, hd)
        out, first, ws = torch.empty_like(q), torch.empty_like(q), cache.c.workspace(nkv * hpk)
        cache.c.attention(q, n, first, ws)
        own, stream, w = rrr.Context(0), torch.cuda.Stream(), nkv * hpk * hd
        calls[i] = KV4Call(own.h, ctypes.addressof(cache.c.desc), nkv * hpk, rrr.ffi.F32, q.data_ptr(), w, n.data_ptr(),
                           out.data_ptr(), w, ws.data_ptr(), ws.nbytes, stream.cuda_stream)
        keep.append((q, out, first, ws, own, stream))
    torch.cuda.synchronize()
    code = repeat(ctypes.cast(rrr.ffi.lib().rrr_attention_kv4, ctypes.c_void_p), calls, 30000)
    torch.cuda.synchronize()
    assert code == 0, [rrr.ffi.last_error(x[4].h) for x in keep]
    for _, out, first, _, own, _ in keep:
        assert torch.equal(out, first) and own.device_error() == 0
        own.close()
