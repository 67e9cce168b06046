"""A step of speculative decoding over the 4-bit cache: rrr_kv4_append, rrr_attention_tree_kv4,
rrr_verify_drafts.

CPU: refusals through the C ABI and the Python host, and the 64-bit formulas that the GPU tests
hold the kernels to (a walk and a chain by hand).
GPU: every operator against its formula in 64 bits (u = 2^-24 is half a step of f32, h(t) half a
step of the type):

  append  the pages are, bit for bit, those of rrr_kv4_store from K in 64 bits rounded to 32; q without norms
          that of rrr_qk_norm_rope. A value read back is off by half a step d of its group, by the
          roundings of m and d to f16 (h16 |m|, 15 h16 d) and by the rotated value's own error,
          32 u (|a| + |b|) af.
  tree    a score carries (hd + 16) u A of the sums (A = sum |q k| scale) and, of a cached row, h16 A:
          its key is rounded to f16 from its code. A weight 2^x is off by twice that (it and the maximum) and
          8 u. Weights are rounded to f16, those of drafted rows to the type, cached values to f16: h16 +
          h(t) of max |v| each, and 64 u of the sums. (With f16 rows keys and weights lose less: a test of its own.)
  verify  whole numbers: equal.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from test_serving import (CACHE_BAD, DT, FINE, ROWS, U, Cache, _cache, _no_gpu, cu_of, gen, half_step, host_ctx,  # noqa: F401
                          ints, normal, ref_qk, within)

H16 = half_step(torch.float16)


# ------------------------------------------------------------------ formulas
def ancestors(parents):
    """Per row the rows that it sees: itself and its ancestors."""
    seen = []
    for i, p in enumerate(parents):
        seen.append([i] + (seen[p] if 0 <= p < i else []))
    return seen


def ref_tree(q, k, v, kc, vc, parents, scale):
    """One sequence in 64 bits: q [n, nh, hd], k, v [n, nkv, hd], cached kc, vc [len, nkv, hd]: out, and A per row
    and head: over the cached rows and over all."""
    n, nh, hd = q.shape
    rep = nh // k.shape[1]
    out, A, Ac = torch.zeros(n, nh, hd, dtype=torch.float64, device=q.device), *(torch.zeros(n, nh, device=q.device) for _ in range(2))
    for i, seen in enumerate(ancestors(parents)):
        kk, vv = (torch.cat((c, x[seen])).repeat_interleave(rep, 1).transpose(0, 1) for c, x in ((kc, k), (vc, v)))
        s = (kk @ q[i, :, :, None])[..., 0] * scale
        mag = (kk.abs() @ q[i].abs()[:, :, None])[..., 0] * scale
        A[i], Ac[i] = mag.amax(-1), (mag[:, :len(kc)].amax(-1) if len(kc) else 0)
        out[i] = (torch.softmax(s, -1)[:, None] @ vv)[:, 0]
    return out, A, Ac


def ref_verify(logits, tokens, parents, uniforms, temperature, draft=None):
    """One sequence by its definition, numpy in 64 bits: path, next token."""
    def p_of(x):
        x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
        if not (x > -np.inf).any():
            return None
        if temperature == 0:
            return np.where(np.arange(len(x)) == x.argmax(), 1.0, 0.0)
        with np.errstate(all="ignore"):
            e = np.exp((x - x.max()) / np.float64(temperature))
        return e / e.sum()

    def weights_of(x):  # p before its division, so that equal ones are summed without a rounding (750 of 3,000
        x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))  # are a quarter)
        return p_of(x) if temperature == 0 else np.exp((x - x.max()) / np.float64(temperature))

    def drawn(w, u):
        total = np.cumsum(w)
        return int(np.nonzero((total > u * total[-1]) & (w > 0))[0][0])

    u = uniforms.astype(np.float64)
    path, at = [0], 0
    while True:
        p = p_of(logits[at])
        if p is None:
            return path, -1
        if draft is None:
            t = drawn(weights_of(logits[at]), u[at, 1])
            child = [i for i in range(at + 1, len(tokens)) if parents[i] == at and tokens[i] == t]
            if not child:
                return path, t
            at = child[0]
        else:
            if at + 1 == len(tokens):
                return path, drawn(weights_of(logits[at]), u[at, 1])
            x, q = int(tokens[at + 1]), p_of(draft[at + 1])
            fine = 0 <= x < len(p) and (p[x] == 1 if temperature == 0 else u[at + 1, 0] * (q[x] if q is not None else 0) < p[x])
            if not fine:
                rest = np.maximum(p - q, 0) if q is not None and temperature != 0 else p
                return path, drawn(rest if rest.sum() > 0 else weights_of(logits[at]), u[at, 1])
            at += 1
        path.append(at)


def random_tree(rng, n, kind):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return ([-1] + [0] * (n - 1))[:n]
    return ([-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)])[:n]


# ------------------------------------------------------------------ CPU
def test_formulas_by_hand():
    assert ancestors([-1, 0, 0, 1, 3]) == [[0], [1, 0], [2, 0], [3, 1, 0], [4, 3, 1, 0]]
    x = np.log(np.array([[0.1, 0.2, 0.7], [0.5, 0.25, 0.25], [0.2, 0.2, 0.6]], np.float32))
    u = np.array([[0.0, 0.25], [0.5, 0.6], [0.5, 0.1]], np.float32)
    # row 0 draws token 1 (0.1 <= 0.25 < 0.3); its child 2 has it and draws 0
    assert ref_verify(x, [0, 2, 1], [-1, 0, 0], u, 1.0) == ([0, 2], 0)
    # a chain: token 0 at p 0.1 against q 0.5, u = 0.5: refused; the rest is (0, 0, 0.4)
    q = np.log(np.array([[1, 1, 1], [0.5, 0.2, 0.3], [1, 1, 1]], np.float32))
    assert ref_verify(x, [0, 0, 1], None, u, 1.0, q) == ([0], 2)
    assert ref_verify(x, [0, 2, 0], None, u, 0.0, q) == ([0, 1, 2], 2)


@pytest.mark.parametrize("over,code", CACHE_BAD + [
    ({}, FINE), ({"rows": 0, "qkv": None}, FINE), ({"q": None, "qs": 0}, FINE), ({"pos": 64}, FINE), ({"halves": 1}, FINE),
    ({"q": None, "path": 1024, "counts": 2048}, FINE), ({"path": 1024, "counts": 2048}, -1), ({"q": None, "path": 1024}, -1),
    ({"q": None, "counts": 1024}, -1), ({"in_type": 2}, -2), ({"out_type": 14}, -2), ({"qkv": None}, -1), ({"cu": None}, -1),
    ({"lens": None}, -1), ({"rows": -1}, -3), ({"halves": 2}, -1), ({"halves": 1, "rd": 100}, -3), ({"rd": 95}, -3),
    ({"a_nkv": 1}, -3), ({"a_hd": 64}, -3), ({"theta": 0.0}, -1), ({"eps": math.nan}, -1), ({"stride": 1016}, -3),
    ({"stride": 1 << 39}, -3), ({"qs": 504}, -3), ({"qkv": 4100}, -4), ({"q": (1 << 20) + 8}, -4), ({"stride": 1028}, -4),
    ({"pos": 66}, -4), ({"kg": 2}, -4), ({"q": 4096}, -1), ({"q": (1 << 30) + 4096}, -1), ({"qkv": (1 << 30) + 4096}, -1)])
def test_kv4_append_refusals(rrr, host_ctx, over, code):  # noqa: F811
    _no_gpu()
    a = dict(nh=4, a_nkv=2, a_hd=128, rd=96, theta=1e4, seq=16, in_type=0, qkv=4096, stride=1024, rows=2, cu=64, lens=128,
             path=None, counts=None, pos=None, qg=None, kg=None, eps=1e-5, halves=0, out_type=30, q=1 << 20, qs=512)
    a.update({k: v for k, v in over.items() if k in a})
    d = rrr.ffi.AttnDesc(a["nh"], a["a_nkv"], a["a_hd"], a["rd"], a["theta"], 1.0, None, 0, a["seq"])
    f = rrr.ffi.lib().rrr_kv4_append
    args = (ctypes.byref(_cache(rrr, **over)), a["in_type"], a["qkv"], a["stride"], a["rows"], a["cu"], a["lens"], a["path"],
            a["counts"], a["pos"], a["qg"], a["kg"], a["eps"], a["halves"], a["out_type"], a["q"], a["qs"], None)
    assert f(host_ctx, ctypes.byref(d), *args) == code, rrr.ffi.last_error(host_ctx)
    assert f(host_ctx, None, *args) == -1 and f(None, ctypes.byref(d), *args) == -1
    assert f(host_ctx, ctypes.byref(d), None, *args[1:]) in (-1, code)


@pytest.mark.parametrize("over,code", CACHE_BAD + [
    ({}, FINE), ({"rows": 0, "q": None, "k": None, "v": None, "out": None}, FINE), ({"parents": None}, FINE),
    ({"head_major": True}, FINE), ({"type": 0}, -2), ({"heads": 5}, -3), ({"heads": 18}, -3), ({"heads": 0}, -3),
    ({"rows": -1}, -3), ({"rows": (1 << 24) + 1}, -3), ({"q": None}, -1), ({"k": None}, -1), ({"v": None}, -1),
    ({"out": None}, -1), ({"cu": None}, -1), ({"lens": None}, -1), ({"ws": None}, -1), ({"q_row": 120}, -3),
    ({"k_head": 120}, -3), ({"v_row": 1 << 39}, -3), ({"out_row": 0}, -3), ({"scale": -1.0}, -1), ({"scale": math.nan}, -1),
    ({"scale": math.inf}, -1), ({"q": (1 << 20) + 8}, -4), ({"k_row": 260}, -4), ({"parents": 1026}, -4),
    ({"ws": (1 << 24) + 8}, -4), ({"ws_bytes": -1}, -11), ({"out": 1 << 20}, -1), ({"out": (1 << 24) + 128}, -1),
    ({"ws": 1 << 30}, -1), ({"ws": 2 << 20}, -1)])
def test_attention_tree_refusals(rrr, host_ctx, over, code):  # noqa: F811
    _no_gpu()
    a = dict(heads=6, type=30, rows=7, scale=0.0, q=1 << 20, k=2 << 20, v=3 << 20, cu=512, parents=1024, lens=2048, out=4 << 20,
             ws=1 << 24, ws_bytes=0, q_row=768, q_head=128, k_row=256, k_head=128, v_row=256, v_head=128, out_row=768,
             out_head=128)
    a.update({k: v for k, v in over.items() if k in a})
    if "head_major" in over:
        a.update(q_row=128, q_head=7 * 128, out_row=128, out_head=7 * 128)
    L, need = rrr.ffi.lib(), ctypes.c_int64()
    assert L.rrr_tree_workspace(host_ctx, ctypes.byref(_cache(rrr)), 6, 7, ctypes.byref(need)) == 0 and need.value > 0
    assert L.rrr_tree_workspace(host_ctx, ctypes.byref(_cache(rrr)), 6, 7, None) == -1
    d = rrr.ffi.TreeDesc(
        a["type"], a["heads"], a["rows"], a["scale"], a["q_row"], a["q_head"], a["k_row"], a["k_head"], a["v_row"], a["v_head"],
        a["out_row"], a["out_head"])
    args = (a["q"], a["k"], a["v"], a["cu"], a["parents"], a["lens"], a["out"], a["ws"], need.value + a["ws_bytes"], None)
    c = ctypes.byref(_cache(rrr, **over))
    assert L.rrr_attention_tree_kv4(host_ctx, c, ctypes.byref(d), *args) == code, rrr.ffi.last_error(host_ctx)
    assert L.rrr_attention_tree_kv4(host_ctx, c, None, *args) == -1
    assert L.rrr_attention_tree_kv4(None, c, ctypes.byref(d), *args) == -1


@pytest.mark.parametrize("over,code", [
    ({}, FINE), ({"draft": 8 << 20}, FINE), ({"parents": None}, FINE), ({"temp": None}, FINE), ({"n_seqs": 0}, FINE),
    ({"rows": 0, "logits": None, "tokens": None, "u": None, "path": None}, FINE), ({"logits": (1 << 20) + 4}, FINE),
    ({"type": 12}, -2), ({"rows": -1}, -3), ({"vocab": 0}, -3), ({"n_seqs": -1}, -3), ({"n_seqs": 65536}, -3),
    ({"rows": 1 << 24, "vocab": 1 << 28, "ls": 1 << 28}, -3), ({"ls": 999}, -3), ({"ls": 1 << 39}, -3),
    ({"draft": 8 << 20, "parents": 1024}, -1), ({"draft": 8 << 20, "ds": 999}, -3), ({"logits": None}, -1),
    ({"tokens": None}, -1), ({"u": None}, -1), ({"path": None}, -1), ({"cu": None}, -1), ({"counts": None}, -1),
    ({"next": None}, -1), ({"ws": None}, -1), ({"logits": (1 << 20) + 2}, -4), ({"u": 8194}, -4), ({"ws": (1 << 24) + 8}, -4),
    ({"ws_bytes": -1}, -11), ({"path": 4096}, -1), ({"counts": (1 << 20) + 64}, -1), ({"next": 1 << 24}, -1),
    ({"counts": 20480, "next": 20484}, -1)])
def test_verify_drafts_refusals(rrr, host_ctx, over, code):  # noqa: F811
    _no_gpu()
    a = dict(type=0, logits=1 << 20, ls=1000, draft=None, ds=1000, rows=7, vocab=1000, n_seqs=2, cu=512, tokens=4096,
             parents=1024 if "draft" not in over else None, u=8192, temp=12288, path=16384, counts=20480, next=24576,
             ws=1 << 24, ws_bytes=0)
    a.update(over)
    L, need = rrr.ffi.lib(), ctypes.c_int64()
    assert L.rrr_verify_workspace(host_ctx, 7, 1000, 2, 1, None) == -1
    assert L.rrr_verify_workspace(None, 7, 1000, 2, 1, ctypes.byref(need)) == -1
    assert L.rrr_verify_workspace(host_ctx, 7, 1000, 2, a["draft"] is not None, ctypes.byref(need)) == 0
    assert L.rrr_verify_drafts(
        host_ctx, a["type"], a["logits"], a["ls"], a["draft"], a["ds"], a["rows"], a["vocab"], a["n_seqs"], a["cu"], a["tokens"],
        a["parents"], a["u"], a["temp"], a["path"], a["counts"], a["next"], a["ws"], need.value + a["ws_bytes"],
        None) == code, rrr.ffi.last_error(host_ctx)


def test_python_host_refuses_what_the_kernels_cannot_take(rrr):
    class Ctx:  # refused before the library is asked
        h, device = None, 0
    E, z = rrr.RRRError, torch.zeros
    i3 = z(3, dtype=torch.int32)
    with pytest.raises(E, match="cuda:0"):
        rrr.verify_drafts(Ctx, z(3, 9), i3, i3, z(3, 2), i3, i3, i3, i3)
    with pytest.raises(E, match="contiguous"):
        rrr.verify_drafts(Ctx, z(3, 18)[:, ::2], i3, i3, z(3, 2), i3, i3, i3, i3)
    c = object.__new__(rrr.KV4Cache)
    c.ctx, c.n_kv_heads, c.head_dim, c.n_seqs = Ctx, 2, 128, 2
    with pytest.raises(E, match="the cache holds"):
        c.append(rrr.ffi.AttnDesc(4, 1, 128, 96, 1e4, 1.0, None, 0, 16), z(3, 6 * 128), i3, i3)
    with pytest.raises(E, match="are needed"):
        c.append(rrr.ffi.AttnDesc(4, 2, 128, 96, 1e4, 1.0, None, 0, 16), z(3, 6 * 128), i3, i3)
    with pytest.raises(E, match="are needed"):
        c.attention_tree(z(3, 4, 64), z(3, 2, 128), z(3, 2, 128), i3, i3, i3, z(3, 4, 64), i3)
    with pytest.raises(E, match="one type"):
        c.attention_tree(z(3, 4, 128).half(), z(3, 2, 128), z(3, 2, 128), i3, i3, i3, z(3, 4, 128).half(), i3)


# ------------------------------------------------------------------ append
def append_inputs(rrr, g, rows, nh, nkv, hd, rd, kind, top=1 << 20):
    wide = torch.empty(rows, (nh + 2 * nkv) * hd + 24, dtype=DT[kind], device="cuda")  # rows with a gap
    qkv = wide[:, 8:8 + (nh + 2 * nkv) * hd]
    qkv.copy_(normal(g, rows, (nh + 2 * nkv) * hd) * torch.exp(normal(g, rows, 1)))
    factors = torch.rand(max(rd // 2 - 3, 1), device="cuda", generator=g) + 0.75 if rd > 8 else None
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, rd, 10000.0, 1.25, None if factors is None else factors.data_ptr(),
                            0 if factors is None else factors.numel(), top)
    return qkv, factors, desc


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv,rd,halves", [
    (128, 24, 8, 96, False), (128, 24, 8, 96, True), (64, 3, 3, 64, True), (64, 8, 1, 6, False), (64, 4, 2, 36, True),
    (256, 8, 2, 128, False), (256, 5, 5, 112, True), (128, 1, 1, 0, False), (128, 2, 1, 24, True)])
@pytest.mark.parametrize("kinds", [("f32", "bf16"), ("bf16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("new,held", [([1], [1]), ([5, 0, 130, 1], [70, 64, 130, 65]), ([64, 63, 7], [64, 191, 13])])
def test_kv4_append(rrr, ctx, hd, nh, nkv, rd, halves, kinds, new, held):
    """q without norms: the bits of rrr_qk_norm_rope (f32). The pages: the bits of rrr_kv4_store with K normed and rotated in 64
    bits and rounded to 32. q with norms: within its rounding and 32 bits' errors. What is read back: within half a step."""
    g, rows, cu = gen(sum(held) + hd), sum(new), cu_of(new)
    qkv, factors, desc = append_inputs(rrr, g, rows, nh, nkv, hd, rd, kinds[0])
    pos = ints([h - n + i for n, h in zip(new, held) for i in range(n)])
    lens = ints(held)
    want, got = (Cache(rrr, ctx, nkv, hd, held, 3) for _ in range(2))
    kv = [torch.empty(rows, nkv, hd, device="cuda") for _ in range(2)]
    q = [torch.full((rows, nh, hd), 7.0, dtype=DT[kinds[1]], device="cuda") for _ in range(2)]
    q32 = torch.empty(rows, nh, hd, device="cuda")

    def store(at, gammas=(None, None)):
        refs, mags = ref_qk(qkv, at, nh, nkv, hd, rd, 10000.0, 1.25, factors, gammas, float(np.float32(1e-5)), halves)
        want.c.store(refs[1].float().contiguous(), refs[2].float().contiguous(), cu, lens)
        return refs, mags
    rrr.qk_norm_rope(ctx, desc, qkv, pos, q32, kv[0], kv[1], halves=halves)
    store(pos)
    got.c.append(desc, qkv, cu, lens, q[0], halves=halves)
    assert torch.equal(got.pages, want.pages)
    assert torch.equal(q[0], q32.to(DT[kinds[1]]))
    # the rows' own positions, and without q
    far = (pos.long() * 37 + 11).int()
    store(far)
    got.c.append(desc, qkv, cu, lens, positions=far, halves=halves)
    assert torch.equal(got.pages, want.pages)
    # norms
    gammas = [torch.rand(hd, device="cuda", generator=g) + 0.5 for _ in range(2)]
    got.c.append(desc, qkv, cu, lens, q[1], q_gamma=gammas[0], k_gamma=gammas[1], halves=halves)
    refs, mags = store(pos, gammas)
    assert torch.equal(got.pages, want.pages)
    out = DT[kinds[1]]
    rounding = 0.0 if out == torch.float32 else half_step(out)
    within(q[1], refs[0], refs[0].abs() * rounding * 1.01 + 32 * U * mags[0] + (2.0 ** -25 if out == torch.float16 else 1e-30))
    back = [torch.empty(rows, nkv, hd, device="cuda") for _ in range(2)]
    got.c.load(cu, lens, *back)
    for x, ref, mag in zip(back, refs[1:], mags[1:]):
        grp = ref.unflatten(-1, (-1, 32))
        low, high = grp.amin(-1, keepdim=True), grp.amax(-1, keepdim=True)
        err = 64 * U * mag.unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
        d = (high - low) / 15
        bound = (0.5 * d * (1 + H16) + low.abs() * H16 + 15 * H16 * d + 2 * err + 2.0 ** -24).expand(grp.shape).flatten(-2)
        within(x, ref, bound)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(128, 6, 2), (64, 8, 8), (256, 2, 1)])
def test_kv4_append_of_accepted_rows(rrr, ctx, hd, nh, nkv):
    """path and counts: the chosen rows alone, as if they were packed by themselves; nothing else changes."""
    g, rng = gen(hd), np.random.default_rng(hd)
    new, before = [16, 1, 0, 9, 128, 3], [60, 0, 5, 62, 1, 200]
    picks = [sorted(rng.choice(range(1, n), min(n - 1, 5), replace=False).tolist()) if n > 1 else [] for n in new]
    paths = [[0] + p if n else [] for p, n in zip(picks, new)]
    paths[5] = []  # nothing accepted
    taken = [len(p) for p in paths]
    held = [a + b for a, b in zip(taken, before)]
    cu, flat = np.cumsum([0] + new), []
    qkv, _, desc = append_inputs(rrr, g, sum(new), nh, nkv, hd, 64, "bf16")
    path = ints([x for p, n in zip(paths, new) for x in p + [-7] * (n - len(p))])
    for s, p in enumerate(paths):
        flat += [int(cu[s]) + i for i in p]
    want, got = (Cache(rrr, ctx, nkv, hd, [h + 9 for h in held], 3) for _ in range(2))
    want.c.append(desc, qkv[flat].contiguous(), cu_of(taken), ints(held))
    got.c.append(desc, qkv, cu_of(new), ints(held), path=path, counts=ints(taken))
    assert torch.equal(got.pages, want.pages)
    assert ctx.device_error() == 0


@pytest.mark.gpu
def test_kv4_append_leaves_out_what_does_not_exist(rrr, ctx):
    """Bad paths, counts, positions and pages are recorded, and only their rows are missing."""
    nh, nkv, hd, new = 4, 2, 128, [4, 3, 2]
    g = gen(5)
    qkv, _, desc = append_inputs(rrr, g, 9, nh, nkv, hd, 96, "f32", top=50)
    cu, held = cu_of(new), [70, 3, 2]
    full = Cache(rrr, ctx, nkv, hd, held, 3)
    full.c.append(desc, qkv, cu, ints(held))  # positions 66.. of sequence 0 are past max_seq = 50
    assert ctx.device_error() == 6
    blank = Cache(rrr, ctx, nkv, hd, held, 3)
    pages = set(full.table[0].tolist())
    assert all(torch.equal(full.pages[i], blank.pages[i]) for i in pages)
    assert not torch.equal(full.pages, blank.pages)

    def one(path, counts, lens=held, table=None):
        c = Cache(rrr, ctx, nkv, hd, held, 3)
        if table is not None:
            c.c.page_table.copy_(torch.from_numpy(table))
        c.c.append(desc, qkv, cu, ints(lens), path=ints(path), counts=ints(counts), positions=ints([1] * 9))
        return c, ctx.device_error()
    fine, code = one([0, 1, 2, 3, 0, 1, 2, 0, 1], [4, 3, 2])
    assert code == 0
    got, code = one([0, 9, -1, 3, 0, 1, 2, 0, 1], [4, 3, 2])  # two rows that the sequence does not have
    assert code == 6
    out = [torch.empty(9, nkv, hd, device="cuda") for _ in range(4)]
    got.c.load(cu, ints(held), *out[:2])
    fine.c.load(cu, ints(held), *out[2:])
    for x, y in ((out[0], out[2]), (out[1], out[3])):
        same = (x == y).flatten(1).all(1).tolist()
        assert [i for i in range(9) if not same[i]] == [1, 2]
    got, code = one([0, 1, 2, 3, 0, 1, 2, 0, 1], [5, 3, -1])  # counts that no sequence has
    assert code == 6 and all(torch.equal(got.pages[i], blank.pages[i]) for s in (0, 2) for i in got.table[s].tolist())
    got, code = one([0, 1, 2, 3, 0, 1, 2, 0, 1], [4, 3, 2], lens=[70, 2, 200])  # more rows than there are places
    assert code == 6
    table = fine.table.copy()
    table[1, 0] = 1 << 20
    got, code = one([0, 1, 2, 3, 0, 1, 2, 0, 1], [4, 3, 2], table=table)
    assert code == 6 and torch.equal(got.pages[fine.table[0]], fine.pages[fine.table[0]])


# ------------------------------------------------------------------ tree
def check_tree(rrr, ctx, hd, nh, nkv, kind, lens, trees, seed=0, size=1.0, scale=0.0, cache=None):
    g, t = gen(seed + hd), DT[kind]
    cache = cache or Cache(rrr, ctx, nkv, hd, [max(n, 1) for n in lens], 3)
    cu, total = cu_of(lens), sum(lens)
    if total:
        strong = torch.exp(0.5 * normal(g, nkv, hd))
        cache.c.store(normal(g, total, nkv, hd) * strong, size * normal(g, total, nkv, hd), cu, ints(lens))
    rows = sum(len(x) for x in trees)
    q, k, v = (normal(g, rows, n, hd, dtype=t) for n in (nh, nkv, nkv))
    v *= size
    out = torch.full((rows + 2, nh, hd), 7.0, dtype=t, device="cuda")
    ws = cache.c.tree_workspace(nh, rows)
    parents = ints([p for x in trees for p in x])
    cache.c.attention_tree(q, k, v, cu_of([len(x) for x in trees]), parents, ints(lens), out[:rows], ws, scale=scale)
    kc, vc = (torch.empty(total, nkv, hd, device="cuda") for _ in range(2))
    if total:
        cache.c.load(cu, ints(lens), kc, vc)
    compare_tree(out, q, k, v, kc, vc, lens, trees, kind, scale or hd ** -0.5)
    assert torch.equal(out[rows:], torch.full_like(out[rows:], 7.0))
    assert ctx.device_error() == 0


def compare_tree(out, q, k, v, kc, vc, lens, trees, kind, scale):
    hd, h = q.shape[2], half_step(DT[kind])
    a = b = 0
    for n, tree in zip(lens, trees):
        r = slice(b, b + len(tree))
        ref, A, Ac = ref_tree(q[r].double(), k[r].double(), v[r].double(), kc[a:a + n].double(), vc[a:a + n].double(), tree, scale)
        top = max(float(v[r].abs().max()) if len(tree) else 0.0, float(vc[a:a + n].abs().max()) if n else 0.0)
        s = (hd + 16) * U * A + H16 * Ac
        bound = (2 * torch.expm1(2 * s) + H16 + h + (n / 64 + 64) * U) * top
        within(out[r], ref, ref.abs() * h * 1.01 + bound[..., None] + 2.0 ** -25)
        a, b = a + n, b + len(tree)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,per", [(64, 8), (128, 3), (128, 8), (256, 2)])
def test_attention_tree_of_f16_rows(rrr, ctx, hd, per):
    """With f16 rows only the values and the result are rounded to f16: independent errors of one distribution, in the mean
    square sqrt(2) times those of the result's rounding alone (about 2 where keys and weights were rounded too)."""
    rng, g, lens = np.random.default_rng(hd), gen(hd + per), [3000, 1500, 40]
    trees = [random_tree(rng, n, "tree") for n in (16, 8, 5)]
    cache, cu = Cache(rrr, ctx, 1, hd, lens, 3), cu_of(lens)
    cache.c.store(normal(g, sum(lens), 1, hd) * torch.exp(0.5 * normal(g, 1, hd)), normal(g, sum(lens), 1, hd), cu, ints(lens))
    q, k, v = (normal(g, 29, n, hd, dtype=torch.float16) for n in (per, 1, 1))
    out = torch.empty_like(q)
    cache.c.attention_tree(q, k, v, cu_of([16, 8, 5]), ints([p for x in trees for p in x]), ints(lens), out, cache.c.tree_workspace(per, 29))
    kc, vc = (torch.empty(sum(lens), 1, hd, device="cuda") for _ in range(2))
    cache.c.load(cu, ints(lens), kc, vc)
    a = b = 0
    for n, tree in zip(lens, trees):
        r = slice(b, b + len(tree))
        ref, _, _ = ref_tree(q[r].double(), k[r].double(), v[r].double(), kc[a:a + n].double(), vc[a:a + n].double(), tree, hd ** -0.5)
        assert (out[r].double() - ref).norm() < 1.5 * (ref.half().double() - ref).norm()
        a, b = a + n, b + len(tree)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(128, 24, 8), (64, 8, 1), (64, 5, 5), (256, 6, 2), (256, 8, 1), (128, 8, 8), (128, 7, 1)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lens,nodes,shape", [
    ([1], [1], "chain"), ([17, 0, 64, 65, 1, 127, 128, 129], [3, 5, 0, 1, 16, 17, 2, 31], "tree"), ([1023], [6], "chain"),
    ([700, 3, 0, 300], [128, 64, 100, 33], "tree"), ([3000, 1, 130], [8, 60, 8], "star")])
def test_attention_tree(rrr, ctx, hd, nh, nkv, kind, lens, nodes, shape):
    rng = np.random.default_rng(len(lens))
    check_tree(rrr, ctx, hd, nh, nkv, kind, lens, [random_tree(rng, n, shape) for n in nodes])


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(128, 6, 2), (64, 8, 1), (256, 2, 2)])
def test_attention_tree_of_many_sequences_and_of_a_long_one(rrr, ctx, hd, nh, nkv):
    rng = np.random.default_rng(hd)
    lens = rng.integers(0, 300, 150).tolist()
    check_tree(rrr, ctx, hd, nh, nkv, "bf16", lens, [random_tree(rng, int(n), "tree") for n in rng.integers(0, 20, 150)])
    check_tree(rrr, ctx, hd, nh, nkv, "f16", [30001, 2], [random_tree(rng, 24, "tree"), [-1, 0]])


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_tree_strides_and_chains(rrr, ctx, hd):
    """Parts of QKV rows, heads of rows; parents None is a chain."""
    nh, nkv, lens, nodes = 6, 2, [100, 7], [9, 4]
    g, rows = gen(hd), 13
    cache = Cache(rrr, ctx, nkv, hd, lens, 3)
    cache.c.store(normal(g, 107, nkv, hd), normal(g, 107, nkv, hd), cu_of(lens), ints(lens))
    qkv = normal(g, rows, nh + 2 * nkv, hd, dtype=torch.bfloat16)
    q, k, v = qkv[:, :nh], qkv[:, nh:nh + nkv], qkv[:, nh + nkv:]
    cu, ws = cu_of(nodes), cache.c.tree_workspace(nh, rows)
    parents = ints([i - 1 for n in nodes for i in range(n)])
    want = cache.c.attention_tree(q, k, v, cu, parents, ints(lens), torch.empty(rows, nh, hd, device="cuda", dtype=torch.bfloat16), ws)
    got = torch.empty(nh, rows, hd, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    head_major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    cache.c.attention_tree(*head_major, cu, None, ints(lens), got, ws)
    assert torch.equal(got, want)
    kc, vc = (torch.empty(107, nkv, hd, device="cuda") for _ in range(2))
    cache.c.load(cu_of(lens), ints(lens), kc, vc)
    compare_tree(want, q, k, v, kc, vc, lens, [[i - 1 for i in range(n)] for n in nodes], "bf16", hd ** -0.5)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 8, 1), (128, 6, 2), (256, 3, 1)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_attention_tree_values_that_are_not_finite(rrr, ctx, hd, nh, nkv, kind):
    """Drafted rows that a row does not see may hold anything; who sees them gets what the formula says."""
    t, g, parents = DT[kind], gen(hd), [-1, 0, 0, 1, 2, 3, 4]
    lens, rows = [90], len(parents)
    cache = Cache(rrr, ctx, nkv, hd, lens, 3)
    cache.c.store(normal(g, 90, nkv, hd), normal(g, 90, nkv, hd), cu_of(lens), ints(lens))
    kc, vc = (torch.empty(90, nkv, hd, device="cuda") for _ in range(2))
    cache.c.load(cu_of(lens), ints(lens), kc, vc)
    for which, value in (("v", math.inf), ("v", math.nan), ("k", math.nan), ("k", math.inf), ("v", -math.inf)):
        q, k, v = (normal(g, rows, n, hd, dtype=t) for n in (nh, nkv, nkv))
        q = q.abs()  # an infinite key gives an infinite score of its own sign
        (v if which == "v" else k)[3, :, hd // 2] = value  # of row 3: rows 3 and 5 see it
        out = torch.empty(rows, nh, hd, dtype=t, device="cuda")
        cache.c.attention_tree(q, k, v, cu_of([rows]), ints(parents), ints(lens), out, cache.c.tree_workspace(nh, rows))
        ref, _, _ = ref_tree(q.double(), k.double(), v.double(), kc.double(), vc.double(), parents, hd ** -0.5)
        fine = torch.isfinite(ref)
        assert torch.equal(fine, torch.isfinite(out)), (which, value)
        assert torch.equal(torch.isnan(ref), torch.isnan(out)), (which, value)
        clean = [0, 1, 2, 4, 6]
        kk, vv = k.clone(), v.clone()
        kk[3] = vv[3] = 0
        compare_tree(out[clean], q[clean], kk[clean], vv[clean], kc, vc, lens, [[-1, 0, 0, 2, 3]], kind, hd ** -0.5)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_tree_rows_that_hold_nothing_never_count(rrr, ctx, hd):
    """Places behind a sequence's rows and pages of nobody hold NaN; the last page is partly filled."""
    rng = np.random.default_rng(1)
    for fill in (0xFF, 0x7E):
        cache = Cache(rrr, ctx, 2, hd, [64, 200, 1, 129], 3, fill=fill)
        check_tree(rrr, ctx, hd, 6, 2, "bf16", [33, 130, 0, 129], [random_tree(rng, n, "tree") for n in (5, 3, 9, 1)], cache=cache)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(64, 8, 1), (128, 6, 2), (256, 3, 1)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("size", [1e4, 1e-2, 1e-4])
def test_attention_tree_small_and_large_values(rrr, ctx, hd, nh, nkv, kind, size):
    check_tree(rrr, ctx, hd, nh, nkv, kind, [300, 20], [[-1, 0, 0, 1], [-1, 0]], size=size)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_tree_groups_beyond_f16(rrr, ctx, hd):
    """A group from -60,000 to 200,000: values that f16 does not hold."""
    g, nh, nkv, lens = gen(hd), 3, 1, [70]
    cache = Cache(rrr, ctx, nkv, hd, lens, 3)
    k, v = normal(g, 70, nkv, hd) * 1e-4, normal(g, 70, nkv, hd)
    k[5, :, 3], k[5, :, 4] = -6e4, 2e5
    v[9, :, 3], v[9, :, 4] = -6e4, 2e5
    cache.c.store(k, v, cu_of(lens), ints(lens))
    cache.c.load(cu_of(lens), ints(lens), k, v)
    q, kd, vd = (normal(g, 2, n, hd, dtype=torch.bfloat16) * s for n, s in ((nh, 1e-4), (nkv, 1.0), (nkv, 1.0)))
    out = torch.empty(2, nh, hd, dtype=torch.bfloat16, device="cuda")
    cache.c.attention_tree(q, kd, vd, cu_of([2]), None, ints(lens), out, cache.c.tree_workspace(nh, 2))
    compare_tree(out, q, kd, vd, k, v, lens, [[-1, 0]], "bf16", hd ** -0.5)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("step", [0.0, 1.0, 4.0, 7.9, 40.0, -7.9])
def test_attention_tree_maxima_that_grow_from_block_to_block(rrr, ctx, hd, step):
    """Keys whose scores grow with the row: the largest weight moves on in every block."""
    g, nh, nkv, n = gen(hd), 4, 2, 900
    cache = Cache(rrr, ctx, nkv, hd, [n], 3)
    one = torch.zeros(hd, device="cuda")
    one[::32] = 1.0  # one value per group: the others stay small
    grow = (torch.arange(n, device="cuda") // 64).float() * step / 16
    k = 0.05 * normal(g, n, nkv, hd) + (grow[:, None, None] * one)
    v = normal(g, n, nkv, hd)
    cache.c.store(k, v, cu_of([n]), ints([n]))
    cache.c.load(cu_of([n]), ints([n]), k, v)
    q = (0.1 * normal(g, 5, nh, hd) + 16 * one / (hd / 32)).to(torch.bfloat16)
    kd, vd = (normal(g, 5, nkv, hd, dtype=torch.bfloat16) for _ in range(2))
    out = torch.empty(5, nh, hd, dtype=torch.bfloat16, device="cuda")
    tree = [-1, 0, 0, 2, 1]
    cache.c.attention_tree(q, kd, vd, cu_of([5]), ints(tree), ints([n]), out, cache.c.tree_workspace(nh, 5), scale=1.0)
    compare_tree(out, q, kd, vd, k, v, [n], [tree], "bf16", 1.0)
    assert ctx.device_error() == 0


@pytest.mark.gpu
def test_attention_tree_bad_arguments_on_the_device(rrr, ctx):
    """Trees of more than 128 rows stay as they were; parents, lengths and pages out of range are recorded."""
    g, hd, nh, nkv = gen(2), 128, 6, 2
    lens, nodes = [40, 70], [129, 3]
    cache = Cache(rrr, ctx, nkv, hd, lens, 3)
    cache.c.store(normal(g, 110, nkv, hd), normal(g, 110, nkv, hd), cu_of(lens), ints(lens))
    kc, vc = (torch.empty(110, nkv, hd, device="cuda") for _ in range(2))
    cache.c.load(cu_of(lens), ints(lens), kc, vc)
    q, k, v = (normal(g, 132, n, hd, dtype=torch.bfloat16) for n in (nh, nkv, nkv))
    ws = cache.c.tree_workspace(nh, 132)

    def run(nodes, parents, lens, table=None):
        out = torch.full((132, nh, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        if table is not None:
            cache.c.page_table.copy_(torch.from_numpy(table))
        cache.c.attention_tree(q, k, v, cu_of(nodes), parents, ints(lens), out, ws)
        return out, ctx.device_error()
    out, code = run(nodes, None, lens)
    assert code == 6 and bool((out[:129] == 7).all())
    compare_tree(out[129:], q[129:], k[129:], v[129:], kc[40:], vc[40:], [70], [[-1, 0, 1]], "bf16", hd ** -0.5)
    for bad in (2, 5, -2, 1 << 30):
        out, code = run([3, 3], ints([-1, 0, bad, -1, 0, 0] + [0] * 126), lens)
        assert code == 6
        compare_tree(out, q, k, v, kc, vc, lens, [[-1, 0, -1], [-1, 0, 0]], "bf16", hd ** -0.5)
        assert bool((out[6:] == 7).all())
    for bad in (-1, 129, 1 << 30):
        out, code = run([3, 3], None, [bad, 70])
        assert code == 6
        compare_tree(out, q, k, v, kc[40:], vc[40:], [0, 70], [[-1, 0, 1]] * 2, "bf16", hd ** -0.5)
    table = cache.table.copy()
    table[1, 0] = -3
    out, code = run([3, 3], None, lens, table)
    assert code == 6
    compare_tree(out, q, k, v, torch.cat((kc[:40], kc[104:])), torch.cat((vc[:40], vc[104:])), [40, 6], [[-1, 0, 1]] * 2, "bf16", hd ** -0.5)


# ------------------------------------------------------------------ verify
def verify_inputs(g, rng, vocab, trees, kind, draft):
    rows = sum(len(t) for t in trees)
    logits = 2 * normal(g, rows, vocab)
    logits.scatter_add_(1, torch.randint(0, vocab, (rows, 5), device="cuda", generator=g), 6 + normal(g, rows, 5))
    logits = logits.to(DT[kind])
    cu = np.cumsum([0] + [len(t) for t in trees])
    up = [int(cu[n]) + max(p, 0) for n, t in enumerate(trees) for p in t]
    guess = (logits[up].float() + 0.5 * normal(g, rows, vocab)).to(DT[kind])
    noise = -torch.rand(rows, vocab, device="cuda", generator=g).clamp_min(1e-20).log().neg().log()
    tokens = (guess.float() + noise).argmax(-1).int()
    return logits, guess if draft else None, tokens, torch.rand(rows, 2, device="cuda", generator=g)


def check_verify(rrr, ctx, logits, draft, tokens, u, trees, temperature, chains=False):
    rows, n = sum(len(t) for t in trees), len(trees)
    path = torch.full((rows + 3,), 77, dtype=torch.int32, device="cuda")
    counts, following = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    ws = rrr.verify_workspace(ctx, rows, logits.shape[1], n, draft is not None)
    ws.fill_(0xFF)
    parents = None if draft is not None or chains else ints([p for t in trees for p in t])
    heat = None if temperature is None else torch.tensor(temperature, dtype=torch.float32, device="cuda")
    rrr.verify_drafts(ctx, logits, tokens, cu_of([len(t) for t in trees]), u, path[:rows], counts, following, ws, draft=draft,
                      parents=parents, temperature=heat)
    x, y, t, uu = (None if z is None else z.float().cpu().numpy() for z in (logits, draft, tokens.double(), u))
    at, want = 0, ([], [], [])
    for s, tree in enumerate(trees):
        r = slice(at, at + len(tree))
        p, token = ([], -1) if not tree else ref_verify(
            x[r], tokens[r].tolist(), tree, uu[r], 1.0 if heat is None else float(heat[s]), None if y is None else y[r])
        want[0].extend(p + [-1] * (len(tree) - len(p)))
        want[1].append(len(p))
        want[2].append(token)
        at += len(tree)
    assert path.tolist() == want[0] + [77] * 3
    assert counts.tolist() == want[1]
    assert following.tolist() == want[2]
    assert ctx.device_error() == 0
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 1023, 4097, 32064, 200064])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mode", ["tree", "chain", "draft"])
def test_verify_drafts(rrr, ctx, vocab, kind, mode):
    g, rng = gen(vocab), np.random.default_rng(vocab)
    nodes = [7, 1, 0, 12, 3] if vocab > 5000 else [7, 1, 0, 12, 3, 40, 5, 8, 2, 9]
    trees = [random_tree(rng, n, "tree" if mode == "tree" else "chain") for n in nodes]
    logits, draft, tokens, u = verify_inputs(g, rng, vocab, trees, kind, mode == "draft")
    heat = [0.0 if i % 4 == 3 else 0.5 + 0.2 * i for i in range(len(trees))]
    want = check_verify(rrr, ctx, logits, draft, tokens, u, trees, heat, chains=mode == "chain")
    assert vocab < 3 or 0 < sum(want[1]) < sum(nodes)  # some stand and some do not
    check_verify(rrr, ctx, logits, draft, tokens, u, trees, None, chains=mode == "chain")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("draft", [False, True])
def test_verify_drafts_rows_at_any_place(rrr, ctx, kind, draft):
    """Rows that begin at any element of 16 bytes, rows with a gap, and rows past the sequences' end."""
    g, rng = gen(3), np.random.default_rng(3)
    trees = [random_tree(rng, n, "chain") for n in (3, 6, 2)]
    for vocab, pitch, off in ((1027, 1027, 1), (2049, 2053, 3), (5000, 5001, 5), (4096, 4096, 0)):
        logits, y, tokens, u = verify_inputs(g, rng, vocab, trees, kind, draft)

        def placed(x, off):
            if x is None:
                return None
            room = torch.full((11 * pitch + 16,), math.nan, dtype=x.dtype, device="cuda")
            got = room[off:off + 11 * pitch].view(11, pitch)[:, :vocab]
            got.copy_(x)
            return got
        check_verify(rrr, ctx, placed(logits, off), placed(y, 7 - off), tokens, u, trees, [0.7, 1.0, 0.0])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_verify_drafts_borders(rrr, ctx, kind):
    """Masked, infinite and missing logits, equal ones, the ends of u, twins among the children, tokens
    that no vocabulary has, extreme temperatures."""
    vocab, g = 3000, gen(1)
    inf, nan = math.inf, math.nan
    base = normal(g, 6, vocab).to(DT[kind])
    base[0] = -inf
    base[0, [7, 2999]] = 1.0  # two tokens of one half each
    base[1, ::2] = nan
    base[2, 5] = base[2, 2500] = inf  # the two share the whole
    base[3] = -inf  # nothing
    base[4] = 0.25  # all equal
    base[5, :] = -inf
    base[5, 1234] = -100.0
    for u1 in (0.0, 0.25, 0.49999997, 0.5, 0.75, 1 - 2.0 ** -24):
        u = torch.full((6, 2), u1, device="cuda")
        for heat in (1.0, 0.0, 1e-30, 1e30, 0.01):
            for row in range(6):  # each row as a sequence of its own, and with children
                check_verify(rrr, ctx, base[[row]], None, ints([0]), u[:1], [[-1]], [heat])
                tokens = ints([0, 7, 2999, 7, 5, 2500])
                check_verify(rrr, ctx, base[[row, 1, 2, 3, 4, 5]], None, tokens, u, [[-1, 0, 0, 0, 0, 0]], [heat])
                check_verify(rrr, ctx, base[[row, 1, 2, 3, 4, 5]], None, ints([0, 7, -1, vocab, 1 << 30, 7]), u, [[-1, 0, 0, 0, 1, 1]], [heat])
    # chains: a draft without any chance, one equal to the target, one that is empty
    for u0 in (0.0, 0.5, 1 - 2.0 ** -24):
        u = torch.full((3, 2), u0, device="cuda")
        for x, y in ((base[[4, 4, 1]], base[[4, 4, 4]]), (base[[0, 1, 2]], base[[0, 5, 4]]), (base[[4, 2, 0]], base[[4, 4, 3]]),
                     (base[[1, 4, 4]], base[[3, 1, 1]])):
            for tokens in ([0, 7, 2999], [0, -5, 7], [0, 1234, 5], [0, vocab, 0]):
                for heat in (1.0, 0.0, 0.3):
                    check_verify(rrr, ctx, x, y, ints(tokens), u, [[-1, 0, 1]], [heat])


@pytest.mark.gpu
def test_verify_drafts_keeps_the_targets_distribution(rrr, ctx):
    """Of 20,000 chains of one draft the first tokens come out as the target's p, whatever the draft's q: each
    count within 6 standard deviations."""
    g, n, vocab = gen(9), 20000, 12
    p, q = torch.softmax(normal(g, vocab), -1), torch.softmax(1.5 * normal(g, vocab), -1)
    logits, draft = (x.log()[None].expand(2 * n, vocab).contiguous() for x in (p, q))
    tokens = torch.zeros(n, 2, dtype=torch.int32, device="cuda")
    tokens[:, 1] = torch.multinomial(q.expand(n, vocab), 1, generator=g)[:, 0].int()
    path, counts, following = torch.empty(2 * n, dtype=torch.int32, device="cuda"), *(torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
    rrr.verify_drafts(ctx, logits, tokens.flatten(), ints(range(0, 2 * n + 1, 2)), torch.rand(2 * n, 2, device="cuda", generator=g),
                      path, counts, following, rrr.verify_workspace(ctx, 2 * n, vocab, n, True), draft=draft)
    first = torch.where(counts == 2, tokens[:, 1], following)
    got = torch.bincount(first.long(), minlength=vocab).double()
    assert float(((got - n * p.double()).abs() / (n * p * (1 - p)).double().sqrt()).max()) < 6
    assert ctx.device_error() == 0


@pytest.mark.gpu
def test_verify_drafts_bad_arguments_on_the_device(rrr, ctx):
    """Bad row starts, parents and temperatures are recorded."""
    g, vocab = gen(4), 500
    logits, u, tokens = normal(g, 6, vocab), torch.rand(6, 2, device="cuda", generator=g), ints([0] * 6)

    def run(cu, parents, heat, draft=None):
        path = torch.full((6,), 77, dtype=torch.int32, device="cuda")
        counts, following = (torch.full((2,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
        rrr.verify_drafts(ctx, logits, tokens, ints(cu), u, path, counts, following,
                          rrr.verify_workspace(ctx, 6, vocab, 2, draft is not None), draft=draft, parents=parents,
                          temperature=torch.tensor(heat, device="cuda"))
        return path.tolist(), counts.tolist(), following.tolist(), ctx.device_error()
    for draft in (None, logits):
        for cu in ([0, 3, 7], [-1, 3, 6], [0, 4, 3]):
            path, counts, following, code = run(cu, None, [1.0, 1.0], draft)
            assert code == 6 and 0 in counts and -1 in following
        for heat in (-1.0, math.nan, math.inf):
            got = run([0, 3, 6], None, [heat, 1.0], draft)
            assert got[3] == 6 and got[:3] == run([0, 3, 6], None, [0.0, 1.0], draft)[:3]
    best = int(logits[0].argmax())
    tokens = ints([0, best, best, 0, 0, 0])
    for bad in (1, 4, -2, 1 << 30):
        path, counts, following, code = run([0, 3, 6], ints([-1, bad, 0, -1, 0, 0]), [0.0, 1.0])
        assert code == 6 and path[:2] == [0, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("chains", [False, True])
def test_verify_drafts_of_overlapping_sequences(rrr, ctx, chains):
    """Row starts that go back: recorded; every token is one of the vocabulary's, or -1, whatever the workspace held."""
    g, vocab = gen(9), 700
    logits, u, tokens = normal(g, 6, vocab), torch.rand(6, 2, device="cuda", generator=g), ints([0] * 6)
    draft = normal(g, 6, vocab) if chains else None
    for cu in ([0, 4, 2, 6], [2, 6, 0, 5], [5, 6, 1, 1], [0, 6, 3, 6]):
        for heat in (1.0, 0.0):
            path, n = torch.full((6,), 77, dtype=torch.int32, device="cuda"), len(cu) - 1
            counts, following = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
            ws = rrr.verify_workspace(ctx, 6, vocab, n, chains)
            ws.fill_(0x3F)
            rrr.verify_drafts(ctx, logits, tokens, ints(cu), u, path, counts, following, ws, draft=draft,
                              temperature=torch.full((n,), heat, device="cuda"))
            assert ctx.device_error() == 6
            assert all(-1 <= t < vocab for t in following.tolist()) and all(0 <= c <= 6 for c in counts.tolist())


@pytest.mark.gpu
def test_steps_on_two_streams_at_once(rrr, ctx):
    """Each stream has its cache and its workspaces: the bits of the calls made one after another."""
    hd, nh, nkv, vocab, lens, nodes = 128, 6, 2, 5000, [900, 33, 2000], [7, 1, 12]
    rng, jobs = np.random.default_rng(3), []
    for seed in range(2):
        g, cu, total = gen(40 + seed), cu_of(nodes), sum(nodes)
        cache = Cache(rrr, ctx, nkv, hd, [n + 16 for n in lens], 3)
        cache.c.store(normal(g, sum(lens), nkv, hd), normal(g, sum(lens), nkv, hd), cu_of(lens), ints(lens))
        trees = [random_tree(rng, n, "tree") for n in nodes]
        qkv, factors, desc = append_inputs(rrr, g, total, nh, nkv, hd, 96, "bf16")
        logits, _, tokens, u = verify_inputs(g, rng, vocab, trees, "f32", False)
        jobs.append(dict(cache=cache, cu=cu, parents=ints([p for t in trees for p in t]), lens=ints(lens), qkv=qkv, desc=desc, factors=factors,
                         q=normal(g, total, nh, hd, dtype=torch.bfloat16), k=normal(g, total, nkv, hd, dtype=torch.bfloat16),
                         v=normal(g, total, nkv, hd, dtype=torch.bfloat16), logits=logits, tokens=tokens, u=u, after=ints([n + 7 for n in lens]),
                         path=torch.empty(total, dtype=torch.int32, device="cuda"), pages=cache.pages.clone()))
    torch.cuda.synchronize()

    def run(j, out):
        j["cache"].c.attention_tree(j["q"], j["k"], j["v"], j["cu"], j["parents"], j["lens"], out["o"], out["ws"])
        rrr.verify_drafts(ctx, j["logits"], j["tokens"], j["cu"], j["u"], out["path"], out["counts"], out["next"], out["vws"], parents=j["parents"])
        j["cache"].c.append(j["desc"], j["qkv"], j["cu"], j["after"], path=out["path"], counts=out["counts"])

    def fresh(j):
        total, i = j["q"].shape[0], dict(dtype=torch.int32, device="cuda")
        j["cache"].pages.copy_(j["pages"])
        return dict(o=torch.zeros_like(j["q"]), ws=j["cache"].c.tree_workspace(nh, total), vws=rrr.verify_workspace(ctx, total, vocab, 3, False),
                    path=torch.zeros(total, **i), counts=torch.zeros(3, **i), next=torch.zeros(3, **i))
    want = []
    for j in jobs:
        out = fresh(j)
        run(j, out)
        want.append([out[x].clone() for x in ("o", "path", "counts", "next")] + [j["cache"].pages.clone()])
    outs, streams = [fresh(j) for j in jobs], [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(3):
        for j, out, stream in zip(jobs, outs, streams):
            with torch.cuda.stream(stream):
                j["cache"].pages.copy_(j["pages"])
                run(j, out)
    torch.cuda.synchronize()
    for j, out, w in zip(jobs, outs, want):
        assert all(torch.equal(a, b) for a, b in zip([out[x] for x in ("o", "path", "counts", "next")] + [j["cache"].pages], w))
    assert ctx.device_error() == 0


# ------------------------------------------------------------------ together
def step_of(rrr, ctx, cache, desc, halves, s, graph=False):
    """One step on device values alone: rotated rows of the trees, their attention, verification, the accepted rows
    appended, lengths advanced."""
    rrr.qk_norm_rope(ctx, desc, s["qkv"], s["pos"], s["q"], s["k"], s["v"], halves=halves)
    cache.attention_tree(s["q"], s["k"], s["v"], s["cu"], s["parents"], s["lens"], s["out"], s["ws"])
    rrr.verify_drafts(ctx, s["logits"], s["tokens"], s["cu"], s["u"], s["path"], s["counts"], s["next"], s["vws"],
                      parents=s["parents"], temperature=s["heat"])
    s["lens"] += s["counts"]
    cache.append(desc, s["qkv"], s["cu"], s["lens"], path=s["path"], counts=s["counts"], halves=halves)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,rd,halves", [(128, 96, False), (64, 64, True), (256, 128, False)])
def test_steps_of_speculative_decoding(rrr, ctx, hd, rd, halves):
    """Prompts appended, then steps of trees: eager and replayed from one captured graph with other values, the same bits; each
    step's attention against 64 bits, the cache's rows against a plain append of the accepted rows."""
    nh, nkv, vocab, g, rng = 6, 2, 700, gen(hd), np.random.default_rng(hd)
    prompts, nodes = [50, 1, 127], [8, 5, 12]
    rows, n_seqs, top = sum(nodes), 3, 1000
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, rd, 10000.0, 1.0, None, 0, top)
    caches = [Cache(rrr, ctx, nkv, hd, [400] * 3, 3) for _ in range(3)]
    prompt = normal(g, sum(prompts), (nh + 2 * nkv) * hd)
    for c in caches:
        c.c.append(desc, prompt, cu_of(prompts), ints(prompts), torch.empty(sum(prompts), nh, hd, device="cuda"), halves=halves)
    bf = torch.bfloat16

    def state(cache):
        e = torch.empty
        i32 = dict(dtype=torch.int32, device="cuda")
        return dict(q=e(rows, nh, hd, dtype=bf, device="cuda"), k=e(rows, nkv, hd, dtype=bf, device="cuda"),
                    v=e(rows, nkv, hd, dtype=bf, device="cuda"), out=e(rows, nh, hd, dtype=bf, device="cuda"),
                    ws=cache.tree_workspace(nh, rows), vws=rrr.verify_workspace(ctx, rows, vocab, n_seqs, False), path=e(rows, **i32),
                    counts=e(n_seqs, **i32), next=e(n_seqs, **i32), cu=cu_of(nodes), lens=ints(prompts), qkv=e(rows, (nh + 2 * nkv) * hd, device="cuda"),
                    pos=e(rows, **i32), parents=e(rows, **i32), logits=e(rows, vocab, device="cuda"), tokens=e(rows, **i32),
                    u=e(rows, 2, device="cuda"), heat=torch.tensor([1.0, 0.0, 0.6], device="cuda"))
    eager, replayed = state(caches[0].c), state(caches[1].c)
    graph = None
    accepted = 0
    for step in range(5):
        trees = [random_tree(rng, n, "tree") for n in nodes]
        depth = [len(a) - 1 for t in trees for a in ancestors(t)]
        of = np.repeat(np.arange(n_seqs), nodes)
        held = eager["lens"].tolist()
        new = dict(qkv=normal(g, rows, (nh + 2 * nkv) * hd), pos=ints([held[s] + d for s, d in zip(of, depth)]),
                   parents=ints([p for t in trees for p in t]))
        new["logits"], _, new["tokens"], new["u"] = verify_inputs(g, rng, vocab, trees, "f32", False)
        for s in (eager, replayed):
            for name, t in new.items():
                s[name].copy_(t)
        before = [torch.empty(sum(held), nkv, hd, device="cuda") for _ in range(2)]
        caches[0].c.load(cu_of(held), ints(held), *before)
        step_of(rrr, ctx, caches[0].c, desc, halves, eager)
        if graph is None:
            saved = replayed["lens"].clone(), caches[1].pages.clone()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step_of(rrr, ctx, caches[1].c, desc, halves, replayed)
            replayed["lens"].copy_(saved[0])
            caches[1].pages.copy_(saved[1])
        graph.replay()
        for name in ("out", "path", "counts", "next", "lens"):
            assert torch.equal(eager[name], replayed[name]), (step, name)
        assert torch.equal(caches[0].pages, caches[1].pages)
        compare_tree(eager["out"], eager["q"], eager["k"], eager["v"], *before, held, trees, "bf16", hd ** -0.5)
        taken, path = eager["counts"].tolist(), eager["path"].tolist()
        accepted += sum(taken) - n_seqs
        cu = np.cumsum([0] + nodes)
        flat = [int(cu[s]) + path[cu[s] + i] for s in range(n_seqs) for i in range(taken[s])]
        caches[2].c.append(desc, new["qkv"][flat].contiguous(), cu_of(taken), eager["lens"], halves=halves)
        assert torch.equal(caches[0].pages, caches[2].pages)
    assert accepted > 0
    assert ctx.device_error() == 0
