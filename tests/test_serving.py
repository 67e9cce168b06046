"""The packed-batch operators: rrr_qk_norm_rope, rrr_attention_packed, rrr_kv4_store /
rrr_kv4_load, rrr_attention_kv4.

CPU: refusals through the C ABI (on a host-made context: arguments are checked before the
device is touched) and through the Python host; the page layout's index formulas.
GPU: every operator against its formula in 64 bits, bounds per element derived from the
roundings that it makes (u = 2^-24 is half a step of f32, h(t) half a step of the type):

  qk      norm and rotation are at most 11 roundings in the inverse root (13 in the sum of
          squares count half; then mean, eps, root, divide), 2 products, 3 of the rotation, and
          the sine is off by at most 2^-24 turns * 2 pi + 2 u: 32 u (|a| + |b|) af in all.
  kv4     store and load are the formula's own f32 operations: bit for bit.
  decode  a score of n = hd products carries at most 48 u sum |q k| scale (16 + 16 products of
          an MMA chain, 2 per group, the split's 2^-22, scale); a weight 2^x is off by that twice
          (it and the maximum) and 8 u (the exponential's 2^-22, the split): the result by 2
          weights' errors times max |v|, and (rows / 64 + 64) u of the sums.
  packed  the same with hd + 16 roundings per score, and h(t) max |v| of the rounded weights.
"""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
ROWS = 64
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------ formulas in 64 bits
def ref_qk(qkv, pos, nh, nkv, hd, rd, theta, af, factors, gammas, eps, halves):
    """q, k, v in 64 bits and the bound's |a| + |b| of every value."""
    x = qkv.double().reshape(qkv.shape[0], nh + 2 * nkv, hd)
    f = float(np.float32(theta)) ** (-2.0 * torch.arange(rd // 2, dtype=torch.float64) / max(rd, 1))
    if factors is not None:
        n = min(len(factors), rd // 2)
        f[:n] /= factors[:n].double().cpu()
    ang = pos.double().cpu()[:, None] * f
    c, s = (ang.cos() * float(np.float32(af))).to(x.device), (ang.sin() * float(np.float32(af))).to(x.device)
    outs, mags = [], []
    for i, (a, b) in enumerate(((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv))):
        y = x[:, a:b].clone()
        mag = y.abs()
        if i < 2:
            if gammas[i] is not None:
                y = gammas[i].double() * y / (y.pow(2).mean(-1, keepdim=True) + float(np.float32(eps))).sqrt()
            mag = y.abs()
            e = torch.arange(rd // 2)
            ia, ib = (e, e + rd // 2) if halves else (2 * e, 2 * e + 1)
            p, q = y[..., ia].clone(), y[..., ib].clone()
            y[..., ia] = p * c[:, None] - q * s[:, None]
            y[..., ib] = p * s[:, None] + q * c[:, None]
            mag[..., ia] = mag[..., ib] = (p.abs() + q.abs()) * max(af, 1.0)
        outs.append(y)
        mags.append(mag)
    return outs, mags


def np_quantise(x):
    """codes, d, m (f16) of f32 rows [..., hd], with the operations of the formula."""
    x = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    with np.errstate(all="ignore"):
        m = np.clip(lo, -65504, 65504).astype(np.float16)
        d = np.minimum((hi - lo) / np.float32(15), np.float32(65504)).astype(np.float16)
        d32, m32 = d.astype(np.float32), m.astype(np.float32)
        c = np.where(d32 > 0, (x - m32) / np.where(d32 > 0, d32, 1), np.float32(0))
        c = np.clip(np.rint(c), 0, 15)
    c = np.where(bad, 0, c).astype(np.int64)
    return c, np.where(bad, np.float16(np.nan), d)[..., 0], np.where(bad, np.float16(np.nan), m)[..., 0], bad[..., 0]


def np_values(x):
    c, d, m, bad = np_quantise(x)
    v = c.astype(np.float32) * d.astype(np.float32)[..., None] + m.astype(np.float32)[..., None]
    return v.reshape(x.shape)


def page_indices(hd, row):
    """Byte-level places of row `row` in a block: [(codes u32 index, nibble)] for K, [(u16
    index, nibble)] for V per element; f16 indices of d, K's m, V's m per group."""
    j_ = min(hd // 32, 4)
    k, v = [], []
    for e in range(hd):
        P, i, w = e // 32 // j_, e // 32 % j_, e % 32
        k.append((((P * 64 + row) * 4 + w // 8) * j_ + i, w % 8))
        t = row % 8 // 2
        word = ((((P * 4 + row // 16) * 2 + row % 16 // 8) * 8 + w % 8) * 4 + t) * j_ + i
        v.append((2 * word + row % 2, w // 8))
    g = hd // 32
    return k, v, [row * g + j for j in range(g)], [((row // 2) * g + j) * 2 + row % 2 for j in range(g)]


def read_block(block, hd):
    """K and V [64, hd] f32 that a block (uint8 numpy) stands for, by the header's formulas."""
    kw, vw = block[:32 * hd].view(np.uint32), block[40 * hd:72 * hd].view(np.uint16)
    kd, km = block[32 * hd:36 * hd].view(np.float16), block[36 * hd:40 * hd].view(np.float16)
    vd, vm = block[72 * hd:76 * hd].view(np.float16), block[76 * hd:80 * hd].view(np.float16)
    K, V = np.empty((64, hd), np.float32), np.empty((64, hd), np.float32)
    for r in range(64):
        k, v, s, sm = page_indices(hd, r)
        for e in range(hd):
            j = e // 32
            K[r, e] = np.float32((int(kw[k[e][0]]) >> (4 * k[e][1])) & 15) * np.float32(kd[s[j]]) + np.float32(km[s[j]])
            V[r, e] = np.float32((int(vw[v[e][0]]) >> (4 * v[e][1])) & 15) * np.float32(vd[s[j]]) + np.float32(vm[sm[j]])
    return K, V


def ref_attention(q, k, v, seen, scale):
    """q [nh, hd] x k, v [rows, nkv, hd] (64 bits), the first `seen` rows: out [nh, hd] and A =
    max over rows of sum |q k| scale per head."""
    nh, nkv = q.shape[0], k.shape[1]
    kk, vv = (x[:seen].repeat_interleave(nh // nkv, 1).transpose(0, 1) for x in (k, v))
    s = (kk @ q[:, :, None])[..., 0] * scale
    A = ((kk.abs() @ q.abs()[:, :, None])[..., 0] * scale).amax(-1)
    return (torch.softmax(s, -1)[:, None] @ vv)[:, 0], A


# ------------------------------------------------------------------ CPU
@pytest.fixture(scope="module")
def host_ctx(rrr, tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host") / "host_ctx.so")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I/usr/local/cuda/include",
                    os.path.join(ROOT, "tests", "cpp", "host_ctx.cpp"), "-o", so], check=True)
    L = ctypes.CDLL(so)
    L.host_ctx_new.restype = ctypes.c_void_p
    L.host_ctx_free.argtypes = [ctypes.c_void_p]
    c = L.host_ctx_new()
    yield ctypes.c_void_p(c)
    L.host_ctx_free(c)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_page_layout_has_a_place_for_every_value(hd):
    k_seen, v_seen, s_seen, m_seen = set(), set(), set(), set()
    for r in range(64):
        k, v, s, m = page_indices(hd, r)
        k_seen.update(k)
        v_seen.update(v)
        s_seen.update(s)
        m_seen.update(m)
    assert k_seen == {(w, n) for w in range(64 * hd // 8) for n in range(8)}
    assert v_seen == {(w, n) for w in range(64 * hd // 4) for n in range(4)}
    assert s_seen == m_seen == set(range(2 * hd))


def _qk_args(rrr, **over):
    a = dict(nh=4, nkv=2, hd=128, rd=96, theta=1e4, seq=16, in_type=0, qkv=4096, stride=1024, rows=2, pos=64, qg=None,
             kg=None, eps=1e-5, halves=0, out_type=30, q=1 << 20, qs=512, k=2 << 20, ks=256, v=3 << 20, vs=256)
    a.update(over)
    d = rrr.ffi.AttnDesc(a["nh"], a["nkv"], a["hd"], a["rd"], a["theta"], 1.0, None, 0, a["seq"])
    return (ctypes.byref(d), a["in_type"], a["qkv"], a["stride"], a["rows"], a["pos"], a["qg"], a["kg"], a["eps"],
            a["halves"], a["out_type"], a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], None)


FINE = -5  # the arguments pass and the missing device is met


def _no_gpu():
    if torch.cuda.is_available():
        pytest.skip("addresses are made up: host only")


@pytest.mark.parametrize("over,code", [
    ({}, FINE), ({"v": None, "vs": 0}, FINE), ({"rows": 0}, FINE), ({"halves": 1}, FINE),
    ({"in_type": 2}, -2), ({"out_type": 14}, -2), ({"qkv": None}, -1), ({"pos": None}, -1), ({"q": None}, -1),
    ({"k": None}, -1), ({"rows": -1}, -3), ({"halves": 2}, -1), ({"halves": 1, "rd": 100}, -3), ({"rd": 95}, -3),
    ({"rd": 130}, -3), ({"hd": 96}, -3), ({"nh": 3}, -3), ({"nh": 18}, -3), ({"theta": 0.0}, -1), ({"eps": -1.0}, -1),
    ({"eps": math.nan}, -1), ({"stride": 1016}, -3), ({"qs": 504}, -3), ({"ks": 248}, -3), ({"vs": 248}, -3),
    ({"qkv": 4100}, -4), ({"q": (1 << 20) + 8}, -4), ({"stride": 1028}, -4), ({"ks": 260}, -4), ({"qg": 2}, -4),
    # in place: their own parts of qkv, one type and stride
    ({"out_type": 0, "q": 4096, "qs": 1024, "k": 4096 + 4 * 512, "ks": 1024, "v": 4096 + 4 * 768, "vs": 1024}, FINE),
    ({"out_type": 0, "q": 4096, "qs": 1024, "k": 4096 + 4 * 768, "ks": 1024}, -1),
    ({"out_type": 30, "q": 4096, "qs": 1024}, -1), ({"q": 4096 + 1024 * 4}, -1), ({"k": 1 << 20}, -1),
    # one buffer of [q | k | v] rows
    ({"q": 1 << 20, "qs": 1024, "k": (1 << 20) + 1024, "ks": 1024, "v": (1 << 20) + 1536, "vs": 1024}, FINE),
    ({"q": 1 << 20, "qs": 1024, "k": (1 << 20) + 1008, "ks": 1024, "v": (1 << 20) + 1536, "vs": 1024}, -1),
])
def test_qk_norm_rope_refusals(rrr, host_ctx, over, code):
    _no_gpu()
    assert rrr.ffi.lib().rrr_qk_norm_rope(host_ctx, *_qk_args(rrr, **over)) == code, rrr.ffi.last_error(host_ctx)


def _cache(rrr, **over):
    a = dict(pages=1 << 30, n_pages=8, nkv=2, hd=128, table=1 << 12, n_seqs=3, most=4, stride=4)
    a.update({k: v for k, v in over.items() if k in a})
    return rrr.ffi.KV4Desc(a["pages"], a["n_pages"], a["nkv"], a["hd"], a["table"], a["n_seqs"], a["most"], a["stride"])


CACHE_BAD = [({"pages": None}, -1), ({"table": None}, -1), ({"hd": 96}, -3), ({"nkv": 0}, -3), ({"n_pages": -1}, -3),
             ({"stride": 3}, -3), ({"n_seqs": 1 << 30}, -3), ({"most": -1}, -3), ({"most": 1 << 26, "stride": 1 << 26}, -3),
             ({"pages": (1 << 30) + 8}, -4), ({"table": 4098}, -4)]


@pytest.mark.parametrize("over,code", CACHE_BAD + [
    ({}, FINE), ({"rows": 0}, FINE), ({"type": 8}, -2), ({"k": None}, -1), ({"v": None}, -1), ({"cu": None}, -1),
    ({"lens": None}, -1), ({"rows": -2}, -3), ({"ks": 248}, -3), ({"vs": 0}, -3), ({"k": (1 << 20) + 8}, -4),
    ({"ks": 260}, -4), ({"k": (1 << 30) + 1024}, -1)])
def test_kv4_store_and_load_refusals(rrr, host_ctx, over, code):
    _no_gpu()
    a = dict(type=30, k=1 << 20, ks=256, v=2 << 20, vs=256, rows=5, cu=256, lens=512)
    a.update({k: v for k, v in over.items() if k in a})
    c = _cache(rrr, **over)
    L = rrr.ffi.lib()
    args = (a["type"], a["k"], a["ks"], a["v"], a["vs"], a["rows"], a["cu"], a["lens"], None)
    assert L.rrr_kv4_store(host_ctx, ctypes.byref(c), *args) == code
    # load may leave one of k and v out, and writes: they must not overlap each other
    if over not in ({"k": None}, {"v": None}, {"vs": 0}):
        assert L.rrr_kv4_load(host_ctx, ctypes.byref(c), *args) == code
    assert L.rrr_kv4_load(host_ctx, ctypes.byref(_cache(rrr)), 30, None, 0, 2 << 20, 256, 5, 256, 512, None) == FINE
    assert L.rrr_kv4_load(host_ctx, ctypes.byref(_cache(rrr)), 30, None, 0, None, 0, 5, 256, 512, None) == -1
    assert L.rrr_kv4_load(host_ctx, ctypes.byref(_cache(rrr)), 30, 1 << 20, 256, (1 << 20) + 256, 256, 5, 256, 512,
                          None) == -1


@pytest.mark.parametrize("over,code", CACHE_BAD + [
    ({}, FINE), ({"type": 12}, -2), ({"heads": 5}, -3), ({"heads": 18}, -3), ({"heads": 0}, -3), ({"q": None}, -1),
    ({"lens": None}, -1), ({"out": None}, -1), ({"ws": None}, -1), ({"qs": 760}, -3), ({"os": 760}, -3),
    ({"scale": -1.0}, -1), ({"scale": math.nan}, -1), ({"scale": math.inf}, -1), ({"q": (1 << 20) + 8}, -4),
    ({"os": 772}, -4), ({"ws": (1 << 24) + 8}, -4), ({"ws_bytes": -1}, -11), ({"out": 1 << 20}, -1),
    ({"out": (1 << 24) + 256}, -1), ({"ws": 1 << 30}, -1)])
def test_attention_kv4_refusals(rrr, host_ctx, over, code):
    _no_gpu()
    a = dict(heads=6, type=0, q=1 << 20, qs=768, lens=512, scale=0.0, out=2 << 20, os=768, ws=1 << 24, ws_bytes=0)
    a.update({k: v for k, v in over.items() if k in a})
    L = rrr.ffi.lib()
    need = ctypes.c_int64()
    assert L.rrr_kv4_workspace(host_ctx, ctypes.byref(_cache(rrr)), 6, ctypes.byref(need)) == 0 and need.value > 0
    assert L.rrr_kv4_workspace(host_ctx, ctypes.byref(_cache(rrr)), 6, None) == -1
    c = _cache(rrr, **over)
    assert L.rrr_attention_kv4(host_ctx, ctypes.byref(c), a["heads"], a["type"], a["q"], a["qs"], a["lens"], a["scale"],
                               a["out"], a["os"], a["ws"], need.value + a["ws_bytes"], None) == code


@pytest.mark.parametrize("over,code", [
    ({}, FINE), ({"q_rows": 0, "q": None, "out": None}, FINE), ({"kv_rows": 0, "k": None, "v": None}, FINE),
    ({"n_seqs": 0}, FINE), ({"head_major": True}, FINE), ({"type": 0}, -2), ({"hd": 32}, -3), ({"nh": 5}, -3),
    ({"nh": 0}, -3), ({"n_seqs": -1}, -3), ({"q_rows": -1}, -3), ({"kv_rows": 1 << 31}, -3), ({"causal": 2}, -1),
    ({"scale": -0.5}, -1), ({"scale": math.nan}, -1), ({"q": None}, -1), ({"k": None}, -1), ({"v": None}, -1),
    ({"out": None}, -1), ({"cu_q": None}, -1), ({"cu_kv": None}, -1), ({"q_row": 0}, -3), ({"k_head": 64}, -3),
    ({"v_row": 260}, -4), ({"q": (1 << 20) + 8}, -4), ({"out_row": 128}, -3), ({"out": 1 << 20}, -1),
    ({"out": 4 << 20}, -1)])
def test_attention_packed_refusals(rrr, host_ctx, over, code):
    _no_gpu()
    a = dict(type=30, nh=4, nkv=2, hd=128, n_seqs=2, causal=1, scale=0.0, q_rows=9, kv_rows=11, q_row=512, q_head=128,
             k_row=256, k_head=128, v_row=256, v_head=128, out_row=512, out_head=128, q=1 << 20, k=2 << 20, v=4 << 20,
             out=8 << 20, cu_q=256, cu_kv=512)
    a.update(over)
    if a.pop("head_major", False):
        a.update(q_row=128, q_head=9 * 128, out_row=128, out_head=9 * 128)
    d = rrr.ffi.PackedDesc(*(a[f] for f in ("type", "nh", "nkv", "hd", "n_seqs", "causal", "scale", "q_rows", "kv_rows",
                                            "q_row", "q_head", "k_row", "k_head", "v_row", "v_head", "out_row",
                                            "out_head")))
    L = rrr.ffi.lib()
    assert L.rrr_attention_packed(host_ctx, ctypes.byref(d), a["q"], a["k"], a["v"], a["cu_q"], a["cu_kv"], a["out"],
                                  None) == code, rrr.ffi.last_error(host_ctx)
    assert L.rrr_attention_packed(host_ctx, None, 0, 0, 0, 0, 0, 0, None) == -1
    assert L.rrr_attention_packed(None, ctypes.byref(d), 0, 0, 0, 0, 0, 0, None) == -1


def test_empty_arrays_may_be_null_and_sizes_have_an_end(rrr, host_ctx):
    """What has no element has no address in many frameworks; counts past what one launch or a page
    number holds are refused before anything is launched."""
    _no_gpu()
    L, ref = rrr.ffi.lib(), ctypes.byref
    none = dict(qkv=None, pos=None, q=None, k=None, v=None, rows=0)
    assert L.rrr_qk_norm_rope(host_ctx, *_qk_args(rrr, **none)) == FINE
    no_seqs = _cache(rrr, table=None, n_seqs=0)
    no_pages = _cache(rrr, pages=None, n_pages=0, table=None, most=0, stride=0)
    many = _cache(rrr, n_pages=1 << 31)
    for f in (L.rrr_kv4_store, L.rrr_kv4_load):
        assert f(host_ctx, ref(no_seqs), 30, None, 256, None, 256, 0, None, None, None) == FINE
        assert f(host_ctx, ref(no_pages), 30, 1 << 20, 256, 2 << 20, 256, 5, 256, 512, None) == FINE
        assert f(host_ctx, ref(many), 30, 1 << 20, 256, 2 << 20, 256, 5, 256, 512, None) == -3
    far = 1 << 40
    assert L.rrr_qk_norm_rope(host_ctx, *_qk_args(rrr, stride=far)) == -3
    assert L.rrr_kv4_store(host_ctx, ref(_cache(rrr)), 30, 1 << 20, far, 2 << 20, 256, 5, 256, 512, None) == -3
    assert L.rrr_attention_kv4(host_ctx, ref(_cache(rrr)), 6, 0, 1 << 20, far, 512, 0.0, 2 << 20, 768, 1 << 24, 1 << 40,
                               None) == -3
    need = ctypes.c_int64()
    for c in (no_seqs, no_pages):
        assert L.rrr_kv4_workspace(host_ctx, ref(c), 6, ref(need)) == 0
        q = (None, 768, None) if c is no_seqs else (1 << 20, 768, 512)
        assert L.rrr_attention_kv4(host_ctx, ref(c), 6, 0, *q, 0.0, None if c is no_seqs else 2 << 20, 768, 1 << 24,
                                   need.value, None) == FINE
    d = rrr.ffi.PackedDesc(30, 4, 2, 128, 0, 1, 0.0, 0, 0, *(512, 128, 256, 128, 256, 128, 512, 128))
    assert L.rrr_attention_packed(host_ctx, ref(d), None, None, None, None, None, None, None) == FINE
    # 65,535 heads times 2^24 / 256 tiles of rows
    w = 65535 * 64
    d = rrr.ffi.PackedDesc(30, 65535, 65535, 64, 1, 1, 0.0, 1 << 24, 1, w, 64, w, 64, w, 64, w, 64)
    assert L.rrr_attention_packed(host_ctx, ref(d), 1 << 12, 1 << 60, 1 << 61, 256, 512, 1 << 62, None) == -3


def test_python_host_refuses_what_the_kernels_cannot_take(rrr):
    class Ctx:  # refused before the library is asked
        h, device = None, 0
    E = rrr.RRRError
    d = rrr.ffi.AttnDesc(4, 2, 128, 96, 1e4, 1.0, None, 0, 16)
    pos, z = torch.zeros(3, dtype=torch.int32), torch.zeros
    with pytest.raises(E, match="cuda:0"):
        rrr.qk_norm_rope(Ctx, d, z(3, 8, 128), pos, z(3, 4, 128), z(3, 2, 128))
    with pytest.raises(E, match="qkv"):
        rrr.qk_norm_rope(Ctx, d, z(3, 7, 128), pos, z(3, 4, 128), z(3, 2, 128))
    with pytest.raises(E, match="needed"):
        rrr.attention_packed(Ctx, z(3, 4, 128), z(3, 2, 128), z(3, 2, 64), pos, pos, z(3, 4, 128))
    with pytest.raises(E, match="one type"):
        rrr.attention_packed(Ctx, z(3, 4, 128).half(), z(3, 2, 128), z(3, 2, 128), pos, pos, z(3, 4, 128))
    with pytest.raises(E, match="contiguous"):
        t = z(3, 4, 256).half()[..., ::2]
        rrr.attention_packed(Ctx, t, z(3, 2, 128).half(), z(3, 2, 128).half(), pos, pos, t)
    with pytest.raises(E, match="pages"):
        rrr.KV4Cache(Ctx, z(4, 2, 80 * 64, dtype=torch.uint8), z(1, 4, dtype=torch.int32), 128)
    with pytest.raises(E, match="page_table"):
        rrr.KV4Cache(Ctx, z(4, 2, 80 * 128, dtype=torch.uint8), z(4, dtype=torch.int32), 128)
    assert rrr.KV4Cache.page_shape(5, 2, 64) == (5, 2, 5120)


# ------------------------------------------------------------------ GPU helpers
def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cu_of(lens):
    return ints([0] + list(np.cumsum(lens)))


def normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


class Cache:
    """Pages of random order for sequences of at most `lens` rows, filled by rrr_kv4_store."""

    def __init__(self, rrr, ctx, nkv, hd, most, seed, n_extra=3, first_page=0, fill=0xA5):
        per = max(1, max(-(-n // ROWS) for n in most))
        order = np.random.default_rng(seed).permutation(per * len(most) + n_extra)[:per * len(most)] + first_page
        self.table = order.reshape(len(most), per).astype(np.int32)
        self.pages = torch.full(rrr.KV4Cache.page_shape(first_page + per * len(most) + n_extra, nkv, hd), fill,
                                dtype=torch.uint8, device="cuda")
        self.c = rrr.KV4Cache(ctx, self.pages, torch.from_numpy(self.table).cuda(), hd)


def within(got, ref, bound):
    """Every element within its bound (and as finite as the formula's)."""
    got, ref = got.double(), ref.double()
    fine = torch.isfinite(ref)
    assert torch.equal(fine, torch.isfinite(got)), "non-finite values differ"
    worst = ((got - ref).abs() / bound.clamp_min(1e-300))[fine]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, f"{float(worst.max())} of the bound"


# ------------------------------------------------------------------ qk
@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv,rd,halves", [
    (128, 24, 8, 96, False), (128, 24, 8, 96, True), (64, 3, 3, 64, True), (64, 8, 1, 6, False), (256, 8, 2, 128, False),
    (256, 5, 5, 112, True), (128, 1, 1, 0, False), (128, 2, 1, 128, True)])
@pytest.mark.parametrize("kinds", [("f32", "f32"), ("f32", "bf16"), ("bf16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("rows", [1, 37, 700])
def test_qk_norm_rope(rrr, ctx, hd, nh, nkv, rd, halves, kinds, rows):
    g = gen(rows + hd)
    heads = nh + 2 * nkv
    wide = torch.empty(rows, heads * hd + 24, dtype=DT[kinds[0]], device="cuda")  # rows with a gap
    qkv = wide[:, 8:8 + heads * hd]
    qkv.copy_(normal(g, rows, heads * hd) * torch.exp(2 * normal(g, rows, 1)))
    top = 1 << 20
    pos = torch.randint(0, top, (rows,), generator=g, device="cuda", dtype=torch.int32)
    pos[0] = top - 1 if rows > 1 else 5
    norm = rows != 37
    gammas = [torch.rand(hd, device="cuda", generator=g) + 0.5 if norm else None for _ in range(2)]
    if rows == 700:
        gammas[1] = None
    factors = torch.rand(max(rd // 2 - 3, 1), device="cuda", generator=g) + 0.75 if rd > 8 else None
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, rd, 10000.0, 1.25, None if factors is None else factors.data_ptr(),
                            0 if factors is None else factors.numel(), top)
    out = DT[kinds[1]]
    outs = [torch.full((rows, n, hd), 7.0, dtype=out, device="cuda") for n in (nh, nkv, nkv)]
    rrr.qk_norm_rope(ctx, desc, qkv, pos, *outs, q_gamma=gammas[0], k_gamma=gammas[1], eps=1e-5, halves=halves)
    refs, mags = ref_qk(qkv, pos, nh, nkv, hd, rd, 10000.0, 1.25, factors, gammas, 1e-5, halves)
    for got, ref, mag, copied in zip(outs, refs, mags, (0, 0, 1)):
        rounding = 0.0 if out == torch.float32 else half_step(out)
        bound = ref.abs() * rounding * 1.01 + (0 if copied else 32 * U) * mag
        if out == torch.float16:
            bound = bound + 2.0 ** -25  # its subnormals
        within(got, ref, bound + 1e-30)
    assert ctx.device_error() == 0


@pytest.mark.gpu
def test_qk_norm_rope_in_place_and_against_rope_kv_store(rrr, ctx):
    """In place gives the same bits; at small positions the framework's own RoPE (angle in 32
    bits) is met within its angle's rounding; rows of other positions stay as they were."""
    g = gen(3)
    nh, nkv, hd, rows = 6, 2, 128, 5
    x = normal(g, rows, (nh + 2 * nkv) * hd)
    pos = ints([0, 1, 2, 3, 4])
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, 96, 10000.0, 1.190238, None, 0, 64)
    outs = [torch.empty(rows, n, hd, device="cuda") for n in (nh, nkv, nkv)]
    rrr.qk_norm_rope(ctx, desc, x, pos, *outs)
    y = x.clone()
    parts = [y[:, a * hd:b * hd] for a, b in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv))]
    rrr.qk_norm_rope(ctx, desc, y, pos, *parts)
    assert torch.equal(y, torch.cat([o.flatten(1) for o in outs], 1))
    z = x.clone()
    kc, vc = (torch.zeros(64, nkv * hd, dtype=torch.float16, device="cuda") for _ in range(2))
    L = rrr.ffi.lib()
    ctx.check(L.rrr_rope_kv_store(ctx.h, ctypes.byref(desc), z.data_ptr(), z.shape[1], rows, 0, None, kc.data_ptr(),
                                  vc.data_ptr(), None))
    assert float((y - z).abs().max()) < 4 * 5 * U * 1.2 * float(x.abs().max()) * 8
    bad = ints([3, -1, 64, 2 ** 31 - 1, 0])
    w = torch.full_like(outs[0], 9.0)
    rrr.qk_norm_rope(ctx, desc, x, bad, w, outs[1])
    assert ctx.device_error() == 6 and ctx.device_error() == 0
    assert bool((w[1:4] == 9).all()) and bool((w[0] != 9).any()) and bool((w[4] != 9).any())


# ------------------------------------------------------------------ cache rows
@pytest.mark.gpu
@pytest.mark.parametrize("hd,nkv", [(64, 1), (128, 8), (256, 3)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,held", [([1], [1]), ([5, 0, 130, 1], [70, 64, 130, 65]), ([64, 63], [64, 191])])
def test_kv4_store_and_load(rrr, ctx, hd, nkv, kind, new, held):
    g = gen(hd + nkv)
    cache = Cache(rrr, ctx, nkv, hd, held, 5)
    before = cache.pages.clone()
    rows, extra = sum(new), 2
    wide = [normal(g, rows + extra, nkv * hd + 16, dtype=DT[kind]) * 3 for _ in range(2)]
    k, v = wide[0][:, 8:8 + nkv * hd], wide[1][:, 16:]
    k[0, :32] = 0.5                    # a group of one value
    v[0, 32:64] = torch.linspace(-0.0, 1e-6, 32, device="cuda").to(DT[kind])
    if kind != "f16":
        v[rows - 1, :3] = torch.tensor([1e30, -1e30, 7e4], device="cuda").to(DT[kind])
    cache.c.store(k, v, cu_of(new), ints(held))
    assert ctx.device_error() == 0
    pages, was = cache.pages.cpu().numpy(), before.cpu().numpy()
    want = {}
    cu = np.cumsum([0] + new)
    for s in range(len(new)):
        for i in range(new[s]):
            p = held[s] - new[s] + i
            want.setdefault(int(cache.table[s, p // ROWS]), {})[p % ROWS] = cu[s] + i
    kn, vn = (x[:rows].float().cpu().numpy().reshape(rows, nkv, hd) for x in (k, v))
    kq, vq = np_quantise(kn), np_quantise(vn)
    for page in range(pages.shape[0]):
        for h in range(nkv):
            blk = was[page, h].copy()
            kw, vw = blk[:32 * hd].view(np.uint32), blk[40 * hd:72 * hd].view(np.uint16)
            kd, km = blk[32 * hd:36 * hd].view(np.float16), blk[36 * hd:40 * hd].view(np.float16)
            vd, vm = blk[72 * hd:76 * hd].view(np.float16), blk[76 * hd:80 * hd].view(np.float16)
            for r, src in want.get(page, {}).items():
                ki, vi, s, sm = page_indices(hd, r)
                for places, words, codes in ((ki, kw, kq[0][src, h].ravel()), (vi, vw, vq[0][src, h].ravel())):
                    w, n = np.array([a for a, _ in places]), np.array([4 * b for _, b in places])
                    words[np.unique(w)] = 0
                    np.bitwise_or.at(words, w, (codes << n).astype(words.dtype))
                kd[s], km[s], vd[s], vm[sm] = kq[1][src, h], kq[2][src, h], vq[1][src, h], vq[2][src, h]
            assert np.array_equal(blk, pages[page, h]), (page, h)
    # back, with the rows behind the last sequence untouched
    back = [torch.full((rows + extra, nkv, hd), 11.0, device="cuda") for _ in range(2)]
    cache.c.load(cu_of(new), ints(held), *back)
    for got, x in zip(back, (kn, vn)):
        assert np.array_equal(got[:rows].cpu().numpy(), np_values(x)) and bool((got[rows:] == 11).all())
    only = torch.zeros(rows, nkv, hd, dtype=torch.bfloat16, device="cuda")
    cache.c.load(cu_of(new), ints(held), v=only)
    assert torch.equal(only, back[1][:rows].bfloat16())
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:overflow")  # some minima are beyond f16
def test_kv4_store_at_the_borders_between_codes(rrr, ctx):
    """Values half way between two codes and the next ones above and below, for steps of all sizes
    and minima far from zero: the division of the formula decides, bit by bit."""
    pick, hd, rows = np.random.default_rng(5), 128, 960
    x = np.empty((rows, hd // 32, 32), np.float32)
    for r in range(rows):
        for j in range(hd // 32):
            d = np.float32(np.float16(2.0 ** pick.uniform(-20, 10)))
            m = np.float32(np.float16(d * pick.choice([0, 1, -7.3, 100.0, -3000.0])))
            half = (m + d * (pick.integers(0, 15, 30) + 0.5).astype(np.float32)).astype(np.float32)
            step = pick.integers(-2, 3, 30)
            for _ in range(2):
                half = np.where(step > 0, np.nextafter(half, np.float32(np.inf)), np.where(step < 0, np.nextafter(half, np.float32(-np.inf)), half))
                step -= np.sign(step)
            x[r, j] = pick.permutation(np.concatenate([[m, m + 15 * d], half]).astype(np.float32))
    x = x.reshape(rows, 1, hd)
    t = torch.from_numpy(x).cuda()
    cache = Cache(rrr, ctx, 1, hd, [rows], 2)
    back = [torch.empty_like(t) for _ in range(2)]
    cache.c.store(t, t, ints([0, rows]), ints([rows]))
    cache.c.load(ints([0, rows]), ints([rows]), *back)
    for b in back:
        assert np.array_equal(b.cpu().numpy(), np_values(x), equal_nan=True)


@pytest.mark.gpu
def test_kv4_rows_that_are_not_finite_and_places_that_do_not_exist(rrr, ctx):
    cache = Cache(rrr, ctx, 1, 64, [70, 70], 1)
    x = normal(gen(1), 4, 64)
    x[0, 3], x[1, 40], x[2, 0] = math.nan, math.inf, -math.inf
    cache.c.store(x, x, ints([0, 4, 4]), ints([70, 70]))
    back = [torch.zeros(4, 1, 64, device="cuda") for _ in range(2)]
    cache.c.load(ints([0, 4, 4]), ints([70, 70]), *back)
    bad = torch.tensor([[1, 0], [0, 1], [1, 0], [0, 0]], device="cuda").bool().repeat_interleave(32, 1)
    for b in back:
        assert torch.equal(b[:, 0].isnan(), bad)
    was = cache.pages.clone()
    cache.c.store(x, x, ints([0, 4, 4]), ints([3, 70]))       # a row before the start
    assert ctx.device_error() == 6
    assert not torch.equal(cache.pages, was)                   # the others are stored
    was = cache.pages.clone()
    for lens, table in (([200, 70], None), ([70, 70], [[0, -1], [0, 1]]), ([70, 70], [[0, 10 ** 6], [0, 1]])):
        c = cache.c if table is None else rrr.KV4Cache(ctx, cache.pages, ints(table), 64)
        c.store(x, x, ints([0, 4, 4]), ints(lens))
        assert ctx.device_error() == 6 and torch.equal(cache.pages, was)


# ------------------------------------------------------------------ decode
def filled(rrr, ctx, nkv, hd, lens, seed, kind=torch.float32, spread=1.0, **over):
    """A cache with random rows and its K and V in 64 bits per sequence."""
    g = gen(seed)
    cache = Cache(rrr, ctx, nkv, hd, lens, seed, **over)
    rows = sum(lens)
    k = normal(g, rows, nkv, hd) * torch.exp(0.5 * normal(g, nkv, hd)) * spread
    v = normal(g, rows, nkv, hd) + 0.3
    cache.c.store(k, v, cu_of(lens), ints(lens))
    kk, vv = torch.empty(rows, nkv, hd, device="cuda"), torch.empty(rows, nkv, hd, device="cuda")
    cache.c.load(cu_of(lens), ints(lens), kk, vv)
    cu = np.cumsum([0] + list(lens))
    return cache, [(kk[a:b].double(), vv[a:b].double()) for a, b in zip(cu, cu[1:])]


def check_decode(got, q, kv, scale, t):
    for s, (k, v) in enumerate(kv):
        if k.shape[0] == 0:
            assert bool((got[s] == 0).all())
            continue
        ref, A = ref_attention(q[s].double(), k, v, k.shape[0], scale)
        err = U * (2 * (48 * A + 8) + k.shape[0] / 64 + 64)
        bound = err[:, None] * float(v.abs().max()) + (0.0 if t == torch.float32 else half_step(t) * 1.01) * ref.abs()
        within(got[s], ref, bound + (2.0 ** -25 if t == torch.float16 else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(128, 24, 8), (64, 8, 1), (64, 5, 5), (256, 6, 2), (256, 8, 1), (128, 8, 8)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens", [[1], [17, 0, 64, 65, 1, 16, 15], [1023], [3000, 1, 130, 700]])
def test_attention_kv4(rrr, ctx, hd, nh, nkv, kind, lens):
    t = DT[kind]
    cache, kv = filled(rrr, ctx, nkv, hd, lens, hd + len(lens))
    g = gen(11)
    wide = normal(g, len(lens), nh * hd + 16, dtype=t)
    q = wide[:, 8:8 + nh * hd].unflatten(1, (nh, hd))
    if len(lens) > 1:
        q[1] = 0.0
        q[2] *= 1e-3
    out = torch.full((len(lens), nh * hd + 8), 5.0, dtype=t, device="cuda")
    o = out[:, :nh * hd].unflatten(1, (nh, hd))
    ws = cache.c.workspace(nh).fill_(0xff)  # whatever it holds
    for scale in (0.0, 0.31):
        cache.c.attention(q, ints(lens), o, ws, scale=scale)
        check_decode(o, q, kv, scale or 1 / math.sqrt(hd), t)
    again = torch.empty_like(o)
    cache.c.attention(q, ints(lens), again, ws, scale=0.31)
    assert torch.equal(o, again) and bool((out[:, nh * hd:] == 5).all())
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("hpk", [5, 6, 7, 8])
def test_attention_kv4_query_heads_per_kv_head(rrr, ctx, hd, hpk):
    lens, nkv = [130, 1, 0, 1000], 3
    cache, kv = filled(rrr, ctx, nkv, hd, lens, hpk)
    q = normal(gen(hpk), len(lens), nkv * hpk, hd)
    out = torch.empty_like(q)
    cache.c.attention(q, ints(lens), out, cache.c.workspace(nkv * hpk).fill_(0xff))
    check_decode(out, q, kv, 1 / math.sqrt(hd), torch.float32)


@pytest.mark.gpu
def test_attention_kv4_long_context_and_offsets_over_32_bits(rrr, ctx):
    """One sequence of 70,001 rows on pages that lie past 4 GB."""
    first = 53000
    cache, kv = filled(rrr, ctx, 8, 128, [70001], 2, first_page=first)
    assert first * 8 * 80 * 128 > 2 ** 32
    q = normal(gen(5), 1, 24, 128)
    out = torch.empty_like(q)
    cache.c.attention(q, ints([70001]), out, cache.c.workspace(24))
    check_decode(out, q, kv, 1 / math.sqrt(128), torch.float32)


@pytest.mark.gpu
def test_attention_kv4_many_sequences(rrr, ctx):
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 200, 700)]
    cache, kv = filled(rrr, ctx, 2, 64, lens, 3)
    q = normal(gen(6), len(lens), 4, 64, dtype=torch.bfloat16)
    out = torch.empty_like(q)
    cache.c.attention(q, ints(lens), out, cache.c.workspace(4))
    check_decode(out, q, kv, 1 / 8, torch.bfloat16)


@pytest.mark.gpu
def test_attention_kv4_rows_that_hold_nothing_never_count(rrr, ctx):
    """NaN and infinite scales in the rest of a page, pages that do not exist, lengths outside."""
    lens = [33, 70, 1]
    cache, kv = filled(rrr, ctx, 2, 128, lens, 4, fill=0xFF)  # 0xffff is a NaN scale
    q = normal(gen(7), 3, 6, 128)
    out, ws = torch.empty_like(q), cache.c.workspace(6)
    cache.c.attention(q, ints(lens), out, ws)
    check_decode(out, q, kv, 1 / math.sqrt(128), torch.float32)
    good = out.clone()
    cache.c.attention(q, ints([33, -1, 10 ** 9]), out, ws)
    assert ctx.device_error() == 6
    assert torch.equal(out[0], good[0]) and bool((out[1:] == 0).all())
    table = cache.table.copy()
    table[1, 1] = 10 ** 6
    c = rrr.KV4Cache(ctx, cache.pages, torch.from_numpy(table).cuda(), 128)
    c.attention(q, ints(lens), out, ws)
    assert ctx.device_error() == 6
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    ref, _ = ref_attention(q[1].double(), kv[1][0], kv[1][1], 64, 1 / math.sqrt(128))
    assert float((out[1] - ref).abs().max()) < 1e-4  # its first page alone
    # values that are there do count: a NaN row makes its sequence NaN and no other
    x = torch.full((1, 2, 128), math.nan, device="cuda")
    cache.c.store(x, x, ints([0, 0, 1, 1]), ints(lens))
    cache.c.attention(q, ints(lens), out, ws)
    assert bool(out[1].isnan().all()) and torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])


@pytest.mark.gpu
def test_attention_kv4_extreme_scores(rrr, ctx):
    """Scores of thousands (one weight takes all), tiny and huge queries, large values."""
    cache, kv = filled(rrr, ctx, 1, 128, [500, 500, 500], 8, spread=30.0)
    q = normal(gen(9), 3, 2, 128) * torch.tensor([20.0, 1e-20, 1e20], device="cuda")[:, None, None]
    out = torch.empty_like(q)
    cache.c.attention(q, ints([500] * 3), out, cache.c.workspace(2))
    # 1e-20: the mean; 1e20: the row of the largest score
    mean = kv[1][1].mean(0)[0]
    assert float((out[1] - mean).abs().max()) < 1e-4
    for h in range(2):
        best = int((kv[2][0][:, 0] @ q[2, h].double()).argmax())
        assert float((out[2, h] - kv[2][1][best, 0]).abs().max()) < 1e-4
        best = (kv[0][0][:, 0] @ q[0, h].double()).topk(2)
        if float(best.values[0] - best.values[1]) / math.sqrt(128) > 50:
            assert float((out[0, h] - kv[0][1][int(best.indices[0]), 0]).abs().max()) < 1e-4


# ------------------------------------------------------------------ prompts
def check_packed(got, q, k, v, lq, lk, causal, scale, before=None):
    t = q.dtype
    cq, ck = np.cumsum([0] + list(lq)), np.cumsum([0] + list(lk))
    nh, hd = q.shape[1:]
    for s in range(len(lq)):
        a, b = cq[s], cq[s + 1]
        if a == b:
            continue
        kk, vv = k[ck[s]:ck[s + 1]].double(), v[ck[s]:ck[s + 1]].double()
        hpk = nh // k.shape[1]
        kk, vv = (x.repeat_interleave(hpk, 1).transpose(0, 1) for x in (kk, vv))  # [nh, lk, hd]
        qq = q[a:b].double().transpose(0, 1)
        n = kk.shape[1]
        seen = torch.ones(b - a, n, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril(n - (b - a))
        some = seen.any(-1)
        sc = (qq @ kk.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        A = (qq.abs() @ kk.abs().transpose(1, 2) * scale * seen).amax(-1) if n else torch.zeros(nh, b - a, device="cuda")
        p = torch.softmax(sc, -1) if n else sc
        ref = torch.where(some[:, None], (p.nan_to_num(0) if not bool(some.all()) else p) @ vv, 0.0) if n else torch.zeros_like(qq)
        top = float(vv.abs().max()) if n else 0.0
        err = U * (2 * ((hd + 16) * A + 8) + n / 16 + 64) + half_step(t) * 1.01
        bound = err[..., None] * top + half_step(t) * 1.01 * ref.abs() + (2.0 ** -25 if t == torch.float16 else 0)
        within(got[a:b].transpose(0, 1), ref, bound)
        assert bool((got[a:b][~some] == 0).all())
    if before is not None:
        assert torch.equal(got[cq[-1]:], before[cq[-1]:])


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(128, 6, 2), (64, 8, 1), (256, 4, 2), (128, 3, 3)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lq,lk", [
    ([1], [1]), ([127, 1, 0, 130, 64], None), ([513], None), ([5, 1, 300, 0], [400, 129, 301, 7]),
    ([10, 200, 3], [4, 0, 3]), ([128, 256, 129], None), ([700], [1500])])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_packed(rrr, ctx, hd, nh, nkv, kind, lq, lk, causal):
    t, g = DT[kind], gen(sum(lq) + hd)
    lk = lq if lk is None else lk
    extra = 3
    q, k, v = (normal(g, sum(n) + extra, h, hd, dtype=t) for n, h in ((lq, nh), (lk, nkv), (lk, nkv)))
    # rows that belong to no sequence hold anything
    for x, n in ((k, lk), (v, lk)):
        x[sum(n):] = math.nan
    out = torch.full_like(q, 3.0)
    before = out.clone()
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), out, causal=causal)
    check_packed(out, q, k, v, lq, lk, causal, 1 / math.sqrt(hd), before)
    again = before.clone()
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), again, causal=causal)
    assert torch.equal(out, again)
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nh", [43, 100, 128, 130])
def test_attention_packed_many_query_heads_per_kv_head(rrr, ctx, hd, nh):
    g, lq, lk, t = gen(nh), [3, 70, 1], [3, 200, 300], torch.bfloat16
    q, k, v = (normal(g, sum(n), h, hd, dtype=t) for n, h in ((lq, nh), (lk, 1), (lk, 1)))
    out = torch.full_like(q, 3.0)
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), out)
    check_packed(out, q, k, v, lq, lk, True, 1 / math.sqrt(hd))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [128, 256])
def test_attention_packed_many_blocks(rrr, ctx, hd):
    """Long enough for every ring to go round several times, and for maxima that keep growing: the
    sums of a row are rescaled in every block."""
    g, n, t = gen(hd), 2300, torch.bfloat16
    q, k, v = (normal(g, n, h, hd, dtype=t) for h in (2, 1, 1))
    k *= torch.linspace(0.05, 6, n, device="cuda")[:, None, None].to(t)
    out = torch.empty_like(q)
    rrr.attention_packed(ctx, q, k, v, cu_of([n]), cu_of([n]), out)
    check_packed(out, q, k, v, [n], [n], True, 1 / math.sqrt(hd))
    again = torch.empty_like(q)
    rrr.attention_packed(ctx, q, k, v, cu_of([n]), cu_of([n]), again)
    assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["qkv rows", "heads of rows", "odd pitch"])
def test_attention_packed_strides(rrr, ctx, layout):
    g, nh, nkv, hd, lens = gen(4), 4, 2, 128, [100, 257]
    rows, t = sum(lens), torch.bfloat16
    if layout == "qkv rows":
        x = normal(g, rows, nh + 2 * nkv, hd, dtype=t)
        q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
        out = torch.empty(rows, nh, hd, dtype=t, device="cuda")
    elif layout == "heads of rows":
        q, k, v, out = (normal(g, h, rows, hd, dtype=t).transpose(0, 1) for h in (nh, nkv, nkv, nh))
    else:
        q, k, v, out = (normal(g, rows + 1, h + 1, hd + 8, dtype=t)[1:, :h, 8:] for h in (nh, nkv, nkv, nh))
    rrr.attention_packed(ctx, q, k, v, cu_of(lens), cu_of(lens), out, scale=0.2)
    check_packed(out, q, k, v, lens, lens, True, 0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_packed_masked_values_that_are_not_finite(rrr, ctx, hd):
    """Infinite and NaN keys and values reach the rows that see them and no others; rows of
    queries that are NaN stay to themselves."""
    g, nh, nkv, lens = gen(8), 2, 1, [200, 150]
    t = torch.float16
    q, k, v = (normal(g, 350, h, hd, dtype=t) for h in (nh, nkv, nkv))
    v[77, 0, 5], v[300, 0, 9], k[120, 0, 3], q[20, 1, 0] = math.inf, math.nan, math.nan, math.nan
    out = torch.empty_like(q)
    rrr.attention_packed(ctx, q, k, v, cu_of(lens), cu_of(lens), out)
    kf, vf, qf = k.clone(), v.clone(), q.clone()
    vf[77, 0, 5], vf[300, 0, 9], kf[120, 0, 3], qf[20, 1, 0] = 0, 0, 0, 0
    plain = torch.empty_like(q)
    rrr.attention_packed(ctx, qf, kf, vf, cu_of(lens), cu_of(lens), plain)
    want = plain.clone()
    want[77:200, :, 5] = math.inf
    want[120:200] = math.nan
    want[300:, :, 9] = math.nan
    want[20, 1] = math.nan
    assert torch.equal(want.isnan(), out.isnan()) and torch.equal(want.isinf(), out.isinf())
    fine = torch.isfinite(want)
    assert float((out - plain)[fine].float().abs().max()) <= 4 * half_step(t) * float(v.nan_to_num(0, 0, 0).abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_packed_many_values_that_are_not_finite(rrr, ctx, hd):
    """Values of every later row infinite in one place, before and behind what a row sees: the rows
    that see none keep theirs, the others are infinite there and nowhere else. One infinite key, or
    NaN queries of every row, leave NaN rows; none of these takes the time of a row by row pass."""
    g, nh, nkv, n = gen(9), 4, 2, 1500
    q, k, v = (normal(g, n, h, hd, dtype=torch.bfloat16) for h in (nh, nkv, nkv))
    plain, out = torch.empty_like(q), torch.empty_like(q)
    cu = ints([0, n])
    rrr.attention_packed(ctx, q, k, v, cu, cu, plain)
    vf = v.clone()
    vf[700:, 1, 3] = math.inf
    rrr.attention_packed(ctx, q, k, vf, cu, cu, out)
    want = plain.clone()
    want[700:, 2:, 3] = math.inf
    assert torch.equal(torch.isinf(want), torch.isinf(out)) and not bool(out.isnan().any())
    fine = torch.isfinite(want)
    assert float((out - plain)[fine].float().abs().max()) <= 4 * half_step(torch.bfloat16) * float(v.abs().max())
    for x in (k, q):
        kept = x.clone()
        x[100 if x is k else slice(None), 0, 1] = math.nan
        rrr.attention_packed(ctx, q, k, v, cu, cu, out)
        heads = slice(0, nh // nkv) if x is k else slice(0, 1)
        first = 100 if x is k else 0
        assert bool(out[first:, heads].isnan().all())
        want = plain.clone()
        want[first:, heads] = math.nan
        assert torch.equal(want.isnan(), out.isnan())
        x.copy_(kept)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(128, 24, 8), (64, 24, 8), (128, 4, 1), (64, 5, 5), (256, 4, 2)])
@pytest.mark.parametrize("lq,lk", [([1], [3000]), ([37], [2111]), ([100], [2048]), ([3, 0, 50], [2500, 900, 2600]), ([700], [1600])])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_packed_few_rows_on_many(rrr, ctx, hd, nh, nkv, lq, lk, causal):
    """Few tiles: the KV rows of one are shared by several CTAs, some of which see none of them."""
    g, t = gen(sum(lq) + hd), torch.bfloat16
    q, k, v = (normal(g, sum(n) + 2, h, hd, dtype=t) for n, h in ((lq, nh), (lk, nkv), (lk, nkv)))
    k[sum(lk):], v[sum(lk):] = math.nan, math.inf
    out = torch.full_like(q, 3.0)
    before = out.clone()
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), out, causal=causal)
    check_packed(out, q, k, v, lq, lk, causal, 1 / math.sqrt(hd), before)
    again = before.clone()
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), again, causal=causal)
    assert torch.equal(out, again) and ctx.device_error() == 0
    # an infinite value that the last row alone sees, in one head
    if causal and len(lq) == 1 and lq[0] > 1:
        v[lk[0] - 1, 0, 7] = math.inf
        rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), again)
        want = out.clone()
        want[lq[0] - 1, :nh // nkv, 7] = math.inf
        assert torch.equal(want.isinf(), again.isinf()) and not bool(again[:lq[0]].isnan().any())
        fine = torch.isfinite(want)
        assert float((again - out)[fine].float().abs().max()) <= 4 * half_step(t) * float(v[:lk[0]].nan_to_num(0, 0, 0).abs().max())


@pytest.mark.gpu
def test_attention_packed_bad_row_starts(rrr, ctx):
    q = normal(gen(1), 64, 2, 64, dtype=torch.float16)
    out = torch.full_like(q, 2.0)
    for cu_q, cu_kv in (([0, 65], [0, 64]), ([0, 64], [0, 65]), ([5, 3], [0, 64]), ([-1, 64], [0, 64]), ([0, 64], [9, 3])):
        rrr.attention_packed(ctx, q, q, q, ints(cu_q), ints(cu_kv), out)
        assert ctx.device_error() == 6 and bool((out == 2).all())
    rrr.attention_packed(ctx, q, q[:0], q[:0], ints([0, 64]), ints([0, 0]), out)
    assert ctx.device_error() == 0 and bool((out == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_packed_shared_items_on_two_streams_and_with_bad_row_starts(rrr, ctx, hd):
    g, t = gen(hd), torch.float16
    q, k, v = (normal(g, n, 2, hd, dtype=t) for n in (50, 3000, 3000))
    out = torch.full_like(q, 2.0)
    for cu_q, cu_kv in (([0, 51], [0, 3000]), ([0, 50], [0, 3001]), ([5, 3], [0, 3000]), ([-1, 50], [0, 3000]), ([0, 50], [9, 3])):
        rrr.attention_packed(ctx, q, k, v, ints(cu_q), ints(cu_kv), out)
        assert ctx.device_error() == 6 and bool((out == 2).all())
    streams, outs = [torch.cuda.Stream() for _ in range(3)], [torch.empty_like(q) for _ in range(3)]
    cq, ck = ints([0, 50]), ints([0, 3000])
    rrr.attention_packed(ctx, q, k, v, cq, ck, out)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o in zip(streams, outs):
            rrr.attention_packed(ctx, q, k, v, cq, ck, o, stream=s)
    torch.cuda.synchronize()
    check_packed(out, q, k, v, [50], [3000], True, 1 / math.sqrt(hd))
    assert all(torch.equal(o, out) for o in outs) and ctx.device_error() == 0


@pytest.mark.gpu
def test_attention_packed_large_scores(rrr, ctx):
    """Scores in the thousands: the running maximum keeps every weight at or below one."""
    g, lens = gen(2), [300]
    q, k, v = (normal(g, 300, 1, 128, dtype=torch.bfloat16) for _ in range(3))
    q, k = q * 40, k * 40
    out = torch.empty_like(q)
    rrr.attention_packed(ctx, q, k, v, cu_of(lens), cu_of(lens), out)
    s = q[:, 0].double() @ k[:, 0].double().T / math.sqrt(128)
    s = s.masked_fill(~torch.ones_like(s).tril().bool(), -math.inf)
    top = s.topk(2, -1)
    sure = (top.values[:, 0] - top.values[:, 1]) > 40
    best = v[top.indices[:, 0], 0]
    assert int(sure.sum()) > 200 and torch.equal(out[sure, 0], best[sure])


# ------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("hd,rd,halves,norm", [(128, 96, False, False), (64, 64, True, True)])
def test_a_batch_from_its_prompts_to_its_tokens(rrr, ctx, hd, rd, halves, norm):
    """Prompts through norm + rotation, cache and packed attention, a continued prompt over its
    loaded prefix, then single tokens over the 4-bit cache, in a captured graph too."""
    nh, nkv, t = 6, 2, torch.bfloat16
    g = gen(hd)
    width = (nh + 2 * nkv) * hd
    prompts, tokens = [90, 1, 200], 3
    most = [n + 40 + tokens for n in prompts]
    cache = Cache(rrr, ctx, nkv, hd, most, 3, fill=0)
    gammas = [torch.rand(hd, device="cuda", generator=g) + 0.5 if norm else None for _ in range(2)]
    desc = rrr.ffi.AttnDesc(nh, nkv, hd, rd, 10000.0, 1.19, None, 0, 4096)
    hist = [[] for _ in prompts]  # dequantised K, V of every sequence, 64 bits

    def step(rows_of, positions, held, kv_from_cache):
        rows = sum(rows_of)
        qkv = normal(g, rows, width)
        pos = ints(positions)
        q, k, v = (torch.empty(rows, n, hd, dtype=t, device="cuda") for n in (nh, nkv, nkv))
        rrr.qk_norm_rope(ctx, desc, qkv, pos, q, k, v, q_gamma=gammas[0], k_gamma=gammas[1], halves=halves)
        refs, mags = ref_qk(qkv, pos, nh, nkv, hd, rd, 10000.0, 1.19, None, gammas, 1e-5, halves)
        for got, ref, mag in zip((q, k, v), refs, mags):
            within(got, ref, ref.abs() * half_step(t) * 1.01 + 32 * U * mag + 1e-30)
        cache.c.store(k, v, cu_of(rows_of), ints(held))
        return q, k, v

    q, k, v = step(prompts, [i for n in prompts for i in range(n)], prompts, False)
    out = torch.empty_like(q)
    rrr.attention_packed(ctx, q, k, v, cu_of(prompts), cu_of(prompts), out)
    check_packed(out, q, k, v, prompts, prompts, True, 1 / math.sqrt(hd))
    # a continued prompt: the new rows see the cache's values of the old ones
    more = [40, 0, 17]
    held = [a + b for a, b in zip(prompts, more)]
    q, _, _ = step(more, [p + i for p, n in zip(prompts, more) for i in range(n)], held, True)
    kk, vv = (torch.empty(sum(held), nkv, hd, dtype=t, device="cuda") for _ in range(2))
    cache.c.load(cu_of(held), ints(held), kk, vv)
    out = torch.empty_like(q)
    rrr.attention_packed(ctx, q, kk, vv, cu_of(more), cu_of(held), out)
    check_packed(out, q, kk, vv, more, held, True, 1 / math.sqrt(hd))
    # single tokens: eager, then the same calls as a graph that replays with other lengths
    n = len(prompts)
    qkv, lens, pos = torch.empty(n, width, device="cuda"), ints(held), ints(held)
    q, k, v = (torch.empty(n, h, hd, dtype=t, device="cuda") for h in (nh, nkv, nkv))
    out, ws, cu = torch.empty_like(q), cache.c.workspace(nh), cu_of([1] * n)

    def token(stream):
        rrr.qk_norm_rope(ctx, desc, qkv, pos, q, k, v, q_gamma=gammas[0], k_gamma=gammas[1], halves=halves, stream=stream)
        cache.c.store(k, v, cu, lens, stream=stream)
        cache.c.attention(q, lens, out, ws, stream=stream)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    for i in range(tokens):
        held = [h + 1 for h in held]
        qkv.copy_(normal(g, n, width))
        lens.copy_(ints(held))
        pos.copy_(ints([h - 1 for h in held]))
        torch.cuda.synchronize()
        if i == 0:
            token(None)
        elif i == 1:
            with torch.cuda.graph(graph, stream=side):
                token(torch.cuda.current_stream())
            graph.replay()
        else:
            graph.replay()
        torch.cuda.synchronize()
        kk, vv = (torch.empty(sum(held), nkv, hd, device="cuda") for _ in range(2))
        cache.c.load(cu_of(held), ints(held), kk, vv)
        c = np.cumsum([0] + held)
        check_decode(out, q, [(kk[a:b].double(), vv[a:b].double()) for a, b in zip(c, c[1:])], 1 / math.sqrt(hd), t)
        new = [x[h - 1] for x, h in ((kk[a:b], b - a) for a, b in zip(c, c[1:]))]
        assert torch.equal(torch.stack(new).cpu(), torch.from_numpy(np_values(k.float().cpu().numpy())))
    assert ctx.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_captured_calls_replay_with_other_lengths(rrr, ctx, hd):
    """One graph of prompt attention and one of a decode step over batches of other shapes: lengths
    and row starts are the device's, so nothing of the capture's batch may remain."""
    g, nh, nkv, t = gen(hd), 6, 2, torch.bfloat16
    batches = [([40, 300, 7], [40, 300, 7]), ([1, 1, 1], [500, 0, 130]), ([0, 600, 0], [0, 600, 0]), ([129, 200, 30], [140, 333, 30])]
    q, k, v = (normal(g, 700, h, hd, dtype=t) for h in (nh, nkv, nkv))
    cq, ck, out = ints([0] * 4), ints([0] * 4), torch.empty_like(q)
    lens = [[5, 0, 64], [3000, 1, 700], [0, 0, 0], [64, 2999, 65]]
    cache, kv = filled(rrr, ctx, nkv, hd, [3000] * 3, hd)
    dq, dlens = normal(g, 3, nh, hd), ints([0] * 3)
    dout, ws = torch.empty_like(dq), cache.c.workspace(nh).fill_(0xff)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        stream = torch.cuda.current_stream()
        rrr.attention_packed(ctx, q, k, v, cq, ck, out, stream=stream)
        cache.c.attention(dq, dlens, dout, ws, stream=stream)
    for (lq, lk), n in zip(batches, lens):
        out.fill_(2.0)
        before = out.clone()
        cq.copy_(cu_of(lq))
        ck.copy_(cu_of(lk))
        dlens.copy_(ints(n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_packed(out, q, k, v, lq, lk, True, 1 / math.sqrt(hd), before)
        check_decode(dout, dq, [(a[:m], b[:m]) for (a, b), m in zip(kv, n)], 1 / math.sqrt(hd), torch.float32)
    assert ctx.device_error() == 0


@pytest.mark.gpu
def test_two_streams_with_a_workspace_each(rrr, ctx):
    cache, kv = filled(rrr, ctx, 8, 128, [9000, 300], 6)
    q = [normal(gen(i), 2, 24, 128) for i in range(2)]
    outs, ws = [torch.empty_like(x) for x in q], [cache.c.workspace(24) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    lens = ints([9000, 300])
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            cache.c.attention(q[i], lens, outs[i], ws[i], stream=streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        check_decode(outs[i], q[i], kv, 1 / math.sqrt(128), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nh,nkv", [(128, 3, 1), (64, 8, 2), (256, 2, 2)])
def test_attention_packed_many_sequences(rrr, ctx, hd, nh, nkv):
    """More sequences than one search over lengths takes, and more items than the GPU has SMs."""
    r = np.random.default_rng(hd)
    lq = [int(x) for x in r.integers(0, 90, 300)]
    lk = [int(x) + int(y) for x, y in zip(lq, r.integers(0, 200, 300))]
    g, t = gen(hd), torch.bfloat16
    q, k, v = (normal(g, sum(n), h, hd, dtype=t) for n, h in ((lq, nh), (lk, nkv), (lk, nkv)))
    out = torch.full_like(q, 3.0)
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), out)
    check_packed(out, q, k, v, lq, lk, True, 1 / math.sqrt(hd))
    lq, lk = lq[:40] + [1500], lk[:40] + [2100]
    q, k, v = (normal(g, sum(n), h, hd, dtype=t) for n, h in ((lq, nh), (lk, nkv), (lk, nkv)))
    out = torch.full_like(q, 3.0)
    rrr.attention_packed(ctx, q, k, v, cu_of(lq), cu_of(lk), out)
    check_packed(out, q, k, v, lq, lk, True, 1 / math.sqrt(hd))
