"""The packed-batch operators where a plain comparison of random values sees little: arrays that
share a buffer, calls of two host threads. Formulas and helpers are test_serving.py's."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

from test_serving import DT, FINE, ROOT, _no_gpu, cu_of, filled, gen, host_ctx, ints, normal  # noqa: F401


class KV4Call(ctypes.Structure):  # tests/cpp/two_threads.cpp
    _fields_ = [("ctx", ctypes.c_void_p), ("cache", ctypes.c_void_p), ("n_heads", ctypes.c_int), ("type", ctypes.c_int),
                ("q", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("kv_lens", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_int64), ("stream", ctypes.c_void_p)]


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


# ------------------------------------------------------------------ GPU
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
    for _, out, first, _, own, _ in keep:
        assert code == 0, rrr.ffi.last_error(own.h)
        assert torch.equal(out, first) and own.device_error() == 0
        own.close()
