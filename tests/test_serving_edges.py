"""The packed-batch operators where a plain comparison of random values sees little: calls of two
host threads. Formulas and helpers are test_serving.py's."""
import ctypes
import os
import subprocess

import pytest
import torch

from test_serving import ROOT, filled, gen, ints, normal


class KV4Call(ctypes.Structure):  # tests/cpp/two_threads.cpp
    _fields_ = [("ctx", ctypes.c_void_p), ("cache", ctypes.c_void_p), ("n_heads", ctypes.c_int), ("type", ctypes.c_int),
                ("q", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("kv_lens", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("out_stride", ctypes.c_int64), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_int64), ("stream", ctypes.c_void_p)]


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
