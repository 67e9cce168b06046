"""Two host threads with a context each on one GPU, in kernels whose shared memory depends on the
batch: the limit that a launch needs is the function's, not the context's."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class GemmCall(ctypes.Structure):  # tests/cpp/two_threads.cpp
    _fields_ = [("ctx", ctypes.c_void_p), ("w", ctypes.c_void_p), ("x", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("m", ctypes.c_int), ("k", ctypes.c_int), ("n", ctypes.c_int), ("qtype", ctypes.c_int),
                ("stream", ctypes.c_void_p)]


@pytest.fixture(scope="module")
def two_threads(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("two") / "two_threads.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-pthread",
                    os.path.join(ROOT, "tests", "cpp", "two_threads.cpp"), "-o", so], check=True)
    return ctypes.CDLL(so)


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["q4_k", "q5_k", "q6_k", "logits"])
def test_batches_of_16_and_256_rows(rrr, ctx, torch_cuda, two_threads, case):
    torch, L, k, n = torch_cuda, rrr.ffi.lib(), 2048, 256
    qtype = {"q4_k": rrr.ffi.Q4_K, "q5_k": rrr.ffi.Q5_K, "q6_k": rrr.ffi.Q6_K, "logits": 0}[case]
    if qtype:
        block = {12: 144, 13: 176, 14: 210}[qtype]
        w = torch.empty(n * k // 256 * block, dtype=torch.uint8, device="cuda")
        ctx.check(L.rrr_fill_kquant_random(ctx.h, qtype, w.data_ptr(), n * k // 256, 5, None))
        entry, repeat = L.rrr_gemm_kq_batched_path, two_threads.repeat_gemm_kq_tc
    else:
        w = torch.randn(n, k, device="cuda")
        entry, repeat = L.rrr_logits_f32_batched, two_threads.repeat_logits
    calls, keep = (GemmCall * 2)(), []
    for i, m in enumerate((16, 256 if qtype else 128)):
        x = torch.randn(m, k, device="cuda").to(torch.bfloat16 if qtype else torch.float32)
        y, first, own, stream = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda"), rrr.Context(0), torch.cuda.Stream()
        if qtype:
            ctx.check(entry(ctx.h, qtype, w.data_ptr(), x.data_ptr(), first.data_ptr(), m, k, n, None, 1, None))
        else:
            ctx.check(entry(ctx.h, w.data_ptr(), x.data_ptr(), first.data_ptr(), first.data_ptr(), m, n, k, None, 0.0, None))
        calls[i] = GemmCall(own.h, w.data_ptr(), x.data_ptr(), y.data_ptr(), m, k, n, qtype, stream.cuda_stream)
        keep.append((x, y, first, own, stream))
    torch.cuda.synchronize()
    code = repeat(ctypes.cast(entry, ctypes.c_void_p), calls, 30000)
    torch.cuda.synchronize()
    assert code == 0, [rrr.ffi.last_error(x[3].h) for x in keep]
    for _, y, first, own, _ in keep:
        assert torch.equal(y, first) and own.device_error() == 0
        own.close()
