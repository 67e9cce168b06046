"""Python host of the packed-batch operators of include/rrr_cuda.h on torch CUDA tensors:
per-head norms with rotation of QKV rows, packed prompt attention, and the 4-bit KV cache
with its decode attention. The rows of the sequences of a batch lie one after another; cu is
an int32 tensor of n_seqs + 1 ascending row starts.

Tensors are checked for device, type, shape and contiguity of their last dimension; the C ABI
checks strides, alignment and overlap. `stream`: a torch stream, an int, or None (torch's current
stream of the context's GPU); a tensor made on another stream is the caller's to order."""
from __future__ import annotations

import ctypes
import struct
from ctypes import byref, c_int64

from . import ffi
from .engine import _stream as _handle

PAGE_ROWS = 64
_TYPES: dict = {}  # torch dtype -> GGML type id
_INTS: set = set()  # torch dtypes of 32-bit integers
_torch = None
# The fields of a PackedDesc, packed: a third of the time of its constructor
_packed = struct.Struct("@6if10q").pack


def _type(t, what: str) -> int:
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: ffi.F32, torch.float16: ffi.F16, torch.bfloat16: ffi.BF16})
    got = _TYPES.get(t.dtype)
    if got is None:
        raise ffi.RRRError(-2, f"{what}: float32, float16 or bfloat16 is needed, got {t.dtype}")
    return got


def _fail(code: int, message: str):
    raise ffi.RRRError(code, message)


def _stream(ctx: ffi.Context, stream):
    global _torch
    if stream is not None:
        return _handle(stream)
    if _torch is None:
        import torch as _torch
    return _torch._C._cuda_getCurrentRawStream(ctx.device)  # current_stream() without its object


def _on(ctx: ffi.Context, t, what: str):
    """t's device address, checked to be on the context's GPU."""
    if t.get_device() != ctx.device:
        _fail(-1, f"{what}: a tensor on cuda:{ctx.device} is needed, got one on {t.device}")
    return t.data_ptr()


def _ints(ctx: ffi.Context, t, n: int, what: str):
    if t.dtype not in _INTS or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        if not _INTS:
            import torch
            _INTS.update({torch.int32, torch.uint32})
            return _ints(ctx, t, n, what)
        _fail(-3, f"{what}: a contiguous int32[{n}] is needed, got {t.dtype}{list(t.shape)}")
    return _on(ctx, t, what)


def _heads(ctx: ffi.Context, t, heads: int, hd: int, what: str, rows: int | None = None):
    """[rows, heads, hd] (or [rows, heads * hd]) with the heads of a row next to each other:
    (address, rows, row stride)."""
    shape = t.shape
    n = shape[0]
    if len(shape) == 3:
        fine = shape[1] == heads and shape[2] == hd
    else:
        fine = len(shape) == 2 and shape[1] == heads * hd
    row = heads * hd
    if not t.is_contiguous():
        stride = t.stride()
        fine = fine and stride[-1] == 1 and (len(shape) == 2 or heads == 1 or stride[1] == hd)
        if n > 1:
            row = stride[0]
    if not fine or (rows is not None and n != rows):
        _fail(-3, f"{what}: rows [{'rows' if rows is None else rows}, {heads}, {hd}] with their heads next to "
                  f"each other are needed, got {list(shape)} with strides {list(t.stride())}")
    return _on(ctx, t, what), n, row


def _strides(t, rows: int, heads: int, hd: int, what: str):
    """Row and head strides of [rows, heads, hd]; the stride of a dimension of one is free."""
    if t.is_contiguous():
        return heads * hd, hd
    row, head, one = t.stride()
    if one != 1:
        _fail(-3, f"{what}: the values of a head must be contiguous")
    return row if rows > 1 else heads * hd, head if heads > 1 else hd


def qk_norm_rope(ctx: ffi.Context, desc: ffi.AttnDesc, qkv, positions, q, k, v=None, *, q_gamma=None,
                 k_gamma=None, eps: float = 1e-5, halves: bool = False, stream=None) -> None:
    """rrr_qk_norm_rope: QKV rows [rows, (n_heads + 2 n_kv) * hd] -> q, k (and v) rows of
    their own type, query and key heads normed (gammas given) and rotated for positions[row]."""
    nh, nkv, hd = desc.n_heads, desc.n_kv_heads, desc.head_dim
    pin, rows, sin = _heads(ctx, qkv, nh + 2 * nkv, hd, "qkv")
    pq, _, sq = _heads(ctx, q, nh, hd, "q", rows)
    pk, _, sk = _heads(ctx, k, nkv, hd, "k", rows)
    pv, _, sv = (None, 0, 0) if v is None else _heads(ctx, v, nkv, hd, "v", rows)
    out = _type(q, "q")
    if k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        _fail(-2, "q, k and v must have one type")
    gammas = [None, None]
    for i, (g, name) in enumerate(((q_gamma, "q_gamma"), (k_gamma, "k_gamma"))):
        if g is not None:
            if _type(g, name) != ffi.F32 or g.numel() != hd or not g.is_contiguous():
                _fail(-3, f"{name}: a contiguous float32[{hd}] is needed")
            gammas[i] = _on(ctx, g, name)
    rc = ffi.lib().rrr_qk_norm_rope(
        ctx.h, byref(desc), _type(qkv, "qkv"), pin, sin, rows, _ints(ctx, positions, rows, "positions"),
        gammas[0], gammas[1], eps, 1 if halves else 0, out, pq, sq, pk, sk, pv, sv, _stream(ctx, stream))
    if rc:
        ctx.check(rc)


def attention_packed(ctx: ffi.Context, q, k, v, cu_q, cu_kv, out, *, causal: bool = True,
                     scale: float = 0.0, stream=None):
    """rrr_attention_packed: q, out [q_rows, n_heads, hd], k, v [kv_rows, n_kv, hd] (any row
    and head strides) of one 16-bit type; causal rows are the last ones of their sequence."""
    qd, kd = q.shape, k.shape
    if len(qd) != 3 or len(kd) != 3 or v.shape != kd or out.shape != qd or kd[2] != qd[2]:
        _fail(-3, f"q and out [rows, heads, hd], k and v [rows, heads, hd] are needed, got {list(qd)}, "
                  f"{list(out.shape)}, {list(kd)}, {list(v.shape)}")
    kind = _type(q, "q")
    if not (q.dtype == k.dtype == v.dtype == out.dtype):
        _fail(-2, "q, k, v and out must have one type")
    rows, heads, hd = qd
    held, kvh, _ = kd
    n = cu_q.shape[0]
    d = ffi.PackedDesc.from_buffer_copy(_packed(
        kind, heads, kvh, hd, max(n - 1, 0), 1 if causal else 0, scale, rows, held, *_strides(q, rows, heads, hd, "q"),
        *_strides(k, held, kvh, hd, "k"), *_strides(v, held, kvh, hd, "v"), *_strides(out, rows, heads, hd, "out")))
    rc = ffi.lib().rrr_attention_packed(ctx.h, byref(d), _on(ctx, q, "q"), _on(ctx, k, "k"), _on(ctx, v, "v"),
                                        _ints(ctx, cu_q, n, "cu_q"), _ints(ctx, cu_kv, n, "cu_kv"),
                                        _on(ctx, out, "out"), _stream(ctx, stream))
    if rc:
        ctx.check(rc)
    return out


class KV4Cache:
    """A 4-bit KV cache (rrr_kv4_cache): pages uint8 [n_pages, n_kv_heads, 80 * head_dim] of 64
    rows each, page_table int32 [n_seqs, max_pages]. Holds both tensors; the table's values
    may change between calls."""

    def __init__(self, ctx: ffi.Context, pages, page_table, head_dim: int):
        if pages.dim() != 3 or pages.shape[2] != 80 * head_dim or pages.element_size() != 1 or not pages.is_contiguous():
            _fail(-3, f"pages: a contiguous uint8 [n_pages, n_kv_heads, {80 * head_dim}] is needed, got "
                      f"{pages.dtype}{list(pages.shape)}")
        if page_table.dim() != 2 or page_table.element_size() != 4 or page_table.is_floating_point() or \
                (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            _fail(-3, "page_table: an int32 [n_seqs, max_pages] is needed")
        self.ctx, self.pages, self.page_table, self.head_dim = ctx, pages, page_table, head_dim
        n_seqs, most = page_table.shape
        self.n_seqs, self.n_kv_heads = n_seqs, pages.shape[1]
        stride = page_table.stride(0) if n_seqs > 1 else most
        self.desc = ffi.KV4Desc(_on(ctx, pages, "pages"), pages.shape[0], pages.shape[1], head_dim,
                                _on(ctx, page_table, "page_table"), n_seqs, most, stride)
        self._desc = byref(self.desc)

    @staticmethod
    def page_shape(n_pages: int, n_kv_heads: int, head_dim: int):
        return (n_pages, n_kv_heads, 80 * head_dim)

    def _rows(self, k, v, cu_rows, kv_lens):
        given = k if k is not None else v
        rows = given.shape[0]
        out = []
        for t, name in ((k, "k"), (v, "v")):
            if t is None:
                out += [None, 0]
                continue
            if t.dtype != given.dtype:
                _fail(-2, "k and v must have one type")
            p, _, s = _heads(self.ctx, t, self.n_kv_heads, self.head_dim, name, rows)
            out += [p, s]
        return (_type(given, "k"), *out, rows, _ints(self.ctx, cu_rows, self.n_seqs + 1, "cu_rows"),
                _ints(self.ctx, kv_lens, self.n_seqs, "kv_lens"))

    def store(self, k, v, cu_rows, kv_lens, stream=None) -> None:
        """rrr_kv4_store: packed rows [rows, n_kv, hd] become the last ones of their sequences,
        which have kv_lens rows then."""
        rc = ffi.lib().rrr_kv4_store(self.ctx.h, self._desc, *self._rows(k, v, cu_rows, kv_lens),
                                     _stream(self.ctx, stream))
        if rc:
            self.ctx.check(rc)

    def load(self, cu_rows, kv_lens, k=None, v=None, stream=None) -> None:
        """rrr_kv4_load: the last rows of every sequence, dequantised, into packed rows."""
        if k is None and v is None:
            _fail(-1, "load: k or v is needed")
        rc = ffi.lib().rrr_kv4_load(self.ctx.h, self._desc, *self._rows(k, v, cu_rows, kv_lens),
                                    _stream(self.ctx, stream))
        if rc:
            self.ctx.check(rc)

    def workspace(self, n_heads: int):
        """A workspace for `attention`; calls that can run at the same time need one each."""
        import torch
        n = c_int64()
        self.ctx.check(ffi.lib().rrr_kv4_workspace(self.ctx.h, byref(self.desc), n_heads, byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=self.pages.device)

    def attention(self, q, kv_lens, out, workspace, scale: float = 0.0, stream=None):
        """rrr_attention_kv4: q, out [n_seqs, n_heads, hd], one query row per sequence."""
        if q.dim() != 3 or out.shape != q.shape:
            _fail(-3, f"q and out [n_seqs, n_heads, hd] are needed, got {list(q.shape)} and {list(out.shape)}")
        if out.dtype != q.dtype:
            _fail(-2, "q and out must have one type")
        heads = q.shape[1]
        pq, _, sq = _heads(self.ctx, q, heads, self.head_dim, "q", self.n_seqs)
        po, _, so = _heads(self.ctx, out, heads, self.head_dim, "out", self.n_seqs)
        rc = ffi.lib().rrr_attention_kv4(
            self.ctx.h, self._desc, heads, _type(q, "q"), pq, sq, _ints(self.ctx, kv_lens, self.n_seqs, "kv_lens"),
            scale, po, so, _on(self.ctx, workspace, "workspace"), workspace.nbytes, _stream(self.ctx, stream))
        if rc:
            self.ctx.check(rc)
        return out
