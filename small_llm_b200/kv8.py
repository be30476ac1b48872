"""The 8-bit paged KV cache over torch tensors: block tables and slot maps, append, read back, attention.

Host layer of the sllm_k_block_tables / sllm_k_kv8_* / sllm_k_attn_kv8 entry points of include/sllm.h, which say what each call
computes.  Tensors live on one CUDA device; calls run on torch's current stream of that device, allocate nothing but their
results and workspace (from torch's allocator, so they can be captured into a CUDA graph) and never wait for the GPU.

    pages, scales = kv8.empty_cache(n_pages, kv_heads, head_dim)        # one layer
    kv8.block_tables(before, after, table, ring, pool_in, pool_out, cu_tok, tok_seq, tok_pos, slot_map)
    kv8.append(k, v, slot_map, pages, scales)                           # k, v: [n_tok, kv_heads, head_dim]
    out = kv8.attention(q, pages, scales, table, tok_seq, tok_pos, cu_tok, max_new=..., max_len=...)

Bad arguments raise ValueError; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C

import torch

from .api import _raise, load_library

PAGE, BLOCK = 64, 16
MAX_SEQS = 8192
_ROWS = {torch.bfloat16: 0, torch.float32: 1}
_HEAD_DIMS = (16, 32, 64, 128)


class _Layer(C.Structure):
    _fields_ = [("pages", C.c_void_p), ("scales", C.c_void_p), ("n_pages", C.c_uint64), ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32)]


class _Tables(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("len_before", "len_after", "table", "ring", "pool_in", "pool_out", "cu_tok", "tok_seq", "tok_pos", "slot_map")] + [
        ("n_pages", C.c_uint64), ("n_seq", C.c_uint32), ("table_width", C.c_uint32), ("max_tok", C.c_uint32)]


class _Rows(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("slot_map", C.c_void_p), ("k_stride", C.c_uint64), ("v_stride", C.c_uint64), ("n_tok", C.c_uint32),
                ("dtype", C.c_uint32)]


class _Attn(C.Structure):
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("q_stride", C.c_uint64), ("out_stride", C.c_uint64)] + [
        (n, C.c_void_p) for n in ("table", "tok_seq", "tok_pos", "cu_tok", "status")] + [
        (n, C.c_uint32) for n in ("n_tok", "n_seq", "table_width", "n_heads", "max_new", "max_len", "dtype")] + [("scale", C.c_float)]


_fns = None
_workspaces: dict[tuple, int] = {}       # sizes of the call, device included -> bytes of workspace


def _lib():
    global _fns
    if _fns is None:
        lib = load_library()
        p = C.c_void_p
        lib.sllm_k_block_tables.argtypes = [p, p]
        lib.sllm_k_kv8_append.argtypes = lib.sllm_k_kv8_read.argtypes = [p, p, p]
        lib.sllm_k_attn_kv8_workspace.argtypes = [p, p, C.POINTER(C.c_uint64)]
        lib.sllm_k_attn_kv8.argtypes = [p, p, p, C.c_uint64, p]
        _fns = lib
    return _fns


def _need(ok: bool, why: str):
    if not ok:
        raise ValueError(why)


def _call(dev: torch.device, fn, *args):
    """fn(*args, stream) on `dev`, which need not be the current device."""
    i = dev.index
    if torch.cuda.current_device() != i:
        with torch.cuda.device(i):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        _raise(rc, _lib().sllm_last_error(None).decode())


def _ints(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, dev: torch.device) -> int:
    if t.dtype != dtype or t.shape != shape or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {dev}")
    return t.data_ptr()


def _layer(pages: torch.Tensor, scales: torch.Tensor) -> _Layer:
    _need(pages.is_cuda, "pages must be a CUDA tensor: this package has no CPU path")
    s = pages.shape
    _need(pages.dtype == torch.int8 and len(s) == 5 and s[2] == 2 and s[3] == PAGE and pages.is_contiguous(),
          "pages must be a contiguous int8 tensor [n_pages][kv_heads][2][64][head_dim]")
    _need(s[4] in _HEAD_DIMS, "head_dim must be 16, 32, 64 or 128")
    _need(s[0] > 0 and s[1] > 0, "a cache has at least one page and one head")
    return _Layer(pages.data_ptr(), _ints("scales", scales, torch.float32, (s[0], s[1], 2, PAGE // BLOCK), pages.device), s[0], s[1], s[4])


def _rows(name: str, t: torch.Tensor, n: int, heads: int, head_dim: int, dev: torch.device) -> int:
    """The distance between rows, in elements."""
    _need(t.shape == (n, heads, head_dim) and t.device == dev, f"{name} must be [{n}, {heads}, {head_dim}] on {dev}")
    st = t.stride()
    row = heads * head_dim
    _need(n == 0 or (st[2] == 1 and (heads == 1 or st[1] == head_dim) and (n == 1 or st[0] >= row)),
          f"{name}: the heads of a row must be contiguous, and rows must not overlap")
    return st[0] if n > 1 else row


def empty_cache(n_pages: int, kv_heads: int, head_dim: int, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """pages and scales of one layer that stands for zeros."""
    _need(head_dim in _HEAD_DIMS, "head_dim must be 16, 32, 64 or 128")
    return (torch.zeros(n_pages, kv_heads, 2, PAGE, head_dim, dtype=torch.int8, device=device),
            torch.zeros(n_pages, kv_heads, 2, PAGE // BLOCK, device=device))


def block_tables(len_before, len_after, table, ring, pool_in, pool_out, cu_tok, tok_seq, tok_pos, slot_map) -> None:
    """Tables, token lists and slot map of a step from the lengths before and after it (int32 [n_seq]); see sllm_k_block_tables.

    table int32 [n_seq, width] and ring int32 [n_pages] are updated; pool_in int64 [4] = {head, free, -, -} is read and pool_out
    int64 [4] = {head, free, entries, status} written (another tensor); cu_tok int32 [n_seq + 1], tok_seq and tok_pos int32 [max_tok]
    and slot_map int64 [max_tok] are written whole."""
    dev = table.device
    _need(table.is_cuda, "table must be a CUDA tensor: this package has no CPU path")
    _need(table.dim() == 2 and ring.dim() == 1 and tok_seq.dim() == 1, "table must be [n_seq, width], ring and tok_seq of one dimension")
    n, width = table.shape
    room = tok_seq.shape
    i32, i64 = torch.int32, torch.int64
    a = _Tables(_ints("len_before", len_before, i32, (n,), dev), _ints("len_after", len_after, i32, (n,), dev), _ints("table", table, i32, (n, width), dev),
                _ints("ring", ring, i32, ring.shape, dev), _ints("pool_in", pool_in, i64, (4,), dev), _ints("pool_out", pool_out, i64, (4,), dev),
                _ints("cu_tok", cu_tok, i32, (n + 1,), dev), _ints("tok_seq", tok_seq, i32, room, dev), _ints("tok_pos", tok_pos, i32, room, dev),
                _ints("slot_map", slot_map, i64, room, dev), ring.shape[0], n, width, room[0])
    if room[0] == 0:                     # empty tensors have no address: any will do, nothing is written
        a.tok_seq = a.tok_pos = a.cu_tok
        a.slot_map = a.pool_out
    _call(dev, _lib().sllm_k_block_tables, C.byref(a))


def append(k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor) -> None:
    """Rows k, v [n_tok, kv_heads, head_dim] (bf16 or fp32, any row stride) into the cache at slot_map int64 [n_tok]; see sllm_k_kv8_append."""
    c = _layer(pages, scales)
    dev, n = pages.device, k.shape[0]
    _need(k.dtype in _ROWS and v.dtype == k.dtype, "k and v must both be bfloat16 or float32")
    r = _Rows(k.data_ptr(), v.data_ptr(), _ints("slot_map", slot_map, torch.int64, (n,), dev), _rows("k", k, n, c.kv_heads, c.head_dim, dev),
              _rows("v", v, n, c.kv_heads, c.head_dim, dev), n, _ROWS[k.dtype])
    if n:
        _call(dev, _lib().sllm_k_kv8_append, C.byref(c), C.byref(r))


def read(slots: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows (k, v), [n, kv_heads, head_dim] each, that the cache stands for at slots int64 [n]; zeros for a slot outside the pool."""
    c = _layer(pages, scales)
    _need(slots.dim() == 1, "slots must have one dimension")
    _need(dtype in _ROWS, "dtype must be bfloat16 or float32")
    dev, n = pages.device, slots.shape[0]
    at = _ints("slots", slots, torch.int64, (n,), dev)
    kv = torch.empty(2, n, c.kv_heads, c.head_dim, dtype=dtype, device=dev)
    k, v = kv.unbind(0)
    row = c.kv_heads * c.head_dim
    if n:
        _call(dev, _lib().sllm_k_kv8_read, C.byref(c), C.byref(_Rows(k.data_ptr(), v.data_ptr(), at, row, row, n, _ROWS[dtype])))
    return k, v


def attention(q: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, tok_seq: torch.Tensor, tok_pos: torch.Tensor,
              cu_tok: torch.Tensor | None = None, *, max_new: int = 0, max_len: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of q [n_tok, n_heads, head_dim] (bf16 or fp32, any row stride) over the cache; see sllm_k_attn_kv8.

    Token t attends positions 0 .. tok_pos[t] of sequence tok_seq[t] (int32 [n_tok]) through table int32 [n_seq, width].  max_new and
    max_len are the most tokens a sequence has in the list and the most positions any has: they choose how the work is cut
    (0: not known).  Rows of tokens with tok_seq < 0 are left as they are, so give `out` where a list is padded."""
    c = _layer(pages, scales)
    dev = pages.device
    _need(q.dim() == 3 and table.dim() == 2, "q must be [n_tok, n_heads, head_dim], table [n_seq, width]")
    n, heads = q.shape[0], q.shape[1]
    _need(q.dtype in _ROWS, "q must be bfloat16 or float32")
    _need(heads > 0 and heads % c.kv_heads == 0, "n_heads must be a multiple of kv_heads")
    n_seq, width = table.shape
    q_stride = _rows("q", q, n, heads, c.head_dim, dev)
    if out is None:
        out = torch.empty(n, heads, c.head_dim, dtype=q.dtype, device=dev)
    _need(out.dtype == q.dtype, "out must have q's dtype")
    _need(0 <= max_new < 1 << 31 and 0 <= max_len < 1 << 31, "max_new and max_len must not be negative")
    _need(scale is None or scale != 0, "scale must not be 0")
    i32 = torch.int32
    a = _Attn(q.data_ptr(), out.data_ptr(), q_stride, _rows("out", out, n, heads, c.head_dim, dev), _ints("table", table, i32, (n_seq, width), dev),
              _ints("tok_seq", tok_seq, i32, (n,), dev), _ints("tok_pos", tok_pos, i32, (n,), dev),
              None if cu_tok is None else _ints("cu_tok", cu_tok, i32, (n_seq + 1,), dev), None if status is None else _ints("status", status, i32, (1,), dev),
              n, n_seq, width, heads, max_new, max_len, _ROWS[q.dtype], scale or 0.0)
    if n == 0:
        return out
    lib = _lib()
    key = (dev.index, c.kv_heads, c.head_dim, n, n_seq, width, heads, max_new, max_len, q.dtype, cu_tok is None)
    need = _workspaces.get(key)
    if need is None:
        got = C.c_uint64()
        _call(dev, lambda *x: lib.sllm_k_attn_kv8_workspace(*x[:-1]), C.byref(c), C.byref(a), C.byref(got))
        if len(_workspaces) > 4096:
            _workspaces.clear()
        need = _workspaces[key] = got.value
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(dev, lib.sllm_k_attn_kv8, C.byref(c), C.byref(a), ws.data_ptr() if need else None, need)
    return out
