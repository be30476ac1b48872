"""The 8-bit paged KV cache over torch tensors: block tables and slot maps, append, read back, attention.

Host layer of the sllm_k_block_tables / sllm_k_kv8_* / sllm_k_attn_kv8 entry points of include/sllm.h, which say what each call
computes.  Tensors live on one CUDA device; calls run on torch's current stream of that device, allocate nothing but their
results and workspace (from torch's allocator, so they can be captured into a CUDA graph) and never wait for the GPU.

    pages, scales = kv8.empty_cache(n_pages, kv_heads, head_dim)        # one layer
    kv8.block_tables(before, after, table, ring, pool_in, pool_out, cu_tok, tok_seq, tok_pos, slot_map)
    kv8.append(k, v, slot_map, pages, scales)                           # k, v: [n_tok, kv_heads, head_dim]
    out = kv8.attention(q, pages, scales, table, tok_seq, tok_pos, cu_tok, max_new=..., max_len=...)

PagedCache keeps what a decode loop keeps between steps: the layers' pages, the table, the ring of free pages, the lengths.

    cache = kv8.PagedCache(n_layers, n_seqs, n_pages, kv_heads, head_dim, max_len, max_tok)
    cache.step(len_after)                                               # which sequences grow, shrink or end
    for layer in ...:
        cache.append(layer, k, v)                                       # rows of the step's list, cache.tok_seq / tok_pos / cu_tok
        out = cache.attention(layer, q, max_new=...)

Bad arguments raise ValueError; there is no CPU path.
"""
from __future__ import annotations

import ctypes as C
from struct import Struct

import torch
from torch._C import _cuda_getCurrentRawStream as _raw_stream
from torch._C import _cuda_getDevice as _current_device

from .api import _raise, load_library

PAGE, BLOCK = 64, 16
MAX_SEQS = 8192
_I32, _I64, _I8, _F32 = torch.int32, torch.int64, torch.int8, torch.float32
_ROWS = {torch.bfloat16: 0, torch.float32: 1}
_HEAD_DIMS = (16, 32, 64, 128)

# The structures of include/sllm.h in their field order, packed with native alignment (packing takes a fraction of what filling
# a ctypes structure does, which a decode step would notice).
STRUCTS = {
    "sllm_kv8_layer": ("@QQQII", "pages scales n_pages kv_heads head_dim"),
    "sllm_block_tables": ("@10QQIII0Q", "len_before len_after table ring pool_in pool_out cu_tok tok_seq tok_pos slot_map n_pages n_seq table_width max_tok"),
    "sllm_kv8_rows": ("@QQQQQII", "k v slot_map k_stride v_stride n_tok dtype"),
    "sllm_kv8_attn": ("@QQQQQQQQQIIIIIIIf0Q", "q out q_stride out_stride table tok_seq tok_pos cu_tok status n_tok n_seq table_width n_heads max_new max_len dtype scale"),
}
_pack_layer, _pack_tables, _pack_rows, _pack_attn = (Struct(f).pack for f, _ in STRUCTS.values())

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


def _call(dev: int, fn, *args):
    """fn(*args, stream) on device `dev`, which need not be the current one."""
    if _current_device() != dev:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    else:
        rc = fn(*args, _raw_stream(dev))
    if rc:
        _raise(rc, _lib().sllm_last_error(None).decode())


def _flat(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, dev: int) -> int:
    """The address of a contiguous tensor of this type and shape on this device."""
    if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous() or t.shape != shape:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{dev}")
    return t.data_ptr()


def _layer(pages: torch.Tensor, scales: torch.Tensor) -> tuple[bytes, int, int, int]:
    """The packed layer, its device, heads and head_dim."""
    s = pages.shape
    if not (pages.is_cuda and pages.dtype is _I8 and len(s) == 5 and s[2] == 2 and s[3] == PAGE and s[4] in _HEAD_DIMS and s[0] > 0 and s[1] > 0 and pages.is_contiguous()):
        _need(pages.is_cuda, "pages must be a CUDA tensor: this package has no CPU path")
        _need(len(s) != 5 or s[4] in _HEAD_DIMS, "head_dim must be 16, 32, 64 or 128")
        raise ValueError("pages must be a contiguous int8 tensor [n_pages][kv_heads][2][64][head_dim] with at least one page and one head")
    dev, n, h, d = pages.get_device(), s[0], s[1], s[4]
    return _pack_layer(pages.data_ptr(), _flat("scales", scales, _F32, (n, h, 2, PAGE // BLOCK), dev), n, h, d), dev, h, d


def _rows(name: str, t: torch.Tensor, n: int, heads: int, head_dim: int, dev: int) -> int:
    """The distance between rows, in elements."""
    row = heads * head_dim
    if t.shape != (n, heads, head_dim) or t.get_device() != dev:
        raise ValueError(f"{name} must be [{n}, {heads}, {head_dim}] on cuda:{dev}")
    st = t.stride()
    if n > 0 and not (st[2] == 1 and (heads == 1 or st[1] == head_dim) and (n == 1 or st[0] >= row)):
        raise ValueError(f"{name}: the heads of a row must be contiguous, and rows must not overlap")
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
    _need(table.is_cuda, "table must be a CUDA tensor: this package has no CPU path")
    _need(table.dim() == 2 and ring.dim() == 1 and tok_seq.dim() == 1, "table must be [n_seq, width], ring and tok_seq of one dimension")
    dev = table.get_device()
    n, width = table.shape
    room, n_pages = tok_seq.shape[0], ring.shape[0]
    one, entries = (n,), (room,)
    cu, out = _flat("cu_tok", cu_tok, _I32, (n + 1,), dev), _flat("pool_out", pool_out, _I64, (4,), dev)
    seq, pos, slot = _flat("tok_seq", tok_seq, _I32, entries, dev), _flat("tok_pos", tok_pos, _I32, entries, dev), _flat("slot_map", slot_map, _I64, entries, dev)
    if room == 0:                        # empty tensors have no address: any will do, nothing is written
        seq, pos, slot = cu, cu, out
    _call(dev, _lib().sllm_k_block_tables,
          _pack_tables(_flat("len_before", len_before, _I32, one, dev), _flat("len_after", len_after, _I32, one, dev), _flat("table", table, _I32, (n, width), dev),
                       _flat("ring", ring, _I32, (n_pages,), dev), _flat("pool_in", pool_in, _I64, (4,), dev), out, cu, seq, pos, slot, n_pages, n, width, room))


def append(k: torch.Tensor, v: torch.Tensor, slot_map: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor) -> None:
    """Rows k, v [n_tok, kv_heads, head_dim] (bf16 or fp32, any row stride) into the cache at slot_map int64 [n_tok]; see sllm_k_kv8_append."""
    c, dev, h, d = _layer(pages, scales)
    n, t = k.shape[0], _ROWS.get(k.dtype)
    _need(t is not None and v.dtype is k.dtype, "k and v must both be bfloat16 or float32")
    r = _pack_rows(k.data_ptr(), v.data_ptr(), _flat("slot_map", slot_map, _I64, (n,), dev), _rows("k", k, n, h, d, dev), _rows("v", v, n, h, d, dev), n, t)
    if n:
        _call(dev, _lib().sllm_k_kv8_append, c, r)


def read(slots: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows (k, v), [n, kv_heads, head_dim] each, that the cache stands for at slots int64 [n]; zeros for a slot outside the pool."""
    c, dev, h, d = _layer(pages, scales)
    _need(slots.dim() == 1, "slots must have one dimension")
    t, n = _ROWS.get(dtype), slots.shape[0]
    _need(t is not None, "dtype must be bfloat16 or float32")
    at = _flat("slots", slots, _I64, (n,), dev)
    k = scales.new_empty((n, h, d), dtype=dtype)
    v = torch.empty_like(k)
    if n:
        _call(dev, _lib().sllm_k_kv8_read, c, _pack_rows(k.data_ptr(), v.data_ptr(), at, h * d, h * d, n, t))
    return k, v


def attention(q: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, table: torch.Tensor, tok_seq: torch.Tensor, tok_pos: torch.Tensor,
              cu_tok: torch.Tensor | None = None, *, max_new: int = 0, max_len: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of q [n_tok, n_heads, head_dim] (bf16 or fp32, any row stride) over the cache; see sllm_k_attn_kv8.

    Token t attends positions 0 .. tok_pos[t] of sequence tok_seq[t] (int32 [n_tok]) through table int32 [n_seq, width].  max_new and
    max_len are the most tokens a sequence has in the list and the most positions any has: they choose how the work is cut
    (0: not known).  Rows of tokens with tok_seq < 0 are left as they are, so give `out` where a list is padded.  status int32 [1]
    takes the SLLM_ERR_* code of what the kernels find: a page outside the pool (it is not attended), a wait that gave up (the rows
    are NaN)."""
    c, dev, h, d = _layer(pages, scales)
    _need(q.dim() == 3 and table.dim() == 2, "q must be [n_tok, n_heads, head_dim], table [n_seq, width]")
    n, heads = q.shape[0], q.shape[1]
    n_seq, width = table.shape
    t = _ROWS.get(q.dtype)
    _need(t is not None, "q must be bfloat16 or float32")
    _need(heads > 0 and heads % h == 0, "n_heads must be a multiple of kv_heads")
    q_stride = _rows("q", q, n, heads, d, dev)
    if out is None:
        out = torch.empty((n, heads, d), dtype=q.dtype, device=q.device)
    _need(out.dtype is q.dtype, "out must have q's dtype")
    _need(0 <= max_new < 1 << 31 and 0 <= max_len < 1 << 31, "max_new and max_len must not be negative")
    _need(scale is None or 1.5e-45 < abs(scale) < 3.4e38, "scale must be a finite number other than 0 in fp32")      # as a float 0 it would mean the default
    a = _pack_attn(q.data_ptr(), out.data_ptr(), q_stride, _rows("out", out, n, heads, d, dev), _flat("table", table, _I32, (n_seq, width), dev),
                   _flat("tok_seq", tok_seq, _I32, (n,), dev), _flat("tok_pos", tok_pos, _I32, (n,), dev),
                   0 if cu_tok is None else _flat("cu_tok", cu_tok, _I32, (n_seq + 1,), dev), 0 if status is None else _flat("status", status, _I32, (1,), dev),
                   n, n_seq, width, heads, max_new, max_len, t, scale or 0.0)
    if n == 0:
        return out
    lib = _lib()
    key = (dev, h, d, n, n_seq, width, heads, max_new, max_len, t, cu_tok is None)
    need = _workspaces.get(key)
    if need is None:
        got = C.c_uint64()
        _call(dev, lambda *x: lib.sllm_k_attn_kv8_workspace(*x[:-1]), c, a, C.byref(got))
        if len(_workspaces) > 4096:
            _workspaces.clear()
        need = _workspaces[key] = got.value
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        _call(dev, lib.sllm_k_attn_kv8, c, a, ws.data_ptr(), need)
    else:
        _call(dev, lib.sllm_k_attn_kv8, c, a, None, 0)
    return out


class PagedCache:
    """An 8-bit cache of several layers for up to n_seqs sequences of up to max_len positions (whole pages: rounded up to a multiple
    of 64), and its bookkeeping on the GPU.

    A step names the length that each sequence is to have after it; from then on lists of up to max_tok new positions say where the
    rows of k, v and q belong: row t is position tok_pos[t] of sequence tok_seq[t] (-1 behind the last).  Nothing here waits for the GPU,
    and the buffers stay where they are, so a step with its layers can be captured into a CUDA graph: write the lengths into the
    tensor that the captured step() was given, and the rows into the captured k, v and q, before each replay.

    A step that needs more pages or entries than there are, or a length above max_len, changes nothing and leaves empty lists:
    status() says so (0, or the SLLM_ERR_* code), at the cost of a wait for the GPU, and the next step starts from the lengths before.
    status() also says what attention() found (a page outside the pool, a wait that gave up)."""

    def __init__(self, n_layers: int, n_seqs: int, n_pages: int, kv_heads: int, head_dim: int, max_len: int, max_tok: int, device="cuda"):
        _need(n_layers > 0 and 0 < n_seqs <= MAX_SEQS and n_pages > 0 and max_len > 0 and max_tok > 0, f"counts must be positive, n_seqs at most {MAX_SEQS}")
        self.layers = [empty_cache(n_pages, kv_heads, head_dim, device) for _ in range(n_layers)]
        dev = self.layers[0][0].device
        i32 = dict(dtype=_I32, device=dev)
        self.max_len = max_len
        self.lens = torch.zeros(n_seqs, **i32)
        self.table = torch.full((n_seqs, (max_len + PAGE - 1) // PAGE), -1, **i32)
        self.ring = torch.arange(n_pages, **i32)
        self._pool = torch.tensor([[0, n_pages, 0, 0]] * 2, dtype=_I64, device=dev)
        self.cu_tok = torch.zeros(n_seqs + 1, **i32)
        self.tok_seq, self.tok_pos = torch.full((max_tok,), -1, **i32), torch.full((max_tok,), -1, **i32)
        self.slot_map = torch.full((max_tok,), -1, dtype=_I64, device=dev)
        self._found = torch.zeros(1, **i32)                  # what attention() found

    def step(self, len_after: torch.Tensor) -> None:
        """Moves every sequence to len_after (int32 [n_seqs] on the cache's device; 0 = it has ended) and makes the step's lists."""
        now, then = self._pool.unbind(0)
        block_tables(self.lens, len_after, self.table, self.ring, now, then, self.cu_tok, self.tok_seq, self.tok_pos, self.slot_map)
        torch.where(then[3] == 0, len_after, self.lens, out=self.lens)
        now.copy_(then)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's rows of k and v, [max_tok, kv_heads, head_dim], into a layer."""
        append(k, v, self.slot_map, *self.layers[layer])

    def attention(self, layer: int, q: torch.Tensor, *, max_new: int = 0, max_len: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                  status: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the step's queries [max_tok, n_heads, head_dim] over a layer.  Rows behind the list's last are left as they
        are in `out`, and zeros where it is not given.  What the kernels find goes to `status`, or where that is not given to status()."""
        if out is None:
            out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        return attention(q, *self.layers[layer], self.table, self.tok_seq, self.tok_pos, self.cu_tok, max_new=max_new, max_len=max_len or self.max_len, scale=scale,
                         out=out, status=self._found if status is None else status)

    def status(self) -> int:
        """The code of the last step's refusal, or else of what attention() has found since status() last said so, or else 0."""
        code = int(self._pool[1, 3])
        if code == 0:
            code = int(self._found)
            if code:
                self._found.zero_()
        return code

    def free_pages(self) -> int:
        return int(self._pool[0, 1])
