"""A paged cache of K and V in 4 bits (C interface: include/mlops_paged.h): pages and slots for a step's new tokens (`assign`), quantise-on-write
(`append`), read-back (`read`) and attention over the pages (`attend`).

An engine keeps, on the GPU, one pool per layer (`empty`), one block table ``int32 [batch, width]`` for all layers, the requests' lengths, and a ring
of free page numbers with its two ends. A step of one layer:

    step = paged.assign(table, lengths, added, free, cursor, cache.page_size, tokens)      # once for all layers
    paged.append(cache, k, v, step.slots)                                                  # k, v [tokens, kv_heads, 128]
    out = paged.attend(q, cache, table, step.lengths, step.starts)                         # q, out [tokens, q_heads, 128]

Elements take 4.5 bits: E2M1 codes, an E4M3 scale per 16 channels, an FP32 factor per head. The reference has no paged cache; tensors are BF16 or FP16.
Nothing here synchronises, so that a step can be captured into a CUDA graph.
"""
import ctypes
import struct
from dataclasses import dataclass
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _C

HEAD_DIM = 128
BLOCK, BLOCK_BYTES = 16, 2304  # tokens and bytes of a block of a page, per KV head
_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32


class _Cache(ctypes.Structure):
    """mlops_paged_cache"""
    _fields_ = [("units", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p), ("page_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("pages", ctypes.c_int), ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int)]


class _Assign(ctypes.Structure):
    """mlops_paged_assign_args"""
    _fields_ = [("batch", ctypes.c_int), ("tokens", ctypes.c_int), ("page_size", ctypes.c_int), ("width", ctypes.c_int), ("table_stride", ctypes.c_int64),
                ("table", ctypes.c_void_p), ("held", ctypes.c_void_p), ("added", ctypes.c_void_p), ("ring", ctypes.c_void_p), ("ring_size", ctypes.c_int),
                ("cursor", ctypes.c_void_p), ("slots", ctypes.c_void_p), ("positions", ctypes.c_void_p), ("starts", ctypes.c_void_p),
                ("lengths", ctypes.c_void_p), ("moved", ctypes.c_void_p)]


class _Attend(ctypes.Structure):
    """mlops_paged_attend_args"""
    _fields_ = [("batch", ctypes.c_int), ("tokens", ctypes.c_int), ("q_heads", ctypes.c_int), ("type", ctypes.c_int), ("q", ctypes.c_void_p),
                ("q_token_stride", ctypes.c_int64), ("q_head_stride", ctypes.c_int64), ("out", ctypes.c_void_p), ("out_token_stride", ctypes.c_int64),
                ("out_head_stride", ctypes.c_int64), ("lse", ctypes.c_void_p), ("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64),
                ("width", ctypes.c_int), ("lengths", ctypes.c_void_p), ("starts", ctypes.c_void_p), ("scale", ctypes.c_float)]


_lib, _vp, _int, _i64 = _C._lib, ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
_lib.mlops_paged_assign.argtypes = [_vp, _vp]
_lib.mlops_paged_append.argtypes = [_vp, _int, _int, _vp, _i64, _i64, _vp, _i64, _i64, _vp, _vp]
_lib.mlops_paged_read.argtypes = [_vp, _int, _int, _vp, _vp, _vp, _vp]
_lib.mlops_paged_attend.argtypes = [_vp, _vp, _vp, ctypes.c_size_t, _vp]
_lib.mlops_paged_attend_scratch_bytes.argtypes = [_vp, _int]
_lib.mlops_paged_attend_scratch_bytes.restype = ctypes.c_size_t
_lib.mlops_paged_last_error.restype = ctypes.c_char_p
# the structures as the calls below pass them: their bytes (a third of the host's time that ctypes takes to fill one; addresses of 0 are null)
_CACHE, _ASSIGN, _ATTEND = struct.Struct("@PPPqqiii4x"), struct.Struct("@iiiiqPPPPiPPPPPP"), struct.Struct("@iiiiPqqPqqPPqiPPf4x")
assert (_CACHE.size, _ASSIGN.size, _ATTEND.size) == (ctypes.sizeof(_Cache), ctypes.sizeof(_Assign), ctypes.sizeof(_Attend))

_scratch = _C._ScratchPool(torch.zeros)  # (zeros at first; every call leaves its counters as it found them)


def _raise(status, what):
    message = _lib.mlops_paged_last_error().decode()
    if status == _C.INVALID_VALUE:
        raise ValueError(message)
    raise RuntimeError(f"{what} failed: {message}")


@dataclass
class PagedCache:
    """A pool of pages for one layer."""
    units: torch.Tensor    # uint8 [pages, kv_heads, page_size / 16, 2304]; the last two dimensions dense
    k_scale: torch.Tensor  # float32 [kv_heads]: the heads' factors, positive
    v_scale: torch.Tensor

    @property
    def pages(self) -> int:
        return self.units.size(0)

    @property
    def page_size(self) -> int:
        return self.units.size(2) * BLOCK


class Step(NamedTuple):
    """What `assign` says of a step's new tokens. The tensors are for `append` (slots), a rotary embedding (positions) and `attend` (lengths, starts);
    `lengths` and `cursor` are the next call's."""
    slots: torch.Tensor      # int32 [tokens]: where each token is stored in the pool, -1: nowhere
    positions: torch.Tensor  # int32 [tokens]: its position in its request
    starts: torch.Tensor     # int32 [batch + 1]: request b's tokens are starts[b] .. starts[b + 1] - 1
    lengths: torch.Tensor    # int32 [batch]: tokens of each request, the new ones among them
    cursor: torch.Tensor     # int64 [3]: the ring's head and tail after the call, and how many pages were missing


def empty(pages: int, kv_heads: int, page_size: int = 64, *, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
          device="cuda") -> PagedCache:
    """A pool of ``pages`` pages of ``page_size`` tokens (a multiple of 16). ``k_scale``, ``v_scale``: float32 [kv_heads] factors that bring the heads'
    values into the scales' range (a block of 16 channels is stored well where its largest value is between 0.1 and 2688 times the factor); default 1."""
    if pages <= 0 or kv_heads <= 0 or page_size <= 0 or page_size % BLOCK:
        raise ValueError(f"expected pages, kv_heads > 0 and a page_size that is a multiple of {BLOCK}; got {pages}, {kv_heads}, {page_size}")
    if pages * page_size >= 1 << 31:
        raise ValueError(f"a pool has fewer than 2^31 slots; {pages} pages of {page_size} tokens are more")
    one = torch.ones((kv_heads,), dtype=_F32, device=device)
    scales = [one.clone() if s is None else s.to(device=device, dtype=_F32).contiguous() for s in (k_scale, v_scale)]
    return PagedCache(torch.zeros((pages, kv_heads, page_size // BLOCK, BLOCK_BYTES), dtype=torch.uint8, device=device), *scales)


def _pool(c):
    """A pool's arrays, checked: the structure that names them to the library, its pages' KV heads, its device's index."""
    u, ks, vs = c.units, c.k_scale, c.v_scale
    index = u.get_device()
    if not 0 <= index == ks.get_device() == vs.get_device():
        raise ValueError(f"the arrays of a paged cache have to live on the same CUDA device (units: {u.device}, scales: {ks.device}, {vs.device})")
    shape, strides = u.shape, u.stride()
    if u.dtype is not torch.uint8 or len(shape) != 4 or shape[3] != BLOCK_BYTES or strides[3] != 1 or (strides[2] != BLOCK_BYTES and shape[2] > 1):
        raise ValueError(f"units has to be a uint8 [pages, kv_heads, blocks, {BLOCK_BYTES}] tensor with dense pages; it is {u.dtype} {tuple(shape)}, strides {strides}")
    pages, heads, blocks, _ = shape
    if not (ks.dtype is vs.dtype is _F32 and ks.shape == vs.shape == (heads,) and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"k_scale and v_scale have to be contiguous float32 [{heads}] tensors; they are {ks.dtype} {tuple(ks.shape)} and {vs.dtype} {tuple(vs.shape)}")
    return _CACHE.pack(u.data_ptr(), ks.data_ptr(), vs.data_ptr(), strides[0], strides[1], pages, blocks * BLOCK, heads), heads, index


def _ints(x, index, what, size=None, dtype=_I32):
    shape = x.shape
    if x.get_device() != index or x.dtype is not dtype or len(shape) != 1 or not x.is_contiguous() or (size is not None and shape[0] != size):
        raise ValueError(f"{what}: expected a contiguous {dtype} [{'n' if size is None else size}] tensor on cuda:{index}; it is {x.dtype} {tuple(shape)} on {x.device}")
    return x.data_ptr()


def _table(x, index):
    shape, strides = x.shape, x.stride()
    if x.get_device() != index or x.dtype is not _I32 or len(shape) != 2 or (strides[1] != 1 and shape[1] > 1):
        raise ValueError(f"table: expected an int32 [batch, width] tensor with dense rows on cuda:{index}; it is {x.dtype} {tuple(shape)} on {x.device}")
    batch, width = shape
    return x.data_ptr(), (strides[0] if batch > 1 else width), batch, width


def _rows(x, index, what, heads=None):
    """[tokens, heads, 128] rows as the library reads them (dense channels, 16-byte pieces aligned), their shape, strides and type"""
    kind, shape = _TYPES.get(x.dtype), x.shape
    if x.get_device() != index or kind is None or len(shape) != 3 or shape[2] != HEAD_DIM or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what}: expected a bfloat16 or float16 [tokens, {'heads' if heads is None else heads}, {HEAD_DIM}] tensor on cuda:{index}; it is {x.dtype} {tuple(shape)} on {x.device}")
    by_token, by_head, by_channel = x.stride()
    if shape[0] == 1:  # (a stride that nothing is reached by may be any number, and stays what it is in a copy)
        by_token = 0
    if shape[1] == 1:
        by_head = 0
    if by_channel != 1 or by_token % 8 or by_head % 8 or x.data_ptr() % 16:
        x = torch.empty(shape, dtype=x.dtype, device=x.device).copy_(x)
        by_token, by_head, _ = x.stride()
    return x, shape, by_token, by_head, kind


def _on(index):
    """Whether ``index`` is the current device (calls are made on their tensors' device)."""
    return torch._C._cuda_getDevice() == index


def assign(table: torch.Tensor, held: torch.Tensor, added: torch.Tensor, free: torch.Tensor, cursor: torch.Tensor, page_size: int, tokens: int) -> Step:
    """Pages and slots for ``added[b]`` new tokens of every request b, which holds ``held[b]``.

    New pages are taken from the ring ``free`` (int32, from ``cursor[0]`` up to ``cursor[1]``, both counted without end and taken modulo the ring's
    size), in the order of the requests, and entered into ``table`` (int32 [batch, width], in place). ``tokens``: rows of the step, at least the sum of
    ``added``; rows behind it get slot and position -1. (Where it is less, the tokens behind it are not added: ``Step.starts`` ends at ``tokens``, ``Step.lengths``
    are without them, and the pages that they would have needed count as missing.) Where the ring runs out or a request outgrows its row, entries and slots are -1 and
    ``Step.cursor[2]`` counts the pages that were missing. A request's pages are given back by ``free[tail % size ...] = table[b, :n]`` and advancing
    the tail, ``cursor[1]``."""
    index = table.get_device()
    if index < 0:
        raise ValueError(f"table: expected a CUDA tensor, not one on {table.device}")
    if not _on(index):
        with torch.cuda.device(index):
            return assign(table, held, added, free, cursor, page_size, tokens)
    entries, stride, batch, width = _table(table, index)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"tokens may not be negative; it is {tokens}")
    if cursor.dim() != 1 or cursor.size(0) not in (2, 3):
        raise ValueError(f"cursor: expected int64 [2] (head, tail) or a Step's; it has shape {tuple(cursor.shape)}")
    held_at, added_at, free_at, cursor_at = _ints(held, index, "held", batch), _ints(added, index, "added", batch), _ints(free, index, "free"), _ints(cursor, index, "cursor", None, _I64)
    moved = torch.empty_like(cursor) if cursor.size(0) == 3 else cursor.new_empty(3)
    words = held.new_empty(2 * tokens + 2 * batch + 1)
    at = words.data_ptr()
    status = _lib.mlops_paged_assign(_ASSIGN.pack(batch, tokens, page_size, width, stride, entries, held_at, added_at, free_at, free.size(0), cursor_at, at, at + 4 * tokens,
                                                  at + 8 * tokens, at + 8 * tokens + 4 * batch + 4, moved.data_ptr()), _C._raw_stream(index))
    if status:
        _raise(status, "mlops_paged_assign")
    return Step(*words.split_with_sizes([tokens, tokens, batch + 1, batch]), moved)


def append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> PagedCache:
    """Quantise ``k, v [tokens, kv_heads, 128]`` (BF16 or FP16, slices of a fused projection as they are) into the pool's ``slots`` (int32 [tokens]; a
    slot outside the pool, -1 for instance: the token is left out). The slots of the pool have to be distinct: what two tokens of one slot leave there may be
    a mixture of both. In place; the cache is also returned."""
    pool, heads, index = _pool(cache)
    if not _on(index):
        with torch.cuda.device(index):
            return append(cache, k, v, slots)
    k, shape, k_by_token, k_by_head, kind = _rows(k, index, "k", heads)
    v, v_shape, v_by_token, v_by_head, v_kind = _rows(v, index, "v", heads)
    tokens = shape[0]
    if v_shape[0] != tokens or v_kind != kind:
        raise ValueError(f"k and v have to be alike; k is {k.dtype} {tuple(k.shape)}, v is {v.dtype} {tuple(v.shape)}")
    status = _lib.mlops_paged_append(pool, tokens, kind, k.data_ptr(), k_by_token, k_by_head, v.data_ptr(), v_by_token, v_by_head,
                                     _ints(slots, index, "slots", tokens), _C._raw_stream(index))
    if status:
        _raise(status, "mlops_paged_append")
    return cache


def read(cache: PagedCache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """What the pool holds in ``slots`` (int32 [tokens]): K and V as ``[tokens, kv_heads, 128]``, rounded once to ``dtype`` (BF16 or FP16). Zeros for a
    slot outside the pool."""
    pool, heads, index = _pool(cache)
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"dtype has to be bfloat16 or float16, not {dtype}")
    if not _on(index):
        with torch.cuda.device(index):
            return read(cache, slots, dtype)
    where, tokens = _ints(slots, index, "slots"), slots.size(0)
    k = torch.empty((tokens, heads, HEAD_DIM), dtype=dtype, device=slots.device)
    v = torch.empty_like(k)
    status = _lib.mlops_paged_read(pool, tokens, kind, where, k.data_ptr(), v.data_ptr(), _C._raw_stream(index))
    if status:
        _raise(status, "mlops_paged_read")
    return k, v


def attend(q: torch.Tensor, cache: PagedCache, table: torch.Tensor, lengths: torch.Tensor, starts: Optional[torch.Tensor] = None, *, scale: float = 0.0,
           return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of the requests' newest tokens over their pages.

    ``q [tokens, q_heads, 128]`` BF16 or FP16, ``table`` int32 [batch, width], ``lengths`` int32 [batch]: tokens that each request has in the pool, the
    queries' own among them. ``starts`` int32 [batch + 1]: the rows of request b are ``starts[b] .. starts[b + 1] - 1``, its newest tokens; None: one
    query per request. Row i of n sees the request's tokens up to ``lengths[b] - n + i``. Returns ``[tokens, q_heads, 128]`` of q's type, zeros for a
    row that sees nothing and for rows of no request, before ``starts[0]`` and behind ``starts[batch]``; with ``return_lse`` also the natural log-sum-exp of the rows' scaled scores, float32
    [tokens, q_heads] (-inf for such rows). ``scale`` 0 selects 1/sqrt(128)."""
    pool, kv_heads, index = _pool(cache)
    if not _on(index):
        with torch.cuda.device(index):
            return attend(q, cache, table, lengths, starts, scale=scale, return_lse=return_lse)
    q, (tokens, heads, _), by_token, by_head, kind = _rows(q, index, "q")
    entries, stride, batch, width = _table(table, index)
    where = _ints(lengths, index, "lengths", batch)
    begins = 0 if starts is None else _ints(starts, index, "starts", batch + 1)
    out = q.new_empty((tokens, heads, HEAD_DIM))
    lse = q.new_empty((tokens, heads), dtype=_F32) if return_lse else None
    call = _ATTEND.pack(batch, tokens, heads, kind, q.data_ptr(), by_token, by_head, out.data_ptr(), heads * HEAD_DIM, HEAD_DIM, lse.data_ptr() if return_lse else 0,
                        entries, stride, width, where, begins, scale)
    stream = _C._raw_stream(index)
    scratch = _scratch.get(q.device, stream, max(16, _lib.mlops_paged_attend_scratch_bytes(call, kv_heads)))
    with scratch.lock:
        status = _lib.mlops_paged_attend(call, pool, scratch.pointer, scratch.bytes, stream)
    if status:
        _raise(status, "mlops_paged_attend")
    return (out, lse) if return_lse else out
