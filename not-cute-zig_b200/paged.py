"""Paged key-value cache on sm_100a (include/ncz_paged.h): the step from the
forward over whole slices (module `flash`) to generating token by token.

    cache = Cache(k_pages, v_pages)                 # [pages, page_size, kv_heads, head_dim]
    plan(held, added, free_pages, free_count, block_table, seq_lens, slots, page_size=16)
    append(k, v, slots, cache)                      # the new tokens' K/V rows into their slots
    decode(q, cache, block_table, seq_lens, o, scale=0.125)

The reference has no cache and no decoding step (its attention takes whole K/V
slices, src/flash.zig:31-70).  Tensors are torch CUDA tensors of one device; calls
run asynchronously on `stream` (default: that device's current stream), whatever
the current device is, and can be captured into CUDA graphs.  Errors raise
FlashError with the library's status code.  A bounded wait that ran out inside decode
is reported by this module's sync_status alone (flash.sync_status and mma.sync_status
are those of the forward and the GEMM).
"""
from __future__ import annotations

import ctypes
from typing import Optional

from . import flash

DTYPE_E4M3 = 3  # NCZ_DTYPE_E4M3

_VP, _SZ, _I32 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32


class _Cache(ctypes.Structure):
    """ncz_paged_cache."""

    _fields_ = [(n, _VP) for n in ("k", "v", "k_scale", "v_scale")] + [(n, _SZ) for n in (
        "num_pages", "page_size", "kv_heads", "head_dim", "k_page_stride", "k_token_stride", "k_head_stride",
        "v_page_stride", "v_token_stride", "v_head_stride")] + [("dtype", _I32)]


class _Plan(ctypes.Structure):
    """ncz_paged_plan_desc."""

    _fields_ = [(n, _VP) for n in ("held", "added", "free_pages", "free_count", "block_table", "seq_lens", "slots",
                                   "positions", "starts", "left", "status")] + [(n, _SZ) for n in (
        "requests", "table_width", "table_stride", "free_capacity", "slot_capacity", "page_size")] + [
        ("device", _I32), ("stream", _VP)]


class _Append(ctypes.Structure):
    """ncz_paged_append_desc."""

    _fields_ = [(n, _VP) for n in ("k", "v", "slots")] + [(n, _SZ) for n in (
        "tokens", "k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride")] + [
        ("in_dtype", _I32), ("device", _I32), ("stream", _VP)]


class _Decode(ctypes.Structure):
    """ncz_paged_decode_desc."""

    _fields_ = [(n, _VP) for n in ("q", "o", "lse", "block_table", "seq_lens")] + [(n, _SZ) for n in (
        "batch", "q_heads", "table_width", "table_stride", "q_batch_stride", "q_head_stride", "o_batch_stride",
        "o_head_stride", "window")] + [("scale", ctypes.c_float), ("q_dtype", _I32), ("o_dtype", _I32),
                                       ("workspace", _VP), ("workspace_bytes", _SZ), ("device", _I32),
                                       ("stream", _VP)]


_SIGNATURES = {
    "ncz_paged_validate": (ctypes.c_int, [ctypes.POINTER(_Cache)]),
    "ncz_paged_plan": (ctypes.c_int, [ctypes.POINTER(_Plan)]),
    "ncz_paged_append": (ctypes.c_int, [ctypes.POINTER(_Cache), ctypes.POINTER(_Append)]),
    "ncz_paged_decode": (ctypes.c_int, [ctypes.POINTER(_Cache), ctypes.POINTER(_Decode)]),
    "ncz_paged_sync_status": (ctypes.c_int, [ctypes.c_int]),
    "ncz_paged_test_set_wait_limit": (ctypes.c_int, [ctypes.c_int, ctypes.c_uint64]),
    "ncz_paged_test_drop_scores": (ctypes.c_int, [ctypes.c_int, ctypes.c_int]),
    "ncz_paged_test_leave_merge": (ctypes.c_int, [ctypes.c_int, ctypes.c_int]),
    "ncz_paged_decode_workspace": (ctypes.c_int, [ctypes.POINTER(_Cache), _SZ, ctypes.c_int, ctypes.POINTER(_SZ)]),
}
_bound: Optional[ctypes.CDLL] = None


def lib() -> ctypes.CDLL:
    global _bound
    if _bound is None:
        handle = flash.lib()
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _bound = handle
    return _bound


_torch = None   # torch, once a call has needed it: importing the package does not
_KINDS: dict = {}  # torch dtype -> ncz_dtype


def _load():
    global _torch
    import torch

    _KINDS.update({torch.float32: flash.DTYPE_F32, torch.float16: flash.DTYPE_F16, torch.bfloat16: flash.DTYPE_BF16,
                   torch.float8_e4m3fn: DTYPE_E4M3})
    _torch = torch
    return torch


def _fail(what: str):
    raise flash.FlashError(5, what)


# Devices are compared by their index (get_device(), -1 on the host) and types by
# identity: half of what Device objects and == cost a call, 10 us with the launch.

def _vector(t, dtype, index: int, what: str, need: int = 0) -> int:
    """Address of a contiguous CUDA vector of the given type on device `index`."""
    if t.dtype is not dtype or t.get_device() != index:
        _fail(f"{what} must be a {dtype} tensor on cuda:{index}")
    if t.dim() != 1 or not t.is_contiguous():
        _fail(f"{what} must be a contiguous vector")
    if need and t.numel() < need:
        _fail(f"{what} holds {t.numel()} elements, needs {need}")
    return t.data_ptr()


def _table(t, index: int, rows: int):
    """(address, width, row stride) of a block table."""
    if t.dtype is not _torch.int32 or t.get_device() != index or t.dim() != 2:
        _fail(f"block_table must be an int32 matrix on cuda:{index}")
    have, width = t.shape
    row, col = t.stride()
    if have < rows:
        _fail(f"block_table has {have} rows, needs {rows}")
    if width > 1 and col != 1:
        _fail("block_table's rows must be contiguous")
    return t.data_ptr(), width, row


def _stream(stream, index: int) -> int:
    """Handle of `stream`, by default of the device's current stream (asked for
    without making a Stream object: 0.1 us instead of 2.2 us a call)."""
    if stream is None:
        return _torch._C._cuda_getCurrentRawStream(index)
    return flash._stream_handle(stream)


class Cache:
    """The two page pools of a cache: k and v [pages, page_size, kv_heads,
    head_dim] with any strides whose last is 1 (a pool with the heads outermost in
    a page is given transposed), float16, bfloat16 or float8_e4m3fn, the last with
    an optional float32 scale per K/V head: an element stands for value * scale.
    Rows must start on 16 bytes.  Checked once, here."""

    def __init__(self, k, v, *, k_scale=None, v_scale=None):
        torch = _torch or _load()
        kinds = _KINDS
        if k.dim() != 4 or v.shape != k.shape:
            _fail("k and v must be [pages, page_size, kv_heads, head_dim] of one shape")
        if not k.is_cuda or v.device != k.device:
            _fail("k and v must be CUDA tensors on one device")
        if k.dtype not in kinds or k.dtype != v.dtype or kinds[k.dtype] == flash.DTYPE_F32:
            _fail("k and v must be float16, bfloat16 or float8_e4m3fn, both the same")
        if k.stride(3) != 1 or v.stride(3) != 1:
            _fail("the elements of a row of k and v must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.dtype, self.index = k.device, k.dtype, k.get_device()
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        self.row = k.shape[2:]
        scales = [None if s is None else _vector(s, torch.float32, self.index, "a scale", self.kv_heads)
                  for s in (k_scale, v_scale)]
        self.struct = _Cache(k.data_ptr(), v.data_ptr(), scales[0], scales[1], *k.shape, *k.stride()[:3],
                             *v.stride()[:3], kinds[k.dtype])
        self.ref = ctypes.byref(self.struct)
        flash._check(lib().ncz_paged_validate(self.ref), "paged.Cache")


def plan(held, added, free_pages, free_count, block_table, seq_lens, slots, *, page_size: int, positions=None,
         starts=None, left=None, status=None, stream=None) -> None:
    """ncz_paged_plan: this step's pages, lengths and slots.

    held, added: int32 [requests], tokens in the cache and new ones.  free_pages:
    int32 stack of free page ids, free_count: int32 [1], how many of them are
    free (pages are taken from free_pages[free_count - 1] downwards).
    block_table: int32 [requests, width], written where pages are taken.
    seq_lens: int32 [requests] (may be `held`); slots: int64, a slot per new token
    in request order, -1 behind the last; positions: int32 like slots, 0 behind;
    starts: int32 [requests + 1]; left: int32 [1], the stack's new count (default:
    free_count itself); status: int32 [4], new tokens, pages taken, requests
    refused, tokens past the slots.  A request is refused (slots -1, everything
    else as it was) when its pages do not fit the table's width or the stack.

    With seq_lens or left in place (left is, by default) 8 SMs do the work: the same time
    for a step of one token each, twice the time for long prompts (98304 new tokens 16.2 us
    instead of 8.8)."""
    torch = _torch or _load()
    device, int32 = held.get_device(), torch.int32
    if not held.is_cuda:
        _fail("held must be a CUDA tensor")
    n, capacity = held.numel(), slots.numel()
    table, width, row = _table(block_table, device, n)
    if positions is not None and positions.numel() < capacity:
        _fail(f"positions holds {positions.numel()} elements, needs {capacity}")
    count = _vector(free_count, int32, device, "free_count", 1)
    desc = _Plan(
        _vector(held, int32, device, "held"), _vector(added, int32, device, "added", n),
        _vector(free_pages, int32, device, "free_pages"), count, table,
        _vector(seq_lens, int32, device, "seq_lens", n), _vector(slots, torch.int64, device, "slots"),
        None if positions is None else _vector(positions, int32, device, "positions"),
        None if starts is None else _vector(starts, int32, device, "starts", n + 1),
        count if left is None else _vector(left, int32, device, "left", 1),
        None if status is None else _vector(status, int32, device, "status", 4),
        n, width, row, free_pages.numel(), capacity, page_size, device, _stream(stream, device))
    flash._check(lib().ncz_paged_plan(ctypes.byref(desc)), "paged.plan")


def append(k, v, slots, cache: Cache, *, stream=None) -> None:
    """ncz_paged_append: rows k[t], v[t] [tokens, kv_heads, head_dim] (any strides
    whose last is 1) to the cache's slots[t] (int64; -1, or any slot outside the
    cache, is skipped; no slot twice).  A float8_e4m3fn cache takes float16 or
    bfloat16 rows and holds x / scale, rounded and saturated; the others take rows
    of their own type.  k and v lie outside the cache, whose K and V are apart."""
    index = cache.index
    shape = k.shape
    if v.shape != shape or shape[1:] != cache.row:
        _fail(f"k and v must be [tokens, {cache.kv_heads}, {cache.head_dim}]")
    dtype = k.dtype
    if k.get_device() != index or v.get_device() != index or v.dtype is not dtype or dtype not in _KINDS:
        _fail(f"k and v must be of one type on {cache.device}")
    k_tok, k_head, k_one = k.stride()
    v_tok, v_head, v_one = v.stride()
    if k_one != 1 or v_one != 1:
        _fail("the elements of a row of k and v must be contiguous")
    tokens = shape[0]
    desc = _Append(k.data_ptr(), v.data_ptr(), _vector(slots, _torch.int64, index, "slots", tokens), tokens, k_tok, k_head,
                   v_tok, v_head, _KINDS[dtype], index, _stream(stream, index))
    flash._check(lib().ncz_paged_append(cache.ref, ctypes.byref(desc)), "paged.append")


def decode_workspace_bytes(cache: Cache, q_heads: int) -> int:
    """ncz_paged_decode_workspace."""
    need = _SZ(0)
    flash._check(lib().ncz_paged_decode_workspace(cache.ref, q_heads, cache.device.index, ctypes.byref(need)),
                 "paged.decode_workspace")
    return need.value


def decode_workspace(cache: Cache, q_heads: int):
    """A workspace for `decode` with this cache and number of query heads, for any
    batch; to be kept and given to every call that cannot run at the same time as
    another one with it (one stream, or one captured graph)."""
    return _torch.empty(decode_workspace_bytes(cache, q_heads), dtype=_torch.uint8, device=cache.device)


def decode(q, cache: Cache, block_table, seq_lens, o, *, scale: float, window: int = 0, lse=None, workspace=None,
           stream=None) -> None:
    """ncz_paged_decode: o[b, h] = softmax(scale * q[b, h] . K) V over the keys of
    request b, query heads h sharing K/V head h // (q_heads // kv_heads).

    q, o: [batch, q_heads, head_dim], any strides whose last is 1, apart; q float16 or
    bfloat16 (the cache's type; either for a float8_e4m3fn cache), o also
    float32.  block_table: int32 [batch, width], seq_lens: int32 [batch].
    window > 0: only the last `window` keys.  Entries that are no page of the
    cache leave their keys out; a row without keys gives o = 0 and lse = -inf.
    lse: float32 [batch, q_heads], receives ln of the softmax's sum.  workspace:
    decode_workspace(cache, q_heads); None allocates one for this call (in a
    captured graph: in the graph's own pool).  The kernel is chosen by the longest row that
    the table's width (or the window) allows: a table no wider than it has to be is faster
    for short rows (one request of 1000 keys 7.1 us, with a table of 131072 keys 9.8)."""
    index, kinds = cache.index, _KINDS
    shape = q.shape
    if len(shape) != 3 or o.shape != shape or shape[2] != cache.head_dim:
        _fail(f"q and o must be [batch, q_heads, {cache.head_dim}]")
    if q.get_device() != index or o.get_device() != index or q.dtype not in kinds or o.dtype not in kinds:
        _fail(f"q and o must be float tensors on {cache.device}")
    batch, heads, _ = shape
    q_batch, q_head, q_one = q.stride()
    o_batch, o_head, o_one = o.stride()
    if q_one != 1 or o_one != 1:
        _fail("the elements of a row of q and o must be contiguous")
    table, width, row = _table(block_table, index, batch)
    if lse is not None and (lse.shape != shape[:2] or lse.get_device() != index or lse.dtype is not _torch.float32
                            or not lse.is_contiguous()):
        _fail(f"lse must be a contiguous float32 tensor [batch, q_heads] on {cache.device}")
    if window < 0:
        _fail("window must not be negative")
    lens = _vector(seq_lens, _torch.int32, index, "seq_lens", batch)
    handle = _stream(stream, index)
    if workspace is None:
        workspace = _call_workspace(cache, heads, stream, handle)
    elif workspace.get_device() != index or not workspace.is_contiguous():
        _fail(f"workspace must be a contiguous tensor on {cache.device}")
    desc = _Decode(q.data_ptr(), o.data_ptr(), None if lse is None else lse.data_ptr(), table, lens, batch, heads,
                   width, row, q_batch, q_head, o_batch, o_head, window, scale, kinds[q.dtype], kinds[o.dtype],
                   workspace.data_ptr(), workspace.nbytes, index, handle)
    flash._check(lib().ncz_paged_decode(cache.ref, ctypes.byref(desc)), "paged.decode")


def _call_workspace(cache: Cache, heads: int, stream, handle: int):
    """A workspace that the caching allocator hands to other work on `stream`
    only after this call's: allocated with that stream current."""
    if stream is None:
        return decode_workspace(cache, heads)
    with _torch.cuda.stream(_torch.cuda.ExternalStream(handle, device=cache.device)):
        return decode_workspace(cache, heads)


def sync_status(device: Optional[int] = None) -> int:
    """Synchronises `device` and raises FlashError(DeviceTimeout) when a bounded
    wait of a decode kernel ran out since the last call."""
    st = lib().ncz_paged_sync_status(-1 if device is None else device)
    flash._check(st, "paged.sync_status")
    return st


def decode_flops(keys: int, q_heads: int, head_dim: int) -> int:
    """Two products of q_heads rows with `keys` keys (over the whole batch)."""
    return 4 * keys * q_heads * head_dim


def decode_bytes(keys: int, batch: int, q_heads: int, kv_heads: int, head_dim: int, cache_bytes: int = 2,
                 q_bytes: int = 2, o_bytes: int = 2) -> int:
    """K and V rows read once per K/V head, q read, o written."""
    return 2 * keys * kv_heads * head_dim * cache_bytes + batch * q_heads * head_dim * (q_bytes + o_bytes)
