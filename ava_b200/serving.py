"""Serving from pages, on torch tensors: the four operators of one scheduling step (include/ava_engine.h, "serving from pages").

    plan            block tables and slot maps from the requests' lengths, pages taken from and given to a free list
    append          the new tokens' keys and values into their pages
    attend          the new tokens' read of their requests' pages (a prompt chunk, a drafted run, a single token)
    verify_drafts   drafted tokens against the target's probabilities

The reference has no counterpart (one growing store per row, design-tests/nn/gpu/src/state.rs:46-49; one token drawn per
step, src/diary.rs:686-718).  Every tensor lives on one CUDA device and is the caller's: nothing is allocated, copied or
waited for, the work is queued on the device's current stream (or `stream`, a cudaStream_t as an int) and may be captured
into a CUDA graph.  Tensors of a wrong type, shape or device raise ValueError, what the library refuses EngineError or
NotApplicable; what only the GPU can see is ORed into `status` (an int32 or uint32 tensor of one element): the bits
NO_PAGES to WAIT_RAN_OUT below.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import engine

NO_PAGES, NO_TABLE, BAD_LENGTH, NO_TOKENS, BAD_PAGE, BAD_TOKEN, NO_MASS, WAIT_RAN_OUT = 1, 2, 4, 8, 16, 32, 64, 128
NO_TOKEN = 0xFFFFFFFF   # -1 in an int32 tensor

_I32, _I64, _F32, _F64, _BF16 = torch.int32, torch.int64, torch.float32, torch.float64, torch.bfloat16
_WORD = (torch.int32, torch.uint32)
_DTYPE = {_F32: 0, _BF16: 1}


class PagedStore(C.Structure):
    """ava_paged_store: keys and values [pages, kv heads, places, channels] in any strides with adjacent channels."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int32), ("n_pages", C.c_int32), ("kv_heads", C.c_int32), ("page_size", C.c_int32),
                ("head_size", C.c_int32), ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("place_stride", C.c_int64)]


def _fail(rc):
    text = engine.lib().ava_serving_last_error().decode()
    if rc == engine.NOT_APPLICABLE:
        raise engine.NotApplicable(text)
    raise engine.EngineError(rc, text)


def _list(t, name, device, shape=None, dtype=_I32):
    """A contiguous tensor's address."""
    if t.dtype is dtype and t.device == device and t.is_contiguous() and (shape is None or t.shape == shape):
        return t.data_ptr()
    raise ValueError(f"{name}: contiguous, {dtype}{'' if shape is None else f', shape {tuple(shape)}'}, on {device}; got {t.dtype} {tuple(t.shape)} on {t.device}")


def _words(t, name, device, shape=None):
    """The same of 32-bit words, signed or not."""
    return _list(t, name, device, shape, t.dtype if t.dtype in _WORD else _WORD)


_MOST = 0x7fffffff   # of numbers that go into 32 bits: ctypes would cut them


def _too_wide(*values):
    raise ValueError(f"{values}: do not fit 32 bits")


def _opt(t, name, device, shape=None, dtype=_I32):
    return None if t is None else _list(t, name, device, shape, dtype)


def _status(t, device):
    return None if t is None else _words(t, "status", device, (1,))


def _cuda(t):
    device = t.device
    if device.type != "cuda":
        raise ValueError("serving operators take CUDA tensors")
    return device


def _stream(stream, device):
    """The device's current stream (the call behind torch.cuda.current_stream, without the object around it: 2 us less)."""
    return torch._C._cuda_getCurrentRawStream(device.index) if stream is None else stream


def _store(k, v):
    shape, stride = k.shape, k.stride()
    if len(shape) != 4 or v.shape != shape or v.stride() != stride or v.dtype is not k.dtype or v.device != k.device or k.dtype not in _DTYPE:
        raise ValueError("k and v pages: [pages, kv heads, places, channels], float32 or bfloat16, with the same strides, on one device")
    if stride[3] != 1 and shape[3] != 1:
        raise ValueError("the channels of a page must be adjacent")
    return PagedStore(k.data_ptr(), v.data_ptr(), _DTYPE[k.dtype], shape[0], shape[1], shape[2], shape[3], stride[0], stride[1], stride[2])


def plan(cached, fresh, table, owned, free_list, free_count, page_size, q_start, slot, *, pos=None, row=None, status=None, trim=False, owned_out=None,
         free_count_out=None, stream=None):
    """The step's lists on the GPU: `table` [rows, max_pages], `owned` [rows] and the stack `free_list` [n_pages] of height
    `free_count` [1] move on (owned and free_count in place unless owned_out / free_count_out are given), `q_start`
    [rows + 1] gets the packed order and `slot` (int64), `pos`, `row` [max_tokens] the tokens' places (-1 behind the last)."""
    if not -_MOST <= page_size <= _MOST:
        _too_wide(page_size)
    device = _cuda(cached)
    rows, tokens = (cached.shape[0],), slot.shape
    if table.dim() != 2 or table.shape[0] != rows[0]:
        raise ValueError("table: [rows, max_pages]")
    rc = engine.lib().ava_paged_plan(
        device.index, _stream(stream, device), _list(cached, "cached", device, rows), _list(fresh, "fresh", device, rows), rows[0], page_size, free_list.shape[0],
        _list(table, "table", device), table.shape[1], _list(owned, "owned", device, rows), _list(owned if owned_out is None else owned_out, "owned_out", device, rows),
        _list(free_list, "free_list", device), _list(free_count, "free_count", device, (1,)),
        _list(free_count if free_count_out is None else free_count_out, "free_count_out", device, (1,)), bool(trim), _list(q_start, "q_start", device, (rows[0] + 1,)),
        _list(slot, "slot", device, None, _I64), _opt(pos, "pos", device, tokens), _opt(row, "row", device, tokens), tokens[0], _status(status, device))
    if rc:
        _fail(rc)


def append(k, v, slot, k_pages, v_pages, *, status=None, stream=None):
    """k and v [tokens, kv heads, channels] (the same strides, adjacent channels: views of a packed q|k|v row are fine) into
    the places `slot` [tokens] (int64) names; negative slots are passed over."""
    device = _cuda(k_pages)
    store = _store(k_pages, v_pages)
    shape, stride = k.shape, k.stride()
    if shape != (slot.shape[0], store.kv_heads, store.head_size) or v.shape != shape or v.dtype is not k.dtype or k.dtype not in _DTYPE or \
            k.device != device or v.device != device:
        raise ValueError("k and v: [tokens, kv heads, channels] of the store, float32 or bfloat16, on its device")
    if (v.stride() != stride and shape[0]) or (stride[2] != 1 and shape[2] != 1):
        raise ValueError("k and v: the same strides, adjacent channels")
    rc = engine.lib().ava_paged_append(device.index, _stream(stream, device), C.byref(store), k.data_ptr(), v.data_ptr(), _DTYPE[k.dtype], stride[0], stride[1],
                                       _list(slot, "slot", device, None, _I64), shape[0], _status(status, device))
    if rc:
        _fail(rc)


def attend_workspace(device, head_size: int) -> int:
    """Bytes of workspace `attend` needs on a device for a head size."""
    index = torch.device(device).index
    n = engine.lib().ava_paged_attend_workspace(torch.cuda.current_device() if index is None else index, head_size)
    if n < 0:
        _fail(engine.ERR_CUDA if head_size in (32, 64, 128) else engine.NOT_APPLICABLE)
    return n


def attend(q, k_pages, v_pages, table, cached, q_start, out, *, max_fresh, workspace, scale, window=0, first=None, lse=None, status=None, stream=None):
    """q [tokens, heads, channels], packed by `q_start` [rows + 1], reads the pages of its requests: token i of request r sees
    the keys first[r] .. cached[r] + i, of them the last `window` if that is not 0.  out like q; lse [tokens, heads] f32.
    max_fresh: the host's largest number of new tokens per request (chooses the kernel).  workspace: a uint8 tensor of
    attend_workspace() bytes, one for each call that may run at the same time."""
    if not (-_MOST <= max_fresh <= _MOST and -_MOST <= window <= _MOST):
        _too_wide(max_fresh, window)
    device = _cuda(q)
    store = _store(k_pages, v_pages)
    shape, stride, to = q.shape, q.stride(), out.stride()
    rows = (cached.shape[0],)
    if len(shape) != 3 or shape[2] != store.head_size or out.shape != shape or out.dtype is not q.dtype or q.dtype not in _DTYPE or out.device != device or \
            k_pages.device != device:
        raise ValueError("q and out: [tokens, heads, channels] of the store, float32 or bfloat16, on its device")
    if (stride[2] != 1 or to[2] != 1) and shape[2] != 1:
        raise ValueError("q and out: adjacent channels")
    if table.dim() != 2 or table.shape[0] != rows[0]:
        raise ValueError("table: [rows, max_pages]")
    rc = engine.lib().ava_paged_attend(
        device.index, _stream(stream, device), C.byref(store), q.data_ptr(), _DTYPE[q.dtype], stride[0], stride[1], shape[1], _list(table, "table", device),
        table.shape[1], _list(cached, "cached", device, rows), _opt(first, "first", device, rows), _list(q_start, "q_start", device, (rows[0] + 1,)), rows[0], shape[0],
        max_fresh, scale, window, out.data_ptr(), to[0], to[1], _opt(lse, "lse", device, shape[:2], _F32), _list(workspace, "workspace", device, None, torch.uint8),
        workspace.numel(), _status(status, device))
    if rc:
        _fail(rc)


def verify_drafts(p, tok, q_start, out, n_out, *, q=None, uniform=None, status=None, stream=None):
    """Drafted tokens against the target's probabilities p [tokens, vocab] (row q_start[r] + i: behind token i of request r;
    tok [tokens] the tokens that were fed, the drafts from q_start[r] + 1 on).  q like p: what the drafts were drawn from
    (None: certain drafts).  uniform [tokens] f64 in [0, 1); None: greedy.  out [rows, max_out] gets the accepted drafts and
    the token behind them, -1 behind that; n_out [rows] their number."""
    device = _cuda(p)
    rows = (n_out.shape[0],)
    for x in (p, q):
        if x is not None and (x.dim() != 2 or x.dtype is not _F32 or x.device != device or x.shape != p.shape or (x.stride(1) != 1 and x.shape[1] != 1)):
            raise ValueError("p and q: [tokens, vocab] float32 with adjacent tokens, on one device")
    if out.dim() != 2 or out.shape[0] != rows[0]:
        raise ValueError("out: [rows, max_out]")
    n, vocab = p.shape
    rc = engine.lib().ava_verify_drafts(
        device.index, _stream(stream, device), p.data_ptr(), max(p.stride(0), vocab), None if q is None else q.data_ptr(), vocab if q is None else max(q.stride(0), vocab),
        _words(tok, "tok", device, (n,)), _list(q_start, "q_start", device, (rows[0] + 1,)), rows[0], n, vocab, _opt(uniform, "uniform", device, (n,), _F64),
        out.shape[1], _words(out, "out", device), _list(n_out, "n_out", device, rows), _status(status, device))
    if rc:
        _fail(rc)
