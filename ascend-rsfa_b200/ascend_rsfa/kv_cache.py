"""A paged cache of K and V in 4 bits, for decoding: what is between attention() on a prompt and the next token.

    kv, weight, position = cache4_empty(pages, heads, page_size, head_dim)      # one per layer
    cache4_append(k, v, kv, table, lengths)              # new rows in; lengths WITH them
    o = cache4_attention(q, kv, table, lengths, scale)   # the new tokens' attention
    lengths = cache4_evict(kv, weight, position, table, lengths, budget, recent)
    k, v = cache4_read(kv, table, lengths, n, dtype)     # back to dense rows, e.g. for attention()

A sequence's slots lie in pages: slot s in page table[b, s // page_size], row s % page_size.  `table` [B, max_pages] and
`lengths` [B] are int32 CUDA tensors, which all layers share; the calls read them on the device and never wait for
the host, so a decoding step can be captured in a CUDA graph.  Rows are quantised in groups of 32 dims with a 16-bit
scale and minimum each, 1.25 bytes per pair of a K and a V element; K goes in as attention is to see it, with its rotary
positions applied (rotary.py).  Head dims 64, 128 and 256, fp16 and bf16; the dtype of q, k and v is the cache's.

Lengths and page numbers out of range make the kernels touch nothing outside; device_status() tells.  The reference has no cache
and no decoding; the kernels are in csrc/cache4_*.cu, without a CPU path.
"""
import ctypes

import torch

from . import _capi
from .flash_attention_forward import _DTYPES
from .rotary import _call, _ordinary, _readable, _rows, _tangent

_lib = _capi.load()
_HEAD_DIMS = (64, 128, 256)


def _strides(*tensors):
    flat = []
    for t in tensors:
        flat.extend(t.stride())
    return (ctypes.c_int64 * len(flat))(*flat)


def cache4_empty(pages, heads, page_size, head_dim, device="cuda"):
    """(kv, weight, position) of an empty cache: uint8 [pages, heads, page_size, 5 head_dim / 4], and fp32 and
    int32 [pages, heads, page_size] for cache4_evict()."""
    if head_dim not in _HEAD_DIMS:
        raise ValueError("head_dim must be 64, 128 or 256")
    if page_size not in (16, 32, 64, 128, 256, 512, 1024):
        raise ValueError("page_size must be a power of two of 16 ... 1024")
    if pages < 1 or heads < 1:
        raise ValueError("a cache needs at least one page and one head")
    shape = (pages, heads, page_size)
    return (torch.zeros(shape + (head_dim * 5 // 4,), dtype=torch.uint8, device=device),
            torch.zeros(shape, dtype=torch.float32, device=device), torch.zeros(shape, dtype=torch.int32, device=device))


def _int32(t, shape, name, device):
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != shape:
        raise ValueError("%s must be an int32 %s tensor on the device of kv" % (name, list(shape)))
    return t


def _cache(kv, table, lengths, dtype, weight=None, position=None):
    """The library's description of a cache, and the tensors it points to that were made here."""
    if kv.dim() != 4 or kv.dtype != torch.uint8 or kv.shape[3] * 4 // 5 not in _HEAD_DIMS or kv.shape[3] % 5:
        raise ValueError("kv must be uint8 [pages, heads, page_size, 5 D / 4] with D = 64, 128 or 256")
    if not kv.is_cuda:
        raise RuntimeError("the cache needs CUDA tensors: this build has no CPU path")
    pages, heads, page_size, rec = kv.shape
    if pages < 1 or heads < 1 or kv.stride(3) != 1 or kv.stride(2) != rec or kv.stride(0) % 16 or kv.stride(1) % 16 or kv.data_ptr() % 16:
        raise ValueError("kv needs contiguous pages of a head, and a base and strides that are multiples of 16 bytes")
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != kv.device or table.shape[1] < 1 or table.stride(1) != 1:
        raise ValueError("table must be an int32 [B, max_pages] tensor with contiguous rows on the device of kv")
    B = table.shape[0]
    lengths = _int32(lengths, (B,), "lengths", kv.device).contiguous()
    c = _capi.Cache4()
    for t, name, want in ((weight, "weight", torch.float32), (position, "position", torch.int32)):
        if t is not None:
            if t.dtype != want or t.device != kv.device or t.shape != kv.shape[:3] or t.stride(2) != 1:
                raise ValueError("%s must be a %s [pages, heads, page_size] tensor with contiguous rows on the device of kv"
                                 % (name, str(want).replace("torch.", "")))
            setattr(c, name, t.data_ptr())
            setattr(c, name + "_stride", (ctypes.c_int64 * 2)(t.stride(0), t.stride(1)))
    c.kv, c.table, c.lengths = kv.data_ptr(), table.data_ptr(), lengths.data_ptr()
    c.kv_stride = (ctypes.c_int64 * 2)(kv.stride(0), kv.stride(1))
    c.table_stride = table.stride(0)
    c.batch, c.heads, c.head_dim, c.page_size, c.pages, c.max_pages = B, heads, rec * 4 // 5, page_size, pages, table.shape[1]
    c.dtype = _DTYPES[dtype]
    return c, lengths


def _check_rows(t, name, c, kv, heads=None):
    if t.dim() != 4 or t.shape[0] != c.batch or t.shape[3] != c.head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError("%s must be [B, heads, S, D] of the cache" % name)
    if t.dtype not in _DTYPES or t.device != kv.device:
        raise ValueError("%s must be float16 or bfloat16 on the device of kv" % name)


def cache4_append(k, v, kv, table, lengths, counts=None, weight=None, position=None, positions=None):
    """Quantises K and V rows [B, heads, S, D] into the last slots of their sequences.

    lengths are the sequences' lengths with the new rows: row j goes to slot lengths[b] - counts[b] + j.
    counts (int32 [B], default S): rows of sequence b that count, the first ones of a padded batch.  Slots below zero
    or behind the pages are left out, so a sequence that is not in use has length 0.
    weight is set to 0 for the new tokens, position to positions [B, S] (int32), the number by which
    cache4_evict() knows the newest ones.
    """
    if _ordinary("cache4_append", k, v, kv, table, lengths, counts, weight, position, positions) is not None:
        return
    if k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _DTYPES:
        raise ValueError("k and v must share one shape and be both float16 or both bfloat16")
    c, lengths = _cache(kv, table, lengths, k.dtype, weight, position)
    _check_rows(k, "k", c, kv, c.heads)
    _check_rows(v, "v", c, kv, c.heads)
    S = k.shape[2]
    if (position is None) != (positions is None):
        raise ValueError("position and positions go together")
    if counts is not None:
        counts = _int32(counts, (c.batch,), "counts", kv.device).contiguous()
    pos_strides = None
    if positions is not None:
        _int32(positions, (c.batch, S), "positions", kv.device)
        pos_strides = _strides(positions)
    if k.numel() == 0:
        return
    kd, vd = _readable(k), _readable(v)
    _call(kv.device, "rsfa_cache4_append", _lib.rsfa_cache4_append, ctypes.byref(c), kd.data_ptr(), vd.data_ptr(), S, _strides(kd, vd),
          None if counts is None else counts.data_ptr(), None if positions is None else positions.data_ptr(), pos_strides)


def cache4_read(kv, table, lengths, n, dtype, starts=None):
    """(k, v): slots starts[b] ... starts[b] + n - 1 (starts: int32 [B], default 0) as dense [B, heads, n, D] rows of the
    cache's dtype; slots that are not in use are zero."""
    if dtype not in _DTYPES:
        raise ValueError("dtype must be float16 or bfloat16")
    done = _ordinary("cache4_read", kv, table, lengths, n, dtype is torch.bfloat16, starts)
    if done is not None:
        return done
    c, lengths = _cache(kv, table, lengths, dtype)
    if starts is not None:
        starts = _int32(starts, (c.batch,), "starts", kv.device).contiguous()
    k, v = (torch.empty((c.batch, c.heads, int(n), c.head_dim), dtype=dtype, device=kv.device) for _ in range(2))
    if k.numel():
        _call(kv.device, "rsfa_cache4_read", _lib.rsfa_cache4_read, ctypes.byref(c), k.data_ptr(), v.data_ptr(), int(n), _strides(k, v),
              None if starts is None else starts.data_ptr())
    return k, v


def _refuse_tangent(q):
    if _tangent(q) is not None:
        raise NotImplementedError("cache4_attention() has no derivative in forward mode")


class _without_gradient(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, kv, table, lengths, sm_scale, counts, weight):
        return cache4_attention(q.detach(), kv, table, lengths, sm_scale, counts=counts, weight=weight, want_lse=True)

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("cache4_attention() has no gradient")


def cache4_attention(q, kv, table, lengths, sm_scale, counts=None, weight=None, want_lse=False):
    """Attention of the sequences' last tokens over the cache: o like q [B, Hq, S, D], or (o, lse).

    Query i of sequence b sees the slots up to lengths[b] - counts[b] + i (counts: int32 [B], default S), so its own row
    has been appended before.  Hq is a multiple of the cache's heads: head h serves query heads h * Hq / heads ... .
    Rows that see nothing - a sequence of length 0, padding behind counts[b] - are zero with an lse of -inf.
    weight: grows, per token and K/V head, by the softmax weights that all query rows of that head give the token.
    lse: [B, Hq, S] fp32, m + log(l).  There is no gradient: a backward pass that reaches the call raises,
    and so does a call with a tangent.
    """
    if torch.is_grad_enabled() and q.requires_grad:
        _refuse_tangent(q)
        o, lse = _without_gradient.apply(q, kv, table, lengths, sm_scale, counts, weight)
        return (o, lse) if want_lse else o
    done = _ordinary("cache4_attention", q, kv, table, lengths, sm_scale, counts, weight, want_lse)
    if done is not None:
        return done if want_lse else done[0]
    _refuse_tangent(q)                   # the native form does not answer for a tensor that has one
    if q.dtype not in _DTYPES:
        raise ValueError("q must be float16 or bfloat16")
    c, lengths = _cache(kv, table, lengths, q.dtype, weight)
    _check_rows(q, "q", c, kv)
    B, Hq, S, D = q.shape
    if Hq % c.heads:
        raise ValueError("q must have a multiple of the cache's %d heads" % c.heads)
    if counts is not None:
        counts = _int32(counts, (B,), "counts", kv.device).contiguous()
    if q.numel() == 0:
        return (torch.empty_like(q), torch.empty((B, Hq, S), dtype=torch.float32, device=q.device)) if want_lse else torch.empty_like(q)
    qd = _readable(q)
    o = _rows(qd)
    lse = torch.empty((B, Hq, S), dtype=torch.float32, device=q.device) if want_lse or weight is not None else None
    with torch.cuda.device(kv.device):
        nbytes = _lib.rsfa_cache4_attention_workspace(ctypes.byref(c), Hq, S)
    if nbytes < 0:
        _capi.check(nbytes, "rsfa_cache4_attention_workspace")
    # the call's own scratch, from the pool of the current stream or of the graph that is being captured
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _call(kv.device, "rsfa_cache4_attention", _lib.rsfa_cache4_attention, ctypes.byref(c), qd.data_ptr(), o.data_ptr(),
          None if lse is None else lse.data_ptr(), Hq, S, _strides(qd, o), None if counts is None else counts.data_ptr(),
          float(sm_scale), ws.data_ptr(), nbytes)
    return (o, lse) if want_lse else o


def cache4_evict(kv, weight, position, table, lengths, budget, recent=0):
    """Cuts every sequence back to `budget` tokens per K/V head, by the weight that cache4_attention() has added up.

    Kept are the tokens at the newest `recent` positions (position > the largest - recent), then the heaviest, the lowest
    slot first among equals.  Kept rows beyond slot `budget` move into the slots that were given up, with their
    weight and position; each head keeps its own choice.  Returns the new lengths, min(lengths, budget); `lengths`
    itself is left for the other layers.  No page may belong to two sequences.
    """
    done = _ordinary("cache4_evict", kv, weight, position, table, lengths, budget, recent)
    if done is not None:
        return done
    budget, recent = int(budget), int(recent)
    if budget < 1 or not 0 <= recent <= budget or budget > 2 ** 31 - 1:
        raise ValueError("cache4_evict() needs 0 <= recent <= budget and a budget of at least 1")
    if weight is None or position is None:
        raise ValueError("cache4_evict() needs weight and position")
    c, lengths = _cache(kv, table, lengths, torch.float16, weight, position)
    out = torch.empty_like(lengths)
    if c.batch == 0:
        return out
    # as many records can move as there are slots within the budget, or beyond it
    nbytes = _lib.rsfa_cache4_evict_workspace(c.batch, c.heads, min(budget, max(c.max_pages * c.page_size - budget, 0)))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=kv.device)
    _call(kv.device, "rsfa_cache4_evict", _lib.rsfa_cache4_evict, ctypes.byref(c), budget, recent, out.data_ptr(), ws.data_ptr(), nbytes)
    return out
