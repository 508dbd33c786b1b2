"""Rotary positions for q and k, in front of attention() or of the 4-bit cache (kv_cache.py).

    table = rotary_table(length, dim)                      # once, or again when the context outgrows it
    q, k = rotary(q, k, table, positions)                  # differentiable, in both modes

on the same [B, H, S, D] fp16 / bf16 CUDA tensors as attention(); the reference applies no positions, its
callers do.  The work is done by hand-written kernels in librsfa_b200.so (csrc/rotary.cu): without the
library, or on a non-CUDA tensor, the calls raise.
"""
import ctypes
import math

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _capi
from .flash_attention_forward import _DTYPES, _current_stream, _dense, _rsfa_torch

_lib = _capi.load()
_native = _rsfa_torch   # the ordinary calls in native code (csrc/torch_binding.cpp), where that is built
if _native is not None:
    _native.bind_ops(*(ctypes.cast(getattr(_lib, "rsfa_" + n), ctypes.c_void_p).value for n in (
        "rotary", "cache4_append", "cache4_read", "cache4_attention_workspace", "cache4_attention",
        "cache4_evict_workspace", "cache4_evict", "strerror")))
_TURNS = {"yarn": (1.0, 32.0), "bands": (1.0, 4.0)}   # usual (low, high) numbers of turns over the original length


def _call(device, what, fn, *args):
    """fn(*args, stream) with `device` current, on its current stream."""
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _current_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _current_stream(device.index))
    if rc != 0:
        _capi.check(rc, what)


def rotary_table(length, dim, base=10000.0, scaling="none", factor=1.0, original_length=0, turns=None,
                 multiplier=None, device=None):
    """[length, dim / 2, 2] fp32 cosines and sines of positions 0 ... length - 1 for rotary(), from angles in 64 bits.

    The angle per position of pair i is base^(-2 i / dim), for long contexts scaled by one of
      "linear"  divided by `factor`,
      "ntk"     base times factor^(dim / (dim - 2)),
      "yarn"    unscaled for the pairs that make more than turns[1] turns over `original_length`, divided by `factor` for
                those below turns[0], a ramp over the pairs between; cosines and sines times 0.1 ln(factor) + 1,
      "bands"   the same with a ramp that is linear in the turns, and no multiplier.
    `multiplier` replaces what cosines and sines are multiplied with.
    """
    if scaling not in _capi.RSFA_ROTARY:
        raise ValueError("scaling must be one of %s" % ", ".join(_capi.RSFA_ROTARY))
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise RuntimeError("rotary_table() needs a CUDA device: this build has no CPU path")
    length, dim = int(length), int(dim)
    if length < 1 or dim < 2 or dim % 2 or dim > 256 or length > 2 ** 31 - 1:
        raise ValueError("rotary_table() needs a positive length and an even dim of 2 ... 256")
    low, high = turns if turns is not None else _TURNS.get(scaling, (0.0, 0.0))
    if multiplier is None:
        multiplier = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and factor > 1 else 1.0
    table = torch.empty((length, dim // 2, 2), dtype=torch.float32, device=device)
    _call(table.device, "rsfa_rotary_table", _lib.rsfa_rotary_table, table.data_ptr(), length, dim, float(base),
          _capi.RSFA_ROTARY[scaling], float(factor), int(original_length), float(low), float(high), float(multiplier))
    return table


def _readable(t):
    """t's rows as the library reads them, copied once if need be."""
    d = _dense(t.detach())
    return d if d.data_ptr() % 16 == 0 else d.clone()


def _rows(t):
    """An output like t whose rows the library can write: dense in t's own order where that is possible."""
    o = torch.empty_like(t)
    if o.stride(-1) == 1 and all(o.shape[i] == 1 or o.stride(i) % 8 == 0 for i in range(3)):
        return o
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _ordinary(what, *args):
    """What the native form of a call returns, None where it is not an ordinary one."""
    if _native is None:
        return None
    done = getattr(_native, what)(*args)
    if type(done) is int:
        _capi.check(done, "rsfa_" + what)
    return done


def _turn(q, k, table, positions, interleaved, inverse):
    done = _ordinary("rotary", q, k, table, positions, interleaved, inverse)
    if done is not None:
        return done
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return torch.empty_like(q), None if k is None else torch.empty_like(k)
    if k is not None and (q.numel() == 0 or k.numel() == 0):       # no heads on one side
        one = _turn(k if q.numel() == 0 else q, None, table, positions, interleaved, inverse)[0]
        return (torch.empty_like(q), one) if q.numel() == 0 else (one, torch.empty_like(k))
    B, Hq, S, D = q.shape
    qd = _readable(q)
    qo = _rows(qd)
    Hk, kd, ko = 0, None, None
    if k is not None:
        Hk, kd = k.shape[1], _readable(k)
        ko = _rows(kd)
    strides = (ctypes.c_int64 * 16)(*qd.stride(), *(kd.stride() if Hk else (0,) * 4), *qo.stride(),
                                    *(ko.stride() if Hk else (0,) * 4))
    pos_strides = None
    if positions is not None:
        st = positions.stride()
        pos_strides = (ctypes.c_int64 * 2)(0 if len(st) == 1 or positions.shape[0] == 1 else st[0], st[-1])
    _call(q.device, "rsfa_rotary", _lib.rsfa_rotary, qd.data_ptr(), kd.data_ptr() if Hk else None, qo.data_ptr(),
          ko.data_ptr() if Hk else None, B, Hq, Hk, S, D, strides, table.data_ptr(), table.shape[0], 2 * table.shape[1],
          None if positions is None else positions.data_ptr(),
          int(positions is not None and positions.dtype == torch.int64), pos_strides, int(interleaved), int(inverse),
          _DTYPES[q.dtype])
    return qo, ko


def _tangent(t):
    return None if t is None else unpack_dual(t).tangent


def _turn_recorded(q, k, table, positions, interleaved, inverse):
    """_turn(), seen by autograd where a gradient is recorded or a tangent carried."""
    if k is not None and (_tangent(q) is None) != (_tangent(k) is None):
        # a node's outputs have tangents together or not at all
        return tuple(_turn_recorded(t, None, table, positions, interleaved, inverse)[0] for t in (q, k))
    if _tangent(q) is None and not (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
        return _turn(q, k, table, positions, interleaved, inverse)
    return _rotary.apply(q, k, table, positions, interleaved, inverse)


class _rotary(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, table, positions, interleaved, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(table, positions)
        ctx.save_for_forward(table, positions)
        ctx.how = (interleaved, inverse)
        return _turn(q, k, table, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        # the transposed rotation of the gradients; it can be differentiated again
        table, positions = ctx.saved_tensors
        interleaved, inverse = ctx.how
        if dq is None:
            if dk is not None:
                dk = _turn_recorded(dk, None, table, positions, interleaved, not inverse)[0]
        else:
            dq, dk = _turn_recorded(dq, dk, table, positions, interleaved, not inverse)
        return dq, dk, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        # tangents turn like what they belong to
        return _turn_recorded(tq, tk, *ctx.saved_tensors, *ctx.how)


def rotary(q, k, table, positions=None, interleaved=False):
    """(q', k'): q [B, Hq, S, D] and k [B, Hk, S, D] (or None) turned by their positions.

    table      from rotary_table(); its dim, at most D, is the part of the head that turns, the rest is copied.
    positions  int32 or int64 CUDA tensor [S], [1, S] or [B, S]; None: 0 ... S - 1.  A row whose position is
               outside the table comes out as NaN, and device_status() tells.
    interleaved  pairs are (2 i, 2 i + 1) instead of (i, i + dim / 2).

    Forward and backward can be captured in a CUDA graph; torch refuses that, for any operation, while a graph of the
    same leaves that was recorded on another stream is alive.
    """
    done = _ordinary("rotary", q, k, table, positions, interleaved, False)
    if done is not None:
        return done
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:])):
        raise ValueError("q and k must be [B, H, S, D] and share B, S and D")
    if q.shape[-1] not in {16, 32, 64, 128, 256}:
        raise ValueError("D must be 16, 32, 64, 128 or 256")
    if not q.is_cuda or (k is not None and not k.is_cuda):
        raise RuntimeError("rotary() needs CUDA tensors: this build has no CPU path")
    if q.dtype not in _DTYPES or (k is not None and k.dtype != q.dtype):
        raise ValueError("q and k must both be float16 or both bfloat16")
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous() or table.numel() == 0:
        raise ValueError("table must be a contiguous float32 [length, dim / 2, 2] tensor")
    if table.requires_grad:
        raise ValueError("rotary() has no gradient for its table")
    if 2 * table.shape[1] > q.shape[-1]:
        raise ValueError("the table turns %d dims, more than a head has" % (2 * table.shape[1]))
    if table.device != q.device or (k is not None and k.device != q.device):
        raise ValueError("q, k and table must live on one device")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
            raise ValueError("positions must be int32 or int64 on the device of q")
        if positions.shape not in ((q.shape[2],), (1, q.shape[2]), (q.shape[0], q.shape[2])):
            raise ValueError("positions must be [S], [1, S] or [B, S]")
    return _turn_recorded(q, k, table, positions, bool(interleaved), False)
