"""Attention of a decoder block over row ranges.

The reference's dense block repeats the key/value heads, forms every score in
memory and adds a [S, S] mask (ram_vram_finetune/adapters/dense.py:142-148).
Here query i sees the keys begin[i] <= j < end[i], one pass over the keys with
a running softmax (csrc/fl_attn.cu) and a backward that forms the scores again
(csrc/fl_attn_bwd.cu).  ``row_ranges`` builds the ranges of causal, document,
prefix, sliding-window and padding masks; scores may be capped by a tanh
(``softcap``) and lowered with the distance (``slopes``).

* ``attend(q, k, v, begin, end, ...)``: autograd in q, k and v.
* ``fwd`` / ``bwd``: the two passes directly, as ``ops.fwd`` / ``ops.bwd``.

CUDA only; no CPU fallback.
"""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _need_cuda, _ptr, on_device, stream_of

MAX_HEAD_DIM = 128
MAX_SOFTCAP = 1024  # the tanh's error times the cap is the score's


def row_ranges(batch, length, *, documents=None, prefix=None, window=None, lengths=None, causal=True, device=None):
    """(begin, end) int32 [batch, length]: the keys that each token of a
    [batch, length] block sees.

    causal: tokens up to itself; else all of them.
    documents: int [batch, length] ids; a token sees its own document only (the
        tokens with its id around it, ids in runs).
    prefix: int [batch]; the first prefix[b] tokens are seen by every token of
        their document.  Not with a window: that is not one range a row.
    window: int >= 1; only the last `window` tokens up to itself (causal masks).
    lengths: int [batch]; tokens from lengths[b] on are padding: they see
        nothing and nothing sees them."""
    if length < 0 or batch < 0:
        raise ValueError("batch and length must not be negative")
    if window is not None and (not causal or window < 1):
        raise ValueError("a window needs a causal mask and a size >= 1")
    if window is not None and prefix is not None:
        raise ValueError("unsupported_capability: a prefix with a window is not one range a row")
    given = [t for t in (documents, prefix, lengths) if t is not None]
    if device is None and given:
        device = given[0].device
    for name, t, shape in (("documents", documents, (batch, length)), ("prefix", prefix, (batch,)),
                           ("lengths", lengths, (batch,))):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {list(shape)}")
    at = torch.arange(length, device=device, dtype=torch.int64).expand(batch, length)
    begin, stop = torch.zeros_like(at), torch.full_like(at, length)
    if documents is not None and length:
        documents = documents.to(at.device)
        change = documents[:, 1:] != documents[:, :-1]
        edge = torch.ones_like(documents[:, :1], dtype=torch.bool)
        begin = at.masked_fill(~torch.cat((edge, change), 1), 0).cummax(1).values
        stop = (at + 1).masked_fill(~torch.cat((change, edge), 1), length).flip(1).cummin(1).values.flip(1)
    end = torch.minimum(at + 1, stop) if causal else stop
    if prefix is not None:
        end = torch.maximum(end, torch.minimum(prefix.to(at)[:, None], stop))
    if window is not None:
        begin = torch.maximum(begin, at + 1 - window)
    if lengths is not None:
        live = lengths.to(at)[:, None]
        end = torch.minimum(end, live).masked_fill(at >= live, 0)
    return begin.to(torch.int32).contiguous(), end.clamp_min(0).to(torch.int32).contiguous()


def _view(x):
    """x where the kernels can read it in place (adjacent columns, 16-byte rows, real strides), else a copy."""
    a, b, c, d = x.stride()
    if d == 1 and a > 0 and b > 0 and c > 0 and not (a | b | c) & 7 and not x.data_ptr() & 15:
        return x
    sh, st = x.shape, (a, b, c)
    if d == 1 and not x.data_ptr() & 15 and all(sh[i] == 1 or (st[i] > 0 and st[i] % 8 == 0) for i in (0, 1, 2)):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, begin, end, scale, softcap, slopes):
    _need_cuda(q, k, v, begin, end)
    bf16 = torch.bfloat16
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4 or t.dtype != bf16:
            raise ValueError(f"{name} must be bf16 [batch, tokens, heads, head size]")
    dev = q.device
    if k.device != dev or v.device != dev or begin.device != dev or end.device != dev or \
            slopes is not None and slopes.device != dev:
        raise ValueError("attention arguments must be on one device")
    B, Sq, Hq, D = q.shape
    ks = k.shape
    Sk, Hkv = ks[1], ks[2]
    if ks != v.shape or ks[0] != B or ks[3] != D:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads do not share {Hkv} key/value heads evenly")
    if D > MAX_HEAD_DIM or D < 8 or D % 8:
        raise ValueError(f"unsupported_capability: head size {D} (multiples of 8 up to {MAX_HEAD_DIM})")
    for name, t in (("begin", begin), ("end", end)):
        if t.dtype != torch.int32 or t.shape != (B, Sq):
            raise ValueError(f"{name} must be int32 [batch, query tokens]")
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.shape != (Hq,)):
        raise ValueError("slopes must be fp32 [query heads]")
    scale = D ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    softcap = float(softcap or 0.0)
    if not 0 <= softcap <= MAX_SOFTCAP or softcap and scale / softcap > 1e30:
        raise ValueError(f"softcap must be 0, or at most {MAX_SOFTCAP} and not too small for the scale")
    return dev, B, Sq, Sk, Hq, Hkv, D, scale, softcap


_Strides3 = ctypes.c_int64 * 9
_Strides4 = ctypes.c_int64 * 12


def fwd(q, k, v, begin, end, *, scale=None, softcap=0.0, slopes=None):
    """(out bf16 [B, Sq, Hq, D], lse fp32 [B, Sq, Hq]) of q [B, Sq, Hq, D] over
    k, v [B, Sk, Hkv, D] (bf16, any views; head h reads key/value head
    h // (Hq // Hkv)).

    begin, end: int32 [B, Sq], the keys each query sees (see ``row_ranges``); a
    query that sees none gets 0 and a log sum of -inf.
    Keys and values before the first or behind the last that a sequence's
    queries see, queries that see none and their gradients may hold anything,
    NaN too; a key in between has to be finite (0 times infinity).
    scale: of q . k, default D ** -0.5.  softcap in (0, 1024]: softcap * tanh(x / softcap).
    slopes: fp32 [Hq]; x -= slopes[h] * |i + Sk - Sq - j|."""
    dev, B, Sq, Sk, Hq, Hkv, D, scale, softcap = _check(q, k, v, begin, end, scale, softcap, slopes)
    out = q.new_empty((B, Sq, Hq, D))
    lse = q.new_empty((B, Sq, Hq), dtype=torch.float32)
    if out.numel() == 0:
        return out, lse
    q, k, v = _view(q), _view(k), _view(v)
    begin, end = begin.contiguous(), end.contiguous()
    if slopes is not None:
        slopes = slopes.contiguous()
    n = _lib.function("fl_attn_fwd_workspace_bytes")(B, Sq, Sk, Hq, Hkv, D)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    _lib.check(on_device(dev, _lib.function("fl_attn_fwd"), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         _Strides3(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]), B, Sq, Sk, Hq, Hkv, D,
                         begin.data_ptr(), end.data_ptr(), scale, softcap, _ptr(slopes), out.data_ptr(),
                         lse.data_ptr(), _ptr(ws), n, stream_of(dev)), "fl_attn_fwd")
    return out, lse


def bwd(dout, q, k, v, out, lse, begin, end, *, scale=None, softcap=0.0, slopes=None):
    """(dq, dk, dv) of fwd(): bf16, contiguous; dk and dv summed over the query
    heads that share them, in a fixed order.  out and lse: what fwd() returned."""
    dev, B, Sq, Sk, Hq, Hkv, D, scale, softcap = _check(q, k, v, begin, end, scale, softcap, slopes)
    if dout.shape != q.shape or out.shape != q.shape or dout.dtype != torch.bfloat16 or out.dtype != torch.bfloat16:
        raise ValueError("dout and out must be bf16 of q's shape")
    if lse.shape != (B, Sq, Hq) or lse.dtype != torch.float32:
        raise ValueError("lse must be fp32 [batch, query tokens, query heads]")
    if dout.device != dev or out.device != dev or lse.device != dev:
        raise ValueError("attention arguments must be on one device")
    dq = q.new_empty((B, Sq, Hq, D))
    dk = q.new_empty((B, Sk, Hkv, D))
    dv = torch.empty_like(dk)
    if dq.numel() + dk.numel() == 0:
        return dq, dk, dv
    q, k, v, dout = _view(q), _view(k), _view(v), _view(dout)
    out, lse = out.contiguous(), lse.contiguous()
    begin, end = begin.contiguous(), end.contiguous()
    if slopes is not None:
        slopes = slopes.contiguous()
    n = _lib.function("fl_attn_bwd_workspace_bytes")(B, Sq, Sk, Hq, Hkv, D)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    _lib.check(on_device(dev, _lib.function("fl_attn_bwd"), dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         _Strides4(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *dout.stride()[:3]),
                         out.data_ptr(), lse.data_ptr(), B, Sq, Sk, Hq, Hkv, D, begin.data_ptr(), end.data_ptr(),
                         scale, softcap, _ptr(slopes), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), n,
                         stream_of(dev)), "fl_attn_bwd")
    return dq, dk, dv


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, begin, end, scale, softcap, slopes):
        out, lse = fwd(q, k, v, begin, end, scale=scale, softcap=softcap, slopes=slopes)
        ctx.scale, ctx.softcap = scale, softcap
        ctx.save_for_backward(q, k, v, out, lse, begin, end, slopes)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, begin, end, slopes = ctx.saved_tensors
        dq, dk, dv = bwd(dout, q, k, v, out, lse, begin, end, scale=ctx.scale, softcap=ctx.softcap, slopes=slopes)
        return dq, dk, dv, None, None, None, None, None


def attend(q, k, v, begin, end, *, scale=None, softcap=0.0, slopes=None):
    """fwd()'s output, differentiable in q, k and v (the ranges and slopes are constants)."""
    if slopes is not None and slopes.requires_grad:
        raise ValueError("unsupported_capability: slopes get no gradient")
    return _Attend.apply(q, k, v, begin, end, scale, softcap, slopes)
