"""Rotary position embedding of queries and keys, with an optional norm of every head.

The reference's dense block norms each head (Qwen3) and rotates queries and
keys in about a dozen elementwise passes (ram_vram_finetune/adapters/dense.py:
131-141, rms at :115-117).  Here both are one pass over the data, forward and
backward (csrc/fl_rotary.cu): the inputs may be strided views of a fused
projection's output, angles are formed from the positions in the kernel, and
each result is rounded once.

* ``rotate(q, k, positions, inv_freq)`` and ``norm_rotate(...)``: autograd.
* ``fwd`` / ``bwd``: the two passes directly, as ``ops.fwd`` / ``ops.bwd``.
* ``frequencies(...)``: inverse frequencies under the usual long-context
  scalings, and the factor that cosines and sines are multiplied by.

CUDA only; no CPU fallback.
"""
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _need_cuda, _ptr, on_device, stream_of

_INTS = {torch.int32: 4, torch.int64: 8}
_WEIGHTS = {torch.bfloat16: 2, torch.float32: 4}
MAX_HEAD_DIM = 256


def frequencies(dim, theta=10000.0, scaling=None):
    """(inv_freq fp32 [dim / 2] on the CPU, factor) for `dim` rotated columns.

    `scaling`: None, or a dict with "type" and its parameters:
      * "linear": factor.  Positions are compressed by it.
      * "llama3": factor, low_freq_factor, high_freq_factor, original_length.
        Wavelengths under original_length / high_freq_factor are kept, those
        over original_length / low_freq_factor divided by `factor`, and blended
        linearly in original_length / wavelength between.
      * "yarn": factor, original_length, beta_fast = 32, beta_slow = 1,
        attention_factor = 0.1 ln(factor) + 1.  Frequencies that turn over
        beta_fast times within original_length are kept, those under beta_slow
        times divided by `factor`, with a linear ramp over the index between.
    """
    if not isinstance(dim, int) or dim < 2 or dim % 2:
        raise ValueError("rotated columns must be a positive even number")
    if not theta > 0:
        raise ValueError("theta must be positive")
    index = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    inv = 1.0 / float(theta) ** index
    if scaling is None:
        return inv.float(), 1.0
    opt = dict(scaling)
    kind = opt.pop("type", None)
    need = {"linear": ("factor",), "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_length"),
            "yarn": ("factor", "original_length")}
    more = {"yarn": ("beta_fast", "beta_slow", "attention_factor")}
    if kind not in need:
        raise ValueError(f"unsupported_capability: rotary scaling {kind!r} (linear, llama3 and yarn are)")
    unknown = set(opt) - set(need[kind]) - set(more.get(kind, ()))
    missing = [n for n in need[kind] if n not in opt]
    if unknown or missing:
        raise ValueError(f"rotary scaling {kind!r}: missing {missing}, unknown {sorted(unknown)}")
    by = float(opt["factor"])
    if not 1.0 <= by < math.inf:
        raise ValueError("rotary scaling factor must be >= 1 and finite")
    if kind == "linear":
        return (inv / by).float(), 1.0
    length = float(opt["original_length"])
    if not 0 < length < math.inf:
        raise ValueError("rotary scaling original_length must be positive and finite")
    if kind == "llama3":
        low, high = float(opt["low_freq_factor"]), float(opt["high_freq_factor"])
        if not high > low > 0:
            raise ValueError("rotary scaling needs high_freq_factor > low_freq_factor > 0")
        turns = length * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return (keep * inv + (1 - keep) * inv / by).float(), 1.0
    if not theta > 1:
        raise ValueError("rotary scaling 'yarn' needs theta > 1")
    fast, slow = float(opt.get("beta_fast", 32.0)), float(opt.get("beta_slow", 1.0))
    if not fast > slow > 0:
        raise ValueError("rotary scaling needs beta_fast > beta_slow > 0")

    def column(turns):  # the (real) pair index whose wavelength turns this often in original_length
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(float(theta)))

    first, last = max(math.floor(column(fast)), 0), min(math.ceil(column(slow)), dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
    factor = opt.get("attention_factor")
    if factor is None:
        factor = 0.1 * math.log(by) + 1.0
    return (inv * (1 - ramp) + inv / by * ramp).float(), float(factor)


def _rows(x, what):
    """x [..., heads, D] as (tensor, token stride, head stride): no copy where
    the leading dimensions have one stride between tokens."""
    if x.dtype != torch.bfloat16:
        raise ValueError(f"{what} must be bf16")
    shape, stride = x.shape, x.stride()
    if len(shape) == 3 and (stride[2] == 1 or shape[2] == 1):
        return x, stride[0], stride[1]
    step, reach, even = 0, 1, stride[-1] == 1
    for n, s in zip(reversed(shape[:-2]), reversed(stride[:-2])):
        if n == 1:
            continue
        if reach == 1:
            step = s
        even = even and s == step * reach
        reach *= n
    if not even:
        x = x.contiguous()
        return x, shape[-2] * shape[-1], shape[-1]
    return x, step, stride[-2]


def _setup(q, k, positions, inv_freq, q_weight, k_weight, eps):
    """Argument checks of both passes and what they share: (tokens, key heads,
    positions, position bytes, inv_freq, rotated columns, weights, weight bytes, eps)."""
    _need_cuda(q, k, positions, inv_freq)
    dev, shape = q.device, q.shape
    if len(shape) < 3:
        raise ValueError("q must be [..., heads, head size]")
    D, lead = shape[-1], shape[:-2]
    kh = 0
    if k is not None:
        ks = k.shape
        if len(ks) != len(shape) or ks[-1] != D or ks[:-2] != lead:
            raise ValueError("q and k must agree in their leading dimensions and head size")
        kh = ks[-2]
    pbytes = _INTS.get(positions.dtype)
    if pbytes is None:
        raise ValueError("positions must be int32 or int64")
    if positions.shape != lead:
        try:
            positions = positions.expand(lead)
        except RuntimeError:
            raise ValueError(f"positions {tuple(positions.shape)} do not fit the tokens {tuple(lead)}") from None
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be fp32 [rotated columns / 2]")
    rot = 2 * inv_freq.shape[0]
    if rot < 2 or rot > D:
        raise ValueError(f"{rot} rotated columns do not fit a head of {D}")
    if D > MAX_HEAD_DIM:
        raise ValueError(f"unsupported_capability: head size {D} > {MAX_HEAD_DIM}")
    if (k is not None and k.device != dev) or positions.device != dev or inv_freq.device != dev:
        raise ValueError("rotary arguments must be on one device")
    wbytes = 0
    if q_weight is not None or k_weight is not None:
        if q_weight is None or (k_weight is None and k is not None):
            raise ValueError("give both norm weights or neither")
        for w in (q_weight, k_weight):
            if w is None:
                continue
            if w.shape != (D,) or w.dtype not in _WEIGHTS or w.dtype != q_weight.dtype:
                raise ValueError("norm weights must be bf16 or fp32 [head size], of one type")
            if w.device != dev:
                raise ValueError("rotary arguments must be on one device")
        if eps is None or not eps >= 0:
            raise ValueError("a norm needs eps >= 0")
        wbytes = _WEIGHTS[q_weight.dtype]
        q_weight = q_weight.contiguous()
        k_weight = None if k_weight is None else k_weight.contiguous()
    return (math.prod(lead), kh, positions.contiguous(), pbytes, inv_freq.contiguous(), rot, q_weight, k_weight,
            wbytes, float(eps or 0.0))


def _like(x):
    """Contiguous uninitialised tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def fwd(q, k, positions, inv_freq, *, interleaved=False, factor=1.0, q_weight=None, k_weight=None, eps=None):
    """(q', k'): q [..., Hq, D] and k [..., Hk, D] (or None), bf16, with the first
    2 * len(inv_freq) columns of every head rotated by positions * inv_freq,
    after an RMS norm of each head when the weights are given.  Contiguous.

    positions: int32 or int64, broadcastable to the leading dimensions.
    interleaved: columns (2p, 2p + 1) pair up, not (p, p + rot / 2).
    factor: multiplies cosine and sine (see ``frequencies``)."""
    T, Hk, positions, pbytes, inv_freq, rot, q_weight, k_weight, wbytes, eps = _setup(q, k, positions, inv_freq,
                                                                                      q_weight, k_weight, eps)
    qr, qt, qh = _rows(q, "q")
    kr, kt, kh = _rows(k, "k") if k is not None else (None, 0, 0)
    yq = _like(q)
    yk = None if k is None else _like(k)
    if T == 0:
        return yq, yk
    dev = q.device
    _lib.check(on_device(dev, _lib.function("fl_rotary_fwd"), qr.data_ptr(), qt, qh, q.shape[-2], _ptr(kr), kt, kh, Hk,
                         T, q.shape[-1], positions.data_ptr(), pbytes, inv_freq.data_ptr(), rot,
                         1 if interleaved else 0, factor, _ptr(q_weight), _ptr(k_weight), wbytes, eps, yq.data_ptr(),
                         _ptr(yk), stream_of(dev)), "fl_rotary_fwd")
    return yq, yk


def bwd(dq, dk, q, k, positions, inv_freq, *, interleaved=False, factor=1.0, q_weight=None, k_weight=None, eps=None,
        weight_grads=False):
    """Gradients of fwd(): (dq, dk, dq_weight, dk_weight) from those of its results.
    q and k are the forward's inputs, read only with a norm; dq and dk may be
    any views.  Weight gradients (fp32 [D], summed in a fixed order) are formed
    with weight_grads=True, else None."""
    if (k is None) != (dk is None):
        raise ValueError("dk goes with k")
    T, Hk, positions, pbytes, inv_freq, rot, q_weight, k_weight, wbytes, eps = _setup(q, k, positions, inv_freq,
                                                                                      q_weight, k_weight, eps)
    if dq.shape != q.shape or k is not None and dk.shape != k.shape:
        raise ValueError("dq and dk must have the shapes of q and k")
    dev = q.device
    if dq.device != dev or dk is not None and dk.device != dev:
        raise ValueError("rotary arguments must be on one device")
    if weight_grads and not wbytes:
        raise ValueError("weight gradients need the norm weights")
    dqr, dqt, dqh = _rows(dq, "dq")
    dkr, dkt, dkh = _rows(dk, "dk") if k is not None else (None, 0, 0)
    qr, qt, qh, kr, kt, kh = None, 0, 0, None, 0, 0
    if wbytes:
        qr, qt, qh = _rows(q, "q")
        if k is not None:
            kr, kt, kh = _rows(k, "k")
    D = q.shape[-1]
    gq = _like(dq)
    gk = None if k is None else _like(dk)
    gqw = gkw = ws = None
    nbytes = 0
    if weight_grads:
        gqw = q.new_zeros(D, dtype=torch.float32) if T == 0 else q.new_empty(D, dtype=torch.float32)
        gkw = None if k is None else gqw.new_zeros(D) if T == 0 else gqw.new_empty(D)
        nbytes = _lib.function("fl_rotary_bwd_workspace_bytes")(D)
        ws = q.new_empty(nbytes, dtype=torch.uint8)
    if T:
        _lib.check(on_device(dev, _lib.function("fl_rotary_bwd"), dqr.data_ptr(), dqt, dqh, _ptr(dkr), dkt, dkh,
                             _ptr(qr), qt, qh, q.shape[-2], _ptr(kr), kt, kh, Hk, T, D, positions.data_ptr(), pbytes,
                             inv_freq.data_ptr(), rot, 1 if interleaved else 0, factor, _ptr(q_weight),
                             _ptr(k_weight), wbytes, eps, gq.data_ptr(), _ptr(gk), _ptr(gqw), _ptr(gkw), _ptr(ws),
                             nbytes, stream_of(dev)), "fl_rotary_bwd")
    return gq, gk, gqw, gkw


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, inv_freq, interleaved, factor, eps):
        ctx.opt = dict(interleaved=interleaved, factor=factor, eps=eps)
        # Without a norm the gradients need no inputs: nothing keeps them alive.
        ctx.has_k, norm = k is not None, q_weight is not None
        ctx.save_for_backward(q if norm else None, k if norm else None, q_weight, k_weight, positions, inv_freq)
        ctx.set_materialize_grads(True)
        yq, yk = fwd(q.detach(), None if k is None else k.detach(), positions, inv_freq, q_weight=q_weight,
                     k_weight=k_weight, **ctx.opt)
        return (yq,) if yk is None else (yq, yk)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        q, k, q_weight, k_weight, positions, inv_freq = ctx.saved_tensors
        if q is None:
            q, k = dq, dk if ctx.has_k else None
        weights = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        gq, gk, gqw, gkw = bwd(dq, dk, q, k, positions, inv_freq, q_weight=q_weight, k_weight=k_weight,
                               weight_grads=weights, **ctx.opt)
        # a key norm's weight without keys has no part in the result: no gradient
        return (gq, gk, gqw.to(q_weight.dtype) if ctx.needs_input_grad[2] else None,
                gkw.to(k_weight.dtype) if ctx.needs_input_grad[3] and gkw is not None else None,
                None, None, None, None, None)


def _constant(inv_freq):
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise ValueError("unsupported_capability: inv_freq gets no gradient")


def rotate(q, k, positions, inv_freq, *, interleaved=False, factor=1.0):
    """fwd() without a norm, differentiable in q and k (positions and frequencies are
    constants).  k None: returns (q', None)."""
    _constant(inv_freq)
    out = _Rotary.apply(q, k, None, None, positions, inv_freq, bool(interleaved), float(factor), None)
    return out[0], out[1] if k is not None else None


def norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, *, eps, interleaved=False, factor=1.0):
    """fwd() with the norm of every head, differentiable in q, k and the norm weights."""
    if q_weight is None:
        raise ValueError("norm_rotate needs the norm weights (rotate has none)")
    _constant(inv_freq)
    out = _Rotary.apply(q, k, q_weight, k_weight, positions, inv_freq, bool(interleaved), float(factor), eps)
    return out[0], out[1] if k is not None else None
