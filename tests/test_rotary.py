"""Rotary embedding of queries and keys, with and without a norm of every head
(spilltune_b200.rotary), against the formulas in 64 bits.

Tolerance: the kernels compute in FP32 and round once, so a result is off by at
most half a bf16 step (2^-8 of the value) plus FP32 error.  A rotated column is
a sum of two products whose factors carry a few roundings each (2^-24): under
32 * 2^-24 < 2e-6 of the pair's magnitude, norm included."""
import math

import pytest
import torch

HALF = torch.finfo(torch.bfloat16).eps / 2
FP32 = 2e-6


def _oracle(x, pos, inv, factor, inter, w=None, eps=0.0):
    """fwd() of one side in float64 (differentiable)."""
    rot = 2 * inv.shape[0]
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    angle = pos.double()[..., None, None] * inv.double()
    c, s = angle.cos() * factor, angle.sin() * factor
    a, rest = y[..., :rot], y[..., rot:]
    l, r = (a[..., 0::2], a[..., 1::2]) if inter else (a[..., :rot // 2], a[..., rot // 2:])
    l, r = c * l - s * r, c * r + s * l
    a = torch.stack((l, r), -1).flatten(-2) if inter else torch.cat((l, r), -1)
    return torch.cat((a, rest), -1)


def _near(got, want, magnitude):
    """Element-wise: half a step of the value plus FP32 error of the pair's magnitude."""
    err = (got.double() - want).abs()
    bound = HALF * want.abs() + FP32 * magnitude
    assert bool((err <= bound).all()), float((err - bound).max())


def _case(T, Hq, Hk, D, rot, inter, norm, first, seed, layout="packed", wdtype=torch.bfloat16, pdtype=torch.int64):
    from spilltune_b200 import rotary
    g = torch.Generator().manual_seed(seed)
    bf = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    if layout == "packed":
        x = bf(T, (Hq + 2 * Hk) * D).cuda()
        q, k = x[:, :Hq * D].view(T, Hq, D), x[:, Hq * D:(Hq + Hk) * D].view(T, Hk, D)
    elif layout == "odd":  # rows that are not 16-byte aligned
        x = bf(T, Hq + Hk, D + 3).cuda()
        q, k = x[:, :Hq, 1:D + 1], x[:, Hq:, 2:D + 2]
    else:  # heads before tokens
        q, k = bf(Hq, T, D).cuda().transpose(0, 1), bf(Hk, T, D).cuda().transpose(0, 1)
    inv, factor = rotary.frequencies(rot, 10000.0, {"type": "yarn", "factor": 4.0, "original_length": 512})
    pos = (first + torch.randperm(T, generator=g)).to(pdtype).cuda()
    qw = kw = None
    if norm:
        qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdtype).cuda() for _ in range(2))
    dq, dk = bf(T, Hq, D).cuda(), bf(T, Hk, D).cuda()
    return q, k, pos, inv.cuda(), factor, qw, kw, dq, dk


CASES = [  # T, Hq, Hk, D, rot, interleaved, norm, first position, layout
    (1, 32, 8, 128, 128, False, False, 8191, "packed"),
    (1, 1, 1, 32, 2, True, True, 0, "packed"),
    (3, 4, 2, 64, 64, True, False, 0, "packed"),
    (257, 14, 2, 80, 40, False, True, 250000, "packed"),
    (61, 6, 3, 96, 96, False, True, 3, "packed"),
    (61, 6, 3, 96, 48, True, True, 3, "packed"),
    (130, 8, 1, 128, 32, False, False, 2000000000, "packed"),
    (1000, 3, 1, 256, 256, False, True, 900000, "packed"),
    (1000, 5, 5, 128, 128, True, True, 17, "heads"),
    (33, 4, 2, 64, 64, False, True, 0, "odd"),
    (33, 4, 2, 72, 36, True, False, 0, "odd"),
    (20, 2, 1, 250, 250, False, True, 5, "packed"),
    (5, 2, 1, 6, 4, False, True, 5, "packed"),
    (5000, 16, 4, 64, 32, False, False, 0, "packed"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("T,Hq,Hk,D,rot,inter,norm,first,layout", CASES)
def test_forward_and_backward(cuda_lib, T, Hq, Hk, D, rot, inter, norm, first, layout):
    from spilltune_b200 import rotary
    q, k, pos, inv, factor, qw, kw, dq, dk = _case(T, Hq, Hk, D, rot, inter, norm, first, T + D, layout)
    opt = dict(interleaved=inter, factor=factor)
    if norm:
        opt.update(q_weight=qw, k_weight=kw, eps=1e-6)
    yq, yk = rotary.fwd(q, k, pos, inv, **opt)
    gq, gk, gqw, gkw = rotary.bwd(dq, dk, q, k, pos, inv, weight_grads=norm, **opt)
    for x, y, dy, g, w, gw in ((q, yq, dq, gq, qw, gqw), (k, yk, dk, gk, kw, gkw)):
        x64 = x.double().requires_grad_(True)
        w64 = None if w is None else w.double().requires_grad_(True)
        want = _oracle(x64, pos, inv, factor, inter, w64, 1e-6)
        grads = torch.autograd.grad(want, [x64] + ([w64] if norm else []), dy.double())
        # a pair's magnitude: bounded by the largest value of its head after the norm
        size = lambda t: t.abs().amax(-1, keepdim=True) * 2 * factor  # noqa: E731
        xn = x64.detach() if w is None else _oracle(x64, pos * 0, inv, 1.0, inter, w64, 1e-6).detach()
        _near(y, want.detach(), size(xn))
        if w is None:
            _near(g, grads[0], size(dy.double()))
        else:
            r = 1 / (x64.detach().pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
            # g w - xh mean(g w xh): both terms are under max|dy| max|w| max(1, max|xh|^2)
            xh = (x64.detach() * r).abs().amax(-1, keepdim=True).clamp_min(1.0)
            _near(g, grads[0], size(dy.double()) * w.double().abs().max() * r * xh * xh * 2)
            # Sums of T * heads terms; the longest chain of additions (a thread's rows, then the
            # row groups, then the blocks) is under 400 long here: 400 * 2^-24 of the terms' magnitudes.
            back = _oracle(dy.double(), -pos, inv, factor, inter)
            terms = (back * (x64.detach() * r)).abs().sum((0, 1))
            assert bool(((gw.double() - grads[1]).abs() <= 400 * 2.0 ** -24 * terms + FP32 * terms).all())


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype,pdtype", [(torch.float32, torch.int32), (torch.bfloat16, torch.int32)])
def test_weight_and_position_types(cuda_lib, wdtype, pdtype):
    from spilltune_b200 import rotary
    q, k, pos, inv, factor, qw, kw, _, _ = _case(37, 4, 2, 64, 64, False, True, 9, 1, wdtype=wdtype, pdtype=pdtype)
    yq, yk = rotary.fwd(q, k, pos, inv, factor=factor, q_weight=qw, k_weight=kw, eps=1e-6)
    for x, y, w in ((q, yq, qw), (k, yk, kw)):
        want = _oracle(x, pos, inv, factor, False, w, 1e-6)
        xn = _oracle(x, pos * 0, inv, 1.0, False, w, 1e-6)
        _near(y, want, xn.abs().amax(-1, keepdim=True) * 2 * factor)


@pytest.mark.gpu
def test_autograd_matches_differences(cuda_lib):
    """The directional derivative of a fixed projection of the results, against a central
    difference of the 64-bit formula (which test_forward_and_backward ties the kernel to)."""
    from spilltune_b200 import rotary
    q, k, pos, inv, factor, qw, kw, dq, dk = _case(19, 4, 2, 64, 32, False, True, 11, 5)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, qw, kw)]
    yq, yk = rotary.norm_rotate(*leaves, pos, inv, eps=1e-6, factor=factor)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    g = torch.Generator().manual_seed(6)
    step = [torch.randn(t.shape, generator=g, dtype=torch.float64).cuda() for t in leaves]

    def at(e):
        a, b, wa, wb = (t.detach().double() + e * s for t, s in zip(leaves, step))
        return float((_oracle(a, pos, inv, factor, False, wa, 1e-6) * dq.double()).sum()
                     + (_oracle(b, pos, inv, factor, False, wb, 1e-6) * dk.double()).sum())

    want = (at(1e-4) - at(-1e-4)) / 2e-4
    parts = [g.double() * s for g, s in zip(grads, step)]
    got = float(sum(p.sum() for p in parts))
    # every gradient element is off by at most half a bf16 step; the difference by O(e^2)
    assert abs(got - want) <= float(sum(HALF * p.abs().sum() for p in parts)) + 1e-5 * abs(want) + 1e-3


@pytest.mark.gpu
def test_only_queries_one_used_result_and_empty(cuda_lib):
    from spilltune_b200 import rotary
    q, k, pos, inv, factor, qw, kw, dq, dk = _case(9, 4, 2, 64, 64, False, False, 2, 7)
    both = rotary.fwd(q, k, pos, inv, factor=factor)
    alone, none = rotary.rotate(q, None, pos, inv, factor=factor)
    assert none is None and torch.equal(alone, both[0])
    ql, kl = (t.detach().clone().requires_grad_(True) for t in (q, k))
    yq, _ = rotary.rotate(ql, kl, pos, inv, factor=factor)
    gq, gk = torch.autograd.grad(yq, (ql, kl), dq)
    assert torch.equal(gq, rotary.bwd(dq, dk, q, k, pos, inv, factor=factor)[0]) and not bool(gk.any())
    e, f = rotary.fwd(q[:0], k[:0], pos[:0], inv)
    assert e.shape == (0, 4, 64) and f.shape == (0, 2, 64)
    w = torch.ones(64, device="cuda")
    _, _, gqw, gkw = rotary.bwd(dq[:0], dk[:0], q[:0], k[:0], pos[:0], inv, q_weight=w, k_weight=w, eps=1e-6,
                                weight_grads=True)
    assert not bool(gqw.any()) and not bool(gkw.any())
    # a gradient that is one number expanded (stride 0 everywhere)
    one = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(q.shape)
    got = rotary.bwd(one, one[:, :2], q, k, pos, inv, factor=factor)[0]
    assert torch.equal(got, rotary.bwd(one.contiguous(), dk, q, k, pos, inv, factor=factor)[0])


@pytest.mark.gpu
def test_batched_positions_other_stream_and_graph(cuda_lib):
    from spilltune_b200 import rotary
    q, k, pos, inv, factor, *_ = _case(24, 4, 2, 64, 64, False, False, 2, 8)
    want = rotary.fwd(q, k, pos, inv, factor=factor)
    q4, k4 = q.view(3, 8, 4, 64), k.view(3, 8, 2, 64)
    got = rotary.fwd(q4, k4, pos.view(3, 8), inv, factor=factor)
    assert torch.equal(got[0].view_as(want[0]), want[0]) and torch.equal(got[1].view_as(want[1]), want[1])
    shared = rotary.fwd(q4, k4, pos[:8], inv)[0]
    assert torch.equal(shared[2], rotary.fwd(q[16:], k[16:], pos[:8], inv)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rotary.fwd(q, k, pos, inv, factor=factor)
    side.synchronize()
    assert torch.equal(other[0], want[0])
    qs = q.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rotary.fwd(qs, k, pos, inv, factor=factor)
    qs.copy_(q.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured[0], rotary.fwd(q.flip(0), k, pos, inv, factor=factor)[0])


def test_frequencies():
    from spilltune_b200 import rotary
    inv, factor = rotary.frequencies(8, 10000.0)
    assert factor == 1.0 and torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001]))
    assert torch.equal(rotary.frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})[0], inv / 4)
    # llama3: kept over 4 turns in 8192, divided by 8 under one, blended between
    opt = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_length": 8192}
    plain = rotary.frequencies(128, 500000.0)[0].double()
    got, factor = rotary.frequencies(128, 500000.0, opt)
    turns = 8192 * plain / (2 * math.pi)
    ratio = got.double() / plain
    assert factor == 1.0
    assert torch.allclose(ratio[turns > 4.01], torch.ones(()).double(), atol=1e-6)
    assert torch.allclose(ratio[turns < 0.99], torch.tensor(0.125).double(), atol=1e-6)
    mid = (turns < 3.99) & (turns > 1.01)
    keep = (turns[mid] - 1) / 3
    assert bool(mid.any()) and torch.allclose(ratio[mid], keep + (1 - keep) / 8, atol=1e-5)
    opt = {"type": "yarn", "factor": 40.0, "original_length": 4096}
    got, factor = rotary.frequencies(64, 10000.0, opt)
    plain = rotary.frequencies(64, 10000.0)[0].double()
    turns = 4096 * plain / (2 * math.pi)
    ratio = got.double() / plain
    assert factor == pytest.approx(0.1 * math.log(40.0) + 1.0)
    assert torch.allclose(ratio[turns > 50], torch.ones(()).double(), atol=1e-6)
    assert torch.allclose(ratio[turns < 0.7], torch.tensor(1 / 40.0).double(), atol=1e-6)
    assert bool((ratio[1:] <= ratio[:-1] + 1e-6).all())
    assert rotary.frequencies(64, 10000.0, {**opt, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("dim,theta,scaling,match", [
    (7, 10000.0, None, "even"), (0, 10000.0, None, "even"), (8, 0.0, None, "theta"),
    (8, 1e4, {"type": "other"}, "unsupported_capability"), (8, 1e4, {"type": "linear"}, "missing"),
    (8, 1e4, {"type": "linear", "factor": 2.0, "beta_fast": 1}, "unknown"), (8, 1e4, {"type": "linear", "factor": 0.5}, ">= 1"),
    (8, 1e4, {"type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0,
              "original_length": 8192}, "high_freq_factor"),
    (8, 1e4, {"type": "yarn", "factor": 8.0, "original_length": 0}, "original_length"),
    (8, 1e4, {"type": "yarn", "factor": 8.0, "original_length": 64, "beta_fast": 1.0, "beta_slow": 2.0}, "beta_fast")])
def test_frequency_refusals(dim, theta, scaling, match):
    from spilltune_b200 import rotary
    with pytest.raises(ValueError, match=match):
        rotary.frequencies(dim, theta, scaling)


def test_no_cpu_fallback():
    from spilltune_b200 import rotary
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        rotary.rotate(q, q, torch.arange(2), torch.ones(32))


def test_c_entry_refusals():
    """Bad arguments are refused before any launch (no GPU needed)."""
    from spilltune_b200 import _lib, build
    build.build()
    p = 4096  # never read: each call is refused first

    def fwd(T=1, Hq=1, Hk=1, D=64, pos=p, pb=8, inv=p, rot=64, qw=None, kw=None, wb=0, eps=0.0, q=p, out=p):
        return _lib.load().fl_rotary_fwd(q, 64, 64, Hq, p, 64, 64, Hk, T, D, pos, pb, inv, rot, 0, 1.0, qw, kw, wb,
                                         eps, out, p, None)

    for bad in (dict(T=-1), dict(Hq=0), dict(Hk=-1), dict(D=1), dict(D=258), dict(rot=3), dict(rot=66), dict(rot=0),
                dict(pb=2), dict(pos=None), dict(inv=None), dict(wb=3), dict(wb=2), dict(wb=2, qw=p),
                dict(wb=2, qw=p, kw=p, eps=-1.0), dict(wb=2, qw=p, kw=p, eps=float("nan")), dict(q=None),
                dict(out=None)):
        assert fwd(**bad) == _lib.FL_ERR_ARG, bad
    assert fwd(T=0) == _lib.FL_OK

    def bwd(wb=0, dqw=None, ws=None, n=0, dq=p, q=p):
        return _lib.load().fl_rotary_bwd(dq, 64, 64, p, 64, 64, q, 64, 64, 1, p, 64, 64, 1, 1, 64, p, 8, p, 64, 0, 1.0,
                                         p if wb else None, p if wb else None, wb, 0.0, p, p, dqw, None, ws, n, None)

    for bad in (dict(dqw=p), dict(wb=2, dqw=p), dict(wb=2, dqw=p, ws=p, n=16), dict(wb=2, dqw=p, ws=p + 2, n=1 << 20),
                dict(dq=None), dict(wb=2, q=None)):
        assert bwd(**bad) == _lib.FL_ERR_ARG, bad


@pytest.mark.gpu
def test_refusals(cuda_lib):
    from spilltune_b200 import rotary
    q, k, pos, inv, factor, qw, kw, dq, dk = _case(6, 4, 2, 64, 64, False, True, 2, 9)
    bad = [(lambda: rotary.fwd(q.float(), k, pos, inv), "bf16"),
           (lambda: rotary.fwd(q, k[:5], pos, inv), "agree"),
           (lambda: rotary.fwd(q, k[..., :32], pos, inv), "agree"),
           (lambda: rotary.fwd(q, k, pos.float(), inv), "int32 or int64"),
           (lambda: rotary.fwd(q, k, pos[:5], inv), "do not fit"),
           (lambda: rotary.fwd(q, k, pos, inv.double()), "inv_freq"),
           (lambda: rotary.fwd(q, k, pos, torch.ones(33, device="cuda")), "do not fit a head"),
           (lambda: rotary.fwd(q, k, pos, inv, q_weight=qw, eps=1e-6), "both norm weights"),
           (lambda: rotary.fwd(q, k, pos, inv, q_weight=qw, k_weight=kw), "eps"),
           (lambda: rotary.fwd(q, k, pos, inv, q_weight=qw, k_weight=kw[:32], eps=1e-6), "norm weights"),
           (lambda: rotary.fwd(q, k, pos, inv, q_weight=qw, k_weight=kw.float(), eps=1e-6), "of one type"),
           (lambda: rotary.norm_rotate(q, k, None, None, pos, inv, eps=1e-6), "needs the norm weights"),
           (lambda: rotary.bwd(dq, None, q, k, pos, inv), "dk goes with k"),
           (lambda: rotary.bwd(dq[:5], dk, q, k, pos, inv), "shapes"),
           (lambda: rotary.bwd(dq, dk, q, k, pos, inv, weight_grads=True), "need the norm weights"),
           (lambda: rotary.fwd(torch.zeros(2, 1, 258, dtype=torch.bfloat16, device="cuda"), None, pos[:2], inv),
            "unsupported_capability")]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()
