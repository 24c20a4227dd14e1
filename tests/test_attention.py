"""Attention over row ranges (spilltune_b200.attention) against the formulas in 64 bits.

Tolerances, element by element, from where the kernels round (h = half a bf16
step, 2^-8 of the value): the results once; p and ds once each, as the operands
of the second products; delta is formed from the rounded output.  FP32 error of
a score is under e = 2^-18 max(1, sum |q k| scale) (D products, the cap and the
distance), and moves p by a factor 1 + e.  So
  |out - o|  <= h |o| + (h + 2 e) sum p |v|
  |dv|:         h |dv| + (h + 2 e) sum p |do|
  |ds|:         (h + 4 e) |ds| + p (sum_d |do| (2 h + 2 e) sum p |v| + 2^-18 sum |do v|)
                (under a cap 2^-11 |ds| more: its factor 1 - tanh^2 waits in fp16, half a step of that)
  |dq|:         h |dq| + scale sum |ds error| |k|, dk alike."""
import pytest
import torch

HALF = torch.finfo(torch.bfloat16).eps / 2


def _ranges(kind, B, Sq, Sk, seed):
    g = torch.Generator().manual_seed(seed)
    at = torch.arange(Sq).expand(B, Sq) + (Sk - Sq)
    begin, end = torch.zeros(B, Sq, dtype=torch.int64), at + 1
    if kind == "all":
        end = torch.full_like(at, Sk)
    elif kind == "window":
        begin = (at - 20).clamp_min(0)
    elif kind == "documents":
        cut = torch.rand(B, Sk, generator=g) < 4.0 / max(Sk, 4)
        cut[:, 0] = True
        first = torch.where(cut, torch.arange(Sk).expand(B, Sk), 0).cummax(1).values
        begin = first[:, Sk - Sq:]
    elif kind == "holes":  # any interval at all, a third of the rows empty, some past the ends
        begin = torch.randint(-5, Sk + 5, (B, Sq), generator=g)
        end = begin + torch.randint(-Sk // 2, Sk + 5, (B, Sq), generator=g)
    elif kind == "none":
        end = begin
    elif kind == "prefix":
        end = torch.maximum(end, torch.full_like(end, Sk // 3))
        end[-1, Sq // 2:] = 0
    return begin.to(torch.int32), end.to(torch.int32)


def _oracle(q, k, v, begin, end, scale, cap, slopes, do=None):
    """{name: (value, bound)} in float64."""
    B, Sq, H, D = q.shape
    Sk, K = k.shape[1:3]
    G = H // K
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(G, 1) for t in (k, v))
    raw = q @ k.mT * scale
    th = torch.tanh(raw / cap) if cap else None
    x = cap * th if cap else raw
    if slopes is not None:
        i = torch.arange(Sq, device=q.device)[:, None] + Sk - Sq
        x = x - slopes.double()[:, None, None] * (i - torch.arange(Sk, device=q.device)).abs()
    j = torch.arange(Sk, device=q.device)
    seen = ((j >= begin[..., None]) & (j < end[..., None]))[:, None]
    x = x.masked_fill(~seen, -torch.inf)
    lse = torch.logsumexp(x, -1) if Sk else torch.full(x.shape[:-1], -torch.inf, dtype=x.dtype, device=x.device)
    p = torch.where(seen, torch.exp(x - lse[..., None].masked_fill(lse[..., None] == -torch.inf, 0.0)), 0.0)
    o = p @ v
    e = 2.0 ** -18 * (q.abs() @ k.abs().mT * scale).clamp_min(1.0)
    e = e.amax(-1, keepdim=True) if Sk else torch.zeros_like(lse[..., None])
    reach = p @ v.abs()
    eo = HALF * o.abs() + (HALF + 2 * e) * reach
    t = lambda a: a.transpose(1, 2)  # noqa: E731
    out = {"out": (t(o), t(eo)), "lse": (t(lse), t(2 * e[..., 0] + 2.0 ** -20 * lse.abs().nan_to_num(posinf=0.0)))}
    if do is None:
        return out
    do = do.double().transpose(1, 2)
    dp = do @ v.mT
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    es = p * ((do.abs() * ((2 * HALF + 2 * e) * reach)).sum(-1, keepdim=True) + 2.0 ** -18 * (do.abs() @ v.abs().mT))
    if cap:
        es = es + (2.0 ** -18 + 2.0 ** -11 * (1 - th * th)) * ds.abs()
        ds = ds * (1 - th * th)
    es = es + (HALF + 4 * e) * ds.abs()
    fold = lambda a: a.unflatten(1, (K, G)).sum(2)  # noqa: E731
    dq, dk, dv = scale * ds @ k, fold(scale * ds.mT @ q), fold(p.mT @ do)
    out["dq"] = (t(dq), t(HALF * dq.abs() + scale * es @ k.abs()))
    out["dk"] = (t(dk), t(HALF * dk.abs() + fold(scale * es.mT @ q.abs())))
    out["dv"] = (t(dv), t(HALF * dv.abs() + fold(((HALF + 2 * e) * p).mT @ do.abs())))
    return out


def _within(name, got, want):
    value, bound = want
    got = got.double()
    assert torch.isfinite(got[torch.isfinite(value)]).all(), name
    if name == "lse":
        assert torch.equal(got == -torch.inf, value == -torch.inf)
        got, value = got.masked_fill(value == -torch.inf, 0.0), value.masked_fill(value == -torch.inf, 0.0)
    over = (got - value).abs() - 1.01 * bound - 1e-30
    assert bool((over <= 0).all()), (name, float(over.max()), int((over > 0).sum()))


def _inputs(B, Sq, Sk, H, K, D, seed, qscale=1.5):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q = (qscale * n(B, Sq, H, D)).to(torch.bfloat16).cuda()
    k, v = (n(B, Sk, K, D).to(torch.bfloat16).cuda() for _ in range(2))
    return q, k, v, n(B, Sq, H, D).to(torch.bfloat16).cuda()


def _both(q, k, v, begin, end, do, cap=0.0, slopes=None, scale=None):
    from spilltune_b200 import _lib, attention
    opt = dict(scale=scale, softcap=cap, slopes=slopes)
    out, lse = attention.fwd(q, k, v, begin, end, **opt)
    got = {"out": out, "lse": lse}
    if do is not None:
        got.update(zip(("dq", "dk", "dv"), attention.bwd(do, q, k, v, out, lse, begin, end, **opt)))
    assert _lib.status() == 0
    return got


CASES = [  # B, Sq, Sk, H, K, D, mask, cap, slopes
    (1, 1, 1, 1, 1, 64, "causal", 0.0, False),
    (1, 2, 2, 2, 1, 128, "causal", 0.0, False),
    (2, 128, 128, 4, 2, 64, "causal", 0.0, False),
    (1, 129, 129, 4, 4, 128, "causal", 0.0, False),
    (2, 300, 300, 8, 1, 128, "documents", 0.0, False),
    (1, 517, 517, 6, 2, 80, "documents", 0.0, False),
    (3, 257, 257, 14, 2, 64, "prefix", 0.0, True),
    (1, 400, 400, 16, 2, 96, "window", 50.0, False),
    (2, 200, 200, 4, 2, 128, "window", 30.0, True),
    (2, 333, 333, 8, 2, 128, "holes", 0.0, False),
    (2, 333, 333, 8, 2, 64, "holes", 20.0, True),
    (1, 130, 130, 2, 2, 64, "none", 0.0, False),
    (1, 100, 900, 4, 1, 128, "causal", 0.0, False),
    (1, 700, 90, 4, 2, 64, "all", 0.0, False),
    (1, 33, 70, 64, 1, 32, "causal", 0.0, False),
    (1, 40, 40, 128, 1, 64, "causal", 0.0, False),
    (1, 60, 60, 5, 5, 8, "causal", 0.0, True),
    (4, 1, 1000, 32, 8, 128, "causal", 0.0, False),
    (1, 1, 5000, 7, 1, 64, "window", 0.0, False),
    (2, 5, 2000, 8, 2, 80, "holes", 50.0, True),
    (1, 1300, 1300, 4, 2, 128, "all", 0.0, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,Sk,H,K,D,mask,cap,slopes", CASES)
def test_forward(cuda_lib, B, Sq, Sk, H, K, D, mask, cap, slopes):
    q, k, v, _ = _inputs(B, Sq, Sk, H, K, D, Sq + Sk + D)
    begin, end = (t.cuda() for t in _ranges(mask, B, Sq, Sk, Sq))
    sl = 2.0 ** -(1.0 + torch.arange(H, device="cuda").float() * 7 / H) if slopes else None
    got = _both(q, k, v, begin, end, None, cap, sl)
    want = _oracle(q, k, v, begin, end, D ** -0.5, cap, sl)
    for name in got:
        _within(name, got[name], want[name])


@pytest.mark.gpu
@pytest.mark.parametrize("B,Sq,Sk,H,K,D,mask,cap,slopes", CASES)
def test_backward(cuda_lib, B, Sq, Sk, H, K, D, mask, cap, slopes):
    q, k, v, do = _inputs(B, Sq, Sk, H, K, D, Sq + Sk + D)
    begin, end = (t.cuda() for t in _ranges(mask, B, Sq, Sk, Sq))
    sl = 2.0 ** -(1.0 + torch.arange(H, device="cuda").float() * 7 / H) if slopes else None
    got = _both(q, k, v, begin, end, do, cap, sl)
    want = _oracle(q, k, v, begin, end, D ** -0.5, cap, sl, do)
    for name in got:
        _within(name, got[name], want[name])
