"""spilltune_b200.attention where delta, the cap's derivative or the operands' rounding decides its results,
element by element against the formulas in 64 bits.

With h = half a bf16 step (2^-8 of the value), er = 2^-18 max(1, sum |q k| scale) the FP32 error of a scaled
product, e = f er + 2^-21 cap + 2^-22 |x| (the largest of a row) that of a score, and ds = p f (dp - delta),
f = 1 - tanh^2 (1 without a cap), the kernels round here:
  p is off by 4 e of itself (its score and its log sum); delta is summed in FP32 from p dp, not taken from the
  rounded output: off by ed = (4 e + 2^-16) sum p sum |do v|; dp by 2^-17 sum |do v| (D products each);
  f by ef = 2^-11 (16 bits) + 2^-20 + 4 er / cap (it changes by 2 f for a change of its argument by 1);
  ds is an operand in bf16, rounded by w = h, or in two parts (few rows and keys) by w = h^2:
  es = f p (ed + 2^-17 sum |do v|) + (w + 4 e + ef) |ds|;  p of out and dv likewise, by (w + 4 e) p.
  dk's terms are off by es |q|; FP32 sums by 2^-14 of their terms; a result is rounded once, by h.
  dq is summed with d0 = do . out in delta's place and corrected by (d0 - delta) times a sum of bf16(p f) k:
  (w + h) p f |d0 - delta| beside es, with d0 from the output that the forward gave.
A backward that took d0 for delta would be off by scale |d0 - delta| |sum p f k|, which is more than these
bounds in the first test's cases (checked beside them)."""
import pytest
import torch

HALF = torch.finfo(torch.bfloat16).eps / 2


def _gradients(q, k, v, begin, end, do, out, cap=0.0, slopes=None, fine=False, half_f=False, coarse=False):
    """{name: (value, bound, value with d0 for delta)} in float64.  fine: operands in two parts; half_f: f in 16
    bits, unscaled; coarse: the values with p and ds rounded to bf16."""
    B, Sq, H, D = q.shape
    Sk, K = k.shape[1:3]
    G, scale = H // K, D ** -0.5
    q, k, v, do, out = (t.double().transpose(1, 2) for t in (q, k, v, do, out))
    k, v = (t.repeat_interleave(G, 1) for t in (k, v))
    raw = q @ k.mT * scale
    x, f = raw, torch.ones_like(raw)
    if cap:
        x = cap * torch.tanh(raw / cap)
        f = torch.cosh(raw / cap) ** -2
        if half_f:
            f = f.half().double()
    j = torch.arange(Sk, device=q.device)
    if slopes is not None:
        i = torch.arange(Sq, device=q.device)[:, None] + Sk - Sq
        x = x - slopes.double()[:, None, None] * (i - j).abs()
    w = HALF * HALF if fine else HALF
    part = (lambda a: a.to(torch.bfloat16).double()) if coarse else (lambda a: a)
    seen = ((j >= begin[..., None]) & (j < end[..., None]))[:, None]
    eraw = 2.0 ** -18 * (q.abs() @ k.abs().mT * scale).clamp_min(1.0)
    e = f * eraw + 2.0 ** -21 * cap + 2.0 ** -22 * x.abs()
    e = e.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    p = torch.softmax(x.masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
    dp, reach = do @ v.mT, do.abs() @ v.abs().mT
    delta = (p * dp).sum(-1, keepdim=True)
    off = (do * out).sum(-1, keepdim=True) - delta
    size = (do.abs() * out.abs()).sum(-1, keepdim=True)
    ds = p * f * (dp - delta)
    ed = (4 * e + 2.0 ** -16) * (p * reach).sum(-1, keepdim=True)
    ef = 2.0 ** -11 + 2.0 ** -20 + 4 * eraw / cap if cap else 0.0
    es = f * p * (ed + 2.0 ** -17 * reach) + (w + 4 * e + ef) * ds.abs()
    eq = es + p * f * ((w + HALF) * off.abs() + 2.0 ** -16 * size)
    fold = lambda a: a.unflatten(1, (K, G)).sum(2)  # noqa: E731
    sums = 2.0 ** -14 * (ds.abs() + p * f * off.abs())
    dq, dk = scale * part(ds) @ k, scale * fold(part(ds).mT @ q)
    o, dv = part(p) @ v, fold(part(p).mT @ do)
    bo = HALF * o.abs() + 1.01 * ((w + 4 * e + 2.0 ** -14) * p) @ v.abs()
    bv = HALF * dv.abs() + 1.01 * fold(((w + 4 * e + 2.0 ** -14) * p).mT @ do.abs())
    bq = HALF * dq.abs() + 1.01 * scale * (eq + sums) @ k.abs()
    bk = HALF * dk.abs() + 1.01 * scale * fold((es + sums).mT @ q.abs())
    wrong = p * f * off
    t = lambda a: a.transpose(1, 2)  # noqa: E731
    return {"out": (t(o), t(bo), None), "dv": (t(dv), t(bv), None), "dq": (t(dq), t(bq), t(dq - scale * wrong @ k)),
            "dk": (t(dk), t(bk), t(dk - scale * fold(wrong.mT @ q)))}


def _short_rows(B, S, width, kind):
    """Documents of `width` tokens seen whole, or the last `width` keys."""
    at = torch.arange(S).expand(B, S)
    if kind == "documents":
        begin, end = at // width * width, (at // width + 1) * width
    else:
        begin, end = at + 1 - width, at + 1
    return begin.clamp_min(0).to(torch.int32), end.clamp_max(S).to(torch.int32)


def _run(q, k, v, begin, end, do, **opt):
    from spilltune_b200 import _lib, attention
    out, lse = attention.fwd(q, k, v, begin, end, **opt)
    dq, dk, dv = attention.bwd(do, q, k, v, out, lse, begin, end, **opt)
    assert _lib.status() == 0
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _check(got, want):
    for n, (value, bound, _) in want.items():
        over = (got[n].double() - value).abs() - bound
        assert bool((over <= 0).all()), (n, float(over.max()), int((over > 0).sum()))


def _fine(Sk):
    """The cases up to 512 keys have at most 2048 rows (tokens x heads): their operands come in two parts."""
    return Sk <= 512


def _common_values(B, S, H, K, D, seed):
    """Values with a large part in common: the output is large beside what sets its keys apart."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    v = 8.0 + 0.5 * n(B, S, K, D)
    return [x.to(torch.bfloat16) for x in (0.5 * n(B, S, H, D), n(B, S, K, D), v, n(B, S, H, D))]


SHORT = [  # B, S, H, K, D, keys to a row, kind, cap, slopes
    (1, 5, 2, 1, 64, 5, "documents", 0.0, False),
    (3, 5, 4, 2, 128, 5, "documents", 0.0, False),
    (2, 130, 4, 2, 64, 2, "documents", 0.0, False),
    (2, 514, 4, 2, 64, 2, "documents", 0.0, False),
    (1, 600, 8, 2, 128, 3, "window", 0.0, False),
    (1, 257, 6, 2, 80, 4, "documents", 0.0, True),
    (1, 524, 3, 1, 80, 4, "documents", 0.0, True),
    (2, 515, 3, 3, 64, 5, "window", 30.0, False),
    (1, 140, 4, 1, 128, 5, "documents", 30.0, True),
    (1, 520, 4, 1, 128, 5, "documents", 30.0, True),
    (1, 600, 7, 7, 96, 20, "window", 0.0, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,K,D,width,kind,cap,slopes", SHORT)
def test_delta_is_not_taken_from_the_rounded_output(cuda_lib, B, S, H, K, D, width, kind, cap, slopes):
    q, k, v, do = (x.cuda() for x in _common_values(B, S, H, K, D, S + D))
    begin, end = (x.cuda() for x in _short_rows(B, S, width, kind))
    sl = 2.0 ** -(1.0 + torch.arange(H, device="cuda").float() * 7 / H) if slopes else None
    got = _run(q, k, v, begin, end, do, softcap=cap, slopes=sl)
    want = _gradients(q, k, v, begin, end, do, got["out"], cap, sl, _fine(S))
    _check(got, want)
    for n in ("dq", "dk"):
        value, bound, wrong = want[n]
        assert bool(((wrong - value).abs() > bound).any()), n


def _saturated(B, S, H, K, D, cap, times, seed):
    """Scores of about `times` caps, mostly within a tenth."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    side = (abs(times) * cap * D ** -0.5) ** 0.5   # q . k D^-1/2 = side^2 D^1/2
    q = side * (1 + 0.1 * n(B, S, H, D)) * (-1 if times < 0 else 1)
    k = side * (1 + 0.05 * n(B, S, K, 1) + 0.1 * n(B, S, K, D))
    return [x.to(torch.bfloat16) for x in (q, k, n(B, S, K, D), n(B, S, H, D))]


SATURATED = [  # B, S, H, K, D, cap, scores in caps, slopes
    (1, 70, 4, 2, 64, 20.0, 6.0, False),
    (1, 70, 4, 2, 128, 30.0, 8.0, False),
    (1, 530, 4, 2, 128, 30.0, 8.0, False),
    (2, 150, 6, 2, 64, 20.0, -7.0, False),
    (1, 140, 2, 2, 80, 50.0, -8.0, False),
    (1, 540, 2, 2, 80, 50.0, -8.0, False),
    (1, 90, 8, 1, 64, 10.0, 7.0, True),
    (1, 600, 4, 4, 64, 20.0, 9.0, False),
    (1, 515, 2, 2, 64, 20.0, 8.0, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,K,D,cap,times,slopes", SATURATED)
def test_gradients_of_scores_far_over_their_cap(cuda_lib, B, S, H, K, D, cap, times, slopes):
    """f = 1 - tanh^2 is 2e-5 at six caps, 6e-8 at nine, to either side: its relative error is what counts.  Held
    as it is in 16 bits it would be off by more than these bounds from 8 caps on."""
    q, k, v, do = (x.cuda() for x in _saturated(B, S, H, K, D, cap, times, S + D))
    begin, end = (x.cuda() for x in _short_rows(B, S, 4, "window"))
    sl = 2.0 ** -(4.0 + torch.arange(H, device="cuda").float() * 4 / H) if slopes else None
    got = _run(q, k, v, begin, end, do, softcap=cap, slopes=sl)
    want = _gradients(q, k, v, begin, end, do, got["out"], cap, sl, _fine(S))
    _check(got, want)
    coarse = _gradients(q, k, v, begin, end, do, got["out"], cap, sl, half_f=True)
    for n in ("dq", "dk"):
        assert bool(((coarse[n][0] - want[n][0]).abs() > want[n][1]).any()) or abs(times) < 8, n


FEW = [  # B, S, H, K, D, keys to a row, kind, cap, slopes
    (1, 4, 2, 1, 128, 4, "documents", 0.0, False),
    (1, 3, 8, 8, 64, 3, "documents", 0.0, False),
    (2, 128, 4, 2, 64, 128, "window", 0.0, False),
    (3, 5, 4, 2, 128, 5, "window", 0.0, True),
    (1, 130, 7, 1, 80, 40, "window", 0.0, False),
    (1, 512, 2, 1, 64, 200, "window", 50.0, True),
    (1, 250, 8, 2, 128, 250, "documents", 20.0, False),
    (4, 4, 56, 8, 64, 4, "documents", 0.0, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,K,D,width,kind,cap,slopes", FEW)
def test_few_results_are_rounded_once(cuda_lib, B, S, H, K, D, width, kind, cap, slopes):
    """Up to 2048 rows over up to 512 keys, p and ds come in two parts: with a single one the results would be
    off by more than these bounds."""
    g = torch.Generator().manual_seed(S + H)
    n = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    q, k, v, do = n(B, S, H, D), n(B, S, K, D), n(B, S, K, D), n(B, S, H, D)
    begin, end = (x.cuda() for x in _short_rows(B, S, width, kind))
    sl = 2.0 ** -(1.0 + torch.arange(H, device="cuda").float() * 7 / H) if slopes else None
    got = _run(q, k, v, begin, end, do, softcap=cap, slopes=sl)
    want = _gradients(q, k, v, begin, end, do, got["out"], cap, sl, True)
    _check(got, want)
    coarse = _gradients(q, k, v, begin, end, do, got["out"], cap, sl, True, coarse=True)
    for name in want:
        # dv, dk: a sum over all queries; where it has hundreds of terms their roundings average out
        assert bool(((coarse[name][0] - want[name][0]).abs() > want[name][1]).any()) or S > 100, name
