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
    (1, 45, 300, 64, 1, 64, "causal", 0.0, True),
    (1, 150, 150, 256, 2, 64, "documents", 30.0, True),
    (1, 500, 500, 16, 1, 128, "holes", 0.0, True),
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


@pytest.mark.gpu
def test_strided_views_are_read_in_place(cuda_lib):
    """Views of one projection's output, heads before tokens, and rows that have to be copied."""
    B, S, H, K, D = 2, 140, 4, 2, 64
    q, k, v, do = _inputs(B, S, S, H, K, D, 3)
    begin, end = (t.cuda() for t in _ranges("causal", B, S, S, 0))
    want = _both(q, k, v, begin, end, do)
    x = torch.cat([t.flatten(2) for t in (q, k, v)], -1)
    a, b, c = x.split([H * D, K * D, K * D], -1)
    views = (a.unflatten(-1, (H, D)), b.unflatten(-1, (K, D)), c.unflatten(-1, (K, D)))
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:D + 1] for t in (q, k, v)]
    for q2, k2, v2 in (views, heads_first, odd):
        got = _both(q2, k2, v2, begin, end, do.transpose(1, 2).contiguous().transpose(1, 2))
        assert all(torch.equal(got[n], want[n]) for n in want)
    one = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(do.shape)
    assert all(torch.equal(x, y) for x, y in zip(_both(q, k, v, begin, end, one).values(),
                                                 _both(q, k, v, begin, end, one.contiguous()).values()))
    cols = torch.stack((begin, end), -1)
    got = _both(q, k, v, cols[..., 0], cols[..., 1], do)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.gpu
def test_values_out_of_sight(cuda_lib):
    """Keys that no row sees: infinities and NaN in their k and v leave forward and backward alone, as far as
    they lie in 128-key tiles that no row of the 128-row tile sees.  Scores of hidden keys inside a seen tile may
    be anything (NaN keys with finite values)."""
    B, S, H, K, D = 1, 512, 2, 2, 64
    q, k, v, do = _inputs(B, S, S, H, K, D, 4)
    begin = torch.full((B, S), 128, dtype=torch.int32, device="cuda")
    end = torch.full((B, S), 300, dtype=torch.int32, device="cuda")
    want = _both(q, k, v, begin, end, do)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, :128], bad_k[:, 384:] = float("nan"), float("inf")
    bad_v[:, :128], bad_v[:, 384:] = float("inf"), float("nan")
    got = _both(q, bad_k, bad_v, begin, end, do)
    assert all(torch.equal(got[n], want[n]) for n in want)
    from spilltune_b200 import attention
    bad_k[:, 300:384] = float("nan")
    out, lse = attention.fwd(q, bad_k, bad_v, begin, end)
    assert torch.equal(out, want["out"]) and torch.equal(lse, want["lse"])


@pytest.mark.gpu
@pytest.mark.parametrize("H,K,D,cap,slopes", [(4, 2, 64, 0.0, False), (8, 2, 128, 0.0, False), (6, 2, 128, 0.0, True),
                                              (8, 1, 80, 30.0, False), (4, 4, 64, 20.0, True)])
def test_padding_that_is_not_finite(cuda_lib, H, K, D, cap, slopes):
    """Keys, values, queries and gradients of padding tokens may be anything, also
    where the padding begins inside a tile: the other results are the same bits."""
    from spilltune_b200 import attention
    B, S = 3, 200
    q, k, v, do = _inputs(B, S, S, H, K, D, 6)
    sl = 2.0 ** -(1.0 + torch.arange(H, device="cuda").float() * 7 / H) if slopes else None
    begin, end = (x.cuda() for x in attention.row_ranges(B, S, lengths=torch.tensor([130, 65, 0])))
    want = _both(q, k, v, begin, end, do, cap, sl)
    bad = [x.clone() for x in (q, k, v, do)]
    for i, x in enumerate(bad):
        for b, live in enumerate((130, 65, 0)):
            x[b, live:] = (float("nan"), float("inf"), float("-inf"))[(b + i) % 3]
    got = _both(*bad[:3], begin, end, bad[3], cap, sl)
    for n in want:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 4])
def test_cache_that_is_not_filled(cuda_lib, Sq):
    """A few tokens over a long cache of which the first and the last rows hold anything."""
    from spilltune_b200 import attention
    B, Sk, H, K, D = 2, 4000, 8, 2, 128
    q, k, v, _ = _inputs(B, Sq, Sk, H, K, D, 7)
    begin = torch.tensor([[5], [70]], dtype=torch.int32, device="cuda").expand(B, Sq)
    end = torch.tensor([[3001], [90]], dtype=torch.int32, device="cuda") + \
        torch.arange(Sq, dtype=torch.int32, device="cuda")
    want = attention.fwd(q, k, v, begin, end)
    for b in range(B):
        for x in (k, v):
            x[b, :int(begin[b, 0])] = float("nan")
            x[b, int(end[b, -1]):] = float("inf")
    got = attention.fwd(q, k, v, begin, end)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_empty_rows_and_rows_behind_the_last(cuda_lib):
    """Rows that see nothing: zero output and gradient, log sum -inf; empty inputs."""
    from spilltune_b200 import attention
    B, S, H, K, D = 2, 200, 4, 2, 64
    q, k, v, do = _inputs(B, S, S, H, K, D, 5)
    begin, end = attention.row_ranges(B, S, lengths=torch.tensor([130, 0]), device="cuda")
    got = _both(q, k, v, begin.cuda(), end.cuda(), do)
    for b, live in ((0, 130), (1, 0)):
        assert not bool(got["out"][b, live:].any()) and bool((got["lse"][b, live:] == -torch.inf).all())
        for n in ("dq", "dk", "dv"):
            assert not bool(got[n][b, live:].any()), n
    short = _both(q[:1, :130], k[:1, :130], v[:1, :130], begin[:1, :130].cuda(), end[:1, :130].cuda(), do[:1, :130])
    assert torch.equal(short["out"], got["out"][:1, :130])
    none = torch.zeros(B, 0, dtype=torch.int32, device="cuda")
    out, lse = attention.fwd(q[:, :0], k, v, none, none)
    assert out.shape == (B, 0, H, D) and lse.shape == (B, 0, H)
    grads = attention.bwd(do[:, :0], q[:, :0], k, v, out, lse, none, none)
    assert grads[0].shape == (B, 0, H, D) and not bool(grads[1].any()) and not bool(grads[2].any())
    zero = torch.zeros(B, S, dtype=torch.int32, device="cuda")
    out, lse = attention.fwd(q, k[:, :0], v[:, :0], zero, zero + 5)
    assert not bool(out.any()) and bool((lse == -torch.inf).all())
    assert not bool(attention.bwd(do, q, k[:, :0], v[:, :0], out, lse, zero, zero)[0].any())


@pytest.mark.gpu
def test_equal_bits_other_stream_and_captured_passes(cuda_lib):
    """Twice the same bits; on a side stream; forward and backward in one graph, replayed on new inputs, with a
    second graph of the same shapes replayed between."""
    from spilltune_b200 import attention
    B, S, H, K, D = 2, 260, 14, 2, 64
    q, k, v, do = _inputs(B, S, S, H, K, D, 6)
    begin, end = (t.cuda() for t in _ranges("causal", B, S, S, 0))
    want = _both(q, k, v, begin, end, do)
    again = _both(q, k, v, begin, end, do)
    assert all(torch.equal(again[n], want[n]) for n in want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _both(q, k, v, begin, end, do)
    side.synchronize()
    assert all(torch.equal(other[n], want[n]) for n in want)

    def captured(q):
        out, lse = attention.fwd(q, k, v, begin, end)
        return (out, *attention.bwd(do, q, k, v, out, lse, begin, end))

    static = [q.clone(), q.clone()]
    graphs, results = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, x in zip(graphs, static):
        with torch.cuda.graph(graph):
            results.append(captured(x))
    static[0].copy_(q.flip(1))
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    flipped = captured(q.flip(1).contiguous())
    assert all(torch.equal(x, y) for x, y in zip(results[0], flipped))
    assert all(torch.equal(x, want[n]) for x, n in zip(results[1], ("out", "dq", "dk", "dv")))


@pytest.mark.gpu
def test_many_tiles(cuda_lib):
    """Enough tiles that every CTA takes several and waits on its pipelines in every order: no wait expires, and
    sampled heads agree with the formulas."""
    B, S, H, K, D = 2, 2048, 32, 8, 128
    q, k, v, do = _inputs(B, S, S, H, K, D, 12)
    for kind in ("causal", "documents"):
        begin, end = (t.cuda() for t in _ranges(kind, B, S, S, 1))
        got = _both(q, k, v, begin, end, do)
        for _ in range(3):
            again = _both(q, k, v, begin, end, do)
            assert all(torch.equal(again[n], got[n]) for n in got)
        for b, h in ((0, 0), (1, 7)):
            part = lambda t, n: t[b:b + 1, :, h * n:(h + 1) * n]  # noqa: E731
            want = _oracle(part(q, 4), part(k, 1), part(v, 1), begin[b:b + 1], end[b:b + 1], D ** -0.5, 0.0, None,
                           part(do, 4))
            for n in got:
                _within(n, part(got[n], 1 if n in ("dk", "dv") else 4), want[n])


@pytest.mark.gpu
def test_two_calls_at_once(cuda_lib):
    """Two streams, each with its own call under way (a split forward and a split backward among them)."""
    cases = []
    for seed, (B, Sq, Sk, H, K) in enumerate(((1, 3, 3000, 8, 2), (1, 600, 600, 14, 2))):
        q, k, v, do = _inputs(B, Sq, Sk, H, K, 64, seed)
        begin, end = (t.cuda() for t in _ranges("causal", B, Sq, Sk, 0))
        cases.append(((q, k, v, begin, end, do), _both(q, k, v, begin, end, do)))
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    from spilltune_b200 import attention
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s, ((q, k, v, begin, end, do), _), g in zip(streams, cases, got):
            with torch.cuda.stream(s):
                out, lse = attention.fwd(q, k, v, begin, end)
                g.append((out, lse, *attention.bwd(do, q, k, v, out, lse, begin, end)))
    torch.cuda.synchronize()
    for (_, want), g in zip(cases, got):
        for r in g:
            assert all(torch.equal(x, want[n]) for x, n in zip(r, ("out", "lse", "dq", "dk", "dv")))


@pytest.mark.gpu
def test_autograd_and_differences(cuda_lib):
    """attend()'s gradients: bwd()'s bits, and a directional derivative against a central difference of the
    64-bit formula (tied to the kernel by test_backward; every element is off by at most its bound there)."""
    from spilltune_b200 import attention
    B, S, H, K, D = 1, 90, 4, 2, 64
    q, k, v, do = _inputs(B, S, S, H, K, D, 8)
    begin, end = (t.cuda() for t in _ranges("documents", B, S, S, 2))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = attention.attend(*leaves, begin, end, softcap=30.0)
    grads = torch.autograd.grad(out, leaves, do)
    want = _both(q, k, v, begin, end, do, cap=30.0)
    assert all(torch.equal(g, want[n]) for g, n in zip(grads, ("dq", "dk", "dv")))
    bounds = _oracle(q, k, v, begin, end, D ** -0.5, 30.0, None, do)
    g = torch.Generator().manual_seed(9)
    step = [torch.randn(t.shape, generator=g, dtype=torch.float64).cuda() for t in leaves]

    def at(e):
        moved = [t.detach().double() + e * s for t, s in zip(leaves, step)]
        return float((_oracle(*moved, begin, end, D ** -0.5, 30.0, None)["out"][0] * do.double()).sum())

    expect = (at(1e-4) - at(-1e-4)) / 2e-4
    got = float(sum((x.double() * s).sum() for x, s in zip(grads, step)))
    room = float(sum((bounds[n][1] * s.abs()).sum() for n, s in zip(("dq", "dk", "dv"), step)))
    assert abs(got - expect) <= room + 1e-5 * abs(expect)


@pytest.mark.gpu
def test_long_rows_and_large_scores(cuda_lib):
    """Scores that grow along the row (the running maximum moves with every tile) and peak above 2^8 of the
    first tile's."""
    B, S, H, K, D = 1, 1500, 2, 1, 128
    q, k, v, do = _inputs(B, S, S, H, K, D, 10, qscale=1.0)
    k = (k.float() * torch.linspace(0.1, 12.0, S, device="cuda")[None, :, None, None]).to(torch.bfloat16)
    begin, end = (t.cuda() for t in _ranges("all", B, S, S, 0))
    got = _both(q, k, v, begin, end, do)
    want = _oracle(q, k, v, begin, end, D ** -0.5, 0.0, None, do)
    for n in got:
        _within(n, got[n], want[n])


def test_row_ranges():
    from spilltune_b200.attention import row_ranges
    begin, end = row_ranges(1, 4)
    assert begin.tolist() == [[0, 0, 0, 0]] and end.tolist() == [[1, 2, 3, 4]]
    assert row_ranges(1, 3, causal=False)[1].tolist() == [[3, 3, 3]]
    docs = torch.tensor([[5, 5, 7, 7, 7, 5]])
    begin, end = row_ranges(1, 6, documents=docs)
    assert begin.tolist() == [[0, 0, 2, 2, 2, 5]] and end.tolist() == [[1, 2, 3, 4, 5, 6]]
    begin, end = row_ranges(1, 6, documents=docs, causal=False)
    assert end.tolist() == [[2, 2, 5, 5, 5, 6]]
    begin, end = row_ranges(1, 6, documents=docs, prefix=torch.tensor([4]))
    assert begin.tolist() == [[0, 0, 2, 2, 2, 5]] and end.tolist() == [[2, 2, 4, 4, 5, 6]]
    begin, end = row_ranges(2, 5, window=2, lengths=torch.tensor([3, 5]))
    assert begin.tolist() == [[0, 0, 1, 2, 3]] * 2 and end.tolist() == [[1, 2, 3, 0, 0], [1, 2, 3, 4, 5]]
    assert all(x.dtype == torch.int32 and x.shape == (2, 0) for x in row_ranges(2, 0, documents=torch.zeros(2, 0)))
    for bad in (dict(window=0), dict(window=3, causal=False), dict(documents=docs[:, :3]),
                dict(prefix=torch.zeros(2)), dict(lengths=torch.zeros(2, 1))):
        with pytest.raises(ValueError):
            row_ranges(1, 6, **bad)
    with pytest.raises(ValueError):
        row_ranges(1, -1)


def test_no_cpu_fallback():
    from spilltune_b200 import attention
    x = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    r = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        attention.attend(x, x, x, r, r)


def test_c_entry_refusals():
    """Bad arguments are refused before any launch (no GPU needed)."""
    import ctypes

    from spilltune_b200 import _lib, build
    build.build()
    lib = _lib.load()
    p = 4096  # never read: each call is refused first
    good = [64 * 4 * 2, 64 * 2, 64] * 4

    def fwd(B=1, Sq=4, Sk=4, Hq=2, Hkv=2, D=64, scale=1.0, cap=0.0, strides=good, q=p, begin=p, out=p, ws=None, n=0):
        s = (ctypes.c_int64 * 12)(*strides) if strides else None
        return lib.fl_attn_fwd(q, p, p, s, B, Sq, Sk, Hq, Hkv, D, begin, p, scale, cap, None, out, p, ws, n, None)

    def bwd(B=1, Sq=4, Sk=4, Hq=2, Hkv=2, D=64, scale=1.0, cap=0.0, strides=good, q=p, begin=p, out=p, ws=p, n=1 << 20):
        s = (ctypes.c_int64 * 12)(*strides) if strides else None
        return lib.fl_attn_bwd(p, q, p, p, s, out, p, B, Sq, Sk, Hq, Hkv, D, begin, p, scale, cap, None, p, p, p, ws, n,
                               None)

    bad = [dict(B=-1), dict(Sq=-1), dict(Sk=-2), dict(Hq=0), dict(Hkv=0), dict(Hq=3), dict(D=4), dict(D=68),
           dict(D=136), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0),
           dict(cap=float("nan")), dict(cap=1e-35), dict(strides=None), dict(strides=[12] + good[1:], B=2), dict(q=None),
           dict(q=p + 8), dict(begin=None), dict(out=None), dict(out=p + 2),
           dict(strides=[good[0], 0, 64] + good[3:]), dict(strides=[good[0], good[1], 36] + good[3:]),
           dict(B=1 << 20), dict(Sq=1 << 31), dict(Hq=1 << 13, Hkv=1 << 13)]
    for call in (fwd, bwd):
        for b in bad:
            assert call(**b) == _lib.FL_ERR_ARG, (call.__name__, b)
    assert bwd(ws=None) == _lib.FL_ERR_ARG and bwd(n=16) == _lib.FL_ERR_ARG and bwd(ws=p + 4) == _lib.FL_ERR_ARG
    long = dict(Sq=1, Sk=4096)
    assert lib.fl_attn_fwd_workspace_bytes(1, 1, 4096, 2, 2, 64) > 0
    assert fwd(**long) == _lib.FL_ERR_ARG and fwd(**long, ws=p, n=64) == _lib.FL_ERR_ARG
    assert fwd(B=0) == _lib.FL_OK and fwd(Sq=0) == _lib.FL_OK and bwd(B=0) == _lib.FL_OK
    assert lib.fl_attn_fwd_workspace_bytes(0, 1, 1, 1, 1, 64) == 0
    assert lib.fl_attn_bwd_workspace_bytes(1, 1, 1, 3, 2, 64) == 0


@pytest.mark.gpu
def test_large_cap(cuda_lib):
    """At the largest cap a score is off by the tanh's error (under 2^-21: an
    exponential, a sum and a reciprocal of half a step to two steps of 2^-24 each
    around 1) times the cap, 2^-11: a probability by less than bf16's half step.
    Larger caps are refused."""
    from spilltune_b200 import attention
    B, S, H, K, D = 1, 150, 4, 2, 64
    q, k, v, _ = _inputs(B, S, S, H, K, D, 8)
    begin, end = (x.cuda() for x in _ranges("causal", B, S, S, 8))
    got = _both(q, k, v, begin, end, None, cap=1024.0)
    want = _oracle(q, k, v, begin, end, D ** -0.5, 1024.0, None)
    assert float((got["lse"].double() - want["lse"][0]).abs().max()) <= 2.0 ** -11 + 2.0 ** -18
    out, vmax = want["out"][0], float(v.double().abs().max())
    # twice the scores' error (numerator and sum), P's and the result's rounding
    assert float((got["out"].double() - out).abs().max()) <= vmax * (2 * 2.0 ** -11 + 2.0 ** -8 + 2.0 ** -8)
    with pytest.raises(ValueError, match="softcap"):
        attention.fwd(q, k, v, begin, end, softcap=1025.0)
    with pytest.raises(ValueError, match="softcap"):
        attention.fwd(q, k, v, begin, end, softcap=float("inf"))


@pytest.mark.gpu
def test_refusals(cuda_lib):
    from spilltune_b200 import attention
    q, k, v, do = _inputs(1, 8, 8, 4, 2, 64, 1)
    r = torch.zeros(1, 8, dtype=torch.int32, device="cuda")
    out, lse = attention.fwd(q, k, v, r, r + 8)
    bad = [(lambda: attention.fwd(q.float(), k, v, r, r), "bf16"),
           (lambda: attention.fwd(q[0], k, v, r, r), "bf16 \\[batch"),
           (lambda: attention.fwd(q, k[..., :32], v, r, r), "do not fit"),
           (lambda: attention.fwd(q, k, v[:, :4], r, r), "do not fit"),
           (lambda: attention.fwd(q[:, :, :3], k, v, r, r), "share"),
           (lambda: attention.fwd(q, k, v, r.long(), r), "begin"),
           (lambda: attention.fwd(q, k, v, r, r[:, :4]), "end"),
           (lambda: attention.fwd(q, k, v, r, r, scale=0.0), "scale"),
           (lambda: attention.fwd(q, k, v, r, r, softcap=-1.0), "softcap"),
           (lambda: attention.fwd(q, k, v, r, r, softcap=1e-35), "softcap"),
           (lambda: attention.fwd(q, k, v, r, r, slopes=torch.ones(2, device="cuda")), "slopes"),
           (lambda: attention.attend(q, k, v, r, r, slopes=torch.ones(4, device="cuda", requires_grad=True)),
            "no gradient"),
           (lambda: attention.bwd(do[:, :4], q, k, v, out, lse, r, r), "q's shape"),
           (lambda: attention.bwd(do, q, k, v, out, lse.double(), r, r), "lse"),
           (lambda: attention.fwd(*(torch.zeros(1, 8, 2, 136, dtype=torch.bfloat16, device="cuda"),) * 3, r, r),
            "unsupported_capability")]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()
