"""Calls of spilltune_b200.attention at the edge of what it takes: scores that are not numbers, masks that are
not one range a row."""
import pytest
import torch


def _inputs(B, Sq, Sk, H, K, D, seed):
    g = torch.Generator().manual_seed(seed)
    bf = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    return bf(B, Sq, H, D), bf(B, Sk, K, D), bf(B, Sk, K, D), bf(B, Sq, H, D)


def _all_keys(B, Sq, Sk):
    begin = torch.zeros(B, Sq, dtype=torch.int32, device="cuda")
    return begin, begin + Sk


MODES = [(0.0, False), (30.0, False), (0.0, True), (30.0, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("cap,slopes", MODES)
@pytest.mark.parametrize("Sq,Sk,H,K,D", [(40, 40, 4, 2, 64), (20, 150, 3, 3, 128), (1, 2000, 8, 2, 64)])
def test_a_key_that_is_not_a_number(cuda_lib, Sq, Sk, H, K, D, cap, slopes):
    """One NaN key that every row sees, at each place among eight neighbouring columns of a score tile: every log
    sum and result of its heads is NaN, and those of the other heads are what they were."""
    from spilltune_b200 import _lib, attention
    q, k, v, _ = _inputs(1, Sq, Sk, H, K, D, Sk)
    begin, end = _all_keys(1, Sq, Sk)
    opt = dict(softcap=cap, slopes=torch.full((H,), 0.01, device="cuda") if slopes else None)
    want = attention.fwd(q, k, v, begin, end, **opt)
    G = H // K
    for at in list(range(8)) + [Sk - 1]:
        bad = k.clone()
        bad[:, at, 0] = float("nan")
        out, lse = attention.fwd(q, bad, v, begin, end, **opt)
        assert bool(lse[:, :, :G].isnan().all()) and bool(out[:, :, :G].isnan().all()), at
        assert torch.equal(lse[:, :, G:], want[1][:, :, G:]) and torch.equal(out[:, :, G:], want[0][:, :, G:]), at
    assert _lib.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cap,slopes", MODES)
@pytest.mark.parametrize("S,H,K,D", [(40, 2, 2, 64), (150, 4, 2, 128)])
def test_a_query_that_is_not_a_number(cuda_lib, S, H, K, D, cap, slopes):
    """A NaN query of one head: NaN in its own row, its own gradient and the gradients of every key it sees (of its
    key/value head), and nowhere else."""
    from spilltune_b200 import _lib, attention
    q, k, v, do = _inputs(1, S, S, H, K, D, S)
    begin, end = _all_keys(1, S, S)
    opt = dict(softcap=cap, slopes=torch.full((H,), 0.01, device="cuda") if slopes else None)
    for at in range(8):
        bad = q.clone()
        bad[:, at, 0] = float("nan")
        out, lse = attention.fwd(bad, k, v, begin, end, **opt)
        dq, dk, dv = attention.bwd(do, bad, k, v, out, lse, begin, end, **opt)
        hit = torch.zeros(1, S, H, dtype=torch.bool, device="cuda")
        hit[:, at, 0] = True
        assert torch.equal(lse.isnan(), hit), at
        for x in (out, dq):
            assert torch.equal(x.isnan(), hit[..., None].expand_as(x)), at
        for x in (dk, dv):
            assert bool(x[:, :, 0].isnan().all()) and not bool(x[:, :, 1:].isnan().any()), at
    assert _lib.status() == 0


def test_a_prefix_with_a_window_is_refused():
    """A token past its window would see the prefix and its last keys: two ranges."""
    from spilltune_b200.attention import row_ranges
    with pytest.raises(ValueError, match="unsupported_capability: .*prefix.*window"):
        row_ranges(1, 10, prefix=torch.tensor([4]), window=2)
    assert row_ranges(1, 4, prefix=torch.tensor([2]))[1].tolist() == [[2, 2, 3, 4]]
    assert row_ranges(1, 4, window=2)[0].tolist() == [[0, 0, 1, 2]]


def test_c_entries_refuse_a_scale_whose_power_of_two_form_overflows():
    """The kernels multiply by scale log2(e): from 2.36e38 on that is infinite, and a score of 0 NaN."""
    import ctypes

    from spilltune_b200 import _lib, build
    build.build()
    lib = _lib.load()
    p, strides = 4096, (ctypes.c_int64 * 12)(*[512, 128, 64] * 4)  # p is never read: each call is refused first
    for scale in (2.5e38, 3.4e38):
        assert lib.fl_attn_fwd(p, p, p, strides, 1, 4, 4, 2, 2, 64, p, p, scale, 0.0, None, p, p, None, 0,
                               None) == _lib.FL_ERR_ARG
        assert lib.fl_attn_bwd(p, p, p, p, strides, p, p, 1, 4, 4, 2, 2, 64, p, p, scale, 0.0, None, p, p, p, p,
                               1 << 20, None) == _lib.FL_ERR_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 70])
def test_offsets_past_32_bits(cuda_lib, Sq):
    """The last keys of the second of two caches of 2^31 elements together and more: results and gradients are those
    of these keys alone, and the other keys' gradients 0."""
    from spilltune_b200 import _lib, attention
    B, Sk, H, K, D, seen = 2, 280_001, 32, 32, 128, 90
    assert (B - 0.5) * Sk * K * D > 2 ** 30 and B * Sk * K * D > 2 ** 31
    q, k0, v0, do = _inputs(B, Sq, seen, H, K, D, 3)
    k, v = (torch.zeros(B, Sk, K, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k[:, Sk - seen:], v[:, Sk - seen:] = k0, v0
    begin = torch.full((B, Sq), Sk - seen, dtype=torch.int32, device="cuda")
    end = torch.full_like(begin, Sk)
    out, lse = attention.fwd(q, k, v, begin, end)
    dq, dk, dv = attention.bwd(do, q, k, v, out, lse, begin, end)
    zero = torch.zeros_like(begin)
    want, wlse = attention.fwd(q, k0, v0, zero, zero + seen)
    grads = attention.bwd(do, q, k0, v0, want, wlse, zero, zero + seen)
    assert _lib.status() == 0
    assert not bool(dk[:, :Sk - seen].any()) and not bool(dv[:, :Sk - seen].any())
    # Other tiles and splits, so other roundings of P or ds and another order.  A rounding to bf16 is off by up to
    # 2^-8, over a binade 1.7e-3 in the mean square; two results with two each differ by twice that, under 2^-7.
    # A log sum is off by up to 2^-17 sum |q k| scale, which is under 8 in the mean of 128 products over 11.3.
    for got, other in ((out, want), (dq, grads[0]), (dk[:, Sk - seen:], grads[1]), (dv[:, Sk - seen:], grads[2])):
        assert float((got.double() - other.double()).norm() / other.double().norm()) < 2.0 ** -7
    assert float((lse - wlse).abs().max()) < 2 * 8 * 2.0 ** -17
