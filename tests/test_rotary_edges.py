"""Calls of spilltune_b200.rotary at the edge of what it takes."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 40])
def test_norm_of_queries_only_with_trainable_weights(cuda_lib, D):
    """Without keys the key norm's weight has no part in the result: the other gradients are those of the call
    without it, and it gets none."""
    from spilltune_b200 import rotary
    g = torch.Generator().manual_seed(D)
    q = torch.randn(21, 3, D, generator=g).to(torch.bfloat16).cuda().requires_grad_(True)
    dq = torch.randn(21, 3, D, generator=g).to(torch.bfloat16).cuda()
    qw = (1 + 0.2 * torch.randn(D, generator=g)).cuda().requires_grad_(True)
    kw = (1 + 0.2 * torch.randn(D, generator=g)).cuda().requires_grad_(True)
    pos, inv = torch.arange(21, device="cuda"), rotary.frequencies(D)[0].cuda()
    y, none = rotary.norm_rotate(q, None, qw, kw, pos, inv, eps=1e-6)
    assert none is None
    got = torch.autograd.grad(y, (q, qw, kw), dq, allow_unused=True)
    want = torch.autograd.grad(rotary.norm_rotate(q, None, qw, None, pos, inv, eps=1e-6)[0], (q, qw), dq)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[2] is None
    alone = torch.autograd.grad(rotary.norm_rotate(q, None, qw.detach(), kw, pos, inv, eps=1e-6)[0], q, dq)
    assert torch.equal(alone[0], want[0])


def test_frequencies_that_want_a_gradient_are_refused():
    """Refused before anything else, so on the CPU too; without a graph they are numbers like any other."""
    from spilltune_b200 import rotary
    q, pos = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.arange(2)
    inv, w = torch.ones(32, requires_grad=True), torch.ones(64)
    for call in (lambda: rotary.rotate(q, q, pos, inv), lambda: rotary.norm_rotate(q, q, w, w, pos, inv, eps=1e-6)):
        with pytest.raises(ValueError, match="unsupported_capability: inv_freq gets no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA tensors"):
            call()


@pytest.mark.parametrize("theta,scaling,match", [
    (1.0, {"type": "yarn", "factor": 4.0, "original_length": 512}, "theta > 1"),
    (0.5, {"type": "yarn", "factor": 4.0, "original_length": 512}, "theta > 1"),
    (1e4, {"type": "yarn", "factor": float("inf"), "original_length": 512}, "factor"),
    (1e4, {"type": "linear", "factor": float("inf")}, "factor"),
    (1e4, {"type": "yarn", "factor": 4.0, "original_length": float("inf")}, "original_length"),
    (1e4, {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_length": float("nan")}, "original_length")])
def test_scalings_without_a_value_are_refused(theta, scaling, match):
    """YaRN's ramp divides by ln(theta); an infinite factor or length leaves frequencies or cosines without a value."""
    from spilltune_b200 import rotary
    with pytest.raises(ValueError, match=match):
        rotary.frequencies(64, theta, scaling)
    assert bool(rotary.frequencies(64, 1.0)[0].eq(1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
def test_offsets_past_32_bits(cuda_lib, norm):
    """The last tokens of 2^31 elements and more: the bits that they give alone, forward and backward."""
    from spilltune_b200 import rotary
    T, H, D, last = 270_000, 64, 128, 40
    assert T * H * D > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    x[-last:] = torch.randn(last, H, D, generator=g, device="cuda").to(torch.bfloat16)
    pos, inv = torch.arange(T, device="cuda"), rotary.frequencies(D)[0].cuda()
    w = torch.rand(D, generator=g, device="cuda") + 0.5
    opt = dict(q_weight=w, eps=1e-6) if norm else {}
    y, _ = rotary.fwd(x, None, pos, inv, **opt)
    assert torch.equal(y[-last:], rotary.fwd(x[-last:], None, pos[-last:], inv, **opt)[0])
    dx = rotary.bwd(y, None, x, None, pos, inv, **opt)[0]
    assert torch.equal(dx[-last:], rotary.bwd(y[-last:], None, x[-last:], None, pos[-last:], inv, **opt)[0])
