"""Rotary, norm and attention together, as a decoder block runs them: over views of one
projection's output, forward and backward, and inside ``packed_dense_block``."""
import os

import numpy as np
import pytest
import torch

import e2e_tiny as t
import oracle.linear as ol
from test_attention import _oracle as attention_oracle
from test_rotary import _oracle as rotary_oracle

GOLDEN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")


@pytest.mark.gpu
@pytest.mark.parametrize("H,K,D,norm", [(8, 2, 128, True), (6, 3, 64, False)])
def test_chain_of_operators(cuda_lib, H, K, D, norm):
    """qkv [B, S, (H + 2 K) D] -> norm, rotation, attention over documents -> gradients of qkv and the
    norm weights, against the same chain in 64 bits.  In norm, q, k and out are rounded once each (2^-9
    of a value on average over its binade, half a step 2^-8 at most), and a score of size x moves p by
    x 2^-8 at most: scores stay under 8 here, so every result is within 8 * 2^-8 + 3 * 2^-8 < 0.045 of
    its norm, and gradients, which carry the same factors twice, within 0.09."""
    from spilltune_b200 import attention, rotary
    from spilltune_b200.dense import FusedAttention
    B, S = 2, 150
    g = torch.Generator().manual_seed(D)
    qkv = torch.randn(B, S, (H + 2 * K) * D, generator=g).to(torch.bfloat16).cuda().requires_grad_(True)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).cuda().requires_grad_(True) for _ in range(2)]
    dout = torch.randn(B, S, H, D, generator=g).to(torch.bfloat16).cuda()
    docs = torch.tensor([[0] * 50 + [1] * 100, [0] * 149 + [1]]).cuda()
    begin, end = attention.row_ranges(B, S, documents=docs)
    pos = torch.arange(S, device="cuda") - begin
    inv, factor = rotary.frequencies(D, 10000.0)
    inv = inv.cuda()

    def split(x):
        q, k, v = x.split([H * D, K * D, K * D], -1)
        return q.unflatten(-1, (H, D)), k.unflatten(-1, (K, D)), v.unflatten(-1, (K, D))

    weights = (*w, 1e-6) if norm else ()
    leaves = [qkv, *w] if norm else [qkv]
    out = FusedAttention(begin, end, factor=factor)(*split(qkv), pos, inv, *weights)
    grads = torch.autograd.grad(out, leaves, dout)
    wide = [x.detach().double().requires_grad_(True) for x in leaves]
    q, k, v = split(wide[0])
    q = rotary_oracle(q, pos, inv, factor, False, wide[1] if norm else None, 1e-6)
    k = rotary_oracle(k, pos, inv, factor, False, wide[2] if norm else None, 1e-6)
    want = attention_oracle(q, k, v, begin, end, D ** -0.5, 0.0, None)["out"][0]
    expect = torch.autograd.grad(want, wide, dout.double())
    assert ol.rel_l2(out.detach(), want.detach()) <= 0.045
    for got, e in zip(grads, expect):
        assert got.shape == e.shape and ol.rel_l2(got, e) <= 0.09


def _block_inputs(H, K, D, hidden, inter, S, B, qk_norm):
    from spilltune_b200 import codec
    g = torch.Generator().manual_seed(7)
    shapes = {"self_attn.q_proj": (H * D, hidden), "self_attn.k_proj": (K * D, hidden),
              "self_attn.v_proj": (K * D, hidden), "self_attn.o_proj": (hidden, H * D),
              "mlp.gate_proj": (inter, hidden), "mlp.up_proj": (inter, hidden), "mlp.down_proj": (hidden, inter)}
    packed = {n: codec.encode_int4_sym(torch.randn(*s, generator=g) * s[1] ** -0.5) for n, s in shapes.items()}
    raw = {n: (1 + 0.1 * torch.randn(hidden, generator=g)).to(torch.bfloat16).cuda()
           for n in ("input_layernorm.weight", "post_attention_layernorm.weight")}
    if qk_norm:
        raw.update({f"self_attn.{n}_norm.weight": (1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).cuda()
                    for n in "qk"})
    x = torch.randn(B, S, hidden, generator=g).to(torch.bfloat16).cuda()
    dy = torch.randn(B, S, hidden, generator=g).to(torch.bfloat16).cuda()
    return packed, raw, x, dy


@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm", [False, True])
def test_block_is_as_near_to_fp32_as_the_eager_form(cuda_lib, qk_norm):
    """packed_dense_block with the fused operators rounds less often than op by op: its output and
    input gradient are no further from the block in FP32 (same decoded weights)."""
    from spilltune_b200 import attention, ops, rotary
    from spilltune_b200.dense import FusedAttention, block_forward, packed_dense_block, part_keys
    H, K, D, hidden, B, S = 8, 2, 64, 512, 2, 200
    packed, raw, x, dy = _block_inputs(H, K, D, hidden, 768, S, B, qk_norm)
    dev = {n: p.to("cuda") for n, p in packed.items()}
    parts = dict(raw)
    for n, p in dev.items():
        pk, sk = part_keys(n + ".weight")
        parts[pk], parts[sk] = p.payload, p.scales
    inv, _ = rotary.frequencies(D, 10000.0)
    inv = inv.cuda()
    pos = torch.arange(S, device="cuda").expand(B, S)
    angle = torch.cat((pos[..., None] * inv,) * 2, -1)
    mask = torch.full((S, S), torch.finfo(torch.bfloat16).min, device="cuda").triu(1)[None, None]
    begin, end = attention.row_ranges(B, S, device="cuda")
    kw = dict(heads=H, kv_heads=K, head_dim=D, eps=1e-6, qk_norm=qk_norm)
    none = dict(lora_q=None, lora_v=None, lora_o=None)

    def run(fn, xin):
        leaf = xin.detach().clone().requires_grad_(True)
        y = fn(leaf)
        return y.detach(), torch.autograd.grad(y, leaf, dy.to(y.dtype))[0]

    fused = run(lambda a: packed_dense_block(a, (pos, inv), None, attention=FusedAttention(begin, end), **kw, **none,
                                             **parts), x)
    eager = run(lambda a: packed_dense_block(a, (angle.cos().bfloat16(), angle.sin().bfloat16()), mask.bfloat16(),
                                             **kw, **none, **parts), x)
    wide = {n: v.float() for n, v in raw.items()}
    dense = {n: ops.dequant(p).float() for n, p in dev.items()}
    exact = run(lambda a: block_forward(a, (angle.cos(), angle.sin()), mask, lambda v, p: v @ dense[p].t(), wide,
                                        **kw), x.float())
    for f, e, w in zip(fused, eager, exact):
        assert ol.rel_l2(f, w) <= ol.rel_l2(e, w)


def test_refusals_without_a_gpu():
    from spilltune_b200.dense import FusedAttention, block_forward
    z = torch.zeros(1, 2, 8, dtype=torch.bfloat16)
    rows = torch.zeros(1, 2, dtype=torch.int32)
    fused = FusedAttention(rows, rows)
    weights = {"input_layernorm.weight": torch.ones(8, dtype=torch.bfloat16)}
    call = lambda mask: block_forward(z, (torch.arange(2), torch.ones(4)), mask, lambda x, p: x, weights, heads=1,  # noqa: E731
                                      kv_heads=1, head_dim=8, eps=1e-6, attention=fused)
    with pytest.raises(ValueError, match="row ranges, not an attention mask"):
        call(torch.zeros(1, 1, 2, 2))
    with pytest.raises(ValueError, match="CUDA tensors"):
        call(None)


@pytest.mark.gpu
def test_trains_like_the_reference(cuda_lib):
    """The tiny Llama of the reference's own training run, streamed from pinned memory, with the fused
    operators in every block: per-step losses and step-1/2 LoRA gradients within the bars of the eager block."""
    from spilltune_b200 import _lib, attention, rotary
    from spilltune_b200.dense import FusedAttention, PackedBlockReloader, packed_dense_block
    from spilltune_b200.streaming import PackedSlotSession
    from test_e2e_tiny_llama import _lora_kwargs, _packed_layers, _snapshot
    fx = np.load(os.path.join(GOLDEN, "tiny_llama_train.npz"))
    dev = torch.device("cuda")
    layers, raw, boundary = _packed_layers()
    session = PackedSlotSession([{k: w.pin_memory() for k, w in layer.items()} for layer in layers], dev, slots=2)
    adapters = t.make_adapters(dev)
    begin, end = attention.row_ranges(1, t.SEQ, device=dev)
    inv, factor = rotary.frequencies(t.HEAD_DIM, t.THETA)
    where = (torch.arange(t.SEQ, device=dev), inv.to(dev))
    fused = FusedAttention(begin, end, factor=factor)

    def functional(hidden_states, position_embeddings, attention_mask, **kw):
        return packed_dense_block(hidden_states, where, None, attention=fused, **kw)

    blocks = []
    for i in range(t.LAYERS):
        kw = {"heads": t.HEADS, "kv_heads": t.KV_HEADS, "head_dim": t.HEAD_DIM, "eps": t.EPS,
              **_lora_kwargs(adapters[i])}
        reloader = PackedBlockReloader(session, i, raw={k: v.to(dev) for k, v in raw[i].items()})
        blocks.append(t.Block(i, functional, kw, reloader, adapters[i]))
    assert _lib.status(reset=True) == 0
    got = {}
    losses = t.train(blocks, boundary["model.embed_tokens.weight"], boundary["model.norm.weight"].to(dev),
                     boundary["lm_head.weight"].to(dev), device=dev, terminal=t.fused_terminal, steps=4,
                     on_step=_snapshot(got))
    torch.cuda.synchronize()
    assert _lib.status() == 0
    session.close()
    assert np.abs(np.array(losses) - fx["losses"][:4]).max() <= 1e-2
    assert got
    for key, val in got.items():
        torch.testing.assert_close(val, torch.from_numpy(fx[key]), rtol=0.06, atol=3e-3, msg=key)
