"""The decoder block's operators between its projections, as cases that can be run and measured.

Three operators: the rotary position embedding of queries and keys ("rotary"), the same with an RMS norm of every
head before it ("norm_rotary"), and attention over row ranges ("attention"): query i of a sequence sees the keys
begin[i] <= j < end[i], which holds causal, document, prefix, sliding-window and padding masks alike; scores may be
capped by a tanh or lowered with the distance.

`own = False` computes the plain forms with elementary torch operations; `own = True` calls spilltune_b200.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token of the Llama-3-8B shape through the rotation: a decode step, all latency.
        {"name": "rotary_one_token", "op": "rotary", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "interleaved": False, "scaling": "llama3", "first": 8191, "train": False},
        # The Llama-3-8B training step's micro-batch: 4 x 2048 tokens, 32 + 8 heads of 128, long-context frequencies.
        {"name": "rotary_llama_train", "op": "rotary", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "interleaved": False, "scaling": "llama3", "first": 0, "train": True},
        # The DeepSeek-V3 shape: 128 query heads' 64 rotated columns (a slice of 192-wide heads) and one shared key
        # head, neighbouring columns paired, YaRN frequencies.
        {"name": "rotary_mla_interleaved", "op": "rotary", "tokens": 4096, "heads": 128, "kv_heads": 1, "dim": 64,
         "rot": 64, "interleaved": True, "scaling": "yarn", "first": 0, "train": True},
        # The Qwen3-30B-A3B shape: 2 x 4096 tokens, 32 + 4 heads of 128, a norm per head; frozen norm weights.
        {"name": "norm_rotary_qwen_train", "op": "norm_rotary", "tokens": 8192, "heads": 32, "kv_heads": 4,
         "dim": 128, "rot": 128, "interleaved": False, "scaling": "none", "first": 0, "train": True, "wgrad": False},
        # An odd row count far into a long context, half of each 80-wide head rotated, trainable norm weights.
        {"name": "norm_rotary_partial_odd", "op": "norm_rotary", "tokens": 1027, "heads": 14, "kv_heads": 2,
         "dim": 80, "rot": 40, "interleaved": False, "scaling": "linear", "first": 250000, "train": True,
         "wgrad": True},
        # The tiny Llama that the end-to-end tests train: 2 x 128 tokens, 4 + 2 heads of 64.
        {"name": "attention_tiny_train", "op": "attention", "batch": 2, "rows": 128, "keys": 128, "heads": 4,
         "kv_heads": 2, "dim": 64, "mask": "causal", "cap": 0.0, "slope": False, "train": True, "shape": 1},
        # The Llama-3-8B training step's attention: 4 sequences of 2048, causal.
        {"name": "attention_llama_train", "op": "attention", "batch": 4, "rows": 2048, "keys": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "mask": "causal", "cap": 0.0, "slope": False, "train": True, "shape": 2},
        # Qwen3-30B-A3B heads over two packed rows of 4096 tokens: several documents to a row.
        {"name": "attention_qwen_documents", "op": "attention", "batch": 2, "rows": 4096, "keys": 4096, "heads": 32,
         "kv_heads": 4, "dim": 128, "mask": "documents", "cap": 0.0, "slope": False, "train": True, "shape": 3},
        # Capped scores and a sliding window.
        {"name": "attention_capped_window", "op": "attention", "batch": 1, "rows": 4096, "keys": 4096, "heads": 16,
         "kv_heads": 8, "dim": 128, "mask": "window", "cap": 50.0, "slope": False, "train": True, "shape": 4},
        # Odd lengths, padding rows, a prefix seen by all, scores lowered with the distance, a head group of 7.
        {"name": "attention_prefix_slope_odd", "op": "attention", "batch": 3, "rows": 777, "keys": 777, "heads": 14,
         "kv_heads": 2, "dim": 64, "mask": "prefix", "cap": 0.0, "slope": True, "train": True, "shape": 5},
        # One long sequence, forward only: the streamed forward pass keeps no graph.
        {"name": "attention_long_forward", "op": "attention", "batch": 1, "rows": 8192, "keys": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "mask": "causal", "cap": 0.0, "slope": False, "train": False, "shape": 6},
        # One new token in each of four sequences over 8192 kept keys: a decode step.
        {"name": "attention_one_token", "op": "attention", "batch": 4, "rows": 1, "keys": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "mask": "causal", "cap": 0.0, "slope": False, "train": False, "shape": 7},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        norm = rng.random() < 0.5
        tokens = _log_int(rng, 1, 16384)
        dim = rng.choice((32, 64, 64, 80, 96, 128, 128, 256))
        rot = dim if rng.random() < 0.6 else rng.choice((dim // 2, dim // 4))
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
        heads = max(1, min(heads, int(8192 * 40 * 128 / (tokens * dim)) - kv_heads))
        case = {"op": "norm_rotary" if norm else "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rot": rot, "interleaved": rng.random() < 0.4,
                "scaling": rng.choice(("none", "linear", "llama3", "yarn")),
                "first": rng.choice((0, 0, 1000, 120000, 900000)), "train": rng.random() < 0.7}
        if norm:
            case["wgrad"] = rng.random() < 0.4
        return case
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
    dim = rng.choice((64, 64, 80, 96, 128, 128))
    if rng.random() < 0.25:
        rows = rng.choice((1, 1, 2, 5, 16))
        batch, keys = rng.choice((1, 2, 4, 8)), _log_int(rng, max(rows, 2), 16384)
        mask, train = rng.choice(("causal", "causal", "window", "all")), False
    else:
        rows = keys = _log_int(rng, 1, 4096)
        batch = rng.choice((1, 1, 2, 3, 4))
        mask = rng.choice(("causal", "documents", "documents", "prefix", "window", "all"))
        train = rng.random() < 0.7 and rows > 1
    while batch > 1 and batch * rows * keys * heads * dim > 4 * 2048 * 2048 * 32 * 128 / 2:
        batch -= 1
    while heads > kv_heads and batch * rows * keys * heads * dim > 4 * 2048 * 2048 * 32 * 128:
        heads -= kv_heads
    return {"op": "attention", "batch": batch, "rows": rows, "keys": keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "mask": mask, "cap": rng.choice((0.0, 0.0, 30.0, 50.0)), "slope": rng.random() < 0.3,
            "train": train, "shape": rng.randrange(1 << 20)}


# ------------------------------------------------------------------ inputs
def _frequencies(case):
    """(inverse frequencies fp32 [rot / 2], factor of cos and sin) under the case's long-context scaling."""
    rot = case["rot"]
    inv = 1.0 / 500000.0 ** (np.arange(0, rot, 2, dtype=np.float64) / rot)
    factor = 1.0
    if case["scaling"] == "linear":
        inv = inv / 8.0
    elif case["scaling"] == "llama3":
        wave = 2 * np.pi / inv
        smooth = np.clip((8192.0 / wave - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        inv = (1 - smooth) * inv / 8.0 + smooth * inv
    elif case["scaling"] == "yarn":
        at = lambda turns: rot * math.log(4096.0 / (turns * 2 * math.pi)) / (2 * math.log(500000.0))  # noqa: E731
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0, 1)
        inv = inv / 40.0 * ramp + inv * (1 - ramp)
        factor = 0.1 * math.log(40.0) + 1.0
    return inv.astype(np.float32), factor


def _ranges(case):
    """begin, end int32 [batch, rows] of a case's mask: made from the case alone, so that its work is known.  Windows
    and documents hold two keys at least: the softmax of a single one is constant, its gradients are zero, and what
    any form computes for them is rounding noise."""
    B, R, S = case["batch"], case["rows"], case["keys"]
    rng = random.Random(case["shape"])
    at = np.arange(R, dtype=np.int64)[None, :] + (S - R)
    begin = np.zeros((B, R), np.int64)
    end = np.broadcast_to(at + 1, (B, R)).copy()
    kind = case["mask"]
    if kind == "all":
        end[:] = S
    elif kind == "window":
        begin = np.maximum(end - max(2, S // 4), 0)
    elif kind == "documents":
        for b in range(B):
            cut = 0
            while cut < S:
                stop = min(S, cut + 2 + int(rng.expovariate(1.0 / max(1.0, S / 6.0))))
                begin[b, cut:stop] = cut
                cut = stop
    elif kind == "prefix":
        for b in range(B):
            prefix, live = rng.randrange(0, S // 2 + 1), S - (rng.randrange(0, S // 3 + 1) if b else 0)
            end[b] = np.maximum(end[b], prefix)
            end[b] = np.minimum(end[b], live)
            begin[b, live:] = 0
            end[b, live:] = 0  # padding: these rows see nothing
    return begin.astype(np.int32), end.astype(np.int32)


def _slopes(case):
    if not case["slope"]:
        return None
    return np.array([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])], np.float32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32)  # noqa: E731
    bf = torch.bfloat16
    s = {"case": case}
    D, H, K = case["dim"], case["heads"], case["kv_heads"]
    if case["op"] != "attention":
        T = case["tokens"]
        if case["interleaved"]:  # the rotated columns of wider heads, and a key of its own
            s["q"] = normal(T, H, 3 * D).to(bf)[..., 2 * D:]
            s["k"] = normal(T, K, D).to(bf)
        else:  # both lie in one projection's output, with the values behind them
            x = normal(T, (H + 2 * K) * D).to(bf)
            s["q"] = x[:, :H * D].view(T, H, D)
            s["k"] = x[:, H * D:(H + K) * D].view(T, K, D)
        inv, s["factor"] = _frequencies(case)
        s["inv"] = torch.from_numpy(inv).to(DEV)
        s["positions"] = case["first"] + torch.arange(T, device=DEV)
        if case["op"] == "norm_rotary":
            s["qw"] = (1 + 0.2 * normal(D)).to(bf)
            s["kw"] = (1 + 0.2 * normal(D)).to(bf)
        if case["train"]:
            s["dq"] = normal(T, H, D).to(bf)
            s["dk"] = normal(T, K, D).to(bf)
        return s
    B, R, S = case["batch"], case["rows"], case["keys"]
    if R == S:  # views of one projection's output
        x = normal(B, S, (H + 2 * K) * D)
        x[..., :H * D] *= 1.5
        x = x.to(bf)
        s["q"] = x[..., :H * D].view(B, S, H, D)
        s["k"] = x[..., H * D:(H + K) * D].view(B, S, K, D)
        s["v"] = x[..., (H + K) * D:].view(B, S, K, D)
    else:
        s["q"] = (1.5 * normal(B, R, H, D)).to(bf)
        s["k"] = normal(B, S, K, D).to(bf)
        s["v"] = normal(B, S, K, D).to(bf)
    begin, end = _ranges(case)
    s["begin"], s["end"] = torch.from_numpy(begin).to(DEV), torch.from_numpy(end).to(DEV)
    slopes = _slopes(case)
    s["slopes"] = None if slopes is None else torch.from_numpy(slopes).to(DEV)
    s["scale"] = D ** -0.5
    if case["train"]:
        s["dout"] = normal(B, R, H, D).to(bf)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _own_attention(s) if case["op"] == "attention" else _own_rotary(s)
    return _plain_attention(s) if case["op"] == "attention" else _plain_rotary(s)


def _own_rotary(s):
    from spilltune_b200 import rotary
    case = s["case"]
    norm = {"q_weight": s["qw"], "k_weight": s["kw"], "eps": 1e-6} if case["op"] == "norm_rotary" else {}
    opt = dict(interleaved=case["interleaved"], factor=s["factor"], **norm)
    q, k = rotary.fwd(s["q"], s["k"], s["positions"], s["inv"], **opt)
    if not case["train"]:
        return {"q": q, "k": k}
    out = {"q": q, "k": k}
    if case.get("wgrad"):
        out["dq"], out["dk"], out["dqw"], out["dkw"] = rotary.bwd(s["dq"], s["dk"], s["q"], s["k"], s["positions"],
                                                                  s["inv"], weight_grads=True, **opt)
    else:
        out["dq"], out["dk"], _, _ = rotary.bwd(s["dq"], s["dk"], s["q"], s["k"], s["positions"], s["inv"], **opt)
    return out


def _own_attention(s):
    from spilltune_b200 import attention
    case = s["case"]
    opt = dict(scale=s["scale"], softcap=case["cap"], slopes=s["slopes"])
    if not case["train"]:
        out, _ = attention.fwd(s["q"], s["k"], s["v"], s["begin"], s["end"], **opt)
        return {"out": out}
    out, lse = attention.fwd(s["q"], s["k"], s["v"], s["begin"], s["end"], **opt)
    dq, dk, dv = attention.bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, s["begin"], s["end"], **opt)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


# ------------------------------------------------------------------ plain forms
def _cos_sin(s):
    # 64 bits: an angle of a far position has lost its fraction in 32
    angle = s["positions"].double()[:, None] * s["inv"].double()[None, :]
    return ((angle.cos() * s["factor"]).float()[:, None, :], (angle.sin() * s["factor"]).float()[:, None, :])


def _turn(x, cos, sin, rot, interleaved):
    """Rotates the first `rot` columns of x [T, heads, D]; -sin turns back."""
    a, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        left, right = a[..., 0::2], a[..., 1::2]
        a = torch.stack((left * cos - right * sin, right * cos + left * sin), -1).flatten(-2)
    else:
        left, right = a[..., :rot // 2], a[..., rot // 2:]
        a = torch.cat((left * cos - right * sin, right * cos + left * sin), -1)
    return torch.cat((a, rest), -1) if rest.shape[-1] else a


def _plain_rotary(s):
    case = s["case"]
    cos, sin = _cos_sin(s)
    norm = case["op"] == "norm_rotary"
    out = {}

    def one(name, x, w, dy):
        x = x.float()
        xn = x
        if norm:
            w = w.float()
            r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            xn = x * r * w
        out[name] = _turn(xn, cos, sin, case["rot"], case["interleaved"]).bfloat16()
        if not case["train"]:
            return
        d = _turn(dy.float(), cos, -sin, case["rot"], case["interleaved"])
        if norm:
            if case["wgrad"]:
                out["d" + name + "w"] = (d * (x * r)).sum((0, 1), dtype=torch.float64).float()
            d = d * w
            d = r * (d - x * r * (d * x * r).mean(-1, keepdim=True))
        out["d" + name] = d.bfloat16()

    one("q", s["q"], s.get("qw"), s.get("dq"))
    one("k", s["k"], s.get("kw"), s.get("dk"))
    return out


def _plain_attention(s):
    case = s["case"]
    B, R, H, D = s["q"].shape
    S, K = s["k"].shape[1:3]
    G, cap = H // K, case["cap"]
    q = s["q"].float().view(B, R, K, G, D).permute(0, 2, 3, 1, 4)
    k = s["k"].float().permute(0, 2, 1, 3)[:, :, None]
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]
    j = torch.arange(S, device=q.device)
    seen = (j >= s["begin"][..., None]) & (j < s["end"][..., None])
    seen = seen[:, None, None]
    x = (q @ k.transpose(-1, -2)) * s["scale"]
    if cap:
        x = torch.tanh(x / cap)
        slope = 1 - x * x if case["train"] else None
        x = x * cap
    if s["slopes"] is not None:
        far = (torch.arange(R, device=q.device)[:, None] + (S - R) - j[None, :]).abs().float()
        x = x - s["slopes"].view(1, K, G, 1, 1) * far
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -math.inf, 0.0))
    del x
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    o = p @ v
    back = lambda t: t.permute(0, 3, 1, 2, 4).reshape(B, R, H, D).bfloat16()  # noqa: E731
    out = {"out": back(o)}
    if not case["train"]:
        return out
    do = s["dout"].float().view(B, R, K, G, D).permute(0, 2, 3, 1, 4)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    d = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    if cap:
        d = d * slope
    d = d * s["scale"]
    out["dq"] = back(d @ k)
    out["dk"] = (d.transpose(-1, -2) @ q).sum(2).permute(0, 2, 1, 3).contiguous().bfloat16()
    out["dv"] = dv.permute(0, 2, 1, 3).contiguous().bfloat16()
    return out


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attention(s) if case["op"] == "attention" else _exact_rotary(s)


def _exact_rotary(s):
    """Each pair of columns as a complex number, turned by exp(i angle); gradients by differentiation."""
    case = s["case"]
    rot, T = case["rot"], case["tokens"]
    angle = s["positions"].double()[:, None] * s["inv"].double()[None, :]
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None, :]
    i = torch.arange(rot // 2, device=DEV)
    left, right = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
    out = {}
    for name in ("q", "k"):
        x = s[name].double().requires_grad_(True)
        w = s[name + "w"].double().requires_grad_(True) if case["op"] == "norm_rotary" else None
        y = x if w is None else w * x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6).sqrt()
        z = torch.complex(y[..., left], y[..., right]) * turn
        y = y.index_copy(-1, left, z.real).index_copy(-1, right, z.imag)
        out[name] = y.detach()
        if case["train"]:
            leaves = [x, w] if case.get("wgrad") else [x]
            grads = torch.autograd.grad(y, leaves, s["d" + name].double())
            out["d" + name] = grads[0]
            if case.get("wgrad"):
                out["d" + name + "w"] = grads[1]
    return out


def _exact_attention(s):
    """One head of one sequence at a time, its softmax differentiated by autograd, all in 64 bits."""
    case = s["case"]
    B, R, S, H, K, D = (case[n] for n in ("batch", "rows", "keys", "heads", "kv_heads", "dim"))
    if B * R * S * H * D > 1.2e12 or R * S > 7e7:
        return None
    new = lambda n, h: torch.zeros(B, n, h, D, dtype=torch.float64, device=DEV)  # noqa: E731
    out = {"out": new(R, H)}
    if case["train"]:
        out.update(dq=new(R, H), dk=new(S, K), dv=new(S, K))
    key = torch.arange(S, device=DEV)[None, :]
    row = torch.arange(R, device=DEV)[:, None] + (S - R)
    for b in range(B):
        hidden = (key < s["begin"][b][:, None]) | (key >= s["end"][b][:, None])
        empty = hidden.all(-1, keepdim=True)
        for h in range(H):
            leaves = [s[n][b, :, i].double().requires_grad_(case["train"])
                      for n, i in (("q", h), ("k", h * K // H), ("v", h * K // H))]
            with torch.set_grad_enabled(case["train"]):
                x = torch.einsum("id,jd->ij", leaves[0], leaves[1]) * s["scale"]
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if s["slopes"] is not None:
                    x = x - s["slopes"][h].double() * (row - key).abs().double()
                x = x.masked_fill(hidden & ~empty, -math.inf).log_softmax(-1).exp()
                y = torch.einsum("ij,jd->id", x.masked_fill(empty, 0.0), leaves[2])
            out["out"][b, :, h] = y.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(y, leaves, s["dout"][b, :, h].double())
                out["dq"][b, :, h] = dq
                out["dk"][b, :, h * K // H] += dk
                out["dv"][b, :, h * K // H] += dv
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] != "attention":
        n = case["tokens"] * (H + K) * D
        norm = case["op"] == "norm_rotary"
        # forward: read x, write y; backward: read dy (and x, for the norm), write dx
        moved = 2 * 2 * n + ((3 if norm else 2) * 2 * n if case["train"] else 0)
        ops = (3 + 4 * norm) * n * (1 + 2 * case["train"])
        return {"bytes": moved + case["tokens"] * 8 + case["rot"] * 2, "flops": ops}
    B, R, S = case["batch"], case["rows"], case["keys"]
    begin, end = _ranges(case)
    pairs = int(np.maximum(end.astype(np.int64) - begin, 0).sum()) * H
    q, kv = B * R * H * D * 2, B * S * K * D * 2
    # forward: q, k, v in, out; backward: those and dout in, three gradients out; 2 products, then 5
    moved = 2 * q + 2 * kv + (4 * q + 4 * kv if case["train"] else 0) + 8 * B * R
    return {"bytes": moved, "flops": pairs * D * (4 + 10 * case["train"])}
