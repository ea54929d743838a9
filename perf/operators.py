"""What is measured of the encoder's layer operators: packed attention, query/key norm with rotary
positions, and the gated feed-forward product with its backward pass.

The model sizes are this repository's own encoder (hidden 768, 12 heads of 64, 32-token queries,
passages of 20..180 tokens) and generic ones (heads of 128 that share keys, hidden 2048).
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------ cases
def _attn(name, dtype, heads, kv_heads, dim, causal, count, shortest, longest, lens_seed):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "causal": causal, "count": count, "shortest": shortest, "longest": longest, "lens_seed": lens_seed}


def _rope(name, dtype, heads, kv_heads, dim, rot, interleaved, norm, tokens, far):
    return {"name": name, "op": "norm_rope", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "interleaved": interleaved, "norm": norm, "tokens": tokens, "far": far}


def _ffn(name, op, dtype, rows, hidden, inner, act):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "hidden": hidden, "inner": inner, "act": act}


def listed():
    return [
        # one query of an interactive search: latency
        _attn("attn_one_query", "fp16", 12, 12, 64, False, 1, 19, 19, 1),
        # passages on their way into the index, packed without padding
        _attn("attn_passages", "fp16", 12, 12, 64, False, 1024, 20, 180, 2),
        # prompts of very different lengths through a causal backbone with grouped heads
        _attn("attn_prompts", "bf16", 32, 8, 128, True, 12, 1, 4096, 3),
        # one long document
        _attn("attn_long", "bf16", 16, 4, 128, True, 1, 16384, 16384, 4),
        # one query of an interactive search: latency
        _rope("rope_one_query", "fp16", 12, 12, 64, 64, False, True, 19, 512),
        # passages; half of each head is rotated, neighbouring pairs
        _rope("rope_passages", "fp16", 12, 12, 64, 32, True, True, 102411, 512),
        # long documents with grouped heads
        _rope("rope_long", "bf16", 32, 8, 128, 128, False, True, 32768, 131072),
        # a single token: the weights are all there is to read
        _ffn("ffn_one_row", "ffn", "bf16", 1, 2048, 5504, "silu"),
        # a few queries in one batch, odd sizes
        _ffn("ffn_queries", "ffn", "fp16", 200, 768, 2056, "gelu"),
        # passages
        _ffn("ffn_passages", "ffn", "bf16", 16384, 2048, 8192, "silu"),
        # fine-tuning on a small batch: forward, then all gradients
        _ffn("ffn_train_small", "ffn_train", "fp16", 1000, 768, 2048, "gelu_tanh"),
        # fine-tuning on passages
        _ffn("ffn_train", "ffn_train", "bf16", 8192, 2048, 5504, "silu"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "norm_rope", "ffn", "ffn_train"))
    dtype = rng.choice(("fp16", "bf16"))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
    heads = kv_heads * rng.choice((1, 2, 3, 4) if kv_heads <= 8 else (1, 2))
    dim = rng.choice((32, 64, 64, 80, 96, 128, 128))
    if op == "attention":
        longest = _log(rng, 1, 8192)
        room = 16 * 16384 ** 2 // (2 * heads * longest ** 2)          # scores that the plain form holds
        count = min(_log(rng, 1, 1024), max(1, room), max(1, 262144 // longest))
        shortest = longest if rng.random() < 0.25 else rng.randint(0, longest)
        return _attn("", dtype, heads, kv_heads, dim, rng.random() < 0.5, count, shortest, longest,
                     rng.randrange(1 << 30))
    if op == "norm_rope":
        rot = 16 * rng.randint(1, dim // 16)
        tokens = min(_log(rng, 1, 131072), (32768 * 40 * 128) // ((heads + kv_heads) * dim))
        return _rope("", dtype, heads, kv_heads, dim, rot, rng.random() < 0.5, rng.random() < 0.75, tokens,
                     _log(rng, 64, 131072))
    hidden = 8 * _log(rng, 8, 512)
    inner = 8 * _log(rng, 8, 1024)
    most = 16384 * 2048 * 8192 if op == "ffn" else 8192 * 2048 * 5504
    rows = max(1, min(_log(rng, 1, 16384), most // (hidden * inner)))
    return _ffn("", op, dtype, rows, hidden, inner, rng.choice(("silu", "gelu", "gelu_tanh")))


def _lens(case):
    rng = random.Random(case["lens_seed"])
    lens = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["count"])]
    lens[rng.randrange(len(lens))] = case["longest"]                 # never no token at all
    return lens


def work(case):
    if case["op"] == "attention":
        H, KV, D = case["heads"], case["kv_heads"], case["dim"]
        lens = _lens(case)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": sum(lens) * (2 * H + 2 * KV) * D * 2 + 4 * (len(lens) + 1), "flops": 4 * D * H * pairs}
    if case["op"] == "norm_rope":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        table = min(case["tokens"], case["far"]) * case["rot"] * 4
        return {"bytes": 4 * values + table + 4 * case["tokens"], "flops": 8 * values}
    M, K, F = case["rows"], case["hidden"], case["inner"]
    if case["op"] == "ffn":
        return {"bytes": 2 * (M * K + 2 * F * K + M * F), "flops": 4 * M * K * F}
    # forward, then both gradients of each product
    return {"bytes": 2 * (2 * M * K + 4 * F * K + 2 * M * F), "flops": 12 * M * K * F}


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = {"case": dict(case)}
    if case["op"] == "attention":
        H, KV, D = case["heads"], case["kv_heads"], case["dim"]
        lens = _lens(case)
        T = sum(lens)
        # q, k, v are views of one projection's output, as a layer leaves them; some heads attend
        # widely and some sharply
        qkv = normal(T, (H + 2 * KV) * D)
        gain = torch.linspace(0.5, 4.0, H, device=dev).repeat_interleave(D)
        qkv[:, :H * D] *= gain
        qkv = qkv.to(dt)
        s["q"] = qkv[:, :H * D].view(T, H, D)
        s["k"] = qkv[:, H * D:(H + KV) * D].view(T, KV, D)
        s["v"] = qkv[:, (H + KV) * D:].view(T, KV, D)
        cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
        cu[1:] = torch.tensor(lens, dtype=torch.int32).cumsum(0)
        s["cu"] = cu.to(dev)
        s["longest"] = max(lens)
    elif case["op"] == "norm_rope":
        H, KV, D, T, R = case["heads"], case["kv_heads"], case["dim"], case["tokens"], case["rot"]
        qkv = (2.0 * normal(T, (H + 2 * KV) * D)).to(dt)
        s["q"] = qkv[:, :H * D].view(T, H, D)
        s["k"] = qkv[:, H * D:(H + KV) * D].view(T, KV, D)
        if case["norm"]:
            s["qw"] = (1.0 + 0.2 * normal(D)).to(dt)
            s["kw"] = (1.0 + 0.2 * normal(D)).to(dt)
        freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)
        angle = torch.arange(case["far"], dtype=torch.float64, device=dev)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        first = torch.randint(0, case["far"], (1,), generator=g, device=dev)
        s["pos"] = ((first + torch.arange(T, device=dev)) % case["far"]).to(torch.int32)
    else:
        M, K, F = case["rows"], case["hidden"], case["inner"]
        s["x"] = normal(M, K).to(dt)
        s["wg"] = (normal(F, K) / math.sqrt(K)).to(dt)
        s["wu"] = (normal(F, K) / math.sqrt(K)).to(dt)
        if case["op"] == "ffn_train":
            s["dh"] = normal(M, F).to(dt)
    return s


# ------------------------------------------------------------------------------------ plain forms
def _plain_attention(q, k, v, cu, longest, causal):
    T, H, D = q.shape
    KV, B, L = k.shape[1], cu.shape[0] - 1, longest
    G = H // KV
    cu = cu.long()
    n = cu[1:] - cu[:-1]
    at = torch.arange(L, device=q.device)
    rows = (cu[:-1, None] + at).clamp(max=T - 1)                       # [B, L]: every sequence padded to L
    qp = q.float()[rows].view(B, L, KV, G, D).permute(0, 2, 3, 1, 4).reshape(B, KV, G * L, D)
    kp = k.float()[rows].permute(0, 2, 3, 1)                           # [B, KV, D, L]
    vp = v.float()[rows].permute(0, 2, 1, 3)                           # [B, KV, L, D]
    s = torch.matmul(qp, kp).view(B, KV, G, L, L).mul_(1.0 / math.sqrt(D))
    seen = (at[None, :] < n[:, None])[:, None, :]                      # [B, 1, L] keys of the sequence
    if causal:
        seen = seen & (at[None, None, :] <= at[None, :, None])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, KV, G * L, L), vp).view(B, KV, G, L, D) / total
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return o.permute(0, 3, 1, 2, 4).reshape(B, L, H, D)[b, t - cu[b]].to(q.dtype)


def _plain_norm_rope(x, w, cos, sin, pos, interleaved):
    R = 2 * cos.shape[1]
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    r = y[..., :R]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = r[..., :R // 2], r[..., R // 2:]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r, y[..., R:]), -1).to(x.dtype)


def _plain_act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)


def _plain_ffn(x, wg, wu, act, dh=None):
    dt = x.dtype
    x, wg, wu = x.float(), wg.float(), wu.float()
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _plain_act(g, act)
    h = (a * u).to(dt)
    if dh is None:
        return h
    dh = dh.float()
    dg, du = dh * u * da, dh * a
    return h, (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)


def run(state):
    s, case = state, state["case"]
    if own:
        from ragrt_b200 import encoder
        if case["op"] == "attention":
            return encoder.packed_attention(s["q"], s["k"], s["v"], s["cu"], causal=case["causal"])
        if case["op"] == "norm_rope":
            return encoder.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["pos"], s.get("qw"), s.get("kw"),
                                        eps=1e-6, interleaved=case["interleaved"])
        if case["op"] == "ffn":
            return encoder.gated_ffn(s["x"], s["wg"], s["wu"], act=case["act"])
        h, gate, up = encoder.gated_ffn(s["x"], s["wg"], s["wu"], act=case["act"], keep=True)
        return (h,) + tuple(encoder.gated_ffn_backward(s["dh"], s["x"], s["wg"], s["wu"], gate, up, act=case["act"]))
    if case["op"] == "attention":
        return _plain_attention(s["q"], s["k"], s["v"], s["cu"], s["longest"], case["causal"])
    if case["op"] == "norm_rope":
        return (_plain_norm_rope(s["q"], s.get("qw"), s["cos"], s["sin"], s["pos"], case["interleaved"]),
                _plain_norm_rope(s["k"], s.get("kw"), s["cos"], s["sin"], s["pos"], case["interleaved"]))
    return _plain_ffn(s["x"], s["wg"], s["wu"], case["act"], s.get("dh"))


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        H, KV, D = case["heads"], case["kv_heads"], case["dim"]
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        ends = s["cu"].tolist()
        if len(ends) * H > 20000:
            return None
        for lo, hi in zip(ends[:-1], ends[1:]):
            for h in range(H):
                q = s["q"][lo:hi, h].double()
                k = s["k"][lo:hi, h * KV // H].double()
                v = s["v"][lo:hi, h * KV // H].double()
                p = q @ k.mT * D ** -0.5
                if case["causal"]:
                    p += torch.full_like(p, -math.inf).triu_(1)
                out[lo:hi, h] = torch.softmax(p, -1) @ v
        return out
    if case["op"] == "norm_rope":
        R = case["rot"]
        cos, sin = s["cos"].double()[s["pos"].long()], s["sin"].double()[s["pos"].long()]
        turn = torch.complex(cos, sin)[:, None]
        outs = []
        for x, w in ((s["q"], s.get("qw")), (s["k"], s.get("kw"))):
            y = x.double()
            if w is not None:
                y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            pairs = y[..., :R].unflatten(-1, (R // 2, 2) if case["interleaved"] else (2, R // 2))
            axis = -1 if case["interleaved"] else -2
            z = torch.complex(pairs.select(axis, 0), pairs.select(axis, 1)) * turn
            y[..., :R] = torch.stack((z.real, z.imag), axis).flatten(-2)
            outs.append(y)
        return tuple(outs)
    leaves = [s[n].double().requires_grad_() for n in ("x", "wg", "wu")]
    x, wg, wu = leaves
    with torch.enable_grad():
        g = torch.nn.functional.linear(x, wg)
        if case["act"] == "silu":
            a = torch.nn.functional.silu(g)
        else:
            a = torch.nn.functional.gelu(g, approximate="tanh" if case["act"] == "gelu_tanh" else "none")
        h = a * torch.nn.functional.linear(x, wu)
        if case["op"] == "ffn":
            return h.detach()
        grads = torch.autograd.grad(h, leaves, s["dh"].double())
    return (h.detach(),) + tuple(grads)
