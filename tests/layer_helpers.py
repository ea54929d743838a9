"""64-bit forms of the encoder's layer operators and the error bounds their tests use.

A rounding to a 16-bit type is off by at most half a step, EPS[dtype] relative to the value
(plus half the smallest fp16 step below the normal range); fp32 work is bounded per operator.
"""
import math

import torch

EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def cu_of(lens, device="cpu"):
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    if lens:
        cu[1:] = torch.tensor(lens, dtype=torch.int32).cumsum(0)
    return cu.to(device)


def attention64(q, k, v, cu, causal, scale=None):
    """(o, bound): the definition in 64 bits over the rows of each sequence, and how far a kernel may be
    off that rounds the weights and the result to q's type.  Rows outside stay NaN."""
    T, H, D = q.shape
    G = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    o = torch.full((T, H, D), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.full_like(o, math.nan)
    e, tiny = EPS[q.dtype], TINY[q.dtype]
    c = cu.tolist()
    for lo, hi in zip(c[:-1], c[1:]):
        n = hi - lo
        if n == 0:
            continue
        see = torch.ones(n, n, dtype=torch.bool, device=q.device)
        if causal:
            see = see.tril()
        for h in range(H):
            a, b, w = q[lo:hi, h].double(), k[lo:hi, h // G].double(), v[lo:hi, h // G].double()
            s = (a @ b.T * scale).masked_fill(~see, -math.inf)
            p = torch.softmax(s, -1)
            o[lo:hi, h] = p @ w
            mass = p @ w.abs()                          # sum of p |v|
            # a score is off by D fp32 roundings of its products' sizes, a weight by that much more
            off = (a.abs() @ b.abs().T * scale).masked_fill(~see, 0).amax(-1, keepdim=True) * (D * 2.0 ** -24)
            # below fp16's normal range a weight (relative to the largest, 1 at least) is off by TINY
            low = tiny * (see.double() @ w.abs())
            bound[lo:hi, h] = 1.02 * (e * o[lo:hi, h].abs() + (e + 2 * off + 2.0 ** -16) * mass + low + tiny)
    return o, bound


def rms_rope64(x, w, cos, sin, pos, eps, interleaved):
    """(y, bound) of one set of heads."""
    R = 2 * cos.shape[1]
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    i = torch.arange(0, R, 2, device=x.device) if interleaved else torch.arange(R // 2, device=x.device)
    j = i + 1 if interleaved else i + R // 2
    out, size = y.clone(), y.abs().clone()
    out[..., i] = y[..., i] * c - y[..., j] * s
    out[..., j] = y[..., j] * c + y[..., i] * s
    size[..., i] = size[..., j] = y[..., i].abs() + y[..., j].abs()
    # fp32: the mean, the root, two products and a sum: far fewer than 64 roundings of 2^-24 each
    return out, 1.001 * EPS[x.dtype] * out.abs() + 2.0 ** -18 * size + TINY[x.dtype]


def act64(g, act):
    """(act, act')"""
    if act == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 0.134145 * g * g)


LIP = 1.2          # |act'| <= 1.13 for the three activations
BEND = 0.8         # |act''| <= 0.798 (gelu at 0)


def ffn64(x, wg, wu, act):
    """(h, g, u, bounds of the three)."""
    e, tiny = EPS[x.dtype], TINY[x.dtype]
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.T, x @ wu.T
    n = (x.shape[1] + 8) * 2.0 ** -24                        # a sum of K products in fp32
    eg, eu = n * (x.abs() @ wg.abs().T), n * (x.abs() @ wu.abs().T)
    a, _ = act64(g, act)
    h = a * u
    # the activation's exp is good to 2^-17 for arguments up to 88
    bh = 1.02 * (e * h.abs() + LIP * eg * u.abs() + (a.abs() + LIP * eg) * eu + 2.0 ** -16 * (g * u).abs() + tiny)
    return h, g, u, bh, 1.02 * eg, 1.02 * eu                 # g and u are kept in fp32


def ffn_backward64(dh, x, wg, wu, gate, up, act):
    """Gradients of the formula at the kept gate and up, and their bounds: dg and du are
    rounded to the type before they are multiplied."""
    e, tiny = EPS[x.dtype], TINY[x.dtype]
    dh, x, wg, wu, g, u = (t.double() for t in (dh, x, wg, wu, gate, up))
    a, d = act64(g, act)
    dg, du = dh * u * d, dh * a
    eg = 1.02 * e * dg.abs() + 2.0 ** -16 * (dh * u).abs() * (1 + g.abs()) + tiny
    eu = 1.02 * e * du.abs() + 2.0 ** -16 * (dh * g).abs() + tiny

    def product(pairs, n):
        """sum of a @ b over (a, error of a, b) with n fp32 roundings, result rounded."""
        y = sum(p @ b for p, _, b in pairs)
        off = sum(ep @ b.abs() + (n + 8) * 2.0 ** -24 * (p.abs() @ b.abs()) for p, ep, b in pairs)
        return y, 1.02 * (e * y.abs() + off + tiny)

    F, M = g.shape[1], g.shape[0]
    dx = product([(dg, eg, wg), (du, eu, wu)], 2 * F)
    dwg = product([(dg.T, eg.T, x)], M)
    dwu = product([(du.T, eu.T, x)], M)
    return dx, dwg, dwu


def check(got, want, bound, what=""):
    """Every value within its bound (NaN in `want`: not looked at)."""
    look = ~torch.isnan(want)
    bad = look & ~((got.double() - want).abs() <= bound)
    if bad.any():
        i = bad.nonzero()[0].tolist()
        i = tuple(i)
        raise AssertionError(f"{what}: {int(bad.sum())} of {int(look.sum())} values off, first at {i}: "
                             f"{got[i].item()} for {want[i].item()} within {bound[i].item()}")
