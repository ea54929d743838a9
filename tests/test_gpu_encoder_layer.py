"""The encoder's layer operators (packed attention, query/key norm with rotary positions, gated
feed-forward and its gradients) against their definitions in 64 bits.  Bounds: layer_helpers.py."""
import math

import pytest
import torch

import layer_helpers as L
from ragrt_b200 import _lib, encoder

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def qkv_of(lens, H, KV, D, dtype, seed, gain=1.0, spare=0):
    """q, k, v as views of one projection's output, with `spare` rows behind the last sequence."""
    T = sum(lens) + spare
    m = torch.randn(T, (H + 2 * KV) * D, generator=gen(seed), device="cuda")
    m[:, :H * D] *= gain
    m = m.to(dtype)
    return (m[:, :H * D].view(T, H, D), m[:, H * D:(H + KV) * D].view(T, KV, D), m[:, (H + KV) * D:].view(T, KV, D))


def flag():
    torch.cuda.synchronize()
    return _lib.lib().ragrt_device_error(1)


# ------------------------------------------------------------------------------------ attention
LENS = [[1], [0, 1, 0], [2, 31, 33], [127, 128, 129], [5, 300, 0, 64, 1], [513], [32] * 9, [1000, 24],
        [255, 1, 257, 0, 0, 640]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [(2, 2, 64), (4, 1, 128), (3, 3, 32), (6, 2, 96), (2, 1, 8), (4, 2, 80)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
def test_attention(lens, heads, causal, dtype):
    q, k, v = qkv_of(lens, *heads, dtype, seed=sum(lens) + heads[2], gain=2.0)
    cu = L.cu_of(lens, "cuda")
    got = encoder.packed_attention(q, k, v, cu, causal=causal)
    want, bound = L.attention64(q, k, v, cu, causal)
    L.check(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads,causal", [([4100], (2, 1, 128), True), ([3000, 1500], (1, 1, 64), False),
                                               ([2048], (4, 2, 64), True), ([4000, 2300], (2, 1, 64), True),
                                               ([700, 5, 1900], (3, 1, 96), False), ([1, 4200], (1, 1, 40), True),
                                               ([130, 0, 3000, 129], (2, 2, 128), True), ([1200], (1, 1, 80), True)])
def test_attention_long(lens, heads, causal, dtype):
    q, k, v = qkv_of(lens, *heads, dtype, seed=5)
    cu = L.cu_of(lens, "cuda")
    want, bound = L.attention64(q, k, v, cu, causal)
    L.check(encoder.packed_attention(q, k, v, cu, causal=causal), want, bound)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n,D", [(700, 64), (700, 128), (3300, 64)])
def test_attention_growing_scores(n, D, causal):
    """Scores that rise along the keys, far beyond one another: the running maximum moves in every block."""
    H = 2
    q, k, v = qkv_of([n], H, H, D, torch.bfloat16, seed=9)
    k = k.clone()
    k[..., 0] = torch.linspace(-60, 60, n, device="cuda")[:, None]
    q = q.clone()
    q[..., 0] = 16.0
    q[300:, 1, 0] = -16.0
    cu = L.cu_of([n], "cuda")
    want, bound = L.attention64(q, k, v, cu, causal)
    L.check(encoder.packed_attention(q, k, v, cu, causal=causal), want, bound)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_keeps_what_is_not_seen_out(causal, D, bad):
    """NaN and infinities of other sequences, of rows behind the last one and (causal) of later rows."""
    lens = [70, 40, 200, 9]
    q, k, v = qkv_of(lens, 4, 2, D, torch.float16, seed=3, spare=30)
    cu = L.cu_of(lens, "cuda")
    clean, bound = L.attention64(q, k, v, cu, causal)
    q, k, v = q.clone(), k.clone(), v.clone()
    for t in (k, v):
        t[70:110] = bad
        t[319:] = bad
        if causal:
            t[250:310] = bad
    q[319:] = bad
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    got = encoder.packed_attention(q, k, v, cu, causal=causal, out=out)
    assert got is out
    seen = torch.ones(349, dtype=torch.bool, device="cuda")
    seen[70:110] = False
    seen[319:] = False
    if causal:
        seen[250:310] = False
    L.check(got[seen], clean[seen], bound[seen])
    assert (got[319:] == 7.0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_attention_keeps_unseen_values_out_of_long_sequences(D):
    """The same for the tiles of long sequences: a neighbour's NaN, and a later row's."""
    lens = [3300, 900, 3300]
    q, k, v = qkv_of(lens, 2, 1, D, torch.float16, seed=13)
    cu = L.cu_of(lens, "cuda")
    clean, bound = L.attention64(q, k, v, cu, True)
    q, k, v = q.clone(), k.clone(), v.clone()
    for t in (k, v):
        t[3300:4200] = math.nan
        t[7490:] = math.inf
    seen = torch.ones(7500, dtype=torch.bool, device="cuda")
    seen[3300:4200] = False
    seen[7490:] = False
    got = encoder.packed_attention(q, k, v, cu, causal=True)
    L.check(got[seen], clean[seen], bound[seen])


def test_attention_spread_of_a_bad_row_is_the_formulas():
    """A NaN that a row does see reaches it, and only the heads that read it."""
    q, k, v = qkv_of([300], 4, 2, 64, torch.float16, seed=4)
    cu = L.cu_of([300], "cuda")
    want, bound = L.attention64(q, k, v, cu, True)
    v = v.clone()
    v[100, 1, 5] = math.nan
    want[100:, 2:, 5] = math.nan                    # by hand: a product with the masked NaN is NaN too
    got = encoder.packed_attention(q, k, v, cu, causal=True)
    assert torch.equal(got.isnan(), want.isnan())
    L.check(got, want, bound)


@pytest.mark.parametrize("first", [0, 5])
def test_attention_leaves_rows_outside(first):
    lens = [60, 100]
    q, k, v = qkv_of(lens, 2, 2, 64, torch.float16, seed=6, spare=140)
    cu = L.cu_of(lens, "cuda") + first
    out = torch.full(q.shape, -3.0, dtype=torch.float16, device="cuda")
    encoder.packed_attention(q, k, v, cu, out=out)
    want, bound = L.attention64(q, k, v, cu, False)
    L.check(out, want, bound)
    assert (out[:first] == -3.0).all() and (out[first + 160:] == -3.0).all() and flag() == 0


def test_attention_strided_output_and_scale():
    q, k, v = qkv_of([150, 31], 3, 1, 64, torch.bfloat16, seed=8)
    wide = torch.zeros(181, 3 * 64 + 40, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 8:8 + 192].view(181, 3, 64)
    cu = L.cu_of([150, 31], "cuda")
    encoder.packed_attention(q, k, v, cu, scale=0.3, out=out)
    want, bound = L.attention64(q, k, v, cu, False, scale=0.3)
    L.check(out, want, bound)
    assert (wide[:, :8] == 0).all() and (wide[:, 200:] == 0).all()


def test_attention_copies_what_it_cannot_read_in_place():
    q, k, v = qkv_of([90], 2, 2, 64, torch.float16, seed=11)
    cu = L.cu_of([90], "cuda")
    want = encoder.packed_attention(q, k, v, cu)
    qt = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)              # head-major storage
    odd = torch.empty(90 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(90, 2, 64).copy_(k)
    assert torch.equal(encoder.packed_attention(qt, odd, v, cu.long()), want)


def test_attention_rows_past_32_bits_of_elements():
    """Rows so far apart that their offsets pass 2^32 elements."""
    T, pitch = 70000, 65536
    if torch.cuda.mem_get_info()[0] < 12e9:
        pytest.skip("needs 9.2 GB")
    big = torch.empty(T * pitch, dtype=torch.float16, device="cuda").view(T, pitch)
    part = torch.randn(T, 4 * 64, generator=gen(2), device="cuda").half()
    big[:, :256] = part
    q, k, v = (big[:, i * 64:(i + 1) * 64].view(T, 1, 64) for i in range(3))
    out = big[:, 192:256].view(T, 1, 64)
    lens = [69000, 1000]
    cu = L.cu_of(lens, "cuda")
    # the long sequence is causal and only its first rows are looked at: the last ones' keys are many
    encoder.packed_attention(q, k, v, cu, causal=True, out=out)
    s = slice(69000, 70000)
    want, bound = L.attention64(q[s], k[s], v[s], L.cu_of([1000]), True)
    L.check(out[s], want, bound)
    want, bound = L.attention64(q[:600], k[:600], v[:600], L.cu_of([600]), True)
    L.check(out[:600], want, bound)
    row = 68999
    p = torch.softmax(q[row, 0].double() @ k[:69000, 0].double().T / 8, -1)
    w = v[:69000, 0].double()
    e = L.EPS[torch.float16]
    b = 1.02 * (e * (p @ w).abs() + (e + 2.0 ** -14) * (p @ w.abs()) + L.TINY[torch.float16] * w.abs().sum(0))
    L.check(out[row, 0], p @ w, b)


@pytest.mark.parametrize("table", [[0, 50, 40, 90], [0, 200], [-5, 90], [0, 90, 30], [2 ** 31 - 1, -2 ** 31]])
def test_attention_bad_table_raises_the_flag(table):
    q, k, v = qkv_of([90], 2, 2, 64, torch.float16, seed=12)
    flag()
    out = torch.zeros_like(q)
    encoder.packed_attention(q, k, v, torch.tensor(table, dtype=torch.int32, device="cuda"), out=out)
    assert flag() == 6
    ok = encoder.packed_attention(q, k, v, L.cu_of([90], "cuda"))
    want, bound = L.attention64(q, k, v, L.cu_of([90]), False)
    L.check(ok, want, bound)
    assert flag() == 0


@pytest.mark.parametrize("D", [16, 24, 40, 72, 104, 120])
def test_attention_other_head_sizes(D):
    lens = [70, 3, 140]
    q, k, v = qkv_of(lens, 3, 1, D, torch.bfloat16, seed=D)
    cu = L.cu_of(lens, "cuda")
    want, bound = L.attention64(q, k, v, cu, True)
    L.check(encoder.packed_attention(q, k, v, cu, causal=True), want, bound)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_many_short_and_empty_sequences(D, causal):
    """More sequences than the search looks at in two steps, most of them of a few rows or none."""
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 4, (2500,), generator=g).tolist() + [0] * 600 + [130] + [0] * 700
    q, k, v = qkv_of(lens, 2, 1, D, torch.float16, seed=20)
    cu = L.cu_of(lens, "cuda")
    want, bound = L.attention64(q, k, v, cu, causal)
    L.check(encoder.packed_attention(q, k, v, cu, causal=causal), want, bound)
    assert flag() == 0


def test_attention_nothing_but_empty_sequences():
    q, k, v = qkv_of([0], 2, 2, 64, torch.float16, seed=1, spare=300)
    out = torch.full(q.shape, 5.0, dtype=torch.float16, device="cuda")
    encoder.packed_attention(q, k, v, torch.zeros(400, dtype=torch.int32, device="cuda"), out=out)
    assert (out == 5.0).all() and flag() == 0
    assert encoder.packed_attention(q[:0], k[:0], v[:0], L.cu_of([0], "cuda")).shape == (0, 2, 64)
    encoder.packed_attention(q, k, v, L.cu_of([], "cuda"), out=out)
    assert (out == 5.0).all()


def test_attention_64_bit_tables():
    q, k, v = qkv_of([90, 11], 2, 2, 64, torch.float16, seed=12)
    cu = L.cu_of([90, 11], "cuda")
    assert torch.equal(encoder.packed_attention(q, k, v, cu.long()), encoder.packed_attention(q, k, v, cu))
    flag()
    far = torch.tensor([0, 90, 2 ** 32 + 101], device="cuda")          # does not come back as 101
    encoder.packed_attention(q, k, v, far)
    assert flag() == 6


def test_attention_on_two_streams_at_once():
    lens = [3000, 40, 1733]                              # two tiles a CTA for heads of 128, one for 64
    sets = [qkv_of(lens, 4, 2, D, torch.float16, seed=D) for D in (64, 128)]
    cu = L.cu_of(lens, "cuda")
    want = [encoder.packed_attention(*s, cu, causal=True) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(encoder.packed_attention(*s, cu, causal=True))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


# ------------------------------------------------------------------------------------ norm + rotary
def tables(n, R):
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    return a.cos().float(), a.sin().float()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,R", [((12, 12, 64), 64), ((12, 12, 64), 32), ((32, 8, 128), 128), ((3, 1, 96), 96),
                                     ((5, 1, 80), 16), ((2, 2, 16), 16), ((1, 1, 256), 256), ((4, 2, 120), 48),
                                     ((7, 1, 24), 16)])
@pytest.mark.parametrize("T", [1, 19, 1000])
def test_norm_rope(T, heads, R, interleaved, dtype):
    H, KV, D = heads
    q, k, _ = qkv_of([T], H, KV, D, dtype, seed=T + D, gain=3.0)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=gen(i), device="cuda")).to(dtype) for i in (1, 2))
    cos, sin = tables(2048, R)
    pos = torch.randint(0, 2048, (T,), generator=gen(7), device="cuda")
    qo, ko = encoder.qk_norm_rope(q, k, cos, sin, pos, qw, kw, eps=1e-5, interleaved=interleaved)
    L.check(qo, *L.rms_rope64(q, qw, cos, sin, pos, 1e-5, interleaved), "q")
    L.check(ko, *L.rms_rope64(k, kw, cos, sin, pos, 1e-5, interleaved), "k")
    q1, k1 = encoder.qk_norm_rope(q, k, cos, sin, pos.int(), None, kw, eps=1e-5, interleaved=interleaved)
    L.check(q1, *L.rms_rope64(q, None, cos, sin, pos, 1e-5, interleaved), "q without a weight")
    assert torch.equal(k1, ko)


def test_norm_rope_in_place_and_zero_rows():
    q, k, v = qkv_of([333], 12, 4, 64, torch.float16, seed=1)
    whole = q._base if q._base is not None else None
    assert whole is not None
    before_v = v.clone()
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    cos, sin = tables(512, 64)
    pos = torch.arange(333, device="cuda")
    q[5] = 0
    qe, ke = encoder.qk_norm_rope(q, k, cos, sin, pos, w, w)
    assert (qe[5] == 0).all()
    qi, ki = encoder.qk_norm_rope(q, k, cos, sin, pos, w, w, q_out=q, k_out=k)
    assert qi is q and ki is k and torch.equal(q, qe) and torch.equal(k, ke) and torch.equal(v, before_v)
    e = torch.empty(0, 12, 64, dtype=torch.float16, device="cuda")
    qz, kz = encoder.qk_norm_rope(e, e, cos, sin, pos[:0], w, w)
    assert qz.shape == (0, 12, 64) and kz.shape == (0, 12, 64)


def test_norm_rope_of_queries_alone():
    q, _, _ = qkv_of([50], 4, 1, 64, torch.float16, seed=3)
    none = torch.empty(50, 0, 64, dtype=torch.float16, device="cuda")
    cos, sin = tables(64, 64)
    pos = torch.arange(50, device="cuda")
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    qo, ko = encoder.qk_norm_rope(q, none, cos, sin, pos, w)
    L.check(qo, *L.rms_rope64(q, w, cos, sin, pos, 1e-6, False))
    assert ko.shape == (50, 0, 64)


@pytest.mark.parametrize("pos", [-1, 512, 2 ** 40])
def test_norm_rope_position_outside_the_table(pos):
    q, k, _ = qkv_of([4], 2, 2, 64, torch.float16, seed=2)
    cos, sin = tables(512, 64)
    at = torch.tensor([3, pos, 7, 0], device="cuda")
    flag()
    qo, _ = encoder.qk_norm_rope(q, k, cos, sin, at)
    assert flag() == 5
    at[1] = 0
    L.check(qo, *L.rms_rope64(q, None, cos, sin, at, 0, False))


# ------------------------------------------------------------------------------------ gated feed-forward
def ffn_inputs(M, F, K, dtype, seed):
    g = gen(seed)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(2 * F, K, generator=g, device="cuda") * 1.5 / math.sqrt(K)).to(dtype)
    dh = torch.randn(M, F, generator=g, device="cuda").to(dtype)
    return x, w[:F], w[F:], dh


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 72, 128])
@pytest.mark.parametrize("others", [[], [700, 1], [3000]])
def test_attention_of_a_single_key_is_its_value(others, dim, dtype):
    """Whatever the score: rows that see one key, alone in a sequence or first of a causal one."""
    lens = [1, 1, 5, 1] + others + [1]
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    g = torch.Generator(device="cuda").manual_seed(dim)
    q, k, v = [torch.randn(cu[-1], h, dim, generator=g, device="cuda").to(dtype) for h in (6, 2, 2)]
    out = encoder.packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), causal=True)
    first = [a for a, n in zip(cu, lens) if n]
    assert torch.equal(out[first], v[first].repeat_interleave(3, 1))


SHAPES = [(1, 128, 64), (1, 2056, 768), (3, 8, 8), (17, 264, 72), (128, 128, 128), (129, 136, 776), (200, 1160, 768),
          (300, 64, 1000), (1000, 520, 264), (8, 1024, 2048), (9, 1000, 520), (64, 776, 512), (2500, 328, 520),
          (130, 1400, 136), (270, 18312, 264), (400, 22000, 264),
          (140, 2824, 1032), (4104, 264, 264), (2100, 1032, 72)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("M,F,K", SHAPES)
def test_gated_ffn(M, F, K, act, dtype):
    x, wg, wu, dh = ffn_inputs(M, F, K, dtype, M + F + K)
    h, gate, up = encoder.gated_ffn(x, wg, wu, act=act, keep=True)
    wh, g, u, bh, bg, bu = L.ffn64(x, wg, wu, act)
    L.check(h, wh, bh, "h")
    L.check(gate, g, bg, "gate")
    L.check(up, u, bu, "up")
    assert torch.equal(encoder.gated_ffn(x, wg, wu, act=act), h)
    for got, (want, bound), what in zip(encoder.gated_ffn_backward(dh, x, wg, wu, gate, up, act=act),
                                        L.ffn_backward64(dh, x, wg, wu, gate, up, act), ("dx", "dwg", "dwu")):
        L.check(got, want, bound, what)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_ffn_extremes(act):
    """Pre-activations far out on both sides, at zero, and infinite inputs."""
    K, F = 64, 128
    x = torch.zeros(6, K, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = torch.tensor([0.0, 100.0, -100.0, 3e4, -3e4, 1e-30], device="cuda")
    x[:, 1] = 1.0
    wg = torch.zeros(F, K, dtype=torch.bfloat16, device="cuda")
    wg[:, 0] = 1.0
    wu = torch.zeros(F, K, dtype=torch.bfloat16, device="cuda")
    wu[:, 1] = 2.0
    h, gate, up = encoder.gated_ffn(x, wg, wu, act=act, keep=True)
    wh, _, _, bh, _, _ = L.ffn64(x, wg, wu, act)
    L.check(h, wh, bh)
    dh = torch.ones_like(h)
    for got, (want, bound) in zip(encoder.gated_ffn_backward(dh, x, wg, wu, gate, up, act=act),
                                  L.ffn_backward64(dh, x, wg, wu, gate, up, act)):
        assert torch.isfinite(got).all()
        L.check(got, want, bound)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_ffn_gradients_against_differences(act):
    """<grad, d> of each input along a random d, against central differences of the 64-bit formula."""
    M, F, K = 40, 72, 56
    x, wg, wu, dh = ffn_inputs(M, F, K, torch.float16, 77)
    _, gate, up = encoder.gated_ffn(x, wg, wu, act=act, keep=True)
    grads = encoder.gated_ffn_backward(dh, x, wg, wu, gate, up, act=act)
    bounds = [b for _, b in L.ffn_backward64(dh, x, wg, wu, gate, up, act)]
    base = [t.double() for t in (x, wg, wu)]
    g, u = gate.double().abs(), up.double().abs()
    _, _, _, _, eg, eu = L.ffn64(x, wg, wu, act)
    # the gradients are taken at the kept gate and up, which are off by eg and eu: dg and du move by at most this
    dg = dh.double().abs() * (L.LIP * eu + u * L.BEND * eg) * 1.05
    du = dh.double().abs() * L.LIP * eg * 1.05
    moved = [dg @ base[1].abs() + du @ base[2].abs(), dg.T @ base[0].abs(), du.T @ base[0].abs()]

    def loss(ts):
        a, _ = L.act64(ts[0] @ ts[1].T, act)
        return (a * (ts[0] @ ts[2].T) * dh.double()).sum()

    for i in range(3):
        d = torch.randn(base[i].shape, generator=gen(i), device="cuda", dtype=torch.float64)
        step = 1e-4
        up_, down_ = list(base), list(base)
        up_[i] = base[i] + step * d
        down_[i] = base[i] - step * d
        want = ((loss(up_) - loss(down_)) / (2 * step)).item()
        got = (grads[i].double() * d).sum().item()
        room = ((bounds[i] + moved[i]) * d.abs()).sum().item()
        size = (grads[i].double() * d).abs().sum().item()
        assert abs(got - want) <= room + 1e-6 * size


def test_gated_ffn_backward_with_less_scratch_or_none():
    """dx's contraction in as many parts as the scratch allows: one, two, all; never differently twice."""
    M, F, K = 70, 1096, 136
    x, wg, wu, dh = ffn_inputs(M, F, K, torch.float16, 21)
    _, gate, up = encoder.gated_ffn(x, wg, wu, keep=True)
    want, bound = L.ffn_backward64(dh, x, wg, wu, gate, up, "silu")[0]
    lib = _lib.lib()
    full = lib.ragrt_enc_gated_ffn_workspace(M, F, K, 1, 0)
    assert 0 < full <= torch.cuda.get_device_properties(0).multi_processor_count * 128 * 128 * 4
    tmp = torch.empty_like(dh), torch.empty_like(dh)
    for nbytes in (0, 1000, 3 * 128 * 64 * 4, 2 * 3 * 128 * 64 * 4, full):
        ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")
        got = []
        for _ in range(2):
            dx = torch.full_like(x, 9.0)
            _lib.check(lib.ragrt_enc_gated_ffn_backward(
                dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gate.data_ptr(), up.data_ptr(),
                tmp[0].data_ptr(), tmp[1].data_ptr(), dx.data_ptr(), None, None, M, F, K, 0, 0,
                ws.data_ptr() if nbytes else None, nbytes, torch.cuda.current_stream().cuda_stream))
            got.append(dx)
        L.check(got[0], want, bound)
        assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("M,F,K", [(4104, 264, 136), (2100, 1032, 72)])
def test_gated_ffn_weight_gradients_with_less_scratch_or_none(M, F, K):
    """As above for the contraction over many rows; alone, beside dx, and with what dx leaves of the scratch."""
    dtype = torch.bfloat16
    x, wg, wu, dh = ffn_inputs(M, F, K, dtype, 22)
    _, gate, up = encoder.gated_ffn(x, wg, wu, keep=True)
    wants = L.ffn_backward64(dh, x, wg, wu, gate, up, "silu")
    lib = _lib.lib()
    full = lib.ragrt_enc_gated_ffn_workspace(M, F, K, 1, 1)
    part = 128 * 128 * 4
    assert full >= 2 * part
    tmp = torch.empty_like(dh), torch.empty_like(dh)
    for nbytes in (0, part, full // 3, full - part, full):
        ws = torch.full((max(nbytes, 16) + 64,), 77, dtype=torch.uint8, device="cuda")
        for with_dx in (False, True):
            got = [torch.full_like(t, 9.0) for t in (x, wg, wu)]
            _lib.check(lib.ragrt_enc_gated_ffn_backward(
                dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gate.data_ptr(), up.data_ptr(),
                tmp[0].data_ptr(), tmp[1].data_ptr(), got[0].data_ptr() if with_dx else None, got[1].data_ptr(),
                got[2].data_ptr(), M, F, K, 0, 1, ws.data_ptr() if nbytes else None, nbytes,
                torch.cuda.current_stream().cuda_stream))
            for g, (want, bound), what in list(zip(got, wants, ("dx", "dwg", "dwu")))[0 if with_dx else 1:]:
                L.check(g, want, bound, what)
            if not with_dx:
                assert bool((got[0] == 9.0).all())
        assert bool((ws[nbytes:] == 77).all())


def test_gated_ffn_gradients_in_parts_on_two_streams_and_in_graphs():
    """The parts' sums of calls that run side by side, or are replayed, do not meet."""
    sets = []
    for seed, (M, F, K) in enumerate([(130, 1400, 136), (2100, 1032, 72), (400, 22000, 264)]):
        x, wg, wu, dh = ffn_inputs(M, F, K, torch.bfloat16, 30 + seed)
        _, gate, up = encoder.gated_ffn(x, wg, wu, keep=True)
        assert _lib.lib().ragrt_enc_gated_ffn_workspace(M, F, K, 1, 1) > 0
        sets.append((dh, x, wg, wu, gate, up))
    want = [encoder.gated_ffn_backward(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(10):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(encoder.gated_ffn_backward(*s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = encoder.gated_ffn_backward(*s)
        graphs.append((g, out))
    for _ in range(3):
        for st, (g, out) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (g, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
            for t in out:
                t.zero_()
        torch.cuda.synchronize()


def test_gated_ffn_partial_gradients_and_no_rows():
    x, wg, wu, dh = ffn_inputs(130, 136, 72, torch.float16, 3)
    _, gate, up = encoder.gated_ffn(x, wg, wu, keep=True)
    keep = gate.clone(), up.clone()
    dx, dwg, dwu = encoder.gated_ffn_backward(dh, x, wg, wu, gate, up)
    a = encoder.gated_ffn_backward(dh, x, wg, wu, gate, up, need_dw=False)
    b = encoder.gated_ffn_backward(dh, x, wg, wu, gate, up, need_dx=False)
    assert a[1] is None and a[2] is None and b[0] is None
    assert torch.equal(a[0], dx) and torch.equal(b[1], dwg) and torch.equal(b[2], dwu)
    assert torch.equal(gate, keep[0]) and torch.equal(up, keep[1])
    h, gate, up = encoder.gated_ffn(x[:0], wg, wu, keep=True)
    assert h.shape == (0, 136)
    dx, dwg, dwu = encoder.gated_ffn_backward(dh[:0], x[:0], wg, wu, gate, up)
    assert dx.shape == (0, 72) and (dwg == 0).all() and (dwu == 0).all() and dwg.shape == wg.shape


def test_gated_ffn_views():
    """Column slices and transposed storage are copied, solid views read in place."""
    x, wg, wu, _ = ffn_inputs(33, 136, 72, torch.bfloat16, 5)
    want = encoder.gated_ffn(x, wg, wu)
    wide = torch.zeros(33, 200, dtype=torch.bfloat16, device="cuda")
    wide[:, 64:136] = x
    assert torch.equal(encoder.gated_ffn(wide[:, 64:136], wg.t().contiguous().t(), wu), want)
    out = torch.empty(33, 136, dtype=torch.bfloat16, device="cuda")
    assert encoder.gated_ffn(x, wg, wu, out=out) is out and torch.equal(out, want)


# ------------------------------------------------------------------------------------ together
def _layer(x, p, cu, pos, cos, sin, H, KV, D, tap=None):
    """One transformer layer on this build's kernels: x [T, hidden] fp16 -> [T, hidden]."""
    T, hid = x.shape
    W = (H + 2 * KV) * D
    qkv = encoder._gemm(x, p["qkv"], None, x.new_empty(T, W), encoder.EPI_BIAS)
    q, k = qkv[:, :H * D].view(T, H, D), qkv[:, H * D:(H + KV) * D].view(T, KV, D)
    v = qkv[:, (H + KV) * D:].view(T, KV, D)
    if tap is not None:
        tap.update(qkv=qkv.clone())
    encoder.qk_norm_rope(q, k, cos, sin, pos, p["qw"], p["kw"], q_out=q, k_out=k)
    ctx = encoder.packed_attention(q, k, v, cu, causal=True)
    y = encoder._gemm(ctx.view(T, H * D), p["o"], None, x.new_empty(T, hid), encoder.EPI_BIAS_RESIDUAL, residual=x)
    h = encoder.gated_ffn(y, p["gate"], p["up"], act="gelu")
    z = encoder._gemm(h, p["down"], None, x.new_empty(T, hid), encoder.EPI_BIAS_RESIDUAL, residual=y)
    if tap is not None:
        tap.update(q=q, k=k, v=v, ctx=ctx, y=y, h=h)
    return z


def _layer_inputs(seed):
    H, KV, D, hid, F = 4, 2, 64, 256, 640
    lens = [20, 180, 1, 0, 77, 122]
    g = gen(seed)
    n = lambda *s, sd=1.0: (torch.randn(*s, generator=g, device="cuda") * sd).half()
    p = {"qkv": n((H + 2 * KV) * D, hid, sd=hid ** -0.5), "qw": 1 + n(D, sd=0.1), "kw": 1 + n(D, sd=0.1),
         "o": n(hid, H * D, sd=(H * D) ** -0.5), "gate": n(F, hid, sd=hid ** -0.5), "up": n(F, hid, sd=hid ** -0.5),
         "down": n(hid, F, sd=F ** -0.5)}
    cos, sin = tables(256, D)
    pos = torch.cat([torch.arange(i) for i in lens]).cuda()
    return n(sum(lens), hid), p, L.cu_of(lens, "cuda"), pos, cos, sin, H, KV, D


def test_layer_of_the_operators_together():
    """Projection, norm + rotary in place, attention, projection + residual, gated feed-forward,
    projection + residual: each operator against 64 bits on what the one before it left."""
    x, p, cu, pos, cos, sin, H, KV, D = _layer_inputs(1)
    tap = {}
    z = _layer(x, p, cu, pos, cos, sin, H, KV, D, tap)
    T = x.shape[0]
    q0, k0 = tap["qkv"][:, :H * D].view(T, H, D), tap["qkv"][:, H * D:(H + KV) * D].view(T, KV, D)
    L.check(tap["q"], *L.rms_rope64(q0, p["qw"], cos, sin, pos, 1e-6, False), "q")
    L.check(tap["k"], *L.rms_rope64(k0, p["kw"], cos, sin, pos, 1e-6, False), "k")
    L.check(tap["ctx"], *L.attention64(tap["q"], tap["k"], tap["v"], cu, True), "ctx")
    wh, _, _, bh, _, _ = L.ffn64(tap["y"], p["gate"], p["up"], "gelu")
    L.check(tap["h"], wh, bh, "h")
    want = tap["h"].double() @ p["down"].double().T + tap["y"].double()
    room = 1.02 * 2.0 ** -11 * want.abs() + 700 * 2.0 ** -24 * (tap["h"].double().abs() @ p["down"].double().abs().T) + 2.0 ** -23
    L.check(z, want, room, "z")


def test_layer_in_two_graphs_and_on_another_stream():
    """Two captured graphs of the layer with their own inputs, replayed in turn and on another stream than
    the one they were captured on, give what eager calls give."""
    sets = [_layer_inputs(s) for s in (2, 3)]
    want = [_layer(*s) for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for s in sets:
        with torch.cuda.stream(side):
            _layer(*s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _layer(*s)
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), w in zip(graphs, want):
            out.zero_()
            g.replay()
            assert torch.equal(out, w)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for g, out in graphs:
            g.replay()
        again = [_layer(*s) for s in sets]
    torch.cuda.synchronize()
    for (g, out), w, a in zip(graphs, want, again):
        assert torch.equal(out, w) and torch.equal(a, w)


def test_gradients_captured_while_eager_ones_live():
    x, wg, wu, dh = ffn_inputs(300, 264, 136, torch.bfloat16, 9)

    def step():
        h, gate, up = encoder.gated_ffn(x, wg, wu, keep=True)
        return (h,) + encoder.gated_ffn_backward(dh, x, wg, wu, gate, up)

    want = step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        for t in got:
            t.zero_()
        g.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert flag() == 0
