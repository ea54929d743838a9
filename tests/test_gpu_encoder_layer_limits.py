"""The encoder's layer operators at the ends of their ranges: the largest sizes, values that are not
finite, steps that follow one another closely.  Bounds: layer_helpers.py."""
import math
import os
import subprocess
import sys

import pytest
import torch

import layer_helpers as L
from ragrt_b200 import _lib, encoder

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def flag():
    torch.cuda.synchronize()
    return _lib.lib().ragrt_device_error(1)


def room_for(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes * 1e9:
        pytest.skip(f"needs {gigabytes} GB")


# ------------------------------------------------------------------------------------ norm + rotary
def test_norm_rope_of_one_token_with_a_million_heads():
    """The heads are dealt out over thousands of warps: heads x warps passes 32 bits."""
    room_for(6)
    H, D, R = 1 << 20, 256, 32
    q, k = (torch.randn(1, H, D, generator=gen(i), device="cuda", dtype=torch.float16) for i in (1, 2))
    w = 1 + 0.2 * torch.randn(D, generator=gen(3), device="cuda").half()
    angle = torch.arange(64, device="cuda")[:, None] * 0.01 * torch.arange(1, R // 2 + 1, device="cuda")
    cos, sin = angle.cos(), angle.sin()
    pos = torch.tensor([37], device="cuda")
    qo, ko = encoder.qk_norm_rope(q, k, cos, sin, pos, w, w)
    n = 1 << 16
    for at in range(0, H, n):
        a, b = encoder.qk_norm_rope(q[:, at:at + n], k[:, at:at + n], cos, sin, pos, w, w)
        assert torch.equal(qo[:, at:at + n], a) and torch.equal(ko[:, at:at + n], b)
    for at in (0, H // 2, H - 1000):
        for x, y in ((q, qo), (k, ko)):
            L.check(y[:, at:at + 1000], *L.rms_rope64(x[:, at:at + 1000], w, cos, sin, pos, 1e-6, False))
    assert flag() == 0


# ------------------------------------------------------------------------------------ attention
def attention64(q, k, v, cu, causal, scale=None):
    """layer_helpers.attention64 with the bound of a divisor that sums the rounded weights: with weights w (1 + d),
    |d| <= e, sum w (1 + d) v / sum w (1 + d) is off from o = sum p v by sum p d (v - o) to first order, which is
    e (sum p |v| + |o|) at most; there it is e sum p |v|, that of the unrounded sum."""
    want, bound = L.attention64(q, k, v, cu, causal, scale)
    return want, bound + 1.02 * L.EPS[q.dtype] * want.abs()


def by_scores(scores, v, D, dtype):
    """q, k, v of one head whose row 0 onwards have score `scores[j]` (in powers of two) for key j."""
    n = scores.shape[0]
    q = torch.zeros(n, 1, D, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    k = torch.zeros(n, 1, D, dtype=dtype, device="cuda")
    k[:, 0, 0] = scores.to(dtype)
    return q, k, v.to(dtype)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_reference_moves_twice_in_a_block(D, causal):
    """The maximum rises by more than 2^8 in both 32-key halves of one block, again and again: the accumulator is
    scaled twice between two products.  Early values are so large that a factor left out shows."""
    n = 320
    j = torch.arange(n, device="cuda")
    scores = (10.0 * (j // 32)).to(torch.bfloat16)          # 2^10 per step: exact
    v = torch.randn(n, 1, D, generator=gen(1), device="cuda") * torch.exp2(-10.0 * (j // 32))[:, None, None]
    q, k, v = by_scores(scores, v, D, torch.bfloat16)
    cu = L.cu_of([n], "cuda")
    scale = math.log(2.0)
    want, bound = attention64(q, k, v, cu, causal, scale=scale)
    for _ in range(20):
        L.check(encoder.packed_attention(q, k, v, cu, causal=causal, scale=scale), want, bound)



@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("T,D", [(700, 64), (700, 128), (2500, 64), (2500, 128), (700, 40)])
def test_attention_what_is_seen_and_not_finite(T, D, causal, dtype):
    """NaN and infinities that rows do see: all of a row whose scores they are in, one column of the rows that see
    them in V.  Nothing else changes."""
    H, KV = 4, 2
    q, k, v = (torch.randn(T, h, D, generator=gen(h + i), device="cuda").to(dtype) for i, h in enumerate((H, KV, KV)))
    cu = L.cu_of([T], "cuda")
    want, bound = attention64(q, k, v, cu, causal)
    seen = lambda row: slice(row if causal else 0, None)
    q[100, 1, 5] = math.nan
    want[100, 1] = math.nan
    v[10, 0, 3], v[20, 0, 3], v[20, 0, 4], v[300, 0, 8] = math.inf, -math.inf, -math.inf, math.nan
    want[seen(10), :2, 3] = math.inf
    want[seen(20), :2, 3] = math.nan
    want[seen(20), :2, 4] = -math.inf
    want[seen(300), :2, 8] = math.nan
    want[100, 1] = math.nan
    k[400, 1, 0] = math.nan
    want[seen(400), 2:] = math.nan
    got = encoder.packed_attention(q, k, v, cu, causal=causal)
    inf = want.isinf()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[inf].double(), want[inf]) and torch.equal(got.isinf(), inf)
    want[inf] = math.nan                                   # looked at
    L.check(got, want, bound)
    assert flag() == 0


@pytest.mark.parametrize("causal", [False, True])
def test_attention_infinity_under_a_weight_that_rounds_to_nothing(causal):
    """A weight far below fp16's smallest times an infinity is an infinity."""
    n = 200
    scores = torch.full((n,), -40.0, device="cuda")
    scores[0] = 0.0
    v = torch.randn(n, 1, 64, generator=gen(4), device="cuda")
    v[50, 0, 2], v[60, 0, 3] = math.inf, -math.inf
    q, k, v = by_scores(scores, v, 64, torch.float16)
    got = encoder.packed_attention(q, k, v, L.cu_of([n], "cuda"), causal=causal, scale=math.log(2.0))
    for col, row, value in ((2, 50, math.inf), (3, 60, -math.inf)):
        sees = slice(row if causal else 0, None)
        assert (got[sees, 0, col] == value).all()
        got[sees, 0, col] = 0
    assert torch.isfinite(got).all()


def test_attention_rows_that_are_not_finite_by_the_formula_are_not_computed_again():
    """They cost a look at V at most (measured: 5 times the time of finite inputs; computed again, 500 times)."""
    T, H, KV, D = 8192, 8, 2, 128
    q, k, v = (torch.randn(T, h, D, generator=gen(h), device="cuda").half() for h in (H, KV, KV))
    cu = L.cu_of([T], "cuda")

    def ms(q, k, v):
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            encoder.packed_attention(q, k, v, cu, causal=True)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    clean = ms(q, k, v)
    for at, what in ((0, slice(None)), (1, 3), (2, 3), (2, slice(T // 2, None))):
        odd = [q, k, v]
        odd[at] = odd[at].clone()
        odd[at][what] = math.nan
        assert ms(*odd) < 25 * clean, (at, what)


def test_attention_many_small_weights_beside_a_large_one():
    """2000 keys whose weights are just under fp16's smallest step relative to the row's largest: each is off by at
    most half that step, as the bound says, so that together they are not lost."""
    n = 2001
    scores = torch.full((n,), -24.03125, device="cuda")
    scores[0] = 0.0078125                                   # 2^-7: both are exact in fp16
    v = torch.ones(n, 1, 64, device="cuda")
    v[0] = 0
    q, k, v = by_scores(scores, v, 64, torch.float16)
    cu, scale = L.cu_of([n], "cuda"), math.log(2.0)
    want, bound = attention64(q, k, v, cu, False, scale=scale)
    L.check(encoder.packed_attention(q, k, v, cu, scale=scale), want, bound)


# ------------------------------------------------------------------------------------ gated feed-forward
@pytest.mark.parametrize("keep", [False, True])
def test_gated_ffn_of_one_row_and_many_columns(keep):
    """More columns than 2^27: a warp per column."""
    room_for(12)
    F, K = (1 << 27) + 64, 8
    x = torch.randn(1, K, generator=gen(1), device="cuda").half()
    part = torch.randn(2, 1 << 20, K, generator=gen(2), device="cuda").half()
    wg, wu = (t.repeat(129, 1)[:F] for t in part)
    h, *kept = (lambda r: r if keep else (r,))(encoder.gated_ffn(x, wg, wu, keep=keep))
    want = encoder.gated_ffn(x, part[0], part[1], keep=keep)
    for got, one in zip((h, *kept), want if keep else (want,)):
        for at in range(0, F, 1 << 20):
            n = min(1 << 20, F - at)
            assert torch.equal(got[0, at:at + n], one[0, :n]), at
    assert flag() == 0


def test_gated_ffn_of_the_longest_sums():
    """2^26 values a sum: as the formula has it and far inside the waits' limit; eight more are refused."""
    room_for(16)
    M, F, K = 8, 8, 1 << 26
    x, w = (torch.zeros(8, K + 8, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = torch.tensor([0, 100, K // 2 + 63, K - 1], device="cuda")
    x[:, at] = torch.randn(M, 4, generator=gen(1), device="cuda").bfloat16()
    w[:, at] = torch.randn(F, 4, generator=gen(2), device="cuda").bfloat16()
    want, _, _, bound, _, _ = L.ffn64(x[:, at], w[:, at], w[:, at], "silu")
    L.check(encoder.gated_ffn(x[:, :K].contiguous(), w[:, :K].contiguous(), w[:, :K].contiguous()), want, bound)
    assert flag() == 0
    with pytest.raises(RuntimeError, match="too long"):
        encoder.gated_ffn(x, w, w)
    dh, kept = torch.zeros(M, K + 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(M, K + 8, device="cuda")
    tall = torch.zeros(K + 8, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="too long"):
        # dx's parts are no more than 16 tiles' worth: without scratch it is one sum
        _lib.check(_lib.lib().ragrt_enc_gated_ffn_backward(
            dh.data_ptr(), x[:, :8].contiguous().data_ptr(), tall.data_ptr(), tall.data_ptr(), kept.data_ptr(),
            kept.data_ptr(), dh.data_ptr(), dh.data_ptr(), torch.zeros_like(x[:, :8]).data_ptr(), None, None, M, K + 8,
            8, 0, 1, None, 0, torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("rows", [1, 4, 40])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_ffn_of_huge_and_infinite_values(act, rows):
    """Pre-activations up to 1e30, whose cubes are beyond fp32, and infinite ones: what the 64-bit formula has."""
    K, F = 64, 128
    values = torch.tensor([1e20, -1e20, 1e30, -1e30, math.inf, -math.inf, math.nan, 3.0], device="cuda")
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, 1] = 1.0, 1.0
    wg = torch.zeros(F, K, dtype=torch.bfloat16, device="cuda")
    wg[:, 0] = values.repeat(F // 8)
    wu = torch.zeros(F, K, dtype=torch.bfloat16, device="cuda")
    wu[:, 1] = 0.5
    h, gate, up = encoder.gated_ffn(x, wg, wu, act=act, keep=True)
    g = wg[:, 0].double()
    a, d = L.act64(g, act)
    room = 1.02 * L.EPS[torch.bfloat16]
    for got, want in ((gate, g), (h, 0.5 * a)):
        want = want.expand(rows, F)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        ok = want.isfinite()
        assert ((got.double() - want)[ok].abs() <= room * want[ok].abs()).all()
        assert torch.equal(got[want.isinf()].double(), want[want.isinf()])
    # gradients of the finite columns, the others out of them
    fine = g.isfinite()
    w1, w2 = wg.clone(), wu.clone()
    w1[~fine], gate[:, ~fine], up[:, ~fine] = 0, 0, 0
    dh = torch.ones(rows, F, dtype=torch.bfloat16, device="cuda")
    dh[:, ~fine] = 0
    dx, dwg, dwu = encoder.gated_ffn_backward(dh, x, w1, w2, gate, up, act=act)
    for got, (want, bound), what in zip((dwg, dwu), L.ffn_backward64(dh, x, w1, w2, gate, up, act)[1:], ("dwg", "dwu")):
        assert torch.isfinite(got).all()
        L.check(got, want, bound, what)


# ------------------------------------------------------------------------------------ captured first calls
FIRST = """
import sys
import torch
sys.path.insert(0, {repo!r})
from ragrt_b200 import encoder
q = torch.randn(70, 2, 64, device="cuda").half()
cu = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
cos = torch.rand(80, 32, device="cuda")
pos = torch.arange(70, device="cuda")
x, w = torch.randn(70, 64, device="cuda").half(), torch.randn(136, 64, device="cuda").half()
dh, kept = torch.randn(70, 136, device="cuda").half(), torch.randn(70, 136, device="cuda")
calls = dict(attention=lambda: encoder.packed_attention(q, q, q, cu), rope=lambda: encoder.qk_norm_rope(q, q, cos, cos, pos),
             ffn=lambda: encoder.gated_ffn(x, w, w), backward=lambda: encoder.gated_ffn_backward(dh, x, w, w, kept, kept))
call = calls[{name!r}]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
graph.replay()
want = call()
torch.cuda.synchronize()
as_tuple = lambda r: r if isinstance(r, tuple) else (r,)
assert all(torch.equal(a, b) for a, b in zip(as_tuple(got), as_tuple(want)))
print("equal")
"""


@pytest.mark.parametrize("name", ["attention", "rope", "ffn", "backward"])
def test_first_call_of_a_process_in_a_graph(name):
    """Nothing has to be called once outside of a capture first."""
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST.format(repo=repo, name=name)], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-3000:]


# ------------------------------------------------------------------------------------ the host's two ways
def test_operators_with_and_without_the_host_binding(monkeypatch):
    q, k, v = (torch.randn(90, h, 64, generator=gen(h), device="cuda").half() for h in (4, 2, 2))
    cu = L.cu_of([33, 57], "cuda")
    cos = torch.rand(90, 32, generator=gen(5), device="cuda")
    x, w = torch.randn(90, 64, generator=gen(6), device="cuda").half(), torch.randn(272, 64, generator=gen(7), device="cuda").half()
    dh = torch.randn(90, 136, generator=gen(8), device="cuda").half()

    def all_of_them():
        h, gate, up = encoder.gated_ffn(x, w[:136], w[136:], act="gelu", keep=True)
        return (encoder.packed_attention(q, k, v, cu, causal=True), *encoder.qk_norm_rope(q, k, cos, cos, torch.arange(90, device="cuda")),
                h, gate, up, *encoder.gated_ffn_backward(dh, x, w[:136], w[136:], gate, up, act="gelu"))

    want = all_of_them()
    assert encoder._bound is not encoder._NoBinding
    monkeypatch.setattr(encoder, "_bound", encoder._NoBinding)
    for a, b in zip(all_of_them(), want):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------ one launch for all gradients
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,F,K", [(3000, 2600, 1000), (6000, 1400, 1000), (5000, 2600, 1496), (9000, 2712, 776)])
def test_gated_ffn_gradients_of_several_rounds_of_pairs(M, F, K, dtype):
    """Tiles of dx and of the weight gradients in one list of large tiles, more than a round of the 74 pairs, the last
    round in part: 48 + 88, 96 + 48, 120 + 132 and 144 + 88 tiles, the border in the first round or the second."""
    x = torch.randn(M, K, generator=gen(M), device="cuda").to(dtype)
    w = (torch.randn(2 * F, K, generator=gen(F), device="cuda") * 1.5 / math.sqrt(K)).to(dtype)
    dh = torch.randn(M, F, generator=gen(K), device="cuda").to(dtype)
    assert _lib.lib().ragrt_enc_gated_ffn_workspace(M, F, K, 1, 1) == 0             # nothing in parts
    _, gate, up = encoder.gated_ffn(x, w[:F], w[F:], keep=True)
    grads = encoder.gated_ffn_backward(dh, x, w[:F], w[F:], gate, up)
    for got, (want, bound), what in zip(grads, L.ffn_backward64(dh, x, w[:F], w[F:], gate, up, "silu"), ("dx", "dwg", "dwu")):
        L.check(got, want, bound, what)
    for a, b in zip(grads, encoder.gated_ffn_backward(dh, x, w[:F], w[F:], gate, up)):
        assert torch.equal(a, b)
    assert flag() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D", [(900, 64), (900, 128), (2600, 64), (2600, 128), (900, 40), (900, 104), (2600, 24)])
def test_attention_rows_before_values_that_are_not_finite(T, D, dtype):
    """Causal, NaN and infinities in V within tiles, in other columns each: the rows before them in the tile are
    those of finite values."""
    H, KV = 4, 2
    q, k, v = (torch.randn(T, h, D, generator=gen(h + i), device="cuda").to(dtype) for i, h in enumerate((H, KV, KV)))
    cu = L.cu_of([T - 7], "cuda")
    want, bound = attention64(q, k, v, cu, True)
    for i, at in enumerate((37, 38, 200, 301, 511, 640, 700, T - 9)):
        v[at, 1, i], v[at, 1, i + 8] = math.nan, math.inf
        want[at:T - 7, 2:, i], want[at:T - 7, 2:, i + 8] = math.nan, math.inf
    v[T - 7:] = math.nan
    out = torch.zeros_like(q)
    encoder.packed_attention(q, k, v, cu, causal=True, out=out)
    seen = slice(0, T - 7)
    inf = want[seen].isinf()
    assert torch.equal(out[seen].isnan(), want[seen].isnan()) and torch.equal(out[seen].isinf(), inf)
    assert (out[seen][inf] == math.inf).all() and (out[T - 7:] == 0).all()
    want[want.isinf()] = math.nan                          # looked at
    L.check(out, want, bound)
    assert flag() == 0


def test_attention_rows_computed_again_share_their_loads():
    """The rows before a NaN in its tile, one after the other and load by load, took 200 times the clean call's time;
    measured now: 30."""
    T, H, KV, D = 8192, 8, 2, 128
    q, k, v = (torch.randn(T, h, D, generator=gen(h), device="cuda").half() for h in (H, KV, KV))
    cu = L.cu_of([T], "cuda")

    def ms(v):
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            encoder.packed_attention(q, k, v, cu, causal=True)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    odd = v.clone()
    odd[4180] = math.nan
    assert ms(odd) < 90 * ms(v)


THREADS = """
import sys, threading
import torch
sys.path.insert(0, {repo!r})
from ragrt_b200 import _lib, encoder
if {python}:
    encoder._bound = encoder._NoBinding                   # ctypes lets go of the interpreter during a call
cu = torch.tensor([0, 30, 700], dtype=torch.int32, device="cuda")
cos = torch.rand(700, 32, device="cuda")
pos = torch.arange(700, device="cuda")
sets = []
for i in range(8):
    g = torch.Generator(device="cuda").manual_seed(i)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
    sets.append((n(700, 4, 64), n(700, 2, 64), n(700, 2, 64), n(700, 128), n(272, 128), n(700, 136)))


def work(q, k, v, x, w, dh):
    a, b = encoder.qk_norm_rope(q, k, cos, cos, pos)
    h, gate, up = encoder.gated_ffn(x, w[:136], w[136:], keep=True)
    return (a, b, encoder.packed_attention(a, b, v, cu, causal=True), h,
            *encoder.gated_ffn_backward(dh, x, w[:136], w[136:], gate, up))


torch.cuda.synchronize()
start, got = threading.Barrier(8), [None] * 8


def run(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        for _ in range(20):
            got[i] = work(*sets[i])
        torch.cuda.current_stream().synchronize()


threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
for s, r in zip(sets, got):
    assert all(torch.equal(a, b) for a, b in zip(work(*s), r))
torch.cuda.synchronize()
assert _lib.lib().ragrt_device_error(0) == 0
print("equal")
"""


@pytest.mark.parametrize("python", [False, True], ids=["binding", "ctypes"])
def test_threads_that_all_make_their_first_calls_at_once(python):
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", THREADS.format(repo=repo, python=python)], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-3000:]
