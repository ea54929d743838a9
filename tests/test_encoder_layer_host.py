"""Refusals of the encoder's layer operators, without a GPU: the C entry points check their arguments
before any CUDA call, the Python entry points every tensor, and outputs apart from inputs."""
import math
import random
import sys
import warnings

import pytest
import torch

import ragrt_b200
from ragrt_b200 import _lib, encoder

P = 0x1000                                              # 16-byte aligned, never touched


def attn(q=P, k=P, v=P, cu=P, out=P, T=8, B=1, H=4, KV=2, D=64, qs=256, ks=128, vs=128, os=256, scale=0.125, causal=0,
         dt=0):
    return _lib.lib().ragrt_enc_packed_attention(q, k, v, cu, out, T, B, H, KV, D, qs, ks, vs, os, scale, causal, dt,
                                                 None)


@pytest.mark.parametrize("kw,what", [
    (dict(dt=2), b"dtype"), (dict(T=-1), b">= 0"), (dict(B=-1), b">= 0"), (dict(H=3), b"multiple of kv_heads"),
    (dict(KV=0), b"kv_heads"), (dict(D=132), b"head_dim"), (dict(D=4), b"head_dim"), (dict(D=60), b"head_dim"),
    (dict(D=0), b"head_dim"), (dict(qs=248), b"strides"), (dict(ks=120), b"strides"), (dict(vs=132), b"strides"),
    (dict(os=-256), b"strides"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(q=None), b"null"), (dict(cu=None), b"null"), (dict(out=None), b"null"),
    (dict(k=P + 8), b"aligned"), (dict(cu=P + 2), b"aligned")])
def test_attention_refusals(kw, what):
    assert attn(**kw) == -1
    assert what in _lib.lib().ragrt_last_error()


def test_nothing_to_do_is_no_error():
    assert attn(T=0, q=None, k=None, v=None, out=None) == 0
    assert attn(B=0, cu=None) == 0
    assert _lib.lib().ragrt_enc_gated_ffn(None, None, None, None, None, None, 0, 128, 64, 0, 0, None) == 0


def rope(q=P, k=P, qw=P, kw=P, cos=P, sin=P, pos=P, pb=8, qo=P, ko=P, T=8, H=4, KV=2, D=64, R=64, n=128, qs=256, ks=128,
         qos=256, kos=128, eps=1e-6, inter=0, dt=0):
    return _lib.lib().ragrt_enc_qk_norm_rope(q, k, qw, kw, cos, sin, pos, pb, qo, ko, T, H, KV, D, R, n, qs, ks, qos,
                                             kos, eps, inter, dt, None)


@pytest.mark.parametrize("kw,what", [
    (dict(dt=-1), b"dtype"), (dict(T=-1), b"T >= 0"), (dict(H=0), b"heads"), (dict(KV=-1), b"heads"),
    (dict(D=264, R=16, qs=4096, ks=4096, qos=4096, kos=4096), b"head_dim"), (dict(D=20, R=16), b"head_dim"),
    (dict(D=8, R=8), b"head_dim"), (dict(R=24), b"rot_dim"), (dict(R=0), b"rot_dim"), (dict(R=80), b"rot_dim"),
    (dict(n=0), b"max_pos"), (dict(pb=2), b"positions"), (dict(qs=200), b"strides"), (dict(kos=132), b"strides"),
    (dict(cos=None), b"null"), (dict(pos=None), b"null"), (dict(k=None), b"null"), (dict(qw=P + 2), b"aligned"),
    (dict(pos=P + 4), b"aligned"), (dict(ko=P + 8), b"aligned")])
def test_norm_rope_refusals(kw, what):
    assert rope(**kw) == -1
    assert what in _lib.lib().ragrt_last_error()


def test_gated_ffn_refusals():
    f, b = _lib.lib().ragrt_enc_gated_ffn, _lib.lib().ragrt_enc_gated_ffn_backward
    last = _lib.lib().ragrt_last_error
    for args, what in [((P, P, P, P, None, None, 4, 60, 64, 0, 0, None), b"multiples of 8"),
                       ((P, P, P, P, None, None, 4, 64, 4, 0, 0, None), b"multiples of 8"),
                       ((P, P, P, P, None, None, -1, 64, 64, 0, 0, None), b"multiples of 8"),
                       ((P, P, P, P, None, None, 4, 64, 64, 3, 0, None), b"activation"),
                       ((P, P, P, P, None, None, 4, 64, 64, 0, 5, None), b"dtype"),
                       ((P, P, P, P, P, None, 4, 64, 64, 0, 0, None), b"together"),
                       ((P, None, P, P, None, None, 4, 64, 64, 0, 0, None), b"null"),
                       ((P, P + 2, P, P, None, None, 4, 64, 64, 0, 0, None), b"aligned")]:
        assert f(*args) == -1 and what in last(), what
    for args, what in [((P,) * 11 + (4, 60, 64, 0, 0, None, 0, None), b"multiples of 8"),
                       ((P,) * 10 + (None, 4, 64, 64, 0, 0, None, 0, None), b"together"),
                       ((None,) + (P,) * 10 + (4, 64, 64, 0, 0, None, 0, None), b"null"),
                       ((P, None) + (P,) * 9 + (4, 64, 64, 0, 0, None, 0, None), b"need x"),
                       ((P, P, None) + (P,) * 8 + (4, 64, 64, 0, 0, None, 0, None), b"needs the weights"),
                       ((P + 8,) + (P,) * 10 + (4, 64, 64, 0, 0, None, 0, None), b"aligned"),
                       ((P,) * 11 + (4, 64, 64, 0, 0, P + 4, 64, None), b"aligned")]:
        assert b(*args) == -1 and what in last(), what


@pytest.fixture
def on_host(monkeypatch):
    """The Python checks alone: tensors stay on the host and no library call is made."""
    monkeypatch.setattr(encoder, "_need_cuda", lambda *ts: None)

    class Stop:
        def __getattr__(self, name):
            raise AssertionError("reached the library")

    monkeypatch.setattr(_lib, "lib", lambda: Stop())


H16 = torch.float16


def test_host_tensors_are_refused():
    q = torch.zeros(4, 2, 64, dtype=H16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    t = torch.zeros(8, 32)
    x, w = torch.zeros(4, 64, dtype=H16), torch.zeros(128, 64, dtype=H16)
    h = torch.zeros(4, 128, dtype=H16)
    for call in (lambda: encoder.packed_attention(q, q, q, cu),
                 lambda: encoder.qk_norm_rope(q, q, t, t, torch.arange(4)),
                 lambda: encoder.gated_ffn(x, w, w), lambda: encoder.gated_ffn_backward(h, x, w, w, h, h)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_python_checks_of_attention(on_host):
    q, k = torch.zeros(8, 4, 64, dtype=H16), torch.zeros(8, 2, 64, dtype=H16)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    for args, what in [((q.float(), k.float(), k.float(), cu), "fp16"), ((q, k, k.bfloat16(), cu), "fp16"),
                       ((q[0], k, k, cu), "wanted"), ((q, k[:7], k[:7], cu), "wanted"), ((q, k, k[:, :1], cu), "wanted"),
                       ((q, k[..., :32], k[..., :32], cu), "wanted"), ((q, k, k, cu[None]), "cu_seqlens"),
                       ((q, k, k, cu[:0]), "cu_seqlens"), ((q, k, k, cu.float()), "cu_seqlens")]:
        with pytest.raises(RuntimeError, match=what):
            encoder.packed_attention(*args)
    for out, what in [(q, "overlaps"), (torch.zeros(8, 4, 32, dtype=H16), "out must be"),
                      (torch.zeros(8, 4, 64, dtype=torch.bfloat16), "out must be"),
                      (torch.zeros(8, 64, 4, dtype=H16).transpose(1, 2), "in place"),
                      (torch.zeros(8 * 256 + 1, dtype=H16)[1:].view(8, 4, 64), "in place")]:
        with pytest.raises(RuntimeError, match=what):
            encoder.packed_attention(q, k, k, cu, out=out)


def test_overlap_of_column_blocks_and_shifted_rows(on_host):
    m = torch.zeros(9, 512, dtype=H16)
    block = lambda r, c, n: m[r:r + 8, c:c + n].view(8, n // 64, 64)
    assert not encoder._overlap(block(0, 0, 256), block(0, 256, 128))
    assert not encoder._overlap(block(0, 384, 128), block(1, 0, 256))
    assert encoder._overlap(block(0, 0, 256), block(0, 192, 128))
    assert encoder._overlap(block(0, 0, 256), block(1, 0, 256))
    assert encoder._overlap(block(0, 256, 128), m.view(18, 256)[:8].view(8, 4, 64))
    assert not encoder._overlap(m[:4], m[4:8]) and not encoder._overlap(m[:0], m)
    assert not encoder._overlap(m[:1, :64], m[:1, 64:])
    cos = torch.zeros(4, 32)
    pos = torch.zeros(8, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="overlaps"):
        encoder.qk_norm_rope(block(0, 0, 256), block(0, 256, 128), cos, cos, pos, q_out=block(1, 0, 256))
    with pytest.raises(RuntimeError, match="overlaps"):
        encoder.qk_norm_rope(block(0, 0, 256), block(0, 256, 128), cos, cos, pos, k_out=block(0, 128, 128))


def test_one_tensor_as_query_and_key_in_place(on_host):
    """Neither may be written over the other, nor the two outputs over one another."""
    q, other = torch.zeros(8, 4, 64, dtype=H16), torch.zeros(8, 4, 64, dtype=H16)
    cos, pos = torch.zeros(4, 32), torch.zeros(8, dtype=torch.int64)
    for outs in (dict(q_out=q), dict(k_out=q), dict(q_out=q, k_out=q), dict(q_out=other, k_out=other)):
        with pytest.raises(RuntimeError, match="overlaps"):
            encoder.qk_norm_rope(q, q, cos, cos, pos, **outs)


def test_python_checks_of_norm_rope(on_host):
    q, k = torch.zeros(8, 4, 64, dtype=H16), torch.zeros(8, 2, 64, dtype=H16)
    cos = torch.zeros(16, 32)
    pos = torch.zeros(8, dtype=torch.int64)
    w = torch.zeros(64, dtype=H16)
    for args, what in [((q, k, cos, cos[:, :16], pos), "cos and sin"), ((q, k, cos.double(), cos.double(), pos), "cos and sin"),
                       ((q, k, cos, cos, pos[:7]), "positions"), ((q, k, cos, cos, pos.float()), "positions"),
                       ((q, k, cos, cos, pos, w[:32]), "norm weight"), ((q, k, cos, cos, pos, w.float()), "fp16"),
                       ((q, k[:7], cos, cos, pos), "wanted"), ((q, k.bfloat16(), cos, cos, pos), "fp16")]:
        with pytest.raises(RuntimeError, match=what):
            encoder.qk_norm_rope(*args)


def test_python_checks_of_gated_ffn(on_host):
    x, w = torch.zeros(4, 64, dtype=H16), torch.zeros(128, 64, dtype=H16)
    h = torch.zeros(4, 128, dtype=H16)
    with pytest.raises(RuntimeError, match="activation"):
        encoder.gated_ffn(x, w, w, act="relu")
    for args in [(x, w, w[:64]), (x[:, :32], w, w), (x[0], w, w)]:
        with pytest.raises(RuntimeError, match="wanted"):
            encoder.gated_ffn(*args)
    with pytest.raises(RuntimeError, match="fp16"):
        encoder.gated_ffn(x, w.bfloat16(), w)
    with pytest.raises(RuntimeError, match="out must be"):
        encoder.gated_ffn(x, w, w, out=h[:3])
    kept = h.float()
    with pytest.raises(RuntimeError, match="must be"):
        encoder.gated_ffn_backward(h[:, :64], x, w, w, kept, kept)
    with pytest.raises(RuntimeError, match="fp32"):
        encoder.gated_ffn_backward(h, x, w, w, h, h)
    square = torch.zeros(128, 64, dtype=H16)
    with pytest.raises(RuntimeError, match="overlaps"):
        encoder.gated_ffn(square, torch.zeros(64, 64, dtype=H16), torch.zeros(64, 64, dtype=H16), out=square)


def test_gated_ffn_sizes_past_32_bits_are_refused():
    big = 0x7FFFFFF8
    f, b = _lib.lib().ragrt_enc_gated_ffn, _lib.lib().ragrt_enc_gated_ffn_backward
    for M, F, K in ((big, 64, 64), (4, big, 64), (4, 64, big)):
        assert f(P, P, P, P, None, None, M, F, K, 0, 0, None) == -1
        assert b"2^31" in _lib.lib().ragrt_last_error()
        assert b(*(P,) * 11, M, F, K, 0, 0, None, 0, None) == -1
        assert b"2^31" in _lib.lib().ragrt_last_error()


def test_binding_is_built_and_loads():
    from ragrt_b200 import _enc_bind
    assert encoder._bind() is _enc_bind


def test_without_the_binding_calls_take_the_way_through_python(monkeypatch):
    """A missing binding is said once; refusals stay what they are."""
    monkeypatch.setattr(encoder, "_bound", None)
    monkeypatch.setitem(sys.modules, "ragrt_b200._enc_bind", None)
    monkeypatch.delattr(ragrt_b200, "_enc_bind", raising=False)
    q, cu = torch.zeros(4, 2, 64, dtype=H16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.warns(RuntimeWarning, match="without their host binding"):
        with pytest.raises(RuntimeError, match="CUDA"):
            encoder.packed_attention(q, q, q, cu)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(RuntimeError, match="CUDA"):
            encoder.gated_ffn(torch.zeros(4, 64, dtype=H16), q[:, 0], q[:, 1])
    x, w, h = torch.zeros(4, 64, dtype=H16), torch.zeros(128, 64, dtype=H16), torch.zeros(4, 128, dtype=H16)
    cos = torch.zeros(4, 32)
    monkeypatch.setattr(encoder, "_need_cuda", lambda *ts: None)
    reached = []

    class Library:
        def __getattr__(self, name):
            reached.append(name)
            return lambda *args: 0

    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(encoder, "_raw_stream", lambda t: 0)
    assert encoder.packed_attention(q, q, q, cu).shape == q.shape
    assert encoder.qk_norm_rope(q, q, cos, cos, torch.arange(4))[1].shape == q.shape
    assert len(encoder.gated_ffn(x, w, w, keep=True)) == 3
    assert encoder.gated_ffn_backward(h, x, w, w, h.float(), h.float())[2].shape == w.shape
    assert reached == ["ragrt_enc_packed_attention", "ragrt_enc_qk_norm_rope", "ragrt_enc_gated_ffn",
                       "ragrt_enc_gated_ffn_workspace", "ragrt_enc_gated_ffn_backward"]


def test_gated_ffn_workspace_is_bounded():
    """Three parts of 64 KiB per SM at most, whatever the sizes; the bound is nearly reached."""
    rng = random.Random(5)
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    size = lambda high: min(high, int(math.exp(rng.uniform(math.log(8), math.log(high + 1)))))
    ws, most = _lib.lib().ragrt_enc_gated_ffn_workspace, 0
    for _ in range(30000):
        M, F, K = size(1 << 20), size(1 << 15) // 8 * 8, size(1 << 14) // 8 * 8
        for dx, dw in ((1, 0), (0, 1), (1, 1)):
            n = ws(M, F, K, dx, dw)
            assert 0 <= n <= 3 * sms * 65536 and n % 16 == 0, (M, F, K, dx, dw, n)
            most = max(most, n)
    assert most > 1.8 * sms * 65536
    assert ws(0, 64, 64, 1, 1) == 0 and ws(100, 64, 64, 0, 0) == 0
