"""The encoder's layer operators at the ends of their ranges: the largest sizes, values that are not
finite, steps that follow one another closely.  Bounds: layer_helpers.py."""
import math

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
    want, bound = L.attention64(q, k, v, cu, causal, scale=scale)
    for _ in range(20):
        L.check(encoder.packed_attention(q, k, v, cu, causal=causal, scale=scale), want, bound)
