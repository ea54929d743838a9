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
