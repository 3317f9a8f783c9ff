"""The rotary append at sizes whose offsets pass 32 bits."""

from __future__ import annotations

import pytest
import torch

from plastic_infer_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("shift", [0, 1], ids=["vector", "generic"])
def test_page_of_more_than_32_bits(shift):
    """One page of 2^20 tokens of 18 heads of 128: head 16 begins 2^31 elements into it."""
    H, S, D, T = 18, 1 << 20, 128, 3
    kp, vp = (torch.zeros((1, H, S, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    assert (H - 1) * S * D > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(3)
    buf = torch.randn(3 * T * H * D + 8, device=DEV, generator=g).bfloat16()[shift:]  # (one off: the generic kernel)
    q, k, v = (buf[i * T * H * D:(i + 1) * T * H * D].view(T, H, D) for i in range(3))
    slots = torch.tensor([0, S - 1, 12345], device=DEV)
    kernels.rope_append(q, k, v, torch.zeros(T, dtype=torch.int64, device=DEV), torch.zeros(0, device=DEV), slots, kp, vp)
    for pool, x in ((kp, k), (vp, v)):
        assert torch.equal(pool[0][:, slots].transpose(0, 1), x)
        pool[0][:, slots] = 0
        assert not any(bool(pool[0, h].any()) for h in range(H))  # nothing else written
    del kp, vp


def test_many_heads():
    """One token's heads are shared out to up to 2048 groups: heads times groups passes 32 bits."""
    Hq, Hkv, D, S = 1_200_000, 1_200_000, 64, 16
    g = torch.Generator(device=DEV).manual_seed(4)
    q = torch.randn((1, Hq, D), device=DEV, generator=g).bfloat16()
    k, v = (torch.randn((1, Hkv, D), device=DEV, generator=g).bfloat16() for _ in range(2))
    kp, vp = (torch.zeros((1, Hkv, S, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    out = kernels.rope_append(q, k, v, torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros(0, device=DEV),
                              torch.tensor([7], device=DEV), kp, vp)
    assert torch.equal(out, q) and torch.equal(kp[0, :, 7], k[0]) and torch.equal(vp[0, :, 7], v[0])
