"""The rotary append's QK-norm where the root mean square overflows fp32 or a row holds an infinity,
on the vector kernel (head sizes of 64, 128) and the generic one (72), into every kind of pool.

The norm's arithmetic is fp32: sqrt(mean(x^2) + eps) is infinite for such a row, every finite
element over it is 0 and an infinity over it is NaN. So the expected values are exact.
"""

from __future__ import annotations

import math

import pytest
import torch

from plastic_infer_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
E4M3 = torch.float8_e4m3fn


def rows(T, H, D, dtype):
    """Row (0, 0) holds an infinity, row (1, 0) is finite with squares past fp32 (where the type
    has such values), the others are ordinary."""
    g = torch.Generator().manual_seed(D)
    x = torch.randn((T, H, D), generator=g)
    x[0, 0, 5] = math.inf
    if dtype != torch.float16:
        x[1, 0] = 1e25 * x[1, 0].sign()
    return x.to(dtype)


@pytest.mark.parametrize("pool", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("D", [64, 128, 72])
def test_rows_whose_root_overflows(D, dtype, pool):
    T, S = 4, 16
    q, k, v = rows(T, 4, D, dtype), rows(T, 2, D, dtype), rows(T, 2, D, dtype)
    w = torch.full((D,), 2.0, dtype=dtype)
    eight = pool == "e4m3"
    kp, vp = (torch.zeros((2, 2, S, D), device=DEV).to(E4M3 if eight else dtype) for _ in range(2))
    scales = [torch.ones((2, 2), device=DEV) for _ in range(2)] if eight else [None, None]
    pos = torch.zeros(T, dtype=torch.int64, device=DEV)  # no turn: rows are the normed rows
    inv = torch.ones(D // 2, device=DEV)
    out = kernels.rope_append(q.to(DEV), k.to(DEV), v.to(DEV), pos, inv, torch.arange(T, device=DEV), kp, vp,
                              w.to(DEV), w.to(DEV), k_scale=scales[0], v_scale=scales[1]).cpu().float()
    kept = kp[0].float().cpu().transpose(0, 1)[:T]  # [T, 2, D]
    if eight:
        kept = kept * scales[0][0].cpu()[None, :, None]
    for got, x in ((out, q), (kept, k)):
        got, x = got.clone(), x.double()
        # the pair of the infinity: NaN * cos - 0 * sin and so on are NaN in both its elements
        other = 5 + D // 2
        assert got[0, 0, 5].isnan() and got[0, 0, other].isnan()
        got[0, 0, 5] = got[0, 0, other] = 0
        assert int(got[0, 0].count_nonzero()) == 0, got[0, 0]
        if dtype != torch.float16:
            assert int(got[1, 0].count_nonzero()) == 0 and got[1, 0].isfinite().all(), got[1, 0]
        # rows beside them are what they are without them
        want = x / (x.square().mean(-1, keepdim=True) + 1e-5).sqrt() * 2
        step = 2.0 ** -4 if eight and got is not out else torch.finfo(dtype).eps / 2
        for t, h in [(0, 1), (1, 1), (2, 0), (3, 1)]:
            size = want[t, h].abs()
            floor = (size.max() * 2.0 ** -17) if eight else torch.finfo(dtype).tiny
            # half a step of the type, and 16 fp32 half-steps for the norm's arithmetic
            assert ((got[t, h] - want[t, h]).abs() <= (step + 2.0 ** -20) * size.clamp(min=float(floor))).all()


@pytest.mark.parametrize("D", [64, 128])
def test_vector_and_generic_kernels_round_alike(D):
    """The same rows, once aligned and once one element off (the generic kernel). What is left
    between them is the order of the sum of squares: 7 of 8 additions at most on the way of an
    element here and D / 16 + 3 there, so the root is equal to 2^-24 * 8 relative, and a value
    rounded to e4m3 differs only where it lies that close to a border: by one step then."""
    T, S, H = 256, 16, 2
    g = torch.Generator().manual_seed(7)
    x = torch.randn((T, 3 * H * D + 8), generator=g)
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(DEV)
    got = []
    for shift in (0, 1):
        buf = torch.zeros(T * x.shape[1] + 8, device=DEV)[shift:shift + x.numel()].view(T, -1)
        buf.copy_(x)
        q, k, v = (buf[:, i * H * D:(i + 1) * H * D].view(T, H, D) for i in range(3))
        kp, vp = (torch.zeros((T // S, H, S, D), device=DEV).to(E4M3) for _ in range(2))
        ks, vs = (torch.ones((T // S, H), device=DEV) for _ in range(2))
        kernels.rope_append(q, k, v, torch.arange(T, device=DEV), kernels.rope_inv_freq(D, 1e4, DEV),
                            torch.arange(T, device=DEV), kp, vp, w, w, k_scale=ks, v_scale=vs)
        got.append((kp.float(), ks, vp.float(), vs))
    (ka, ksa, va, vsa), (kb, ksb, vb, vsb) = got
    assert torch.equal(va, vb) and torch.equal(vsa, vsb) and torch.equal(ksa, ksb)
    diff = (ka - kb).abs()
    assert (diff <= 2.0 ** -3 * torch.maximum(ka.abs(), kb.abs()).clamp(min=2.0 ** -6)).all()
    # a step is 2^-3 relative at most and a value lies within 2^-20 of a border with probability
    # 2^-17: of 65536 values (D = 128) half of one is expected
    assert int((diff > 0).sum()) <= 16
