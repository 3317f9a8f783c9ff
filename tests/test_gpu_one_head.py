"""Tensors of one head whose head axis has any stride ([1, T, D] transposed): the rotary append and the
8-bit attention take them as they are."""

from __future__ import annotations

import pytest
import torch

from plastic_infer_b200 import kernels
from tests._q8 import DEV, E4M3, cache, on_gpu

pytestmark = pytest.mark.gpu


def one_head(T, D, g, dtype=torch.bfloat16):
    x = torch.randn((1, T, D), device=DEV, generator=g).to(dtype)
    return x.transpose(0, 1)  # [T, 1, D], head stride T * D


@pytest.mark.parametrize("eight", [False, True])
def test_append(eight):
    T, D, S = 21, 64, 16
    g = torch.Generator(device=DEV).manual_seed(0)
    q, k, v = (one_head(T, D, g) for _ in range(3))
    pools = [torch.zeros((2, 1, S, D), device=DEV).to(E4M3 if eight else torch.bfloat16) for _ in range(4)]
    sc = [torch.ones((2, 1), device=DEV) for _ in range(4)]
    pos = torch.arange(T, device=DEV)
    inv = kernels.rope_inv_freq(D, 1e4, DEV)
    out = one_head(T, D, g)
    kw = [dict(k_scale=sc[i], v_scale=sc[i + 1]) if eight else {} for i in (0, 2)]
    got = kernels.rope_append(q, k, v, pos, inv, pos, pools[0], pools[1], q_out=out, **kw[0])
    want = kernels.rope_append(q.clone(memory_format=torch.contiguous_format), k.clone(memory_format=torch.contiguous_format),
                               v.clone(memory_format=torch.contiguous_format), pos, inv, pos, pools[2], pools[3], **kw[1])
    assert got is out and torch.equal(got, want)
    for i in (0, 1):
        assert torch.equal(pools[i].view(torch.uint8), pools[i + 2].view(torch.uint8))
        assert torch.equal(sc[i], sc[i + 2])


def test_attention():
    D, S, n = 64, 16, 50
    c = on_gpu(cache([n, 33], 1, D, S, seed=1))
    g = torch.Generator(device=DEV).manual_seed(1)
    pools = (c["k_pool"], c["v_pool"], c["k_scale"], c["v_scale"])
    q, out = one_head(2, D, g), one_head(2, D, g)
    assert kernels.paged_decode_attention_q8(q, *pools, c["tables"], c["lens"], out=out) is out
    assert torch.equal(out, kernels.paged_decode_attention_q8(q.contiguous(), *pools, c["tables"], c["lens"]))
    q, out = one_head(9, D, g), one_head(9, D, g)
    assert kernels.paged_prefill_attention_q8(q, *pools, c["tables"][0], n, n - 9, out=out) is out
    assert torch.equal(out, kernels.paged_prefill_attention_q8(q.contiguous(), *pools, c["tables"][0], n, n - 9))
