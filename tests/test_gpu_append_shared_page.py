"""Rotary append into 8-bit pools where several runs of one call name the same page: that page and its
scales stay as they were, `err` says so, and q and every other page are what they are without them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import quant_kv_oracle as orc
from plastic_infer_b200 import _capi, kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
E4M3 = torch.float8_e4m3fn


def np64(t):
    return t.detach().cpu().float().double().numpy()


def call(slots, D, S, P, Hkv=2, Hq=4, seed=0):
    T = len(slots)
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn((T, h, D), generator=g).bfloat16().to(DEV) for h in (Hq, Hkv, Hkv))
    kp, vp = ((torch.randn((P, Hkv, S, D), generator=g) * 50).to(E4M3).to(DEV) for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-8, -4, (P, Hkv), generator=g).float()).to(DEV) for _ in range(2))
    before = [x.clone() for x in (kp, vp, ks, vs)]
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = kernels.rope_append(q, k, v, torch.zeros(T, dtype=torch.int64, device=DEV), torch.zeros(0, device=DEV),
                              torch.tensor(slots, device=DEV), kp, vp, k_scale=ks, v_scale=vs, err=err)
    return q, k, v, out, before, (kp, vp, ks, vs), int(err.item())


def expect(slots, S, k, before, pool, scale):
    """The oracle's pool and scales over the tokens whose page one run names alone."""
    names = {}
    for t, page, off, n in orc.runs(slots, S):
        names.setdefault(page, []).append((t, n))
    alone = [-1] * len(slots)
    for runs in names.values():
        if len(runs) == 1:
            t, n = runs[0]
            alone[t:t + n] = slots[t:t + n]
    ref, sc = np64(before[pool]), np64(before[scale])
    orc.append_q8(np64(k), alone, ref, sc)
    return ref, sc, [page for page, runs in names.items() if len(runs) > 1]


@pytest.mark.parametrize("D,S", [(128, 16), (64, 32), (80, 16), (128, 8)])
@pytest.mark.parametrize("kind", ["gap", "padding", "order", "twice", "far apart", "none"])
def test_a_page_of_several_runs(kind, D, S):
    P = 1700
    base = [5 * S + i for i in range(6)] + [9 * S + S - 2, 9 * S + S - 1, 11 * S, 11 * S + 1]
    slots = {
        "gap": base + [3 * S + 1, 3 * S + 4],
        "padding": base + [3 * S + 1, -1, 3 * S + 2],
        "order": base + [3 * S + 2, 3 * S + 1],
        "twice": base + [3 * S + 7, 3 * S + 7],
        # more tokens between the two than a tile, a CTA's threads or a page holds
        "far apart": [3 * S + 3] + [(20 + i) * S + i % S for i in range(1600)] + base + [3 * S + 4],
        "none": base + [3 * S + 1, 3 * S + 2],
    }[kind]
    q, k, v, out, before, after, err = call(slots, D, S, P)
    assert err == (0 if kind == "none" else _capi.PI_ERR_PAGE_SHARED)
    assert torch.equal(out, q)
    for rows, pool, scale in ((k, 0, 2), (v, 1, 3)):
        ref, sc, shared = expect(slots, S, rows, before, pool, scale)
        assert shared == ([] if kind == "none" else [3])
        assert np.array_equal(np64(after[pool]), ref) and np.array_equal(np64(after[scale]), sc)
        for page in shared:
            assert torch.equal(after[pool][page].view(torch.uint8), before[pool][page].view(torch.uint8))


def test_many_tokens_on_one_dummy_slot():
    # padding that names a page of its own instead of -1 is reported and harms nothing else
    S, D, P, T = 16, 128, 40, 700
    slots = [2 * S + i for i in range(S)] + [0] * (T - S)
    q, k, v, out, before, after, err = call(slots, D, S, P)
    assert err == _capi.PI_ERR_PAGE_SHARED and torch.equal(out, q)
    for rows, pool, scale in ((k, 0, 2), (v, 1, 3)):
        ref, sc, shared = expect(slots, S, rows, before, pool, scale)
        assert shared == [0]
        assert np.array_equal(np64(after[pool]), ref) and np.array_equal(np64(after[scale]), sc)
