"""Programmatic launch over the 8-bit cache: appends, decode attention (with its merge launch and
without) and prefill (widened and not) in a row give the bits that they give without it, eagerly, in a
graph and with tables that the wrappers have to copy; and every call repeats itself bit for bit."""

from __future__ import annotations

import pytest
import torch

from plastic_infer_b200 import kernels
from tests._q8 import DEV, E4M3, check, reference

pytestmark = pytest.mark.gpu


def inputs(B, L, seed, Hq=16, Hkv=4, D=128, S=16):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, 700, (B,), generator=g, dtype=torch.int32)
    spans = (lens + S) // S + 1
    P = int(spans.sum()) + 2
    order = torch.randperm(P, generator=g).int()
    tables = torch.zeros((B, int(spans.max())), dtype=torch.int32)
    at = 0
    for b in range(B):
        tables[b, :spans[b]] = order[at:at + int(spans[b])]
        at += int(spans[b])
    x = dict(lens=lens + 1, tables=tables,
             q=torch.randn((L, B, Hq, D), generator=g).bfloat16(), k=torch.randn((L, B, Hkv, D), generator=g).bfloat16(),
             v=torch.randn((L, B, Hkv, D), generator=g).bfloat16(), pos=lens.long(),
             slots=tables[torch.arange(B), (lens // S).long()].long() * S + lens.long() % S,
             inv=kernels.rope_inv_freq(D, 1e4),
             kp=(torch.randn((P, Hkv, S, D), generator=g) * 60).to(E4M3), vp=(torch.randn((P, Hkv, S, D), generator=g) * 60).to(E4M3),
             ks=torch.exp2(torch.randint(-8, -5, (P, Hkv), generator=g).float()),
             vs=torch.exp2(torch.randint(-8, -5, (P, Hkv), generator=g).float()),
             chunk=torch.randn((400, Hq, D), generator=g).bfloat16())
    return {k: v.to(DEV) for k, v in x.items()}


def run(x, strided=False):
    """Layers of append and decode over one cache, then a long and a short chunk of request 0."""
    t, n = x["tables"], x["lens"]
    outs = []
    for l in range(x["q"].shape[0]):
        if strided:  # copied anew for every call
            t = torch.stack([x["tables"], torch.full_like(x["tables"], 2 ** 30)], -1)[..., 0]
            n = torch.stack([x["lens"], torch.zeros_like(x["lens"])], -1)[:, 0]
        q = kernels.rope_append(x["q"][l], x["k"][l], x["v"][l], x["pos"], x["inv"], x["slots"], x["kp"], x["vp"],
                                k_scale=x["ks"], v_scale=x["vs"])
        outs += [q, kernels.paged_decode_attention_q8(q, x["kp"], x["vp"], x["ks"], x["vs"], t, n)]
    row = t[0] if not strided else torch.stack([x["tables"][0], torch.zeros_like(x["tables"][0])], -1)[:, 0]
    pools = (x["kp"], x["vp"], x["ks"], x["vs"])
    length = x["first_len"]
    for c in (x["chunk"], x["chunk"][:9]):
        outs.append(kernels.paged_prefill_attention_q8(c, *pools, row, length, 0))
    return outs


@pytest.mark.parametrize("B", [5, 60], ids=["merge launch", "last arriver"])
@pytest.mark.parametrize("strided", [False, True])
def test_same_bits_with_programmatic_launch(B, strided):
    def fresh():
        x = inputs(B, 6, seed=B)
        x["first_len"] = int(x["lens"][0])
        torch.cuda.synchronize()
        return x

    want = run(fresh())
    torch.cuda.synchronize()
    try:
        for on in (False, True):
            kernels.set_programmatic_launch(on)
            x = fresh()
            got = run(x, strided)
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            x = fresh()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = run(x, strided)
            for name in ("kp", "vp"):
                x[name].view(torch.uint8).copy_(fresh()[name].view(torch.uint8))
            for name in ("ks", "vs"):
                x[name].copy_(fresh()[name])
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            del graph
    finally:
        kernels.set_programmatic_launch(False)


def test_result_is_the_oracles():
    x = inputs(5, 1, seed=9)
    x["first_len"] = int(x["lens"][0])
    outs = run(x)
    c = dict(k_pool=x["kp"], v_pool=x["vp"], k_scale=x["ks"], v_scale=x["vs"], tables=x["tables"])
    check(outs[1], *reference(outs[0], c, [int(n) for n in x["lens"]]))
