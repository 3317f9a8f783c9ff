"""GPU parity of decode attention over an 8-bit cache (pi_paged_decode_attn_q8) against the
64-bit oracle; tests/_q8.py derives the bounds."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from plastic_infer_b200 import _capi, kernels
from tests._q8 import DEV, E4M3, TYPES, cache, check, np64, on_gpu, reference

pytestmark = pytest.mark.gpu


def attend(q, c, **kw):
    return kernels.paged_decode_attention_q8(q, c["k_pool"], c["v_pool"], c["k_scale"], c["v_scale"],
                                             c["tables"], c["lens"], **kw)


def queries(B, Hq, D, dtype, seed):
    g = torch.Generator().manual_seed(seed + 100)
    return torch.randn((B, Hq, D), generator=g).to(TYPES[dtype]).to(DEV)


LENS = [[1], [0], [16], [17, 31, 32, 33], [0, 5, 0, 64, 129, 0], [1000], [700, 1, 15, 48, 333]]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("shape", [(1, 4, 128, 16), (2, 8, 128, 16), (2, 1, 64, 32), (1, 5, 64, 16),
                                   (2, 3, 256, 32), (1, 7, 256, 16), (3, 2, 128, 32)], ids=str)
def test_decode_matches_oracle(dtype, lens, shape):
    Hkv, G, D, S = shape
    c = on_gpu(cache(lens, Hkv, D, S, seed=len(lens) + D))
    q = queries(len(lens), Hkv * G, D, dtype, D)
    ref, tol = reference(q, c, lens)
    check(attend(q, c), ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("G", [9, 11, 16, 24])
def test_decode_many_query_heads(dtype, G):
    lens = [40, 0, 257]
    c = on_gpu(cache(lens, 2, 128, 16, seed=G))
    q = queries(3, 2 * G, 128, dtype, G)
    ref, tol = reference(q, c, lens)
    check(attend(q, c), ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(2, 2, 80, 16), (1, 3, 128, 8), (2, 1, 40, 5), (1, 2, 192, 64)], ids=str)
def test_decode_other_shapes(dtype, shape):
    Hkv, G, D, S = shape
    lens = [3, 0, 100, 5 * S]
    c = on_gpu(cache(lens, Hkv, D, S, seed=D))
    q = queries(4, Hkv * G, D, dtype, D)
    ref, tol = reference(q, c, lens)
    check(attend(q, c), ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_decode_many_requests_and_one_long(dtype):
    # cut segments, whole segments and merges in one launch; far more units than warps
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 900, 150)] + [40000]
    c = on_gpu(cache(lens, 2, 128, 16, seed=9))
    q = queries(len(lens), 8, 128, dtype, 9)
    ref, tol = reference(q, c, lens)
    for _ in range(3):  # the workspace's counters return to zero
        check(attend(q, c), ref, tol)


@pytest.mark.parametrize("dtype,G,D,S", [("bf16", 4, 64, 16), ("f16", 8, 128, 32), ("bf16", 2, 256, 16)])
def test_decode_long_streams(dtype, G, D, S):
    # enough units that a part of the stream is handed out in chunks, and every stage of the rings
    # goes round many times; lengths from nothing to many times a CTA's share
    lens = [9000, 1, 0, 4500, 12001, 33, 7000, 5000, 3000, 640]
    c = on_gpu(cache(lens, 8, D, S, seed=14))
    q = queries(len(lens), 8 * G, D, dtype, 14)
    ref, tol = reference(q, c, lens)
    first = attend(q, c)
    check(first, ref, tol)
    for _ in range(5):  # whoever computes which chunk, the result is the same
        assert torch.equal(attend(q, c), first)


def test_decode_more_requests_than_one_launch():
    lens = [int(x) for x in np.random.default_rng(1).integers(0, 60, 2100)]
    c = on_gpu(cache(lens, 1, 64, 16, seed=15))
    q = queries(len(lens), 2, 64, "bf16", 15)
    ref, tol = reference(q, c, lens)
    check(attend(q, c), ref, tol)


@pytest.mark.parametrize("plain_scales", [False, True])
def test_decode_scales(plain_scales):
    # neighbouring pages whose scales differ by many powers of two; scales that are no powers
    # of two, and zeros among them
    lens = [200, 33, 16]
    c = on_gpu(cache(lens, 2, 128, 16, seed=3, spread=6.0, plain_scales=plain_scales))
    q = queries(3, 8, 128, "bf16", 3) * 0.05
    ref, tol = reference(q, c, lens)
    check(attend(q, c), ref, tol)


def test_decode_one_token_outweighs_all():
    # a peaked softmax: all but one weight vanish, and the large scores keep their places
    lens = [500]
    c = on_gpu(cache(lens, 1, 128, 16, seed=4))
    q = queries(1, 4, 128, "f16", 4) * 30
    ref, tol = reference(q, c, lens)
    check(attend(q, c), ref, tol)


def test_decode_strides_scale_out_and_shared_table():
    lens = [90, 17, 64]
    Hkv, G, D, S = 2, 4, 128, 16
    c = on_gpu(cache(lens, Hkv, D, S, seed=5))
    wide = queries(3, Hkv * G + 3, D, "bf16", 5)
    q = wide[:, :Hkv * G]
    out = torch.zeros((3, Hkv * G + 1, D), dtype=torch.bfloat16, device=DEV)
    ref, tol = reference(q, c, lens, scale=0.03)
    got = attend(q, c, scale=0.03, out=out[:, :Hkv * G])
    check(got, ref, tol)
    assert int(out[:, Hkv * G].count_nonzero()) == 0
    # one table for several query rows (stride 0) at different lengths
    shared = dict(c, tables=c["tables"][:1].expand(4, -1), lens=torch.tensor([1, 33, 89, 90], dtype=torch.int32, device=DEV))
    q4 = queries(4, Hkv * G, D, "bf16", 6)
    ref, tol = reference(q4, c, [1, 33, 89, 90], rows_of=[0] * 4)
    check(attend(q4, shared), ref, tol)
    # lengths beyond the table and below zero are cut
    cut = dict(c, tables=c["tables"][:1, :2].contiguous(), lens=torch.tensor([10 ** 6], dtype=torch.int32, device=DEV))
    ref, tol = reference(q4[:1], c, [32])
    check(attend(q4[:1], cut), ref, tol)
    none = dict(cut, lens=torch.tensor([-5], dtype=torch.int32, device=DEV))
    assert int(attend(q4[:1], none).count_nonzero()) == 0
    empty = dict(cut, tables=torch.zeros((1, 0), dtype=torch.int32, device=DEV))
    assert int(attend(q4[:1], empty).count_nonzero()) == 0


@pytest.mark.parametrize("dtype,D,S", [("bf16", 128, 16), ("f32", 128, 16), ("bf16", 80, 16)])
def test_decode_reports_bad_pages(dtype, D, S):
    lens = [100, 64]
    c = on_gpu(cache(lens, 1, D, S, seed=6))
    good = c["tables"].clone()
    q = queries(2, 4, D, dtype, 6)
    for bad in (-1, int(c["k_pool"].shape[0]), 2 ** 31 - 1):
        c["tables"] = good.clone()
        c["tables"][0, 3] = bad
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = attend(q, c, err=err)
        assert int(err.item()) == _capi.PI_ERR_PAGE_RANGE
        ref, tol = reference(q[1:], dict(c, tables=good[1:]), lens[1:])
        check(out[1:], ref, tol)  # the other request is not touched by it
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    attend(q, dict(c, tables=good), err=err)
    assert int(err.item()) == 0


def test_decode_nan_and_infinite_queries():
    lens = [50, 50]
    c = on_gpu(cache(lens, 1, 128, 16, seed=7))
    q = queries(2, 4, 128, "bf16", 7)
    q[0, 1, 5] = math.nan
    q[0, 2, 6] = math.inf
    out = attend(q, c)
    assert out[0, 1].isnan().all() and out[0, 2].isnan().all()
    ref, tol = reference(torch.where(q.isfinite(), q, 0), c, lens)
    keep = [(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (1, 3)]
    for b, h in keep:
        assert (np.abs(np64(out[b, h]) - ref[b, h]) <= tol[b, h]).all()


def test_decode_pool_past_32_bits():
    # pages whose elements lie more than 2^31 from the pool's start
    Hkv, D, S = 8, 128, 16
    P = (2 ** 31 + 2 ** 28) // (Hkv * S * D)
    small = cache([100, 65], Hkv, D, S, seed=8)
    q = queries(2, 32, D, "bf16", 8)
    ref, tol = reference(q, small, [100, 65])
    n = small["k_pool"].shape[0]
    c = dict(lens=small["lens"].to(DEV), tables=(small["tables"] % 2 ** 30 + (P - n)).to(DEV))
    for name in ("k_pool", "v_pool"):
        c[name] = torch.empty((P, Hkv, S, D), dtype=E4M3, device=DEV)
        c[name].view(torch.uint8)[P - n:] = small[name].view(torch.uint8).to(DEV)
    for name in ("k_scale", "v_scale"):
        c[name] = torch.full((P, Hkv), math.nan, device=DEV)
        c[name][P - n:] = small[name].to(DEV)
    check(attend(q, c), ref, tol)


def test_decode_streams_and_graphs():
    lens_a, lens_b = [800, 30, 1200], [64, 2000]
    a, b = on_gpu(cache(lens_a, 2, 128, 16, seed=10)), on_gpu(cache(lens_b, 2, 128, 16, seed=11))
    qa, qb = queries(3, 8, 128, "bf16", 10), queries(2, 8, 128, "bf16", 11)
    ra, rb = reference(qa, a, lens_a), reference(qb, b, lens_b)
    attend(qa, a), attend(qb, b)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):  # two streams at once, without a workspace of the caller's
        for st, q, c in ((s[0], qa, a), (s[1], qb, b)):
            with torch.cuda.stream(st):
                outs.append(attend(q, c))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        check(o, *(ra if i % 2 == 0 else rb))
    graphs = []
    for q, c in ((qa, a), (qb, b)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = attend(q, c)
        graphs.append((g, out))
    for _ in range(10):  # two graphs replayed at once
        for st, (g, _o) in zip(s, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    check(graphs[0][1], *ra)
    check(graphs[1][1], *rb)


def test_decode_with_programmatic_launch():
    lens = [300, 77, 1024]
    c = on_gpu(cache(lens, 2, 128, 16, seed=12))
    q = queries(3, 8, 128, "bf16", 12)
    ref, tol = reference(q, c, lens)
    kernels.set_programmatic_launch(True)
    try:
        outs = [attend(q, c) for _ in range(10)]
        torch.cuda.synchronize()
    finally:
        kernels.set_programmatic_launch(False)
    for o in outs:
        check(o, ref, tol)


def test_append_then_decode():
    # a prompt, then tokens one by one, through the cache that both operators share
    Hq, Hkv, D, S, n0, steps = 8, 2, 128, 16, 43, 9
    g = torch.Generator().manual_seed(13)
    T = n0 + steps
    q, k, v = (torch.randn((T, h, D), generator=g).bfloat16().to(DEV) for h in (Hq, Hkv, Hkv))
    P = -(-T // S) + 2
    kp, vp = (torch.full((P, Hkv, S, D), 0x7F, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    ks, vs = (torch.full((P, Hkv), math.nan, device=DEV) for _ in range(2))
    table = torch.randperm(P, generator=g)[:-(-T // S)]
    slots = (table[torch.arange(T) // S] * S + torch.arange(T) % S).to(DEV)
    inv, rs = kernels.rope_frequencies(D, 1e6, device=DEV)
    pos = torch.arange(T, device=DEV)
    bt = table.int()[None].to(DEV)
    at = 0
    for n in [n0] + [1] * steps:
        sl = slice(at, at + n)
        qr = kernels.rope_append(q[sl], k[sl], v[sl], pos[sl], inv, slots[sl], kp, vp, k_scale=ks, v_scale=vs)
        at += n
        c = dict(k_pool=kp, v_pool=vp, k_scale=ks, v_scale=vs, tables=bt,
                 lens=torch.tensor([at], dtype=torch.int32, device=DEV))
        ref, tol = reference(qr[-1:], c, [at])
        check(attend(qr[-1:], c), ref, tol)
