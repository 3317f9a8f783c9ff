"""GPU parity of several query tokens over an 8-bit cache (pi_paged_prefill_attn_q8) and of the
widened pages (pi_page_dequant) against the 64-bit oracle; tests/_q8.py derives the bounds. The
widening path rounds P to the output type as the tcgen05 prefill does, half a step of which is
what the bounds allow a weight in bf16, and 2^-11 in f16."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from plastic_infer_b200 import _capi, kernels
from tests._q8 import DEV, E4M3, TYPES, cache, check, np64, on_gpu, reference

pytestmark = pytest.mark.gpu


def attend(q, c, kv_len, q_start, **kw):
    return kernels.paged_prefill_attention_q8(q, c["k_pool"], c["v_pool"], c["k_scale"], c["v_scale"],
                                              c["tables"][0], kv_len, q_start, **kw)


def queries(n, Hq, D, dtype, seed):
    g = torch.Generator().manual_seed(seed + 200)
    return torch.randn((n, Hq, D), generator=g).to(TYPES[dtype]).to(DEV)


def expect(q, c, kv_len, q_start, causal=True, scale=None, wide=False):
    n = q.shape[0]
    lens = [min(kv_len, q_start + i + 1) if causal else kv_len for i in range(n)]
    ref, tol = reference(q, c, lens, rows_of=[0] * n, scale=scale)
    if wide and q.dtype == torch.float16:
        # P and the widened K and V are f16 values: half a step more on each of the two products
        tol = tol + 2.0 ** -10 * (np.abs(ref) + tol / 2.0 ** -11)
    return ref, tol


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(1, 4, 128, 16), (2, 1, 64, 32), (1, 5, 128, 16), (2, 8, 64, 16),
                                   (1, 3, 256, 32), (1, 16, 128, 32), (1, 2, 80, 16)], ids=str)
@pytest.mark.parametrize("span", [(1, 0), (2, 0), (17, 0), (33, 100), (3, 31), (7, 1001), (40, 16)], ids=str)
def test_short_chunks(dtype, shape, span):
    Hkv, G, D, S = shape
    n, start = span
    kv_len = start + n
    c = on_gpu(cache([kv_len], Hkv, D, S, seed=n + D))
    q = queries(n, Hkv * G, D, dtype, n)
    ref, tol = expect(q, c, kv_len, start)
    check(attend(q, c, kv_len, start), ref, tol)


@pytest.mark.parametrize("causal,kv_len,start", [(False, 90, 0), (False, 257, 7), (True, 50, 0), (True, 40, 60),
                                                 (True, 0, 0), (False, 0, 5), (True, 65, 30)])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64), ("f16", 256)])
def test_masks(dtype, D, causal, kv_len, start):
    # keys beyond the last query, queries beyond the last key, no key at all
    c = on_gpu(cache([max(kv_len, 1)], 2, D, 16, seed=21))
    q = queries(37, 8, D, dtype, 21)
    ref, tol = expect(q, c, kv_len, start, causal)
    got = attend(q, c, kv_len, start, causal=causal)
    if kv_len == 0:
        assert int(got.count_nonzero()) == 0
    else:
        check(got, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [(8, 4, 128, 16), (2, 8, 64, 32), (4, 16, 128, 32)], ids=str)
@pytest.mark.parametrize("span", [(700, 0), (401, 333)], ids=str)
def test_long_chunks(dtype, shape, span):
    Hkv, G, D, S = shape
    n, start = span
    kv_len = start + n
    c = on_gpu(cache([kv_len], Hkv, D, S, seed=n))
    q = queries(n, Hkv * G, D, dtype, n)
    ref, tol = expect(q, c, kv_len, start, wide=True)
    check(attend(q, c, kv_len, start), ref, tol)


def test_long_chunk_not_causal_and_unaligned():
    Hkv, G, D, S = 4, 4, 128, 16
    c = on_gpu(cache([500], Hkv, D, S, seed=31))
    wide = queries(420, Hkv * G + 1, D, "bf16", 31)
    for q in (wide[:, :Hkv * G], wide.flatten()[4:4 + 420 * Hkv * G * D].view(420, Hkv * G, D)):
        ref, tol = expect(q, c, 500, 0, causal=False, scale=0.05)
        check(attend(q, c, 500, 0, causal=False, scale=0.05), ref, tol)


def test_few_rows_over_a_long_history():
    # cut segments and merges, with rows that see nothing of the last units
    for dtype in ("bf16", "f16"):
        c = on_gpu(cache([30011], 2, 128, 16, seed=32))
        q = queries(50, 8, 128, dtype, 32)
        ref, tol = expect(q, c, 30011, 30011 - 50)
        for _ in range(2):
            check(attend(q, c, 30011, 30011 - 50), ref, tol)


def test_batch_axis_out_and_bad_pages():
    c = on_gpu(cache([200], 2, 128, 16, seed=33))
    for n in (5, 800):
        q = queries(n, 8, 128, "bf16", 33)
        out = torch.zeros((1, n, 8, 128), dtype=torch.bfloat16, device=DEV)
        got = attend(q[None], c, 200, 0, out=out)
        assert got is out
        ref, tol = expect(q, c, 200, 0)
        check(out[0], ref, tol)
        assert attend(q[None], c, 200, 0).shape == (1, n, 8, 128)
        bad = dict(c, tables=c["tables"].clone())
        bad["tables"][0, 4] = -3
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        attend(q, bad, 200, 0, err=err)
        # page 4 holds tokens 64 .. 79: five queries at positions 0 .. 4 see none of them, and a
        # page that no query sees is not read
        assert int(err.item()) == (_capi.PI_ERR_PAGE_RANGE if n > 64 else 0)
    assert attend(queries(0, 8, 128, "bf16", 0), c, 200, 0).shape == (0, 8, 128)


def test_streams_and_graph():
    c = on_gpu(cache([900], 4, 128, 16, seed=34))
    q = [queries(n, 16, 128, "bf16", n) for n in (9, 800)]
    want = [expect(x, c, 900, 900 - x.shape[0]) for x in q]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(s[i]):
                outs.append((i, attend(q[i], c, 900, 900 - q[i].shape[0])))
    torch.cuda.synchronize()
    for i, o in outs:
        check(o, *want[i])
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = attend(q[i], c, 900, 900 - q[i].shape[0])
        for _ in range(3):
            g.replay()
        torch.cuda.synchronize()
        check(o, *want[i])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,S", [(128, 16), (40, 5)])
def test_page_dequant(dtype, D, S):
    g = torch.Generator().manual_seed(D)
    pool = (torch.randn((9, 3, S, D), generator=g) * 100).to(E4M3)
    pool.view(torch.uint8)[1, 2, 0, 3] = 0x7F
    scale = torch.exp2(torch.randint(-3, 3, (9, 3), generator=g).float())
    scale[4, 1] = 2.0 ** 10  # past what f16 holds
    ids = torch.tensor([4, 0, 1, 4, 8], dtype=torch.int32)
    got = kernels.page_dequant(pool.to(DEV), scale.to(DEV), ids.to(DEV), TYPES[dtype])
    ref = np64(pool)[ids] * np64(scale)[ids][:, :, None, None]
    if dtype == "f16":
        ref = np.clip(ref, -65504, 65504)
    assert np.array_equal(np64(got), ref, equal_nan=True)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.ones((2, 3, S, D), dtype=TYPES[dtype], device=DEV)
    kernels.page_dequant(pool.to(DEV), scale.to(DEV), torch.tensor([9, 0], dtype=torch.int32, device=DEV),
                         TYPES[dtype], out=out, err=err)
    assert int(err.item()) == _capi.PI_ERR_PAGE_RANGE
    assert int(out[0].count_nonzero()) == 0 and np.array_equal(np64(out[1]), ref[1])


def test_prompt_then_chunk_through_one_cache():
    # two chunks of a prompt appended and attended, then the whole against one pass
    Hq, Hkv, D, S, n = 8, 2, 128, 16, 300
    g = torch.Generator().manual_seed(40)
    q, k, v = (torch.randn((n, h, D), generator=g).bfloat16().to(DEV) for h in (Hq, Hkv, Hkv))
    P = -(-n // S) + 1
    kp, vp = (torch.full((P, Hkv, S, D), 0x7F, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    ks, vs = (torch.full((P, Hkv), math.nan, device=DEV) for _ in range(2))
    table = torch.randperm(P, generator=g)[:-(-n // S)]
    slots = (table[torch.arange(n) // S] * S + torch.arange(n) % S).to(DEV)
    pos = torch.arange(n, device=DEV)
    inv, rs = kernels.rope_frequencies(D, 1e6, "yarn", 4.0, 64, device=DEV)
    for a, b in ((0, 121), (121, n)):
        qr = kernels.rope_append(q[a:b], k[a:b], v[a:b], pos[a:b], inv, slots[a:b], kp, vp, rope_scale=rs,
                                 interleaved=True, k_scale=ks, v_scale=vs)
        c = dict(k_pool=kp, v_pool=vp, k_scale=ks, v_scale=vs, tables=table.int()[None].to(DEV))
        ref, tol = expect(qr, c, b, a)
        check(attend(qr, c, b, a), ref, tol)
