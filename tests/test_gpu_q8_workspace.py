"""Scratch of the 8-bit attention calls: shared with the 16-bit ones, between streams and threads,
grown and given back."""

from __future__ import annotations

import threading

import pytest
import torch

from plastic_infer_b200 import _capi, kernels
from tests._q8 import DEV, cache, check, on_gpu, reference

pytestmark = pytest.mark.gpu


def queries(B, Hq, D, dtype, seed):
    g = torch.Generator().manual_seed(seed + 300)
    return torch.randn((B, Hq, D), generator=g).to(dtype).to(DEV)


def decode(q, c, **kw):
    return kernels.paged_decode_attention_q8(q, c["k_pool"], c["v_pool"], c["k_scale"], c["v_scale"],
                                             c["tables"], c["lens"], **kw)


def prefill(q, c, kv_len, q_start, **kw):
    return kernels.paged_prefill_attention_q8(q, c["k_pool"], c["v_pool"], c["k_scale"], c["v_scale"],
                                              c["tables"][0], kv_len, q_start, **kw)


def counters(ws):
    return ws.buf[:int(_capi.load().pi_paged_decode_attn_ws_zero_bytes())]


@pytest.mark.parametrize("lens", [[4000], [900] * 40], ids=["merge launch", "last arriver"])
def test_one_workspace_for_both_caches(lens):
    # contexts cut across warps, so partial results are written; the block that the 16-bit kernels
    # (the gather's completion counter at its end) need zeroed stays zero
    c = on_gpu(cache(lens, 8, 128, 16, seed=50))
    q = queries(len(lens), 32, 128, torch.bfloat16, 50)
    ref, tol = reference(q, c, lens)
    ws = kernels.Workspace(DEV)
    k16 = kernels.page_dequant(c["k_pool"], c["k_scale"], torch.arange(c["k_pool"].shape[0], dtype=torch.int32, device=DEV))
    v16 = kernels.page_dequant(c["v_pool"], c["v_scale"], torch.arange(c["k_pool"].shape[0], dtype=torch.int32, device=DEV))
    tables = torch.where(c["tables"] < 2 ** 29, c["tables"], 0)
    alone = kernels.paged_decode_attention(q, k16, v16, tables, c["lens"], workspace=kernels.Workspace(DEV))
    for _ in range(2):
        check(decode(q, c, workspace=ws), ref, tol)
        assert int(counters(ws).count_nonzero()) == 0
        assert torch.equal(kernels.paged_decode_attention(q, k16, v16, tables, c["lens"], workspace=ws), alone)
        assert int(counters(ws).count_nonzero()) == 0
        check(prefill(q[:1], c, lens[0], lens[0] - 1, workspace=ws), *(x[:1] for x in (ref, tol)))
        assert int(counters(ws).count_nonzero()) == 0


def run_threads(jobs, rounds):
    """Every job in a thread of its own, on one stream, `rounds` times; the outputs by job."""
    outs = [[] for _ in jobs]
    failed = []
    go = threading.Barrier(len(jobs))

    def work(i):
        try:
            go.wait()
            for _ in range(rounds):
                outs[i].append(jobs[i]())
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    return outs


@pytest.mark.parametrize("own", [False, True], ids=["hidden", "workspace"])
def test_threads_on_one_stream(own):
    # few segments: a launch that writes partial results and one that merges them; another thread's
    # launches must not come between the two
    ws = kernels.Workspace(DEV) if own else None
    caches = [on_gpu(cache([n], 2, 128, 16, seed=60 + i)) for i, n in enumerate((3000, 2500, 1700))]
    qs = [queries(1, 8, 128, torch.bfloat16, 60 + i) for i in range(3)]
    want = [decode(q, c).clone() for q, c in zip(qs, caches)]
    jobs = [lambda q=q, c=c: decode(q, c, workspace=ws) for q, c in zip(qs, caches)]
    for w, got in zip(want, run_threads(jobs, 300)):
        for o in got:
            assert torch.equal(o, w)


def test_threads_with_long_chunks():
    # widened pages of one request must not be read by another's queries
    lens = (1200, 700, 950)
    caches = [on_gpu(cache([n], 4, 128, 16, seed=70 + i)) for i, n in enumerate(lens)]
    qs = [queries(n // 2, 16, 128, torch.bfloat16, 70 + i) for i, n in enumerate(lens)]
    want = [prefill(q, c, n, n - n // 2).clone() for q, c, n in zip(qs, caches, lens)]
    jobs = [lambda q=q, c=c, n=n: prefill(q, c, n, n - n // 2) for q, c, n in zip(qs, caches, lens)]
    for w, got in zip(want, run_threads(jobs, 60)):
        for o in got:
            assert torch.equal(o, w)


def test_widened_pages_are_given_back():
    # a prompt in growing chunks: nothing of the 16-bit copies stays allocated, and the allocator's
    # blocks behind them are few
    Hkv, D, S, chunk, n = 8, 128, 16, 512, 8192
    c = on_gpu(cache([n], Hkv, D, S, seed=80))
    q = queries(chunk, 32, D, torch.bfloat16, 80)
    side = torch.cuda.Stream()  # a stream whose scratch is its own
    with torch.cuda.stream(side):
        prefill(q[:1], c, 1, 0)  # the decode kernels' scratch
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        before, reserved = torch.cuda.memory_allocated(), torch.cuda.memory_reserved()
        out = torch.empty_like(q)
        for end in range(chunk, n + 1, chunk):
            prefill(q, c, end, end - chunk, out=out)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() <= before + out.numel() * 2 + (1 << 20)
        need = int(_capi.load().pi_paged_prefill_attn_q8_workspace_bytes(chunk, n, 32, Hkv, D, S, _capi.PI_DTYPE_BF16))
        assert torch.cuda.memory_reserved() - reserved <= 4 * need + (16 << 20)
    rows = list(range(0, chunk, 97))
    ref, tol = reference(q[rows], c, [n - chunk + i + 1 for i in rows], rows_of=[0] * len(rows))
    check(out[rows], ref, tol)


def test_lent_scratch_need_not_be_zeroed():
    # rows that are not 16-byte aligned keep to the decode kernels: many segments, whose counters lie
    # in scratch that held something else before
    Hkv, D, S, n = 4, 128, 16, 500
    c = on_gpu(cache([n], Hkv, D, S, seed=81))
    q = queries(420, 16 * D + 4, 1, torch.bfloat16, 81)[:, 4:, 0].unflatten(1, (16, D))
    rows = list(range(0, 420, 41))
    ref, tol = reference(q[rows], c, [n - 420 + i + 1 for i in rows], rows_of=[0] * len(rows))
    for _ in range(2):
        dirty = torch.full((64 << 20,), 0xA5, dtype=torch.uint8, device=DEV)
        del dirty
        check(prefill(q, c, n, n - 420)[rows], ref, tol)


@pytest.mark.parametrize("lens", [[3000], [700] * 40], ids=["merge launch", "last arriver"])
def test_two_graphs_over_a_cold_workspace(lens):
    # neither graph has grown it for the other, nor for an eager call before any replay
    c = on_gpu(cache(lens, 8, 128, 16, seed=90))
    q = queries(len(lens), 32, 128, torch.bfloat16, 90)
    want = decode(q, c).clone()
    ws = kernels.Workspace(DEV)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = decode(q, c, workspace=ws)
        graphs.append((g, out))
    assert ws.buf is None
    assert torch.equal(decode(q, c, workspace=ws), want)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):  # the second first, then both at once
        for s, (g, _out) in zip(streams, reversed(graphs)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _g, out in graphs:
        assert torch.equal(out, want)
    assert torch.equal(decode(q, c, workspace=ws), want)
