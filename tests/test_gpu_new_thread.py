"""The attention calls as the first CUDA work of a host thread.

A new thread has no CUDA context bound to it until a runtime call needs one, and none of a call's
steps before its tensor maps does where all its buffers are given.
"""

from __future__ import annotations

import threading

import pytest
import torch

from plastic_infer_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def in_new_thread(call):
    failed = []

    def work():
        try:
            call()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not failed, failed


@pytest.mark.parametrize("eight", [False, True], ids=["16-bit pools", "8-bit pools"])
def test_decode_and_prefill(eight):
    Hq, Hkv, D, S, P, n = 16, 4, 128, 16, 24, 384
    g = torch.Generator(device=DEV).manual_seed(1)
    dt = torch.float8_e4m3fn if eight else torch.bfloat16
    kp, vp = (torch.randn((P, Hkv, S, D), device=DEV, generator=g).to(dt) for _ in range(2))
    sc = [torch.ones((P, Hkv), device=DEV) for _ in range(2)] if eight else []
    table = torch.arange(P, dtype=torch.int32, device=DEV)
    q = torch.randn((n, Hq, D), device=DEV, generator=g).bfloat16()
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    ws = kernels.Workspace(DEV)
    ws.get(64 << 20)
    decode = kernels.paged_decode_attention_q8 if eight else kernels.paged_decode_attention
    want = decode(q[:1], kp, vp, *sc, table[None], lens)
    kp2, vp2 = kp.clone(), vp.clone()  # pools that no thread has used
    out = torch.empty((1, Hq, D), dtype=torch.bfloat16, device=DEV)
    in_new_thread(lambda: decode(q[:1], kp2, vp2, *sc, table[None], lens, out=out, workspace=ws))
    assert torch.equal(out, want)
    rows = torch.empty((n, Hq, D), dtype=torch.bfloat16, device=DEV)
    kp2, vp2 = kp.clone(), vp.clone()
    if eight:
        in_new_thread(lambda: kernels.paged_prefill_attention_q8(q, kp2, vp2, *sc, table, n, out=rows, workspace=ws))
        assert torch.equal(rows, kernels.paged_prefill_attention_q8(q, kp, vp, *sc, table, n))
    else:
        in_new_thread(lambda: kernels.paged_prefill_attention(q, kp2, vp2, table, n, out=rows))
        assert torch.equal(rows, kernels.paged_prefill_attention(q, kp, vp, table, n))
