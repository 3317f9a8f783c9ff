"""Programmatic launch, host side: the attention kernels read block tables and lengths before they wait
for the launch before them, so the wrappers' own copies of strided ones must not be that launch.

The wrappers run here on CPU tensors with the C call replaced, and every torch operation is recorded:
the last one that runs a kernel before the call must not have written what the call is given.
"""

from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from plastic_infer_b200 import _capi, kernels

E4M3 = torch.float8_e4m3fn
NO_KERNEL = ("view", "slice", "select", "empty", "as_strided", "detach", "expand", "alias", "unsqueeze", "transpose", "t.")


class Recorder(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.last = None  # address that the last kernel wrote

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if isinstance(out, torch.Tensor) and not any(n in str(func) for n in NO_KERNEL):
            self.last = out.data_ptr()
        return out


def tables(kind, B=3, W=4):
    t, lens = torch.zeros((B, 2 * W), dtype=torch.int32)[:, :W], torch.ones(B, dtype=torch.int32)
    if kind in ("tables", "both"):
        t = torch.zeros((B, 2 * W), dtype=torch.int32)[:, ::2]
    if kind in ("lengths", "both"):
        lens = torch.ones(2 * B, dtype=torch.int32)[::2]
    return t, lens


@pytest.mark.parametrize("kind", ["none", "tables", "lengths", "both"])
@pytest.mark.parametrize("op", ["decode", "append", "decode_q8", "prefill_q8"])
def test_the_launch_before_the_attention_is_no_copy_of_its_tables(monkeypatch, op, kind):
    B, Hq, Hkv, D, S, P = 3, 4, 2, 64, 16, 8
    seen = []
    rec = Recorder()

    def call(func, *args):
        seen.append((func, rec.last, args))

    monkeypatch.setattr(_capi, "call", call)
    monkeypatch.setattr(kernels, "_call_on", lambda device, func, *args: call(func, *args))
    monkeypatch.setattr(kernels, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(kernels, "_check_one_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(kernels, "_stream", lambda: 0)
    monkeypatch.setattr(kernels, "workspace_bytes", lambda *a: 256)
    monkeypatch.setattr(kernels, "_q8_decode_workspace_bytes", lambda *a: 256)
    t, lens = tables(kind)
    q = torch.zeros((B, Hq, D), dtype=torch.bfloat16)
    out = torch.zeros_like(q)
    ws = kernels.Workspace(torch.device("cpu"))
    ws.get(256)
    pools16 = [torch.zeros((P, Hkv, S, D), dtype=torch.bfloat16) for _ in range(2)]
    pools8 = [p.to(E4M3) for p in pools16] + [torch.ones((P, Hkv)) for _ in range(2)]
    new = [torch.zeros((B, Hkv, D), dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.zeros(B, dtype=torch.int64)
    with rec:
        if op == "decode":
            kernels.paged_decode_attention(q, *pools16, t, lens, out=out, workspace=ws)
        elif op == "append":
            kernels.paged_decode_attention(q, *pools16, t, lens, out=out, workspace=ws, k_new=new[0], v_new=new[1],
                                           slot_mapping=slots)
        elif op == "decode_q8":
            kernels.paged_decode_attention_q8(q, *pools8, t, lens, out=out, workspace=ws)
        else:
            kernels.paged_prefill_attention_q8(q, *pools8, t[1], 20, out=out, workspace=ws)
    (func, last, args), = seen
    assert last is None or last not in args, func
