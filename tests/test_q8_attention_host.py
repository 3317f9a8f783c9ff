"""Refusals of the 8-bit cache attention: the wrappers' checks and the C entry points' validation."""

from __future__ import annotations

import ctypes
import threading
import time
import weakref

import pytest
import torch

from plastic_infer_b200 import _build, _capi, kernels

E4M3 = torch.float8_e4m3fn


def _args(B=2, Hq=4, Hkv=2, D=64, S=16, P=4):
    z = torch.zeros
    return dict(q=z((B, Hq, D), dtype=torch.bfloat16), k_pool=z((P, Hkv, S, D)).to(E4M3),
                v_pool=z((P, Hkv, S, D)).to(E4M3), k_scale=z((P, Hkv)), v_scale=z((P, Hkv)),
                block_tables=z((B, 3), dtype=torch.int32), ctx_lens=z(B, dtype=torch.int32))


@pytest.mark.parametrize("change,error", [
    (dict(k_pool=torch.zeros(4, 2, 16, 64)), TypeError),
    (dict(v_pool=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)), TypeError),
    (dict(v_pool=torch.zeros(5, 2, 16, 64).to(E4M3)), ValueError),
    (dict(v_pool=torch.zeros(4, 2, 64, 16).to(E4M3).transpose(2, 3)), ValueError),
    (dict(k_scale=torch.zeros(4, 1)), ValueError),
    (dict(v_scale=torch.zeros(4, 2, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 4, 32, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 0, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.float64)), TypeError),
    (dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(block_tables=torch.zeros(3, 3, dtype=torch.int32)), ValueError),
    (dict(ctx_lens=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(ctx_lens=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(), ValueError),  # nothing wrong but the device
])
def test_decode_refuses(change, error):
    with pytest.raises(error):
        kernels.paged_decode_attention_q8(**{**_args(), **change})


def test_decode_c_entry_validates_before_launch():
    _build.build()
    lib = _capi.load()
    a = ctypes.c_void_p(256)
    # out, q, k_pool, v_pool, k_scale, v_scale, tables, bt_stride, max_pages, lens, batch, hq, hkv,
    # d, s, pages, scale, dtype, q_stride, out_stride, workspace, bytes, err, stream
    base = [a, a, a, a, a, a, a, 4, 4, a, 2, 4, 2, 128, 16, 8, 1.0, _capi.PI_DTYPE_BF16, 512, 512,
            None, 0, None, None]

    def rc(**change):
        x = list(base)
        for i, v in change.items():
            x[int(i[1:])] = v
        return lib.pi_paged_decode_attn_q8(*x)

    assert rc(_10=0) == _capi.PI_OK
    assert rc(_17=7) == _capi.PI_ERR_UNSUPPORTED
    assert rc(_17=_capi.PI_DTYPE_E4M3) == _capi.PI_ERR_UNSUPPORTED
    assert rc(_13=264, _18=4096, _19=4096) == _capi.PI_ERR_UNSUPPORTED
    assert rc(_11=5) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_8=-1) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_10=-1) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_18=511) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_19=511) == _capi.PI_ERR_BAD_SHAPE
    for i in (0, 1, 2, 3, 4, 5, 6, 9):
        assert rc(**{f"_{i}": None}) == _capi.PI_ERR_NULL_POINTER, i
    for i in (0, 1, 4, 5, 6, 9):
        assert rc(**{f"_{i}": ctypes.c_void_p(257)}) == _capi.PI_ERR_MISALIGNED, i
    assert rc() == _capi.PI_ERR_WORKSPACE
    assert rc(_20=a, _21=1000) == _capi.PI_ERR_WORKSPACE
    need = lib.pi_paged_decode_attn_q8_workspace_bytes(128)
    assert rc(_20=ctypes.c_void_p(128), _21=need) == _capi.PI_ERR_MISALIGNED
    assert lib.pi_paged_decode_attn_q8_ws_zero_bytes() < need


def _chunk(n=2, **kw):
    a = _args(B=n)
    a.pop("ctx_lens")
    a["block_table"] = a.pop("block_tables")[0]
    return {**a, "kv_len": 20, **kw}


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 4, 32, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 3, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k_pool=torch.zeros(4, 2, 16, 64)), TypeError),
    (dict(k_scale=torch.zeros(2, 4)), ValueError),
    (dict(block_table=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(block_table=torch.zeros(1, 3, dtype=torch.int32)), ValueError),
    (dict(kv_len=49), ValueError),
    (dict(kv_len=-1), ValueError),
    (dict(q_start=-1), ValueError),
    (dict(q_start=2 ** 31), ValueError),
    (dict(), ValueError),
])
def test_prefill_refuses(change, error):
    with pytest.raises(error):
        kernels.paged_prefill_attention_q8(**{**_chunk(), **change})


@pytest.mark.parametrize("args,error", [
    ((torch.zeros(4, 2, 16, 64), torch.zeros(4, 2), torch.zeros(1, dtype=torch.int32)), TypeError),
    ((torch.zeros(4, 2, 16, 64).to(E4M3), torch.zeros(4, 3), torch.zeros(1, dtype=torch.int32)), ValueError),
    ((torch.zeros(4, 2, 16, 64).to(E4M3), torch.zeros(4, 2), torch.zeros(1, dtype=torch.int64)), ValueError),
    ((torch.zeros(4, 2, 16, 64).to(E4M3), torch.zeros(4, 2), torch.zeros(1, dtype=torch.int32),
      torch.float64), TypeError),
    ((torch.zeros(4, 2, 16, 64).to(E4M3), torch.zeros(4, 2), torch.zeros(1, dtype=torch.int32)), ValueError),
])
def test_page_dequant_refuses(args, error):
    with pytest.raises(error):
        kernels.page_dequant(*args)


def test_prefill_c_entries_validate_before_launch():
    _build.build()
    lib = _capi.load()
    a = ctypes.c_void_p(256)
    # out, q, k_pool, v_pool, k_scale, v_scale, table, table_len, q_len, kv_len, q_start, causal, hq,
    # hkv, d, s, pages, scale, dtype, q_stride, out_stride, workspace, bytes, err, stream
    base = [a, a, a, a, a, a, a, 4, 3, 40, 0, 1, 4, 2, 128, 16, 8, 1.0, _capi.PI_DTYPE_BF16, 512, 512, None, 0,
            None, None]

    def rc(**change):
        x = list(base)
        for i, v in change.items():
            x[int(i[1:])] = v
        return lib.pi_paged_prefill_attn_q8(*x)

    assert rc(_8=0) == _capi.PI_OK
    assert rc(_18=_capi.PI_DTYPE_E4M3) == _capi.PI_ERR_UNSUPPORTED
    assert rc(_14=264, _19=4096, _20=4096) == _capi.PI_ERR_UNSUPPORTED
    for change in (dict(_8=-1), dict(_9=65), dict(_9=-1), dict(_10=-1), dict(_12=5), dict(_19=511), dict(_20=511),
                   dict(_10=2 ** 31 - 2)):
        assert rc(**change) == _capi.PI_ERR_BAD_SHAPE, change
    for i in range(7):
        assert rc(**{f"_{i}": None}) == _capi.PI_ERR_NULL_POINTER, i
    for i in (0, 1, 4, 5, 6):
        assert rc(**{f"_{i}": ctypes.c_void_p(257)}) == _capi.PI_ERR_MISALIGNED, i
    assert rc() == _capi.PI_ERR_WORKSPACE
    assert rc(_8=4000) == _capi.PI_ERR_WORKSPACE
    need = lib.pi_paged_prefill_attn_q8_workspace_bytes
    few = need(3, 40, 4, 2, 128, 16, _capi.PI_DTYPE_BF16)
    assert few == lib.pi_paged_decode_attn_q8_workspace_bytes(128)
    assert need(4000, 40, 4, 2, 128, 16, _capi.PI_DTYPE_BF16) >= few + 2 * 3 * 2 * 16 * 128 * 2
    assert need(4000, 40, 4, 2, 128, 16, _capi.PI_DTYPE_F32) == few
    edge = _capi.Q8_FEW_ROWS // 4  # the wrapper asks for more from here on
    assert need(edge, 40, 4, 2, 128, 16, _capi.PI_DTYPE_BF16) == few < need(edge + 1, 40, 4, 2, 128, 16, _capi.PI_DTYPE_BF16)
    d = lib.pi_page_dequant
    assert d(a, a, a, a, 0, 2, 128, 16, 8, 1, None, None) == _capi.PI_OK
    assert d(a, a, a, a, 1, 2, 128, 16, 8, 7, None, None) == _capi.PI_ERR_UNSUPPORTED
    assert d(a, a, a, a, -1, 2, 128, 16, 8, 1, None, None) == _capi.PI_ERR_BAD_SHAPE
    assert d(a, None, a, a, 1, 2, 128, 16, 8, 1, None, None) == _capi.PI_ERR_NULL_POINTER
    assert d(a, a, ctypes.c_void_p(257), a, 1, 2, 128, 16, 8, 1, None, None) == _capi.PI_ERR_MISALIGNED


def test_one_zeroed_block_for_every_decode_attention():
    # 16-bit and 8-bit calls may share a workspace: what either needs zeroed, neither writes over
    _build.build()
    lib = _capi.load()
    assert lib.pi_paged_decode_attn_q8_ws_zero_bytes() == lib.pi_paged_decode_attn_ws_zero_bytes()


@pytest.mark.parametrize("hidden", [False, True], ids=["workspace", "hidden"])
def test_a_call_is_not_split_by_another_thread(monkeypatch, hidden):
    # a call is several launches over one scratch: while one thread is in it, another with the same
    # stream and scratch has to wait (the C call releases the interpreter lock)
    ws = kernels.Workspace(torch.device("cpu"))
    monkeypatch.setattr(kernels, "_check_one_device", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(kernels, "_q8_decode_workspace_bytes", lambda *a: 4096)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 7, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setitem(kernels._q8_ws, (0, 7), ws)
    inside, most, done = [0], [0], []

    def call_on(device, func, *args):
        inside[0] += 1
        most[0] = max(most[0], inside[0])
        time.sleep(0.1)
        inside[0] -= 1
        done.append(func)

    monkeypatch.setattr(kernels, "_call_on", call_on)

    def work():
        a = _args()
        kernels.paged_decode_attention_q8(**a, out=torch.empty_like(a["q"]), workspace=None if hidden else ws)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(done) == 3 and most[0] == 1


def test_workspace_gives_what_was_asked_for(monkeypatch):
    # a thread that finds the buffer large enough gets it, whatever another does meanwhile
    ws = kernels.Workspace(torch.device("cpu"))
    short = []

    def work(n):
        for _ in range(200):
            if ws.get(n).numel() < n:
                short.append(n)

    threads = [threading.Thread(target=work, args=((1 << 20) + 4096 * i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not short


def test_page_dequant_keeps_its_copy_of_the_ids(monkeypatch):
    # strided ids are copied; the copy has to live until the launch is enqueued, or its memory may be
    # another thread's by then
    copies = []
    real = torch.Tensor.contiguous

    def contiguous(t, *a):
        c = real(t, *a)
        if c is not t:
            copies.append(weakref.ref(c))
        return c

    def call_on(device, func, *args):
        assert len(copies) == 1 and copies[0]() is not None and copies[0]().data_ptr() in args

    monkeypatch.setattr(torch.Tensor, "contiguous", contiguous)
    monkeypatch.setattr(kernels, "_check_one_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(kernels, "_call_on", call_on)
    kernels.page_dequant(torch.zeros(4, 2, 16, 64).to(E4M3), torch.ones(4, 2),
                         torch.zeros(6, dtype=torch.int32)[::2])
    assert len(copies) == 1


def test_capture_on_another_device_takes_the_graphs_memory(monkeypatch):
    # q on a device that is not the current one, whose stream is being captured: the scratch must not
    # be the one that eager calls on that stream use
    current = [0]

    class On:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *a):
            current[0] = self.before

    kept = kernels.Workspace(torch.device("cpu"))
    kept.get(1 << 21)
    real_empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: real_empty(*a, **{**k, "device": "cpu"}))
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == 1)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 7, raising=False)
    monkeypatch.setattr(kernels, "_check_one_device", lambda *t: torch.device("cuda", 1))
    monkeypatch.setattr(kernels, "_q8_decode_workspace_bytes", lambda *a: 1 << 21)
    monkeypatch.setitem(kernels._q8_ws, (1, 7), kept)
    _build.build()
    seen = []
    monkeypatch.setattr(kernels, "_call_on", lambda device, func, *args: seen.append(args))
    a = _args()
    kernels.paged_decode_attention_q8(**a, out=torch.zeros_like(a["q"]))
    assert len(seen) == 1 and kept.buf.data_ptr() not in seen[0]


@pytest.mark.parametrize("warm", [False, True])
def test_workspace_under_capture(monkeypatch, warm):
    # a workspace that would have to grow under capture is left alone: memory that only one graph's
    # replays zero must not be what another graph or an eager call finds there
    zero = []

    class Lib:
        def pi_paged_decode_attn_q8_ws_zero_bytes(self):
            zero.append(True)
            return 1024

    ws = kernels.Workspace(torch.device("cpu"))
    if warm:
        ws.get(1 << 21)
    before = ws.buf
    real_empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: real_empty(*a, **{**k, "device": "cpu"}))
    monkeypatch.setattr(_capi, "load", lambda: Lib())
    monkeypatch.setattr(kernels, "_check_one_device", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(kernels, "_q8_decode_workspace_bytes", lambda *a: 1 << 21)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    seen = []
    monkeypatch.setattr(kernels, "_call_on", lambda device, func, *args: seen.append(args))
    a = _args()
    kernels.paged_decode_attention_q8(**a, out=torch.zeros_like(a["q"]), workspace=ws)
    assert ws.buf is before and len(seen) == 1
    assert (before is not None and before.data_ptr() in seen[0]) == warm and bool(zero) != warm


def test_workspace_grows_in_few_steps():
    ws = kernels.Workspace(torch.device("cpu"))
    buffers = set()
    for i in range(1, 41):
        assert ws.get(i << 20).numel() >= i << 20
        buffers.add(ws.buf.numel())
    assert len(buffers) <= 7 and max(buffers) < 2 * (40 << 20)
