"""Refusals of the 8-bit cache attention: the wrappers' checks and the C entry points' validation."""

from __future__ import annotations

import ctypes

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
