"""Host side of the rotary append: frequencies, refusals and the C entry point's validation."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import quant_kv_oracle as orc
from plastic_infer_b200 import _build, _capi, kernels


def test_frequencies():
    plain, one = kernels.rope_frequencies(64, 1e4)
    assert one == 1.0
    want = 1e4 ** -(np.arange(0, 64, 2) / 64)
    np.testing.assert_allclose(plain.numpy(), want, rtol=2 ** -23)
    half, one = kernels.rope_frequencies(64, 1e4, "linear", 4.0)
    np.testing.assert_allclose(half.numpy(), want / 4, rtol=2 ** -23)
    ntk, _ = kernels.rope_frequencies(64, 1e4, "ntk", 4.0)
    np.testing.assert_allclose(ntk[0], want[0], rtol=2 ** -23)
    np.testing.assert_allclose(ntk[-1], want[-1] / 4, rtol=2 ** -22)
    yarn, scale = kernels.rope_frequencies(64, 1e4, "yarn", 4.0, 4096)
    assert scale == pytest.approx(0.1 * math.log(4.0) + 1)
    turns = 4096 * want / (2 * math.pi)
    fast, slow = turns > 40, turns < 0.7
    assert fast.any() and slow.any()
    np.testing.assert_allclose(yarn.numpy()[fast], want[fast], rtol=2 ** -23)
    np.testing.assert_allclose(yarn.numpy()[slow], want[slow] / 4, rtol=2 ** -23)
    assert (yarn.numpy() <= want * (1 + 1e-6)).all() and (yarn.numpy() >= want / 4 * (1 - 1e-6)).all()


@pytest.mark.parametrize("args", [(0, 1e4), (7, 1e4), (64, 1e4, "other"), (64, 1e4, "linear", 0.5),
                                  (2, 1e4, "ntk", 2.0), (64, 1e4, "yarn", 2.0)])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        kernels.rope_frequencies(*args)


def _args(T=3, Hq=4, Hkv=2, D=64, S=16, P=4, dtype=torch.bfloat16, pool=None):
    z = torch.zeros
    return dict(q=z((T, Hq, D), dtype=dtype), k=z((T, Hkv, D), dtype=dtype), v=z((T, Hkv, D), dtype=dtype),
                positions=z(T, dtype=torch.int64), inv_freq=z(D // 2), slot_mapping=z(T, dtype=torch.int64),
                k_pool=z((P, Hkv, S, D), dtype=pool or dtype), v_pool=z((P, Hkv, S, D), dtype=pool or dtype))


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(3, 1, 64, dtype=torch.bfloat16)), ValueError),
    (dict(v=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.zeros(3, 2, 64)), TypeError),
    (dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), ValueError),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(inv_freq=torch.zeros(33)), ValueError),
    (dict(inv_freq=torch.zeros(32, dtype=torch.float64)), ValueError),
    (dict(v_pool=torch.zeros(4, 2, 16, 64)), ValueError),
    (dict(q_norm_weight=torch.ones(64)), ValueError),
    (dict(q_norm_weight=torch.ones(32), k_norm_weight=torch.ones(32)), ValueError),
    (dict(k_scale=torch.ones(4, 2), v_scale=torch.ones(4, 2)), ValueError),
    (dict(q_out=torch.zeros(3, 4, 64)), ValueError),
    (dict(), ValueError),  # nothing wrong but the device
])
def test_append_refuses(change, error):
    with pytest.raises(error):
        kernels.rope_append(**{**_args(), **change})


@pytest.mark.parametrize("scales", [(None, None), (torch.ones(4, 2), None), (torch.ones(4, 1), torch.ones(4, 1)),
                                    (torch.ones(4, 2, dtype=torch.float64),) * 2,
                                    (torch.ones(2, 4).t(), torch.ones(2, 4).t())])
def test_append_8bit_refuses_scales(scales):
    with pytest.raises(ValueError, match="scale"):
        kernels.rope_append(**_args(pool=torch.float8_e4m3fn), k_scale=scales[0], v_scale=scales[1])


def test_c_entry_validates_before_launch():
    _build.build()
    f = _capi.load().pi_rope_append
    a = ctypes.c_void_p(256)
    # q_out, q_out_stride, k_pool, v_pool, k_scale, v_scale, q, q_stride, k, k_stride, v, v_stride,
    # in_dtype, qw, kw, eps, inv_freq, pairs, interleaved, rope_scale, positions, slots, n, hq, hkv,
    # d, s, pages, pool_dtype, err, stream
    base = [a, 256, a, a, None, None, a, 256, a, 128, a, 128, _capi.PI_DTYPE_BF16, None, None, 1e-5,
            a, 32, 0, 1.0, a, a, 4, 4, 2, 64, 16, 8, _capi.PI_DTYPE_BF16, None, None]

    def rc(**change):
        x = list(base)
        for i, v in change.items():
            x[int(i[1:])] = v
        return f(*x)

    assert rc(_22=0) == _capi.PI_OK
    assert rc(_12=9) == _capi.PI_ERR_UNSUPPORTED
    assert rc(_28=9) == _capi.PI_ERR_UNSUPPORTED
    assert rc(_12=_capi.PI_DTYPE_E4M3) == _capi.PI_ERR_UNSUPPORTED
    assert rc(_17=33) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_17=-1) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_22=-1) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_1=255) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_9=100) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_11=100) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_15=-1.0) == _capi.PI_ERR_BAD_SHAPE
    assert rc(_0=None) == _capi.PI_ERR_NULL_POINTER
    assert rc(_16=None) == _capi.PI_ERR_NULL_POINTER
    assert rc(_13=a) == _capi.PI_ERR_NULL_POINTER
    assert rc(_28=_capi.PI_DTYPE_E4M3) == _capi.PI_ERR_NULL_POINTER  # no scales
    assert rc(_6=ctypes.c_void_p(257)) == _capi.PI_ERR_MISALIGNED
    assert rc(_20=ctypes.c_void_p(260)) == _capi.PI_ERR_MISALIGNED


def test_oracle_rounding_is_torchs():
    # the oracle's e4m3 rounding against torch's conversion, over every half-way point
    v = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (v[1:] + v[:-1]) / 2
    x = torch.cat([v, mid, mid * (1 + 1e-6), mid * (1 - 1e-6)])
    x = torch.cat([x, -x])
    assert np.array_equal(orc.e4m3_round(x.numpy()),
                          x.float().to(torch.float8_e4m3fn).double().numpy())
    for top, e in ((448.0, 0), (448.1, 1), (1.75, -8), (1.7500001, -7), (0.0, -118), (1e-44, -118)):
        assert orc.block_exp(np.array([top, -0.1 * top])) == e


def test_c_entry_refuses_misaligned_weights():
    # an address that the type's loads would fault on
    _build.build()
    f = _capi.load().pi_rope_append
    a = ctypes.c_void_p(256)
    for dtype, size in ((_capi.PI_DTYPE_BF16, 2), (_capi.PI_DTYPE_F16, 2), (_capi.PI_DTYPE_F32, 4)):
        for qw, kw in ((256 + size // 2, 256), (256, 256 + size // 2)):
            args = [a, 256, a, a, None, None, a, 256, a, 128, a, 128, dtype, ctypes.c_void_p(qw), ctypes.c_void_p(kw),
                    1e-5, a, 32, 0, 1.0, a, a, 0, 4, 2, 64, 16, 8, dtype, None, None]
            assert f(*args) == _capi.PI_OK  # no tokens: nothing is looked at
            args[22] = 4
            assert f(*args) == _capi.PI_ERR_MISALIGNED


def test_one_head_of_any_stride_is_taken():
    # refused for the device alone: [1, T, D] transposed has a head stride of T * D
    x = torch.zeros((1, 3, 64), dtype=torch.bfloat16).transpose(0, 1)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.rope_append(**{**_args(Hq=1, Hkv=1), "q": x, "k": x, "v": x}, q_out=x.clone(memory_format=torch.preserve_format))
