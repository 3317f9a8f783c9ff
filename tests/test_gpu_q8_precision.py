"""How exact the attention over an 8-bit cache is, held to the arithmetic of the tensor-core kernels.

With x the scores, A the softmax-weighted mean of |V|, L = |scale| sum |q_d k_d| and eps(f16) = 2^-10:
- K and V are widened without loss; q is scaled by a power of two that brings its row's largest
  element into [128, 256) and rounded to f16: exact down to 2^-21 of that element, and half a
  subnormal step (2^-25 against 2^7) below: 2^-32 of it in each product;
- a score's products are exact, their sums fp32, D / 16 MMAs that keep 2^-21 of the largest of their
  17 terms at worst: D / 16 * 17 * 2^-21 L is the worst case, but the terms of one MMA that come near
  the largest are few; 2^-18 L is allowed; scaling and exp2.approx: 2^-20 |x| + 2^-20;
- a shift of the scores by d moves the output by at most 2 d A;
- P is rounded to f16 relative to its unit's largest weight: half a step is 2^-11 of the weight, or 2^-33 of
  the unit's largest (times the larger V scale of its two pages: cases with equal scales here);
- sums of P V and their scaling: 2^-16 A; then half a step of the output's type.
The widening path (many rows) has P in q's type, so 2^-8 in bf16, and P's largest is not its tile's but
up to 2^8 below the running maximum's: no more than the same relative step.

The inputs are made so that these terms show: V rows that cancel, so that the output is far smaller than
A and its own rounding hides nothing; q rows whose largest element meets zeros in K.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import quant_kv_oracle as orc
from plastic_infer_b200 import kernels
from tests._q8 import DEV, E4M3, TYPES, np64

pytestmark = pytest.mark.gpu


def pools(n, Hkv, D, S, seed, cancel, hollow):
    """A request of n tokens in consecutive pages. cancel: V rows come in pairs, one the other's negative,
    whose keys differ in one element, so their weights nearly cancel too. hollow: K's first column is
    zero."""
    g = torch.Generator().manual_seed(seed)
    P = -(-n // S)
    k = torch.randn((Hkv, P * S, D), generator=g) * 40
    v = torch.randn((Hkv, P * S, D), generator=g) * 80
    if cancel:
        v[:, 1::2] = -v[:, ::2]
        k[:, 1::2, 1:] = k[:, ::2, 1:]
    if hollow:
        k[..., 0] = 0
    kp, vp = (x.view(Hkv, P, S, D).transpose(0, 1).contiguous().to(E4M3) for x in (k, v))
    ks, vs = (torch.full((P, Hkv), 2.0 ** -6) for _ in range(2))
    return kp, vp, ks, vs


def bounds(q, kp, vp, ks, vs, lens, p_err):
    """(64-bit outputs, bound on each element) for the query rows over the first lens[i] tokens."""
    B, Hq, D = q.shape
    q64, K, V, a, b = np64(q), np64(kp), np64(vp), np64(ks), np64(vs)
    P, H, S = K.shape[:3]
    t = [np.arange(P)] * B
    ref = orc.attention_q8(q64, K, V, a, b, t, lens)
    mean_abs = orc.attention_q8(q64, K, np.abs(V), a, b, t, lens)
    k = (K * a[:, :, None, None]).transpose(1, 0, 2, 3).reshape(H, -1, D)
    tol = np.zeros_like(ref)
    for i in range(B):
        for h in range(Hq):
            ka, qa = np.abs(k[h // (Hq // H)][:lens[i]]), np.abs(q64[i, h])
            L = float((ka @ qa).max()) / math.sqrt(D)
            low = 2.0 ** -32 * qa.max() * float(ka.sum(-1).max()) / math.sqrt(D)
            d = 2.0 ** -18 * L + low + 2.0 ** -20 * (L + 1)
            tol[i, h] = (2 * d + p_err + 2.0 ** -16) * mean_abs[i, h]
    half = torch.finfo(q.dtype).eps / 2
    return ref, tol + half * np.maximum(np.abs(ref) + tol, torch.finfo(q.dtype).tiny)


def held(got, ref, tol):
    err = np.abs(np64(got) - ref)
    assert (err <= tol).all(), f"{(err / tol).max():.2f} of the bound"


@pytest.mark.parametrize("kind", ["plain", "cancel", "hollow"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,G,D,S", [(2, 4, 128, 16), (32, 8, 128, 16), (100, 1, 64, 32), (1000, 4, 128, 32),
                                     (300, 5, 256, 16)])
def test_decode(dtype, kind, n, G, D, S):
    Hkv, B = 2, 3
    c = pools(n, Hkv, D, S, n + D, kind == "cancel", kind == "hollow")
    g = torch.Generator().manual_seed(n)
    q = torch.randn((B, Hkv * G, D), generator=g)
    if kind == "hollow":
        q[..., 0] = 2.0 ** 9 * 1.7
    q = q.to(TYPES[dtype])
    lens = [n, max(1, n - 1), max(1, n // 2)]
    gpu = [x.to(DEV) for x in c]
    tables = torch.arange(c[0].shape[0], dtype=torch.int32, device=DEV)[None].expand(B, -1)
    got = kernels.paged_decode_attention_q8(q.to(DEV), *gpu, tables, torch.tensor(lens, dtype=torch.int32, device=DEV))
    held(got, *bounds(q, *c, lens, 2.0 ** -11))


@pytest.mark.parametrize("kind", ["plain", "cancel", "hollow"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,start,G,D,S", [(17, 200, 4, 128, 16), (40, 0, 7, 64, 32), (400, 30, 8, 128, 16),
                                              (700, 0, 4, 64, 32)])
def test_prefill(dtype, kind, rows, start, G, D, S):
    Hkv, n = 2, start + rows
    c = pools(n, Hkv, D, S, rows, kind == "cancel", kind == "hollow")
    g = torch.Generator().manual_seed(rows)
    q = torch.randn((rows, Hkv * G, D), generator=g)
    if kind == "hollow":
        q[..., 0] = 2.0 ** 9 * 1.7
    q = q.to(TYPES[dtype])
    wide = rows * Hkv * G > kernels._capi.Q8_FEW_ROWS
    got = kernels.paged_prefill_attention_q8(q.to(DEV), *[x.to(DEV) for x in c],
                                             torch.arange(c[0].shape[0], dtype=torch.int32, device=DEV), n, start)
    take = sorted(set(range(0, rows, 29)) | {rows - 1})
    p_err = torch.finfo(TYPES[dtype]).eps / 2 if wide else 2.0 ** -11
    held(got[take], *bounds(q[take], *c, [start + i + 1 for i in take], p_err))
