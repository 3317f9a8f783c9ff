"""8-bit caches for the attention tests, and the bound their outputs have to keep."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import quant_kv_oracle as orc

DEV = torch.device("cuda", 0)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn


def np64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().float().double().numpy()


def cache(lens, Hkv, D, S, seed, extra=3, width=None, spread=1.0, plain_scales=False):
    """Pools, scales, block tables and lengths for requests of the given lengths. Rows behind a
    request's last token and pages of nobody hold NaN; the tables' unused entries name pages that
    do not exist."""
    g = torch.Generator().manual_seed(seed)
    spans = [-(-n // S) for n in lens]
    P = sum(spans) + extra
    W = max(max(spans, default=1), 1) if width is None else width
    kp, vp = ((torch.randn((P, Hkv, S, D), generator=g) * 80).to(E4M3) for _ in range(2))
    if plain_scales:  # any positive scale, zero among them
        ks, vs = (torch.rand((P, Hkv), generator=g) * 0.02 for _ in range(2))
        vs[::3] = 0.0
    else:
        ks, vs = (torch.exp2(torch.round(torch.randn((P, Hkv), generator=g) * spread) - 7) for _ in range(2))
    order = torch.randperm(P, generator=g)
    tables = torch.full((len(lens), W), 2 ** 30, dtype=torch.int32)
    at = 0
    for b, (n, span) in enumerate(zip(lens, spans)):
        ids = order[at:at + span]
        tables[b, :span] = ids.int()
        at += span
        if n % S:
            for pool in (kp, vp):
                pool.view(torch.uint8)[ids[-1], :, n % S:] = 0x7F
    for pool, sc in ((kp, ks), (vp, vs)):
        pool.view(torch.uint8)[order[at:]] = 0xFF
        sc[order[at:]] = math.nan
    return dict(k_pool=kp, v_pool=vp, k_scale=ks, v_scale=vs, tables=tables,
                lens=torch.tensor(lens, dtype=torch.int32), spans=spans)


def on_gpu(c):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def reference(q, c, lens, rows_of=None, scale=None):
    """(64-bit outputs, the bound on each element) for q [B, Hq, D]; rows_of maps a query row to its
    request (itself unless given).

    With x the scores, A the softmax-weighted mean of |V| and N = D / 32 * parts MMAs per score:
    - a score: an MMA keeps terms to 2^-21 of the largest of 33, which is at most L = sum |q_d k_d|,
      so N * 33 * 2^-21 * L; q's parts miss at most 2^-17 of its largest element in each product
      (bf16 exactly, f16 2^-12 of the element: 2^-12 L); fp32 rounding of the scaling and exp2.approx
      (2^-22) are below 2^-12 * |x| + 2^-20. Shifting scores by d moves the output by at most 2 d A;
    - a weight: two parts keep 2^-8 of it, three 2^-12, and 2^-17 of its unit's largest;
    - the sums of P V: 2^-16 A at most, and half a step of the output type."""
    B, Hq, D = q.shape
    kp, vp = np64(c["k_pool"]), np64(c["v_pool"])
    ks, vs = np64(c["k_scale"]), np64(c["v_scale"])
    tables = c["tables"].cpu().numpy()
    rows_of = list(range(B)) if rows_of is None else rows_of
    t = [tables[r] for r in rows_of]
    q64 = np64(q)
    H, S = kp.shape[1], kp.shape[2]
    sc = 1.0 / math.sqrt(D) if scale is None else scale
    ref = orc.attention_q8(q64, kp, vp, ks, vs, t, lens, scale)
    mean_abs = orc.attention_q8(q64, kp, np.abs(vp), ks, vs, t, lens, scale)
    dt = q.dtype
    parts, p_err = {torch.bfloat16: (2, 2.0 ** -8), torch.float16: (3, 2.0 ** -12),
                    torch.float32: (0, 0.0)}[dt]
    G = Hq // H
    tol = np.zeros_like(ref)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        ids = np.asarray(t[b][:-(-n // S)], dtype=np.int64)
        k = (kp[ids] * ks[ids][:, :, None, None]).transpose(1, 0, 2, 3).reshape(H, -1, D)[:, :n]
        for h in range(Hq):
            qa, ka = np.abs(q64[b, h]), np.abs(k[h // G])
            L = float((ka @ qa).max()) * abs(sc)
            K1 = float(ka.sum(-1).max()) * abs(sc) * qa.max()
            d = max(D // 32 * parts * 33 * 2.0 ** -21, 2.0 ** -17) * L + 2.0 ** -17 * K1 + 2.0 ** -12 * L * (dt != torch.float32) \
                + 2.0 ** -20
            tol[b, h] = (2 * d + p_err + 2.0 ** -15) * mean_abs[b, h]
    half = torch.finfo(dt).eps / 2
    tol += half * np.maximum(np.abs(ref) + tol, torch.finfo(dt).tiny) + 2.0 ** -20 * mean_abs
    return ref, tol


def check(got: torch.Tensor, ref: np.ndarray, tol: np.ndarray) -> None:
    x = np64(got)
    assert np.isfinite(x).all(), "non-finite output"
    err = np.abs(x - ref)
    assert (err <= tol).all(), f"max excess {(err - tol).max():.3e}, max err {err.max():.3e}"
    # the bounds are worst cases; the 2-norm is held to the half steps of output and weights
    norm = np.linalg.norm(ref)
    lim = {torch.bfloat16: 2.0 ** -8 + 2.0 ** -8, torch.float16: 2.0 ** -11 + 2.0 ** -11,
           torch.float32: 2.0 ** -18}[got.dtype]
    assert np.linalg.norm(err) <= lim * norm + 1e-30, f"rel {np.linalg.norm(err) / norm:.3e}"
