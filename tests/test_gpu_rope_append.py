"""GPU parity of the rotary append (pi_rope_append) against the 64-bit oracle.

Tolerances, from the arithmetic: the kernel works in fp32 on inputs it reads exactly, with at
most 3 roundings in the norm's scale and 2 more in applying it, cosine and sine within 2 ulp
plus one rounding for rope_scale, and two products and a sum, so a rotated element is within
16 half-steps (2^-24) of (|a| + |b|) * rope_scale with a, b the normed pair; storing adds half a
step of the output type. 8-bit values are within half an e4m3 step of that, scales and kept rows
are equal bit for bit.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import quant_kv_oracle as orc
from plastic_infer_b200 import _capi, kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
_T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn


def np64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().float().double().numpy()


def half_step(dt: torch.dtype) -> float:
    return torch.finfo(dt).eps / 2


def make(T, Hq, Hkv, D, R, dtype, norm, seed=0, spread=False):
    g = torch.Generator().manual_seed(seed)
    mk = lambda h: torch.randn((T, h, D), generator=g)  # noqa: E731
    q, k, v = mk(Hq), mk(Hkv), mk(Hkv)
    if spread:  # rows of very different sizes, so block scales grow
        k = k * torch.exp(2 * torch.randn((T, Hkv, 1), generator=g))
        v = v * torch.exp(2 * torch.randn((T, Hkv, 1), generator=g))
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(DEV) for _ in range(2)] if norm else [None, None]
    return [x.to(dtype).to(DEV) for x in (q, k, v)] + w


def tolerance(x64: np.ndarray, R: int, il: bool, rs: float, out_dt) -> np.ndarray:
    """16 fp32 half-steps of (|a| + |b|) for each rotated element, of |x| for the others."""
    n = R // 2
    i = 2 * np.arange(n) if il else np.arange(n)
    j = i + 1 if il else i + n
    size = np.abs(x64)
    t = size.copy()
    t[..., i] = t[..., j] = (size[..., i] + size[..., j]) * rs
    return 16 * 2.0 ** -24 * t


def check_rows(got, ref, tol32, dt):
    # half a step is relative down to the smallest normal value and the same absolute size below
    # it: the subnormals are spaced finfo.tiny * finfo.eps apart (2^-24 in f16, whose smallest
    # normal value is 2^-14)
    err = np.abs(got - ref)
    lim = tol32 + half_step(dt) * np.maximum(np.abs(ref) + tol32, torch.finfo(dt).tiny)
    assert (err <= lim).all(), f"max excess {(err - lim).max():.3e}"


SHAPES = [  # D, R, page
    (64, 64, 16), (128, 128, 16), (128, 64, 32), (256, 256, 16), (256, 128, 32), (128, 0, 16),
    (64, 16, 16), (80, 32, 16), (96, 96, 8), (128, 20, 16), (40, 6, 5),
]


def positions_slots(T, pages, S, seed, kind):
    g = np.random.default_rng(seed)
    if kind == "prompt":  # one request: consecutive positions over pages in random order
        start = int(g.integers(0, 5 * S))
        n = (start % S + T + S - 1) // S
        order = g.permutation(pages)[:n]
        rows = start % S + np.arange(T)
        return start + np.arange(T), order[rows // S] * S + rows % S
    slots = g.permutation(pages)[:T] * S + g.integers(0, S, T)  # one token per page
    return g.integers(0, 200000, T), slots


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_matches_oracle(dtype, shape, il):
    D, R, S = shape
    for T, Hq, Hkv, norm, kind in ((1, 4, 1, True, "step"), (37, 6, 3, False, "step"),
                                   (70, 8, 2, True, "prompt")):
        dt = _T[dtype]
        pages = max(T + 3, 8)
        q, k, v, qw, kw = make(T, Hq, Hkv, D, R, dt, norm, seed=T + D)
        pos, slots = positions_slots(T, pages, S, T, kind)
        inv, rs = kernels.rope_frequencies(R, 1e4, "yarn", 4.0, 4096) if R else (torch.zeros(0), 1.0)
        kp = torch.randn((pages, Hkv, S, D), device=DEV).to(dt)
        vp = torch.randn((pages, Hkv, S, D), device=DEV).to(dt)
        k0, v0 = kp.clone(), vp.clone()
        out = kernels.rope_append(q, k, v, torch.from_numpy(pos).to(DEV), inv.to(DEV),
                                  torch.from_numpy(slots).to(DEV), kp, vp, qw, kw,
                                  interleaved=il, rope_scale=rs)
        torch.cuda.synchronize()
        wq = None if qw is None else np64(qw)
        wk = None if kw is None else np64(kw)
        f = inv.double().numpy()
        for x, w, got in ((q, wq, np64(out)), (k, wk, None)):
            ref = orc.rope_rows(np64(x), pos, f, il, rs, w)
            plain = orc.rope_rows(np64(x), pos, f[:0], il, rs, w)
            tol = tolerance(plain, R, il, rs, dt)
            if got is None:
                got = np64(kp[torch.from_numpy(slots // S), :, torch.from_numpy(slots % S)])
            check_rows(got, ref, tol, dt)
        # V bit for bit, and nothing else written
        page, off = torch.from_numpy(slots // S), torch.from_numpy(slots % S)
        assert torch.equal(vp[page, :, off], v)
        k0[page, :, off] = kp[page, :, off]
        v0[page, :, off] = v
        assert torch.equal(kp, k0) and torch.equal(vp, v0)


def test_append_far_positions_keep_their_precision():
    # at position 2^24 - 3 the fp32 product pos * inv_freq is off by up to half a radian
    T, D = 64, 128
    q, k, v, _, _ = make(T, 2, 1, D, D, torch.float32, False)
    pos = np.arange(T) + 2 ** 24 - 3
    inv, _ = kernels.rope_frequencies(D, 1e6)
    kp = torch.zeros((8, 1, 16, D), device=DEV)
    vp = torch.zeros_like(kp)
    out = kernels.rope_append(q, k, v, torch.from_numpy(pos).to(DEV), inv.to(DEV),
                              torch.arange(T, device=DEV), kp, vp)
    ref = orc.rope_rows(np64(q), pos, inv.double().numpy())
    check_rows(np64(out), ref, tolerance(np64(q), D, False, 1.0, None), torch.float32)


def test_append_agrees_with_decode_prologue():
    # where the fp32 angle is exact enough (small positions) the two entry points agree
    T, Hq, Hkv, D, S = 33, 8, 2, 128, 16
    q, k, v, qw, kw = make(T, Hq, Hkv, D, D, torch.bfloat16, True)
    pos = torch.arange(T, device=DEV)
    inv = kernels.rope_inv_freq(D, 1e6, DEV)
    slots = torch.randperm(T, device=DEV) * S
    pools = [torch.zeros((T, Hkv, S, D), dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    a = kernels.decode_prologue(q, k, v, pos, inv, slots, pools[0], pools[1], qw, kw)
    b = kernels.rope_append(q, k, v, pos, inv, slots, pools[2], pools[3], qw, kw)
    for x, y in ((a, b), (pools[0], pools[2])):
        assert (np.abs(np64(x) - np64(y)) <= 2.0 ** -7 * np.abs(np64(y)) + 1e-4).all()
    assert torch.equal(pools[1], pools[3])


def test_append_converts_to_the_pool_type_and_takes_strides():
    T, Hq, Hkv, D, S = 19, 4, 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(5)
    for width in (8 * D, 8 * D + 3):  # the second row stride is odd: the generic kernel
        qkv = torch.randn((T, width), device=DEV, generator=g)
        q = qkv[:, :Hq * D].unflatten(1, (Hq, D))
        k = qkv[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
        v = qkv[:, (Hq + Hkv) * D:8 * D].unflatten(1, (Hkv, D))
        pos = torch.arange(T, device=DEV) + 7
        inv = kernels.rope_inv_freq(D, 1e4, DEV)
        slots = torch.arange(T, device=DEV) + 3
        slots[4] = -1
        kp, vp = (torch.zeros((3, Hkv, S, D), dtype=torch.float16, device=DEV) for _ in range(2))
        wide = torch.zeros((T, Hq + 1, D), dtype=torch.float16, device=DEV)
        out = kernels.rope_append(q, k, v, pos, inv, slots, kp, vp, q_out=wide[:, :Hq])
        assert out.data_ptr() == wide.data_ptr() and int(wide[:, Hq].count_nonzero()) == 0
        ref = orc.rope_rows(np64(q), pos.cpu().numpy(), np64(inv))
        check_rows(np64(out), ref, tolerance(np64(q), D, False, 1.0, None), torch.float16)
        live = slots >= 0
        s = slots[live]
        assert torch.equal(vp[s // S, :, s % S], v[live].half())
        assert int(vp[4 // S, :, 7].count_nonzero()) == 0


def settle(k64, tol, slots, scale, page_size):
    """A block's exponent goes by its largest fp32 value, which is within tol of the exact one: an
    exact amax within tol of 448 * 2^e leaves e and e + 1 both right. The exact value is moved
    across that border, by tol at most, where the kernel's value lay on its other side."""
    for t, page, off, n in orc.runs(slots, page_size):
        for h in range(k64.shape[1]):
            new = k64[t:t + n, h]
            at = np.unravel_index(np.abs(new).argmax(), new.shape)
            top, room, s = abs(new[at]), tol[t:t + n, h][at], scale[page, h]
            if 448 * s < top <= 448 * s + room:
                np.clip(new, -448 * s, 448 * s, out=new)
            elif off == 0 and 224 * s - room <= top <= 224 * s:
                new[at] = np.sign(new[at]) * 224 * s * (1 + 1e-12)


def run_q8(T, Hq, Hkv, D, R, S, dtype, norm, il, kind, seed, steps=1):
    dt = _T[dtype]
    pages = max(2 * T + 6, 16)
    g = torch.Generator().manual_seed(seed)
    kp = (torch.randn((pages, Hkv, S, D), generator=g) * 60).to(E4M3).to(DEV)
    vp = (torch.randn((pages, Hkv, S, D), generator=g) * 60).to(E4M3).to(DEV)
    ks = torch.exp2(torch.randint(-9, -5, (pages, Hkv), generator=g).float()).to(DEV)
    vs = torch.exp2(torch.randint(-9, -5, (pages, Hkv), generator=g).float()).to(DEV)
    rk, rv, rks, rvs = np64(kp), np64(vp), np64(ks), np64(vs)
    q, k, v, qw, kw = make(T, Hq, Hkv, D, R, dt, norm, seed=seed + 1, spread=True)
    pos, slots = positions_slots(T, pages, S, seed, kind)
    inv, rs = kernels.rope_frequencies(R, 1e4, "linear", 2.0) if R else (torch.zeros(0), 1.0)
    out = kernels.rope_append(q, k, v, torch.from_numpy(pos).to(DEV), inv.to(DEV),
                              torch.from_numpy(slots).to(DEV), kp, vp, qw, kw, interleaved=il,
                              rope_scale=rs, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    f = inv.double().numpy()
    k64 = orc.rope_rows(np64(k), pos, f, il, rs, None if kw is None else np64(kw))
    tol = tolerance(orc.rope_rows(np64(k), pos, f[:0], il, rs, None if kw is None else np64(kw)),
                    R, il, rs, None)
    before = rk.copy(), rv.copy()
    settle(k64, tol, slots, np64(ks), S)
    orc.append_q8(k64, slots, rk, rks)
    orc.append_q8(np64(v), slots, rv, rvs)
    return out, dt, (kp, vp, ks, vs), (rk, rv, rks, rvs), before, (k64, tol, np64(v), slots), (q, qw, pos, f, il, rs, R)


@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_append_8bit_matches_oracle(dtype, shape, il):
    D, R, S = shape
    for T, Hq, Hkv, norm, kind in ((1, 2, 1, True, "step"), (29, 4, 3, False, "step"),
                                   (75, 4, 2, True, "prompt"), (700, 2, 2, False, "prompt")):
        out, dt, got, ref, _, (k64, tol, v64, slots), qs = run_q8(
            T, Hq, Hkv, D, R, S, dtype, norm, il, kind, seed=T + D + S)
        kp, vp, ks, vs = got
        rk, rv, rks, rvs = ref
        assert np.array_equal(np64(ks), rks) and np.array_equal(np64(vs), rvs)
        # V comes from exact inputs: equal everywhere, kept rows and untouched rows included
        assert np.array_equal(np64(vp), rv)
        # K: new rows within half an e4m3 step of the fp32 value; every other row equal
        page, off = slots // S, slots % S
        new = np.zeros(rk.shape[:1] + rk.shape[2:3], dtype=bool)
        new[page, off] = True
        g = np64(kp)
        assert np.array_equal(g.transpose(0, 2, 1, 3)[~new], rk.transpose(0, 2, 1, 3)[~new])
        s = rks[page][:, :, None]
        vals = g[page, :, off] * s
        step = np.maximum(2.0 ** -4 * (np.abs(k64) + tol), 2.0 ** -10 * s)
        assert (np.abs(vals - k64) <= tol + step * (1 + 1e-9)).all()
        q, qw, pos, f, il_, rs, R_ = qs
        w = None if qw is None else np64(qw)
        plain = orc.rope_rows(np64(q), pos, f[:0], il_, rs, w)
        check_rows(np64(out), orc.rope_rows(np64(q), pos, f, il_, rs, w),
                   tolerance(plain, R_, il_, rs, dt), dt)


@pytest.mark.parametrize("shape", [(128, 16), (64, 32), (80, 16)])
def test_append_8bit_token_by_token(shape):
    # a request that grows by one token per call: V of the kept rows is rescaled as the oracle
    # does it, step by step, and a page that is taken up again starts anew
    D, S = shape
    Hkv, T = 2, 2 * S + 3
    q, k, v, _, _ = make(T, 2, Hkv, D, D, torch.bfloat16, False, seed=3, spread=True)
    kp, vp = (torch.full((4, Hkv, S, D), 0x7F, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    ks, vs = (torch.full((4, Hkv), math.nan, device=DEV) for _ in range(2))
    rv, rvs = np64(vp), np64(vs)
    inv = kernels.rope_inv_freq(16, 1e4, DEV)
    order = [2, 0, 2]  # the third page is the first one again
    for t in range(T):
        slot = order[t // S] * S + t % S
        kernels.rope_append(q[t:t + 1], k[t:t + 1], v[t:t + 1], torch.tensor([t], device=DEV), inv,
                            torch.tensor([slot], device=DEV), kp, vp, k_scale=ks, v_scale=vs)
        orc.append_q8(np64(v[t:t + 1]), [slot], rv, rvs)
    assert np.array_equal(np64(vs), rvs, equal_nan=True)
    assert np.array_equal(np64(vp), rv, equal_nan=True)


@pytest.mark.parametrize("D", [128, 72])
def test_append_8bit_odd_values(D):
    # zeros, infinities, NaN, the smallest and largest finite values
    S, Hkv = 16, 5
    kp, vp = (torch.zeros((2, Hkv, S, D), dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2))
    ks, vs = (torch.ones((2, Hkv), device=DEV) for _ in range(2))
    rows = torch.zeros((3, Hkv, D))
    rows[:, 1] = 3.0
    rows[1, 1, 5] = math.inf
    rows[2, 1, 6] = -math.inf
    rows[1, 2, 7] = math.nan
    rows[0, 2, 8] = 448.0
    rows[:, 3] = 1e-44
    rows[0, 4] = 3.3e38
    rows[1, 4] = -448.0
    rows = rows.to(DEV)
    slots = torch.arange(3, device=DEV)
    kernels.rope_append(rows, rows, rows, slots, torch.zeros(0, device=DEV), slots, kp, vp,
                        k_scale=ks, v_scale=vs)
    rv, rvs = np.zeros((2, Hkv, S, D)), np.ones((2, Hkv))
    orc.append_q8(np64(rows), [0, 1, 2], rv, rvs)
    for pool, sc in ((kp, ks), (vp, vs)):
        assert np.array_equal(np64(sc), rvs)
        assert np.array_equal(np64(pool), rv, equal_nan=True)


def test_append_padding_and_bad_slots():
    T, Hq, Hkv, D, S, P = 6, 4, 2, 128, 16, 5
    for eight in (False, True):
        q, k, v, _, _ = make(T, Hq, Hkv, D, D, torch.bfloat16, False)
        dt = E4M3 if eight else torch.bfloat16
        kp, vp = (torch.zeros((P, Hkv, S, D), device=DEV).to(dt) for _ in range(2))
        sc = dict(k_scale=torch.ones((P, Hkv), device=DEV), v_scale=torch.ones((P, Hkv), device=DEV)) if eight else {}
        slots = torch.tensor([3, -1, 40, P * S + 4, -7, 2 ** 40], device=DEV)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        pos = torch.arange(T, device=DEV)
        inv = kernels.rope_inv_freq(D, 1e4, DEV)
        out = kernels.rope_append(q, k, v, pos, inv, slots, kp, vp, err=err, **sc)
        assert int(err.item()) == _capi.PI_ERR_SLOT_RANGE
        written = (vp.float() != 0).any(-1).any(1).nonzero().cpu().tolist()
        assert written == [[0, 3], [2, 8]]
        ref = orc.rope_rows(np64(q), pos.cpu().numpy(), np64(inv))  # q of every token
        check_rows(np64(out), ref, tolerance(np64(q), D, False, 1.0, None), torch.bfloat16)


def test_append_in_a_graph_and_on_another_stream():
    T, Hq, Hkv, D, S = 48, 4, 2, 128, 16
    q, k, v, _, _ = make(T, Hq, Hkv, D, D, torch.bfloat16, False)
    pos = torch.arange(T, device=DEV)
    inv = kernels.rope_inv_freq(D, 1e4, DEV)
    slots = torch.arange(T, device=DEV)

    def pools():
        return ([torch.zeros((4, Hkv, S, D), device=DEV).to(E4M3) for _ in range(2)]
                + [torch.ones((4, Hkv), device=DEV) for _ in range(2)])

    a, b = pools(), pools()
    run = lambda p: kernels.rope_append(q, k, v, pos, inv, slots, p[0], p[1], k_scale=p[2], v_scale=p[3])  # noqa: E731
    want = run(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        run(b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    c = pools()
    with torch.cuda.graph(graph):
        got = run(c)
    for p in c[:2]:
        p.view(torch.uint8).fill_(0x7F)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for x, y in zip(a[:2], c[:2]):  # the rows of the three pages that the run fills
        assert torch.equal(x.view(torch.uint8)[:3], y.view(torch.uint8)[:3])
    assert torch.equal(a[2][:3], c[2][:3]) and torch.equal(a[3][:3], c[3][:3])
