"""Tensor-level wrappers over the C ABI (the batched entry points of the hot path).

These are the batched additions behind the reference's single-request API:

  kv_index_copy          one launch writes a whole step's new K/V rows
                         (reference: _write_kv_layer, src/plastic_infer/exec/runner_paged.py:112-129)
  paged_decode_attention one launch attends every request of the batch
                         (reference: paged_attention_v1, src/plastic_infer/exec/attention.py:151-190)
  paged_kv_gather        contiguous gather of one request
                         (reference: gather_paged_kv, src/plastic_infer/exec/attention.py:103-148)
  page_gather / page_scatter
                         pool <-> staging moves for the host store
                         (reference: src/plastic_infer/kv/kv_store.py:258-269, 311-321)
  paged_decode_attention_gather
                         decode attention of one KV-head shard with the all-gather of the
                         per-rank outputs fused in (NVLink peer stores; multi-GPU)
  decode_prologue        QK-norm + RoPE of a step's q/k rows and the K/V slot write, one
                         launch (reference: attention.py:23-95 + _write_kv_layer)
  rope_append            QK-norm + rotary positions (half or interleaved pairs, part of the head,
                         scaled) of any number of tokens and their K/V slot write, one launch;
                         16/32-bit pools, or e4m3 pools with a scale per (page, KV head)
  rope_frequencies       rotary frequencies for rope_append: plain, or scaled for long contexts
  paged_decode_attention_q8
                         decode attention over e4m3 pools with a scale per (page, KV head)
  paged_prefill_attention_q8
                         several query tokens of one request over such pools
  page_dequant           pages of such a pool widened to f32, bf16 or f16
  paged_prefill_attention
                         one request's prefill straight from the pool
                         (reference: _attn_paged, src/plastic_infer/exec/runner_paged.py:36-95)
  expert_slot_copy       MoE expert rows from pinned host banks into device slots, all banks
                         in one launch (reference: fast_index_copy_multi_jit)
  host_stream_attention  one request's attention over host-resident chunks (pinned, read in
                         place) plus a device tail (reference: host_stream_attention_v1,
                         src/plastic_infer/exec/attention.py:193-250)
  set_programmatic_launch
                         programmatic dependent launch for the index-copy, prologue and
                         attention kernels
  set_decode_attn_ring   page-ring depth of plain attention launches (automatic, deep or
                         shallow), so either kernel instance can be run at any size

Pools are the *physical* tensors [num_pages, kv_heads, page_size, head_dim]. Every
function launches on torch's current stream, as the reference's ctypes launch does
(src/plastic_infer/kernel/fast_index_copy.py:185), and raises `KernelError` on a
non-zero status. Inputs must be CUDA tensors (host_stream_attention also reads
page-locked host tensors in place); there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
import threading

import numpy as np
import torch

from . import _capi

_DTYPES = {
    torch.float32: _capi.PI_DTYPE_F32,
    torch.bfloat16: _capi.PI_DTYPE_BF16,
    torch.float16: _capi.PI_DTYPE_F16,
}


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DTYPES[dt]
    except KeyError:
        raise TypeError(f"unsupported KV dtype {dt}; expected float32, bfloat16 or float16")


def _require_cuda(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(
                "plastic_infer_b200 kernels need CUDA tensors (no CPU fallback); got "
                f"{t.device}"
            )


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _err_ptr(err: torch.Tensor | None) -> int | None:
    if err is None:
        return None
    if err.dtype != torch.int32 or not err.is_cuda or err.numel() < 1:
        raise ValueError("err must be a CUDA int32 tensor with at least one element")
    return err.data_ptr()


def _check_pool(pool: torch.Tensor, name: str) -> tuple[int, int, int, int]:
    if pool.dim() != 4 or not pool.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [num_pages, kv_heads, page_size, head_dim] tensor")
    return tuple(pool.shape)  # type: ignore[return-value]


# ---------------------------------------------------------------------------
# a1: slot-mapping index-copy
# ---------------------------------------------------------------------------


def kv_index_copy(
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_new: torch.Tensor,
    v_new: torch.Tensor,
    slot_mapping: torch.Tensor,
    err: torch.Tensor | None = None,
) -> None:
    """pool[slot // S, :, slot % S, :] = new[i] for every i with slot_mapping[i] >= 0.

    k_new / v_new: [n, kv_heads, head_dim] (any token stride, heads contiguous) or
    [1, n, kv_heads, head_dim] as produced by the reference runner.
    slot_mapping: int64 [n] on the pool's device; slot = page_id * page_size + offset.
    """
    P, H, S, D = _check_pool(k_pool, "k_pool")
    if v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype:
        raise ValueError("k_pool and v_pool must have the same shape and dtype")
    if k_new.dim() == 4:
        k_new = k_new.reshape(-1, k_new.shape[-2], k_new.shape[-1])
        v_new = v_new.reshape(-1, v_new.shape[-2], v_new.shape[-1])
    if k_new.shape != v_new.shape or tuple(k_new.shape[1:]) != (H, D):
        raise ValueError(f"k_new/v_new must be [n, {H}, {D}], got {tuple(k_new.shape)}")
    if k_new.dtype != k_pool.dtype or v_new.dtype != k_pool.dtype:
        raise TypeError("new K/V rows must have the pool dtype")
    n = k_new.shape[0]
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (n,):
        raise ValueError("slot_mapping must be int64 of shape [n]")
    _require_cuda(k_pool, v_pool, k_new, v_new, slot_mapping)
    if n == 0:
        return
    # Rows of one token must be [H, D] contiguous and K/V must share one token
    # stride; tokens themselves may be strided (e.g. slices of a fused QKV output).
    if not (k_new.stride(2) == 1 and k_new.stride(1) == D and v_new.stride() == k_new.stride()):
        k_new = k_new.contiguous()
        v_new = v_new.contiguous()
    slot_mapping = slot_mapping.contiguous()
    _capi.call(
        "pi_kv_index_copy",
        k_pool.data_ptr(), v_pool.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
        slot_mapping.data_ptr(), n, H, D, S, P * S, dtype_code(k_pool.dtype), k_new.stride(0),
        _err_ptr(err), _stream(),
    )


# ---------------------------------------------------------------------------
# f1: fused decode prologue (QK-norm + RoPE + slot-mapping write)
# ---------------------------------------------------------------------------


def rope_inv_freq(head_dim: int, base: float, device: torch.device | str = "cpu") -> torch.Tensor:
    """fp32 [head_dim / 2] rotary frequencies 1 / base^(2j / head_dim).

    Computed on the CPU with the expression of build_rope_cache's fp32 table
    (src/plastic_infer/exec/attention.py:68), so pos * inv_freq[j] is exactly the angle
    that table holds at (pos, j); then moved to `device`.
    """
    inv = 1.0 / (base ** (torch.arange(0, head_dim, 2, dtype=torch.float32) / head_dim))
    return inv.to(device)


def decode_prologue(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    q_norm_weight: torch.Tensor | None = None,
    k_norm_weight: torch.Tensor | None = None,
    eps: float = 1e-5,
    q_out: torch.Tensor | None = None,
    err: torch.Tensor | None = None,
) -> torch.Tensor:
    """One launch per layer: QK-norm (optional) + RoPE of the step's q and k rows, and the
    write of the new K/V rows at their slots (the kv_index_copy semantics).

    q [B, Hq, D], k / v [B, Hkv, D]: the projection outputs (heads contiguous; any request
    stride, k and v sharing one, e.g. slices of a fused QKV output). positions int64
    [B]: each request's new-token position. inv_freq fp32 [D/2] (rope_inv_freq).
    slot_mapping int64 [B] (< 0: no K/V row). Returns q_out [B, Hq, D] in the pool dtype.
    Replaces qk_norm + rope_positions + _write_kv_layer of the reference runners
    (src/plastic_infer/exec/attention.py:23-95, src/plastic_infer/exec/runner_paged.py:112-129).
    """
    P, Hkv, S, D = _check_pool(k_pool, "k_pool")
    if v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype:
        raise ValueError("k_pool and v_pool must have the same shape and dtype")
    B, Hq = q.shape[0], q.shape[1]
    if q.dim() != 3 or q.shape[2] != D or tuple(k.shape) != (B, Hkv, D) or k.shape != v.shape:
        raise ValueError(f"q must be [B, Hq, {D}] and k, v [B, {Hkv}, {D}]")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k and v must share one dtype")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.stride(2) != 1 or t.stride(1) != D:
            raise ValueError(f"{name}: heads must be contiguous rows of head_dim elements")
    if k.stride(0) != v.stride(0):
        raise ValueError("k and v must share one request stride")
    if positions.dtype != torch.int64 or positions.shape != (B,):
        raise ValueError("positions must be int64 [B]")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (B,):
        raise ValueError("slot_mapping must be int64 [B]")
    if inv_freq.dtype != torch.float32 or inv_freq.numel() != D // 2:
        raise ValueError(f"inv_freq must be float32 [{D // 2}]")
    if (q_norm_weight is None) != (k_norm_weight is None):
        raise ValueError("give both QK-norm weights or neither")
    _require_cuda(q, k, v, positions, inv_freq, slot_mapping, k_pool, v_pool)
    if q_out is None:
        q_out = torch.empty((B, Hq, D), dtype=k_pool.dtype, device=q.device)
    elif q_out.dtype != k_pool.dtype or tuple(q_out.shape) != (B, Hq, D) or q_out.stride(2) != 1 \
            or q_out.stride(1) != D:
        raise ValueError("q_out must be [B, Hq, D] in the pool dtype with contiguous heads")
    qw = kw = None
    if q_norm_weight is not None:
        qw = q_norm_weight.to(q.dtype).contiguous()
        kw = k_norm_weight.to(q.dtype).contiguous()
        if qw.numel() != D or kw.numel() != D:
            raise ValueError(f"QK-norm weights must have {D} elements")
    positions = positions.contiguous()
    slot_mapping = slot_mapping.contiguous()
    inv_freq = inv_freq.contiguous()
    _capi.call(
        "pi_decode_prologue",
        q_out.data_ptr(), q_out.stride(0), k_pool.data_ptr(), v_pool.data_ptr(),
        q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.stride(0), dtype_code(q.dtype),
        qw.data_ptr() if qw is not None else None, kw.data_ptr() if kw is not None else None,
        float(eps), inv_freq.data_ptr(), positions.data_ptr(), slot_mapping.data_ptr(),
        B, Hq, Hkv, D, S, P * S, dtype_code(k_pool.dtype), _err_ptr(err), _stream(),
    )
    return q_out


# ---------------------------------------------------------------------------
# Rotary append (any number of tokens; 16/32-bit or 8-bit pools)
# ---------------------------------------------------------------------------

ROPE_SCALINGS = ("none", "linear", "ntk", "yarn")


def rope_frequencies(rotary_dim: int, base: float, scaling: str = "none", factor: float = 1.0,
                     trained_len: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                     device: torch.device | str = "cpu") -> tuple[torch.Tensor, float]:
    """(inv_freq fp32 [rotary_dim / 2], rope_scale) for rope_append.

    "none"    1 / base^(2j / rotary_dim), rope_scale 1
    "linear"  every frequency divided by `factor` (positions interpolated)
    "ntk"     base raised to base * factor^(R / (R - 2)): the slowest pair is stretched by
              `factor`, the fastest not at all
    "yarn"    (Peng et al., "YaRN: Efficient Context Window Extension of Large Language Models",
              2023) pairs that turn fewer than beta_slow times in the trained length are divided
              by `factor`, those that turn more than beta_fast times are kept, a linear ramp over
              the pair index in between, which may end past the last pair;
              rope_scale = 0.1 ln(factor) + 1
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"scaling must be one of {ROPE_SCALINGS}, got {scaling!r}")
    if scaling != "none" and not factor >= 1.0:
        raise ValueError("factor must be at least 1")
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = 1.0 / base ** (torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    rope_scale = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if trained_len <= 0:
            raise ValueError("yarn scaling needs trained_len")

        def pair_turning(turns: float) -> float:  # index of the pair with that many turns
            return (rotary_dim * math.log(trained_len / (turns * 2 * math.pi))
                    / (2 * math.log(base)))

        low = max(math.floor(pair_turning(beta_fast)), 0)
        high = min(math.ceil(pair_turning(beta_slow)), rotary_dim - 1)
        ramp = (torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)
        keep = 1.0 - ramp.clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
        rope_scale = 0.1 * math.log(factor) + 1.0
    return inv.float().to(device), rope_scale


def _check_scales(k_scale: torch.Tensor | None, v_scale: torch.Tensor | None, pages: int,
                  heads: int) -> None:
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if t is None or t.dtype != torch.float32 or tuple(t.shape) != (pages, heads) \
                or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 [{pages}, {heads}] tensor: one "
                             "scale per (page, KV head) of an 8-bit pool")


def _check_one_device(*tensors: torch.Tensor | None) -> torch.device:
    """The one CUDA device that every given tensor is on."""
    device = None
    for t in tensors:
        if t is None:
            continue
        if device is None:
            device = t.device
            if device.type != "cuda":
                _require_cuda(t)
        elif t.device != device:
            _require_cuda(t)
            raise ValueError(f"all tensors must be on one device, got {device} and {t.device}")
    return device  # type: ignore[return-value]


def _call_on(device: torch.device, func: str, *args) -> None:
    """_capi.call on the current stream of `device`, with that device current."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if device.index == torch._C._cuda_getDevice():
        _capi.call(func, *args, stream)
        return
    with torch.cuda.device(device):
        _capi.call(func, *args, stream)


def rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    q_norm_weight: torch.Tensor | None = None,
    k_norm_weight: torch.Tensor | None = None,
    eps: float = 1e-5,
    interleaved: bool = False,
    rope_scale: float = 1.0,
    k_scale: torch.Tensor | None = None,
    v_scale: torch.Tensor | None = None,
    q_out: torch.Tensor | None = None,
    err: torch.Tensor | None = None,
) -> torch.Tensor:
    """QK-norm (optional) and rotary positions of T new q and k rows, and the write of the new
    K/V rows at their slots; one launch for a decode step or for whole prompts.

    q [T, Hq, D], k / v [T, Hkv, D]: heads contiguous, any token strides (e.g. slices of a
    fused QKV output). positions int64 [T]; slot_mapping int64 [T] (page * page_size + offset;
    < 0: no K/V row). inv_freq fp32 [R / 2] turns the first R elements of a head
    (rope_frequencies): pairs (j, j + R/2), or (2j, 2j + 1) with `interleaved`; rope_scale
    multiplies cosine and sine. Angles are formed in 64 bits, so far positions keep their
    precision. QK-norm weights are taken in q's dtype, others are rounded to it first, as in
    decode_prologue. Returns q_out [T, Hq, D], which must not overlap the inputs.

    For one token per request, half layout over the whole head and 16/32-bit pools,
    decode_prologue does the same in the same time, with the reference's fp32 angles; take
    rope_append for prompts, far positions, other rotary forms and 8-bit pools.

    16/32-bit pools take the rows in the pool dtype, which is q_out's too. Pools of
    torch.float8_e4m3fn need k_scale and v_scale, fp32 [num_pages, Hkv] (q_out then has q's
    dtype): each (page, head) block has one power-of-two scale, grown as rows arrive; the rows
    of one call in one page must be consecutive tokens with consecutive slots, rows at lower
    offsets are kept (rescaled when the scale grows), rows behind are left as they were
    (include/plastic_kv.h has the formulas). With `err`, a page named in any other way (out of
    order, with gaps or padding between its tokens, a slot twice) is left as it was and `err`
    gets PI_ERR_PAGE_SHARED; without, nobody looks, and what that page ends up with is
    unspecified.
    """
    P, Hkv, S, D = _check_pool(k_pool, "k_pool")
    if v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype:
        raise ValueError("k_pool and v_pool must have the same shape and dtype")
    if not v_pool.is_contiguous():
        raise ValueError("v_pool must be contiguous")
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q must be [T, Hq, {D}], got {tuple(q.shape)}")
    T, Hq = q.shape[0], q.shape[1]
    if tuple(k.shape) != (T, Hkv, D) or k.shape != v.shape:
        raise ValueError(f"k and v must be [{T}, {Hkv}, {D}]")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("q, k and v must share one dtype")
    in_code = dtype_code(q.dtype)
    eight = k_pool.dtype == torch.float8_e4m3fn
    if eight:
        _check_scales(k_scale, v_scale, P, Hkv)
    elif k_scale is not None or v_scale is not None:
        raise ValueError("k_scale and v_scale go with pools of torch.float8_e4m3fn")
    pool_code = _capi.PI_DTYPE_E4M3 if eight else dtype_code(k_pool.dtype)
    out_dtype = q.dtype if eight else k_pool.dtype
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        # (a single head's stride means nothing)
        if t.stride(2) != 1 or (t.stride(1) != D and t.shape[1] != 1):
            raise ValueError(f"{name}: heads must be contiguous rows of head_dim elements")
    if positions.dtype != torch.int64 or positions.shape != (T,):
        raise ValueError("positions must be int64 [T]")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (T,):
        raise ValueError("slot_mapping must be int64 [T]")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > D:
        raise ValueError(f"inv_freq must be float32 [R / 2] with R <= {D}")
    if (q_norm_weight is None) != (k_norm_weight is None):
        raise ValueError("give both QK-norm weights or neither")
    if q_out is None:
        q_out = torch.empty((T, Hq, D), dtype=out_dtype, device=q.device)
    elif q_out.dtype != out_dtype or tuple(q_out.shape) != (T, Hq, D) or q_out.stride(2) != 1 \
            or (q_out.stride(1) != D and Hq != 1):
        raise ValueError(f"q_out must be [T, Hq, D] {out_dtype} with contiguous heads")
    qw = kw = None
    if q_norm_weight is not None:
        qw = q_norm_weight.to(q.dtype).contiguous()
        kw = k_norm_weight.to(q.dtype).contiguous()
        if qw.numel() != D or kw.numel() != D:
            raise ValueError(f"QK-norm weights must have {D} elements")
    device = _check_one_device(q, k, v, positions, inv_freq, slot_mapping, k_pool, v_pool, q_out,
                               qw, kw, k_scale, v_scale, err)
    if T == 0:
        return q_out
    positions = positions.contiguous()
    slot_mapping = slot_mapping.contiguous()
    inv_freq = inv_freq.contiguous()
    # (one token: its stride is never used, and torch may report any)
    row, kv_row = Hq * D, Hkv * D
    strides = (q_out.stride(0), q.stride(0), k.stride(0), v.stride(0)) if T > 1 \
        else (row, row, kv_row, kv_row)
    _call_on(
        device, "pi_rope_append",
        q_out.data_ptr(), strides[0], k_pool.data_ptr(), v_pool.data_ptr(),
        k_scale.data_ptr() if eight else None, v_scale.data_ptr() if eight else None,
        q.data_ptr(), strides[1], k.data_ptr(), strides[2], v.data_ptr(), strides[3], in_code,
        qw.data_ptr() if qw is not None else None, kw.data_ptr() if kw is not None else None,
        float(eps), inv_freq.data_ptr(), inv_freq.shape[0], 1 if interleaved else 0,
        float(rope_scale), positions.data_ptr(), slot_mapping.data_ptr(), T, Hq, Hkv, D, S, P,
        pool_code, _err_ptr(err),
    )
    return q_out


# ---------------------------------------------------------------------------
# f4: MoE expert-slot copy (all banks, one launch)
# ---------------------------------------------------------------------------


def expert_slot_copy(
    dst_ptrs: torch.Tensor,
    src_ptrs: torch.Tensor,
    feat_bytes: torch.Tensor,
    dst_indices: torch.Tensor,
    src_indices: torch.Tensor,
    num_indices: torch.Tensor | None = None,
    err: torch.Tensor | None = None,
) -> None:
    """dst_b[dst_indices[i]] = src_b[src_indices[i]] for every bank b and i < n, one launch.

    The signature of the reference's fast_index_copy_multi_jit
    (src/plastic_infer/kernel/fast_index_copy.py:208-244): dst_ptrs / src_ptrs / feat_bytes
    are int64 [num_banks] CUDA tensors (slot-cache base, host-bank device alias, row
    bytes), the index tensors int32 or int64 CUDA [L], num_indices an optional CUDA
    int64 [1] valid length (n = min(num_indices[0], L)).
    """
    for t, name in ((dst_ptrs, "dst_ptrs"), (src_ptrs, "src_ptrs"), (feat_bytes, "feat_bytes")):
        if t.dtype != torch.int64 or t.dim() != 1:
            raise ValueError(f"{name} must be an int64 [num_banks] tensor")
    if not (dst_ptrs.numel() == src_ptrs.numel() == feat_bytes.numel()):
        raise ValueError("dst_ptrs, src_ptrs and feat_bytes must have one entry per bank")
    if dst_indices.shape != src_indices.shape or dst_indices.dtype != src_indices.dtype \
            or dst_indices.dtype not in (torch.int32, torch.int64) or dst_indices.dim() != 1:
        raise ValueError("dst_indices and src_indices must be matching int32/int64 [L] tensors")
    if num_indices is not None and (num_indices.dtype != torch.int64 or num_indices.numel() < 1):
        raise ValueError("num_indices must be an int64 [1] tensor")
    tensors = [dst_ptrs, src_ptrs, feat_bytes, dst_indices, src_indices]
    if num_indices is not None:
        tensors.append(num_indices)
    _require_cuda(*tensors)
    _capi.call(
        "pi_expert_slot_copy",
        dst_ptrs.contiguous().data_ptr(), src_ptrs.contiguous().data_ptr(),
        feat_bytes.contiguous().data_ptr(), dst_ptrs.numel(), dst_indices.contiguous().data_ptr(),
        src_indices.contiguous().data_ptr(), dst_indices.numel(),
        num_indices.data_ptr() if num_indices is not None else None,
        1 if dst_indices.dtype == torch.int32 else 0, _err_ptr(err), _stream(),
    )


# ---------------------------------------------------------------------------
# a2: paged decode attention
# ---------------------------------------------------------------------------


class Workspace:
    """Zero-initialised device scratch for the paged attention calls, grown on demand.

    The kernels leave the counter region zero on exit, so the buffer is zeroed once
    at allocation. paged_decode_attention, its gather variant and the 8-bit attention
    calls may share one; host_stream_attention keeps no zeroed region and needs one of
    its own. Launches that share one Workspace must be ordered (same stream);
    give concurrent streams their own Workspace. Threads may share one on one stream:
    a call of several launches (the 8-bit attention) holds `lock` from get() until its
    last launch is enqueued, so no other thread's launch comes between them.
    """

    def __init__(self, device: torch.device) -> None:
        self.device = torch.device(device)
        self.buf: torch.Tensor | None = None
        self.lock = threading.RLock()

    def get(self, nbytes: int) -> torch.Tensor:
        with self.lock:
            buf = self.buf
            if buf is None or buf.numel() < nbytes:
                # (twice as large at least: a history that grows call by call is not a buffer a call)
                n = max(nbytes, 1 << 20, 0 if buf is None else 2 * buf.numel())
                self.buf = buf = torch.zeros(n, dtype=torch.uint8, device=self.device)
            return buf


_ws_lock = threading.Lock()
_default_ws: dict[int, Workspace] = {}


def default_workspace(device: torch.device) -> Workspace:
    idx = torch.device(device).index
    if idx is None:
        idx = torch.cuda.current_device()
    with _ws_lock:
        ws = _default_ws.get(idx)
        if ws is None:
            ws = _default_ws[idx] = Workspace(torch.device("cuda", idx))
        return ws


def set_programmatic_launch(enable: bool) -> None:
    """Programmatic dependent launch for every later index-copy and attention launch.

    When on, a kernel may launch while the previous kernel on its stream is still
    running: the attention computes its work split and fetches its first page ids
    (reading only ctx_lens and block_tables) before it waits for that kernel. So the
    kernel launched just before an attention must not write its ctx_lens or
    block_tables. Off by default.
    """
    _capi.call("pi_set_programmatic_launch", 1 if enable else 0)


_RING_MODES = {"auto": _capi.PI_ATTN_RING_AUTO, "deep": _capi.PI_ATTN_RING_DEEP,
               "shallow": _capi.PI_ATTN_RING_SHALLOW}


def set_decode_attn_ring(mode: str) -> None:
    """Page-ring depth of every later plain paged_decode_attention launch.

    "auto" (the default) picks per launch: a two-stage ring with two CTAs per SM when
    batch x block-table width x KV heads is large, else a deep ring (4 stages at
    head_dim <= 128) with one CTA per SM. "deep" and "shallow" force one of them
    (shallow only where two CTAs fit on an SM). Launches with the fused append or the
    peer all-gather always use the deep ring.
    """
    try:
        code = _RING_MODES[mode]
    except KeyError:
        raise ValueError(f"ring mode must be one of {sorted(_RING_MODES)}, got {mode!r}")
    _capi.call("pi_set_decode_attn_ring", code)


def decode_attn_ring_stages(batch: int, bt_stride: int, num_q_heads: int, num_kv_heads: int,
                            head_dim: int, page_size: int, num_pages: int,
                            dtype: torch.dtype) -> int:
    """Ring stages a plain attention launch of this shape would use now (0: SIMT path)."""
    return int(_capi.load().pi_paged_decode_attn_ring_stages(
        batch, bt_stride, num_q_heads, num_kv_heads, head_dim, page_size, num_pages,
        dtype_code(dtype)))


def _early_reads(*tables: torch.Tensor) -> list[torch.Tensor]:
    """Contiguous block tables and lengths of an attention call. The kernel reads them before it
    waits for the launch before it (set_programmatic_launch), so where one had to be copied,
    another launch is put between the copy and the kernel."""
    dense = [t.contiguous() for t in tables]
    if any(d.data_ptr() != t.data_ptr() for d, t in zip(dense, tables)):
        torch.zeros(1, dtype=torch.int32, device=dense[0].device)
    return dense


def workspace_bytes(batch: int, num_q_heads: int, num_kv_heads: int, head_dim: int) -> int:
    return int(_capi.load().pi_paged_decode_attn_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim))


def paged_decode_attention(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: Workspace | None = None,
    err: torch.Tensor | None = None,
    k_new: torch.Tensor | None = None,
    v_new: torch.Tensor | None = None,
    slot_mapping: torch.Tensor | None = None,
) -> torch.Tensor:
    """Decode attention of q [B, Hq, D] over each request's first ctx_lens[b] tokens.

    block_tables: int32 [B, max_pages] page ids; ctx_lens: int32 [B]. Returns
    out [B, Hq, D] in the pool dtype (fp32 softmax/accumulation inside).

    With k_new / v_new [B, Hkv, D] and slot_mapping int64 [B], the step's new rows
    are first written at their slots (the kv_index_copy semantics) in the same
    launch: a whole decode layer's KV path is then one kernel.
    """
    P, Hkv, S, D = _check_pool(k_pool, "k_pool")
    if v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype:
        raise ValueError("k_pool and v_pool must have the same shape and dtype")
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q must be [B, Hq, {D}], got {tuple(q.shape)}")
    B, Hq, _ = q.shape
    if Hq % Hkv != 0:
        raise ValueError(f"num_q_heads {Hq} not a multiple of num_kv_heads {Hkv}")
    if q.dtype != k_pool.dtype:
        raise TypeError("q must have the pool dtype")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise ValueError("block_tables must be int32 [B, max_pages]")
    if ctx_lens.dtype != torch.int32 or ctx_lens.shape != (B,):
        raise ValueError("ctx_lens must be int32 [B]")
    _require_cuda(q, k_pool, v_pool, block_tables, ctx_lens)
    if q.stride(2) != 1 or q.stride(1) != D:
        q = q.contiguous()
    if block_tables.stride(1) != 1 or ctx_lens.stride(0) != 1:  # (rows may be apart)
        block_tables, ctx_lens = _early_reads(block_tables, ctx_lens)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=q.dtype, device=q.device)
    elif out.shape != (B, Hq, D) or out.dtype != q.dtype or out.stride(2) != 1 or out.stride(1) != D:
        raise ValueError("out must be [B, Hq, D] with contiguous heads, pool dtype")
    if B == 0:
        return out
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    nbytes = workspace_bytes(B, Hq, Hkv, D)
    ws = (workspace or default_workspace(q.device)).get(nbytes)
    if k_new is None and v_new is None and slot_mapping is None:
        _capi.call(
            "pi_paged_decode_attn",
            out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
            block_tables.data_ptr(), block_tables.stride(0), ctx_lens.data_ptr(),
            B, Hq, Hkv, D, S, P, float(scale), dtype_code(q.dtype), q.stride(0), out.stride(0),
            ws.data_ptr(), ws.numel(), _err_ptr(err), _stream(),
        )
        return out
    # Fused append: write one new K/V row per request, then attend (one launch).
    if k_new is None or v_new is None or slot_mapping is None:
        raise ValueError("k_new, v_new and slot_mapping go together")
    if k_new.shape != (B, Hkv, D) or v_new.shape != (B, Hkv, D):
        raise ValueError(f"k_new/v_new must be [{B}, {Hkv}, {D}]")
    if k_new.dtype != k_pool.dtype or v_new.dtype != k_pool.dtype:
        raise TypeError("new K/V rows must have the pool dtype")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (B,):
        raise ValueError("slot_mapping must be int64 [B]")
    _require_cuda(k_new, v_new, slot_mapping)
    if not (k_new.stride(2) == 1 and k_new.stride(1) == D and v_new.stride() == k_new.stride()):
        k_new = k_new.contiguous()
        v_new = v_new.contiguous()
    slot_mapping = slot_mapping.contiguous()
    _capi.call(
        "pi_paged_decode_attn_append",
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_new.data_ptr(),
        v_new.data_ptr(), slot_mapping.data_ptr(), k_new.stride(0),
        block_tables.data_ptr(), block_tables.stride(0), ctx_lens.data_ptr(),
        B, Hq, Hkv, D, S, P, float(scale), dtype_code(q.dtype), q.stride(0), out.stride(0),
        ws.data_ptr(), ws.numel(), _err_ptr(err), _stream(),
    )
    return out


# ---------------------------------------------------------------------------
# Attention over an 8-bit cache
# ---------------------------------------------------------------------------

_q8_ws: dict[tuple[int, int], Workspace] = {}
_q8_decode_bytes: dict[tuple[int, int], int] = {}


def _check_q8_pools(k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor) -> tuple[int, int, int, int]:
    P, Hkv, S, D = _check_pool(k_pool, "k_pool")
    if k_pool.dtype != torch.float8_e4m3fn or v_pool.dtype != torch.float8_e4m3fn:
        raise TypeError("the pools must be torch.float8_e4m3fn")
    if v_pool.shape != k_pool.shape or not v_pool.is_contiguous():
        raise ValueError("v_pool must be contiguous and have k_pool's shape")
    _check_scales(k_scale, v_scale, P, Hkv)
    return P, Hkv, S, D


def _capturing(device: torch.device) -> bool:
    """Whether the current stream of `device`, current or not, is being captured."""
    if device.index == torch._C._cuda_getDevice():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _q8_call(device: torch.device, nbytes: int, lent: bool, workspace: Workspace | None,
             err: torch.Tensor | None, func: str, args: tuple) -> None:
    """One q8 attention call on the device's current stream, with `nbytes` of scratch: the
    caller's, or one of the stream's own, so that calls on two streams never share it. A call
    may be several launches that hand data over through the scratch, so it is held against
    other threads until all are enqueued. Under graph capture it comes out of the graph's
    memory, zeroed by the graph: no two graphs share it either. So it does where the caller's
    workspace is too small yet: the workspace is left as it was.

    Scratch for widened pages (`lent`) grows with the history, so it is not kept: torch's
    allocator lends it for the call, in powers of two, that a prompt taken in chunks leaves a few
    blocks behind and not one per chunk. It need not be zeroed."""
    if workspace is not None and torch.device(workspace.device).index not in (None, device.index):
        raise ValueError(f"the workspace is on {workspace.device}, q on {device}")
    lent = lent and workspace is None
    # (a caller's workspace that would have to grow under capture: what it grew by would be zeroed by
    # that graph's replays only)
    capturing = (workspace is None or workspace.buf is None or workspace.buf.numel() < nbytes) \
        and _capturing(device)
    if lent or capturing:
        size = nbytes if capturing else 1 << (nbytes - 1).bit_length()
        buf = torch.empty(size, dtype=torch.uint8, device=device)
        if not lent:
            buf[:int(_capi.load().pi_paged_decode_attn_q8_ws_zero_bytes())].zero_()
        _call_on(device, func, *args, buf.data_ptr(), size, _err_ptr(err))
        return
    if workspace is None:
        stream = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
        workspace = _q8_ws.get(stream)
        if workspace is None:
            with _ws_lock:
                workspace = _q8_ws.setdefault(stream, Workspace(device))
    with workspace.lock:
        buf = workspace.buf
        if buf is None or buf.numel() < nbytes:
            buf = workspace.get(nbytes)
        _call_on(device, func, *args, buf.data_ptr(), buf.numel(), _err_ptr(err))


def _q8_decode_workspace_bytes(device: torch.device, head_dim: int) -> int:
    key = (device.index, head_dim)
    nbytes = _q8_decode_bytes.get(key)
    if nbytes is None:
        with torch.cuda.device(device):
            nbytes = int(_capi.load().pi_paged_decode_attn_q8_workspace_bytes(head_dim))
        _q8_decode_bytes[key] = nbytes
    return nbytes


def paged_decode_attention_q8(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: Workspace | None = None,
    err: torch.Tensor | None = None,
) -> torch.Tensor:
    """Decode attention of q [B, Hq, D] over each request's first ctx_lens[b] tokens of an
    8-bit cache: pools torch.float8_e4m3fn [num_pages, Hkv, page_size, D] with fp32 scales
    [num_pages, Hkv], as rope_append fills them.

    block_tables int32 [B, max_pages], ctx_lens int32 [B]. Returns out [B, Hq, D] in q's dtype
    (bf16, f16 or f32); a request with no context gets zeros. What lies behind a request's last
    token is not used, whatever it holds. Head sizes 64, 128 and 256 with pages of 16 or 32 run
    on the tensor cores in bf16 and f16; everything else (head_dim <= 256) on a plain kernel.
    Without `workspace`, calls on different streams and captured graphs have scratch of their own;
    threads that call on one stream, with or without one, do not disturb each other.
    """
    P, Hkv, S, D = _check_q8_pools(k_pool, v_pool, k_scale, v_scale)
    if q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q must be [B, Hq, {D}], got {tuple(q.shape)}")
    B, Hq, _ = q.shape
    if Hq == 0 or Hq % Hkv != 0:
        raise ValueError(f"num_q_heads {Hq} not a multiple of num_kv_heads {Hkv}")
    code = dtype_code(q.dtype)
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != B:
        raise ValueError("block_tables must be int32 [B, max_pages]")
    if ctx_lens.dtype != torch.int32 or ctx_lens.shape != (B,):
        raise ValueError("ctx_lens must be int32 [B]")
    device = _check_one_device(q, k_pool, v_pool, k_scale, v_scale, block_tables, ctx_lens, out, err)
    if q.stride(2) != 1 or (q.stride(1) != D and Hq != 1) or (B > 1 and q.stride(0) < Hq * D):
        q = q.contiguous()
    if block_tables.stride(1) != 1 or ctx_lens.stride(0) != 1:  # (rows may be apart)
        block_tables, ctx_lens = _early_reads(block_tables, ctx_lens)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=q.dtype, device=device)
    elif out.shape != (B, Hq, D) or out.dtype != q.dtype or out.stride(2) != 1 \
            or (out.stride(1) != D and Hq != 1):
        raise ValueError("out must be [B, Hq, D] with contiguous heads, q's dtype")
    if B == 0:
        return out
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    row = Hq * D
    _q8_call(
        device, _q8_decode_workspace_bytes(device, D), False, workspace, err, "pi_paged_decode_attn_q8",
        (out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(),
         v_scale.data_ptr(), block_tables.data_ptr(), block_tables.stride(0) if B > 1 else 0,
         block_tables.shape[1], ctx_lens.data_ptr(), B, Hq, Hkv, D, S, P, float(scale), code,
         q.stride(0) if B > 1 else row, out.stride(0) if B > 1 else row),
    )
    return out


def paged_prefill_attention_q8(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    kv_len: int,
    q_start: int = 0,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: Workspace | None = None,
    err: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one request's q [q_len, Hq, D] (or [1, q_len, Hq, D]) over the first kv_len
    tokens of its pages in an 8-bit cache (pools and scales as in paged_decode_attention_q8).

    Query i sits at position q_start + i; with `causal` it sees keys j <= q_start + i. Returns
    [q_len, Hq, D] in q's dtype (the input's leading batch axis is kept when given). Long chunks
    widen the request's pages once into the workspace and run the tcgen05 prefill on them; short
    ones, and shapes that it does not take, run the 8-bit decode kernels over several rows. Without
    `workspace` the widened pages are lent by torch's allocator for the call. Widened values and
    the softmax weights on them are of q's dtype (include/plastic_kv.h states what either path
    rounds), so outputs of short and long chunks may differ by that.
    """
    P, Hkv, S, D = _check_q8_pools(k_pool, v_pool, k_scale, v_scale)
    batched = q.dim() == 4
    if batched and q.shape[0] != 1:
        raise ValueError("prefill attends one request: q must be [1, q_len, Hq, D]")
    q3 = q[0] if batched else q
    if q3.dim() != 3 or q3.shape[2] != D:
        raise ValueError(f"q must be [q_len, Hq, {D}]")
    n, Hq = q3.shape[0], q3.shape[1]
    if Hq == 0 or Hq % Hkv != 0:
        raise ValueError(f"num_q_heads {Hq} not a multiple of num_kv_heads {Hkv}")
    code = dtype_code(q3.dtype)
    if block_table.dtype != torch.int32 or block_table.dim() != 1:
        raise ValueError("block_table must be int32 [n]")
    kv_len, q_start = int(kv_len), int(q_start)
    if kv_len > block_table.numel() * S or kv_len < 0 or q_start < 0 or q_start + n > 2 ** 31 - 1:
        raise ValueError("kv_len must be within the block table's pages, q_start not negative")
    device = _check_one_device(q3, k_pool, v_pool, k_scale, v_scale, block_table, out, err)
    if q3.stride(2) != 1 or (q3.stride(1) != D and Hq != 1) or (n > 1 and q3.stride(0) < Hq * D):
        q3 = q3.contiguous()
    if block_table.stride(0) != 1:
        block_table, = _early_reads(block_table)
    if out is None:
        out3 = torch.empty((n, Hq, D), dtype=q3.dtype, device=device)
    else:
        out3 = out[0] if out.dim() == 4 else out
        if out3.shape != (n, Hq, D) or out3.dtype != q3.dtype or out3.stride(2) != 1 \
                or (out3.stride(1) != D and Hq != 1):
            raise ValueError("out must be [q_len, Hq, D] in q's dtype with contiguous heads")
    if n > 0:
        if scale is None:
            scale = 1.0 / math.sqrt(D)
        nbytes = kept = _q8_decode_workspace_bytes(device, D)
        if n * Hq > _capi.Q8_FEW_ROWS:  # (fewer rows need the decode scratch only)
            with torch.cuda.device(device):
                nbytes = int(_capi.load().pi_paged_prefill_attn_q8_workspace_bytes(
                    n, kv_len, Hq, Hkv, D, S, code))
        row = Hq * D
        _q8_call(
            device, nbytes, nbytes > kept, workspace, err, "pi_paged_prefill_attn_q8",
            (out3.data_ptr(), q3.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
             k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), block_table.numel(), n,
             kv_len, q_start, 1 if causal else 0, Hq, Hkv, D, S, P, float(scale), code,
             q3.stride(0) if n > 1 else row, out3.stride(0) if n > 1 else row),
        )
    if out is not None:
        return out
    return out3.unsqueeze(0) if batched else out3


def page_dequant(pool: torch.Tensor, scale: torch.Tensor, page_ids: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
                 err: torch.Tensor | None = None) -> torch.Tensor:
    """out[i, h] = pool[page_ids[i], h] * scale[page_ids[i], h]: pages of an 8-bit pool widened to
    `dtype` (f32, bf16 or f16), [n, Hkv, page_size, D]. Exact in bf16 and f32 for power-of-two
    scales; an f16 value past 65504 becomes 65504."""
    P, Hkv, S, D = _check_pool(pool, "pool")
    if pool.dtype != torch.float8_e4m3fn:
        raise TypeError("the pool must be torch.float8_e4m3fn")
    _check_scales(scale, scale, P, Hkv)
    if page_ids.dtype != torch.int32 or page_ids.dim() != 1:
        raise ValueError("page_ids must be int32 [n]")
    code = dtype_code(dtype)
    n = page_ids.numel()
    device = _check_one_device(pool, scale, page_ids, out, err)
    if out is None:
        out = torch.empty((n, Hkv, S, D), dtype=dtype, device=device)
    elif out.dtype != dtype or tuple(out.shape) != (n, Hkv, S, D) or not out.is_contiguous():
        raise ValueError(f"out must be contiguous [{n}, {Hkv}, {S}, {D}] {dtype}")
    if n:
        page_ids = page_ids.contiguous()  # (kept until the launch is enqueued)
        _call_on(device, "pi_page_dequant", out.data_ptr(), pool.data_ptr(), scale.data_ptr(),
                 page_ids.data_ptr(), n, Hkv, D, S, P, code, _err_ptr(err))
    return out


# ---------------------------------------------------------------------------
# gather_paged_kv and a3: page moves
# ---------------------------------------------------------------------------


def paged_kv_gather(pool: torch.Tensor, block_table: torch.Tensor, num_tokens: int,
                    err: torch.Tensor | None = None) -> torch.Tensor:
    """out[t, h, :] = pool[block_table[t // S], h, t % S, :] -> [num_tokens, H, D]."""
    P, H, S, D = _check_pool(pool, "pool")
    if block_table.dtype != torch.int32 or block_table.dim() != 1:
        raise ValueError("block_table must be int32 [n_pages]")
    if num_tokens > block_table.numel() * S:
        raise ValueError("num_tokens exceeds the block table's pages")
    _require_cuda(pool, block_table)
    out = torch.empty((num_tokens, H, D), dtype=pool.dtype, device=pool.device)
    if num_tokens == 0:
        return out
    _capi.call(
        "pi_paged_kv_gather",
        out.data_ptr(), pool.data_ptr(), block_table.contiguous().data_ptr(), num_tokens, H, D, S,
        P, dtype_code(pool.dtype), _err_ptr(err), _stream(),
    )
    return out


def _page_move(func: str, pool: torch.Tensor, staging: torch.Tensor, page_ids: torch.Tensor,
               pages_per_group: int, err: torch.Tensor | None) -> None:
    P, H, S, D = _check_pool(pool, "pool")
    if page_ids.dtype != torch.int32 or page_ids.dim() != 1:
        raise ValueError("page_ids must be int32 [n]")
    n = page_ids.numel()
    tile_bytes = S * D * pool.element_size()
    if not staging.is_contiguous() or staging.numel() * staging.element_size() < n * H * tile_bytes:
        raise ValueError("staging must be contiguous and hold n * kv_heads * page_size * head_dim elements")
    if pages_per_group <= 0 or n % pages_per_group != 0:
        raise ValueError("page count must be a multiple of pages_per_group")
    _require_cuda(pool, staging, page_ids)
    if n == 0:
        return
    page_ids = page_ids.contiguous()
    if func == "pi_page_gather":
        args = (staging.data_ptr(), pool.data_ptr())
    else:
        args = (pool.data_ptr(), staging.data_ptr())
    _capi.call(func, *args, page_ids.data_ptr(), n, H, tile_bytes, pages_per_group, P,
               _err_ptr(err), _stream())


def page_gather(pool: torch.Tensor, page_ids: torch.Tensor, staging: torch.Tensor,
                pages_per_group: int = 1, err: torch.Tensor | None = None) -> None:
    """staging <- pool pages, grouped head-major (see include/plastic_kv.h)."""
    _page_move("pi_page_gather", pool, staging, page_ids, pages_per_group, err)


def page_scatter(staging: torch.Tensor, page_ids: torch.Tensor, pool: torch.Tensor,
                 pages_per_group: int = 1, err: torch.Tensor | None = None) -> None:
    """pool pages <- staging (inverse of page_gather)."""
    _page_move("pi_page_scatter", pool, staging, page_ids, pages_per_group, err)


# ---------------------------------------------------------------------------
# f3: paged prefill attention
# ---------------------------------------------------------------------------

PREFILL_GROUPS = (1, 2, 4, 8, 16)


def prefill_supported(q: torch.Tensor, k_pool: torch.Tensor) -> bool:
    """Whether pi_paged_prefill_attn covers this q / pool combination."""
    if k_pool.dim() != 4 or q.dim() not in (3, 4):
        return False
    P, Hkv, S, D = k_pool.shape
    Hq = q.shape[-2]
    return (k_pool.dtype in (torch.bfloat16, torch.float16) and q.dtype == k_pool.dtype
            and D in (64, 128) and S in (16, 32) and q.shape[-1] == D and Hq % Hkv == 0
            and Hq // Hkv in PREFILL_GROUPS)


def paged_prefill_attention(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_table: torch.Tensor,
    kv_len: int,
    q_start: int = 0,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    err: torch.Tensor | None = None,
    impl: str = "mma",
) -> torch.Tensor:
    """Prefill attention of one request's q [q_len, Hq, D] (or [1, q_len, Hq, D]) over the
    first kv_len tokens of its pages (block_table: int32 [n] page ids, device).

    Query i sits at position q_start + i; with `causal` it sees keys j <= q_start + i
    (the reference's is_causal when q_start == 0, its offset mask otherwise:
    src/plastic_infer/exec/runner_paged.py:36-95). Returns [q_len, Hq, D] in the pool dtype
    (the input's leading batch axis is kept when given). `impl` picks the kernel: "tc"
    (tcgen05, S and O in tensor memory) or "mma" (mma.sync, accumulators in registers).
    """
    if impl not in ("tc", "mma"):
        raise ValueError(f"impl must be 'tc' or 'mma', got {impl!r}")
    P, Hkv, S, D = _check_pool(k_pool, "k_pool")
    if v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype:
        raise ValueError("k_pool and v_pool must have the same shape and dtype")
    batched = q.dim() == 4
    if batched:
        if q.shape[0] != 1:
            raise ValueError("prefill attends one request: q must be [1, q_len, Hq, D]")
        q3 = q[0]
    else:
        q3 = q
    if q3.dim() != 3 or q3.shape[2] != D:
        raise ValueError(f"q must be [q_len, Hq, {D}]")
    if not prefill_supported(q3, k_pool):
        raise ValueError("shape or dtype not covered by the prefill kernel (bf16/f16, head_dim "
                         "64/128, page 16/32, Hq/Hkv in 1/2/4/8/16)")
    if block_table.dtype != torch.int32 or block_table.dim() != 1:
        raise ValueError("block_table must be int32 [n]")
    q_len, Hq = q3.shape[0], q3.shape[1]
    if kv_len > block_table.numel() * S or kv_len < 0 or q_start < 0:
        raise ValueError("kv_len must be within the block table's pages")
    _require_cuda(q3, k_pool, v_pool, block_table)
    if q3.stride(2) != 1 or q3.stride(1) != D:
        q3 = q3.contiguous()
    if out is None:
        out3 = torch.empty((q_len, Hq, D), dtype=k_pool.dtype, device=q3.device)
    else:
        out3 = out[0] if out.dim() == 4 else out
        if out3.shape != (q_len, Hq, D) or out3.dtype != k_pool.dtype or out3.stride(2) != 1 \
                or out3.stride(1) != D:
            raise ValueError("out must be [q_len, Hq, D] in the pool dtype with contiguous heads")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    block_table = block_table.contiguous()
    dst = out3
    if impl == "tc":
        # the tcgen05 kernel moves q and the output by TMA: 16-byte aligned rows
        if q3.data_ptr() % 16 or q3.stride(0) % 8:
            q3 = q3.clone(memory_format=torch.contiguous_format)
        if dst.data_ptr() % 16 or dst.stride(0) % 8:
            dst = torch.empty((q_len, Hq, D), dtype=k_pool.dtype, device=q3.device)
    _capi.call(
        "pi_paged_prefill_attn_tc" if impl == "tc" else "pi_paged_prefill_attn",
        dst.data_ptr(), q3.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        block_table.data_ptr(), block_table.numel(), q_len, int(kv_len), int(q_start),
        1 if causal else 0, Hq, Hkv, D, S, P, float(scale), dtype_code(k_pool.dtype),
        q3.stride(0), dst.stride(0), _err_ptr(err), _stream(),
    )
    if dst is not out3:
        out3.copy_(dst)
    if out is not None:
        return out
    return out3.unsqueeze(0) if batched else out3


# ---------------------------------------------------------------------------
# f2: attention over host-resident chunks + a device tail, read in place
# ---------------------------------------------------------------------------

_keep_lock = threading.Lock()
_keep: list[tuple[torch.cuda.Event, tuple]] = []
_hs_ws: dict[int, Workspace] = {}


def _keep_until_done(tensors: list[torch.Tensor]) -> None:
    """Hold host tensors a launch reads in place until the launch has run: torch cannot
    see a kernel's reads of pinned memory, and would otherwise recycle the pages."""
    if not tensors or torch.cuda.is_current_stream_capturing():
        return
    ev = torch.cuda.Event()
    ev.record()
    with _keep_lock:
        _keep[:] = [(e, t) for e, t in _keep if not e.query()]
        _keep.append((ev, tuple(tensors)))


def host_stream_attention(
    q: torch.Tensor,
    kv_spans,
    q_start: int = 0,
    causal: bool = True,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    workspace: Workspace | None = None,
    err: torch.Tensor | None = None,
    num_kv_heads: int | None = None,
) -> torch.Tensor:
    """Attention of one request over a KV sequence given as spans, on the host or the GPU.

    q is [q_len, Hq, D] (or [1, q_len, Hq, D]) on the GPU; query i sits at position
    q_start + i. kv_spans is a sequence of (k, v) views shaped [H_kv, T, D] (any strides;
    k and v alike) that concatenate, in order, into the request's keys and values. A span
    lives on the query's GPU or in page-locked host memory, which the kernel reads in
    place over the host link: host chunks are never staged or materialised. With
    `causal`, query i sees keys j <= q_start + i; otherwise every key. Returns
    [q_len, Hq, D] in q's dtype (the leading batch axis is kept when given).

    The pinned spans stay referenced until the launch has run. Under CUDA-graph capture
    the caller keeps them alive for the graph's lifetime.
    """
    batched = q.dim() == 4
    if batched:
        if q.shape[0] != 1:
            raise ValueError("host-stream attention attends one request: q must be [1, q_len, Hq, D]")
        q3 = q[0]
    else:
        q3 = q
    if q3.dim() != 3:
        raise ValueError("q must be [q_len, Hq, D]")
    _require_cuda(q3)
    q_len, Hq, D = q3.shape
    if q_start < 0:
        raise ValueError("q_start must be >= 0")
    if q3.stride(2) != 1 or q3.stride(1) != D:
        q3 = q3.contiguous()
    code = dtype_code(q3.dtype)
    kv_spans = list(kv_spans)
    if len(kv_spans) > _capi.HS_MAX_SPANS:
        raise ValueError(f"at most {_capi.HS_MAX_SPANS} spans per call")
    rows: list[tuple[int, int, int, int, int, int]] = []
    hkv = num_kv_heads
    kv_len = 0
    host: list[torch.Tensor] = []
    for i, (k, v) in enumerate(kv_spans):
        if k.dim() != 3 or k.shape != v.shape or k.stride() != v.stride():
            raise ValueError("each span is a (k, v) pair of [H_kv, T, D] views with equal strides")
        if k.shape[2] != D:
            raise ValueError(f"span {i} has head_dim {k.shape[2]}, q has {D}")
        if hkv is None:
            hkv = k.shape[0]
        elif k.shape[0] != hkv:
            raise ValueError("every span must have the same number of KV heads")
        if k.dtype != q3.dtype or v.dtype != q3.dtype:
            raise TypeError(f"span {i} is {k.dtype}; q is {q3.dtype}")
        if k.is_cuda or v.is_cuda:
            if k.device != q3.device or v.device != q3.device:
                raise ValueError(f"span {i} is on {k.device}, q on {q3.device}")
        else:
            if not (k.is_pinned() and v.is_pinned()):
                raise ValueError(f"host span {i} must be in page-locked memory (Tensor.pin_memory())")
            host += [k, v]
        rows.append((k.data_ptr(), v.data_ptr(), k.shape[1], k.stride(0), k.stride(1), k.stride(2)))
        kv_len += k.shape[1]
    if hkv is None:
        hkv = Hq  # no keys at all: every row is zero
    if Hq % hkv:
        raise ValueError(f"Hq={Hq} is not a multiple of H_kv={hkv}")
    if out is None:
        out3 = torch.empty((q_len, Hq, D), dtype=q3.dtype, device=q3.device)
    else:
        out3 = out[0] if out.dim() == 4 else out
        if out3.shape != (q_len, Hq, D) or out3.dtype != q3.dtype or out3.stride(2) != 1 \
                or out3.stride(1) != D:
            raise ValueError("out must be [q_len, Hq, D] in q's dtype with contiguous heads")
    # pi_kv_span_t[]: six 64-bit fields per span (two addresses, length, three strides)
    table = np.array(rows if rows else [(0, 0, 0, 0, 0, 1)], dtype=np.uint64)
    _host_stream_launch(q3, out3, table, len(kv_spans), hkv, kv_len, q_start, causal, scale,
                        workspace, err)
    _keep_until_done(host)
    if out is not None:
        return out
    return out3.unsqueeze(0) if batched else out3


def _host_stream_launch(q3: torch.Tensor, out3: torch.Tensor, table: np.ndarray, n_spans: int,
                        hkv: int, kv_len: int, q_start: int, causal: bool, scale: float | None,
                        workspace: Workspace | None, err: torch.Tensor | None) -> None:
    q_len, Hq, D = q3.shape
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    nbytes = int(_capi.load().pi_host_stream_attn_workspace_size(q_len, Hq, hkv, D, kv_len))
    ws_ptr = None
    if nbytes:
        if workspace is None:
            idx = q3.device.index
            with _ws_lock:
                workspace = _hs_ws.get(idx)
                if workspace is None:
                    workspace = _hs_ws[idx] = Workspace(q3.device)
        ws_ptr = workspace.get(nbytes).data_ptr()
    _capi.call(
        "pi_host_stream_attn",
        out3.data_ptr(), q3.data_ptr(), q3.stride(0), out3.stride(0), table.ctypes.data,
        n_spans, q_len, int(q_start), 1 if causal else 0, Hq, hkv, D, float(scale),
        dtype_code(q3.dtype), ws_ptr, nbytes, _capi.HS_SPANS_CHECKED, _err_ptr(err), _stream(),
    )


def host_stream_attention_table(q: torch.Tensor, out: torch.Tensor, table: np.ndarray,
                                num_kv_heads: int, q_start: int = 0, causal: bool = True,
                                scale: float | None = None, workspace: Workspace | None = None,
                                err: torch.Tensor | None = None) -> torch.Tensor:
    """host_stream_attention over a span table the caller has already built and checked.

    `table` is a uint64 [n, 6] array, one row per span in sequence order: K address, V
    address, length T, then the element strides of the [H_kv, T, D] views (head, token,
    dim). Every span must be device memory on q's GPU or page-locked host memory, in q's
    dtype with `num_kv_heads` heads and q's head_dim, and stay allocated until the launch
    has run; nothing here re-checks them. This is the per-step path of a decode loop that
    keeps its host chunks' rows across steps (decode.HostStoreDecoder): building the table
    is a few array operations instead of per-span tensor checks. q and out are
    [q_len, Hq, D] on the GPU with contiguous heads.
    """
    if q.dim() != 3 or out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("q and out must both be [q_len, Hq, D] in one dtype")
    if q.stride(2) != 1 or q.stride(1) != q.shape[2] or out.stride(2) != 1 \
            or out.stride(1) != q.shape[2]:
        raise ValueError("q and out need contiguous heads")
    _require_cuda(q, out)
    if table.dtype != np.uint64 or table.ndim != 2 or table.shape[1] != 6 or not table.flags.c_contiguous:
        raise ValueError("table must be a C-contiguous uint64 [n, 6] array")
    n = table.shape[0]
    if n > _capi.HS_MAX_SPANS:
        raise ValueError(f"at most {_capi.HS_MAX_SPANS} spans per call")
    if q.shape[1] % num_kv_heads:
        raise ValueError(f"Hq={q.shape[1]} is not a multiple of H_kv={num_kv_heads}")
    kv_len = int(table[:, 2].sum()) if n else 0
    if n == 0:
        table = np.array([(0, 0, 0, 0, 0, 1)], dtype=np.uint64)
    _host_stream_launch(q, out, table, n, num_kv_heads, kv_len, q_start, causal, scale,
                        workspace, err)
    return out


# ---------------------------------------------------------------------------
# e: decode attention with the all-gather fused in (multi-GPU, peer stores)
# ---------------------------------------------------------------------------


def paged_decode_attention_gather(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_tables: torch.Tensor,
    ctx_lens: torch.Tensor,
    exchange,
    scale: float | None = None,
    workspace: Workspace | None = None,
    err: torch.Tensor | None = None,
) -> torch.Tensor:
    """This rank's heads of decode attention, all-gathered across ranks in-kernel.

    `exchange` is a dist.PeerExchange built for (B, Hq_local, D). Returns the gathered
    [world * B, Hq_local, D] buffer (rank-major), complete (every rank's rows) for the
    work that follows on the current stream: the launch ends only after every rank's
    slice has landed (bounded wait; `err` gets PI_ERR_TIMEOUT if a rank never launches).
    """
    P, Hkv, S, D = _check_pool(k_pool, "k_pool")
    B, Hq, _ = q.shape
    if q.dtype != k_pool.dtype or q.shape[2] != D:
        raise ValueError("q must be [B, Hq_local, D] in the pool dtype")
    if exchange.shape != (exchange.world * B, Hq, D) or exchange.dtype != q.dtype:
        raise ValueError("exchange was built for another shape or dtype")
    _require_cuda(q, k_pool, v_pool, block_tables, ctx_lens)
    q = q.contiguous()
    block_tables, ctx_lens = _early_reads(block_tables, ctx_lens)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    ex = exchange
    slot, g = ex.next_launch()
    gathered = ex.slot_tensor(slot)
    out = gathered[ex.rank * B:(ex.rank + 1) * B]
    nbytes = workspace_bytes(B, Hq, Hkv, D)
    ws = (workspace or default_workspace(q.device)).get(nbytes)
    _capi.call(
        "pi_paged_decode_attn_gather",
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        block_tables.data_ptr(), block_tables.stride(0), ctx_lens.data_ptr(),
        B, Hq, Hkv, D, S, P, float(scale), dtype_code(q.dtype), q.stride(0), out.stride(0),
        ws.data_ptr(), ws.numel(), ctypes.byref(g), _err_ptr(err), _stream(),
    )
    return gathered
