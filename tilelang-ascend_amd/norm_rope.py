"""Norms of query and key heads with the position rotation in the same pass, gfx950.

``qk_norm_rope(q, k, q_weight, k_weight, positions, cos, sin)`` takes a token's
heads as they lie in the projection's output (views of it) and returns the
normed, rotated queries and keys; ``qk_norm_rope_paged`` writes the keys, and the
values beside them, to rows of the paged cache that ``paged_gqa_fwd`` reads, in
the same launch.  Per head: ``y = x / sqrt(mean(x^2) + eps) * weight``, then the
first R = 2 * cos.shape[1] elements rotated in pairs (i, i + R/2), or (2i, 2i+1)
with ``interleaved``; fp32 throughout, rounded once.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

_KINDS = {torch.bfloat16: _lib.KIND_BF16, torch.float16: _lib.KIND_FP16}


def _heads(name: str, t: torch.Tensor, like: torch.Tensor) -> int:
    """Checks a [T, heads, D] argument whose tokens may lie apart; returns the token stride."""
    if t.dim() != 3 or t.shape[0] != like.shape[0] or t.shape[2] != like.shape[2]:
        raise ValueError(f"{name} must be [{like.shape[0]}, heads, {like.shape[2]}], got {tuple(t.shape)}")
    if t.dtype != like.dtype:
        raise ValueError(f"{name} dtype {t.dtype} must equal q dtype {like.dtype}")
    n, D = t.shape[1], t.shape[2]
    if t.stride(2) != 1 or (n > 1 and t.stride(1) != D):
        raise ValueError(f"{name}: a token's heads must be contiguous, got strides {t.stride()}")
    stride = t.stride(0) if t.shape[0] > 1 else n * D
    if stride % 8 != 0 or t.data_ptr() % 16 != 0:
        raise ValueError(f"{name}: tokens must start on 16 bytes (offset and stride multiples of 8 elements)")
    return stride


def _run(q, k, v, q_weight, k_weight, positions, cos, sin, k_cache, v_cache, slots, eps, interleaved):
    if q.dtype not in _KINDS:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    if q.dim() != 3:
        raise ValueError(f"q must be [T, H, D], got {tuple(q.shape)}")
    T, H, D = q.shape
    if D % 8 != 0 or not 8 <= D <= 512:
        raise ValueError(f"the head width must be a multiple of 8 in [8, 512], got {D}")
    dev = _lib.require_device(q, k, v, q_weight, k_weight, positions, cos, sin, k_cache, v_cache, slots)
    strides = [_heads(n, t, q) if t is not None else 0 for n, t in (("q", q), ("k", k), ("v", v))]
    G = k.shape[1]
    if v is not None and v.shape[1] != G:
        raise ValueError(f"v has {v.shape[1]} heads, k has {G}")
    wk = None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if tuple(w.shape) != (D,) or w.dtype not in (q.dtype, torch.float32):
            raise ValueError(f"{name} must be [{D}] in float32 or {q.dtype}, got {tuple(w.shape)} {w.dtype}")
        _lib.require_contiguous(name, w)
        if wk is not None and w.dtype != wk:
            raise ValueError("q_weight and k_weight must have one dtype")
        wk = w.dtype
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"cos and sin must be float32 [positions, R / 2], got {tuple(cos.shape)} {cos.dtype} and "
                         f"{tuple(sin.shape)} {sin.dtype}")
    R = 2 * cos.shape[1]
    if R % 16 != 0 or R > D:
        raise ValueError(f"R = 2 * cos.shape[1] must be a multiple of 16 up to the head width {D}, got {R}")
    _lib.require_contiguous("cos", cos)
    _lib.require_contiguous("sin", sin)

    def ints(name, t):
        if t.numel() != T or t.dtype not in (torch.int32, torch.int64, torch.int16, torch.uint8, torch.int8):
            raise ValueError(f"{name} must hold one integer per token ({T}), got {tuple(t.shape)} {t.dtype}")
        return _lib.saturated_int32(t).contiguous()  # values past 32 bits mark padding, as they did

    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    rows = 0
    with torch.cuda.device(dev):
        positions = ints("positions", positions)
        if k_cache is not None:
            slots = ints("slots", slots)
            for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
                if c.dim() != 4 or tuple(c.shape[2:]) != (G, D) or c.dtype != q.dtype or c.shape != k_cache.shape:
                    raise ValueError(f"{name} must be [blocks, block_size, {G}, {D}] {q.dtype}, got {tuple(c.shape)} "
                                     f"{c.dtype}")
                _lib.require_contiguous(name, c)
            if k_cache.numel() and k_cache.data_ptr() == v_cache.data_ptr():
                raise ValueError("k_cache and v_cache must be caches of their own")
            rows = k_cache.shape[0] * k_cache.shape[1]
        q_out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
        k_out = torch.empty((T, G, D), dtype=q.dtype, device=dev) if k_cache is None else k_cache
        rc = _lib.load_library().dsa_qk_norm_rope(
            _KINDS[q.dtype], _lib.ptr(q), strides[0], _lib.ptr(k), strides[1], _lib.ptr(v), strides[2],
            _lib.ptr(q_weight), _lib.ptr(k_weight), _lib.KIND_FP32 if wk == torch.float32 else _KINDS[q.dtype],
            _lib.ptr(positions), _lib.ptr(cos), _lib.ptr(sin), cos.shape[0], T, H, G, D, R, eps,
            1 if interleaved else 0, _lib.ptr(slots), rows, _lib.ptr(q_out), _lib.ptr(k_out), _lib.ptr(v_cache),
            _lib.stream_handle(dev))
        _lib.check(rc, "dsa_qk_norm_rope")
    return q_out, k_out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                 k_weight: Optional[torch.Tensor], positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                 eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q_out [T, H, D], k_out [T, G, D]) of q [T, H, D] and k [T, G, D] (bf16 or fp16; tokens may lie apart).

    Weights [D] (float32 or q's dtype; None: ones); positions: one integer per token into the rows of cos and sin
    [P, R/2] float32 (R a multiple of 16 up to D).  A position outside [0, P) marks a padding token: rows of zeros.
    """
    res = _lib.host_path().qk_norm_rope(q, k, None, q_weight, k_weight, positions, cos, sin, None, None, None, eps,
                                        interleaved)
    if res is not None:
        return _lib.returned(res, "dsa_qk_norm_rope")
    return _run(q, k, None, q_weight, k_weight, positions, cos, sin, None, None, None, eps, interleaved)


def qk_norm_rope_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor],
                       k_weight: Optional[torch.Tensor], positions: torch.Tensor, cos: torch.Tensor,
                       sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor, *,
                       eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """``qk_norm_rope`` whose keys, and the values v [T, G, D] as they are, go to row ``slots[t]`` of the caches
    [blocks, block_size, G, D] (in place); returns q_out.

    A slot outside [0, blocks * block_size), and any token whose position marks it as padding, writes nothing;
    other rows of the caches are left as they were.  The slots inside must differ from each other.
    """
    res = _lib.host_path().qk_norm_rope(q, k, v, q_weight, k_weight, positions, cos, sin, k_cache, v_cache, slots,
                                        eps, interleaved)
    if res is not None:
        return _lib.returned(res, "dsa_qk_norm_rope")[0]
    for name, t in (("v", v), ("k_cache", k_cache), ("v_cache", v_cache), ("slots", slots)):
        if t is None:
            raise ValueError(f"{name} is required")
    return _run(q, k, v, q_weight, k_weight, positions, cos, sin, k_cache, v_cache, slots, eps, interleaved)[0]
