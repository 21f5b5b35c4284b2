"""Attention of new tokens over a paged cache: grouped heads, chunks and single tokens, gfx950.

``paged_gqa_fwd(q, k_cache, v_cache, block_table, ...)`` returns ``(out, lse)``
for every key a token sees (the dense counterpart of ``sparse_gqa_fwd``):

* q         [T, H, D] packed sequences with ``actual_seq_lengths_query`` as
            inclusive prefix sums (TND), or [B, S, H, D] with lengths per
            sequence or none; D = 64 or 128, bf16 / fp16
* k_cache, v_cache  [blocks, block_size, G, D]; block_table [B, max_blocks]
* out like q, lse fp32 (natural log), [T, H] or [B, S, H]

Sequence b's new tokens are the last of its ``actual_seq_lengths_kv[b]`` tokens,
whose keys and values already lie in the cache.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

_KINDS = {torch.bfloat16: _lib.KIND_BF16, torch.float16: _lib.KIND_FP16}


def paged_gqa_fwd(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                  sm_scale: Optional[float] = None, *, actual_seq_lengths_query: Optional[torch.Tensor] = None,
                  actual_seq_lengths_kv: torch.Tensor = None, is_causal: bool = True,
                  win_left: Optional[int] = None,
                  sinks: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Grouped attention over a paged cache; returns ``(out, lse)``.

    Token i of a sequence with n keys and L new tokens sits at position p = n - L + i and sees the keys j < n with
    j <= p (``is_causal``) and j >= p - win_left (``win_left`` None: all).  ``sinks`` [H] fp32 adds exp(sink) to
    each head's denominator.  sm_scale defaults to D^-0.5.  Rows that see nothing -- padding rows, rows behind the
    last packed sequence -- give out = 0 and lse = -inf (or the sink).  A table entry outside the pool hides its keys.
    Keys that a row does not see do not reach it, whatever the caches hold there (infinities and NaN too); a value
    that it does see and that is not finite makes its column infinite or NaN (NaN where its weight rounds to 0).  Lengths
    stay on the device and are cut to what the table and q hold.  Prefix sums must not decrease (a sequence without
    new tokens repeats the one before it): on the host that is checked; on the device sums that do decrease leave
    rows of out and lse undefined.
    """
    scale = q.shape[-1] ** -0.5 if sm_scale is None and q.dim() >= 3 and q.shape[-1] > 0 else sm_scale
    win = -1 if win_left is None else -2 if win_left == -1 else win_left  # -1: none, in the calls below
    res = _lib.host_path().paged_gqa(q, k_cache, v_cache, block_table, scale, actual_seq_lengths_query,
                                     actual_seq_lengths_kv, is_causal, win, sinks)
    if res is not None:
        return _lib.returned(res, "dsa_paged_gqa_fwd")
    if q.dtype not in _KINDS:
        raise ValueError(f"q must be bfloat16 or float16, got {q.dtype}")
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dtype != q.dtype:
            raise ValueError(f"{name} dtype {c.dtype} must equal q dtype {q.dtype}")
    if q.dim() not in (3, 4) or q.shape[-1] not in (64, 128):
        raise ValueError(f"q must be [T, H, D] or [B, S, H, D] with D = 64 or 128, got {tuple(q.shape)}")
    H, D = q.shape[-2], q.shape[-1]
    if k_cache.dim() != 4 or k_cache.shape[3] != D or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache and v_cache must be [blocks, block_size, kv_group, {D}], got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    num_blocks, block_size, G, _ = k_cache.shape
    if G < 1 or H < 1 or H % G != 0:
        raise ValueError(f"H={H} must be a multiple of kv_group={G}")
    if num_blocks < 1 or block_size < 1:
        raise ValueError(f"the caches must hold at least one row, got {tuple(k_cache.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] < 1 or block_table.shape[1] < 1:
        raise ValueError(f"block_table must be [B, max_blocks], got {tuple(block_table.shape)}")
    if not _lib.is_integer(block_table):
        raise ValueError(f"block_table must hold integers, got {block_table.dtype}")
    B = block_table.shape[0]
    if actual_seq_lengths_kv is None:
        raise ValueError("actual_seq_lengths_kv is required")
    packed = q.dim() == 3
    if packed and actual_seq_lengths_query is None:
        raise ValueError("packed queries need actual_seq_lengths_query (inclusive prefix sums)")
    if not packed and q.shape[0] != B:
        raise ValueError(f"q batch {q.shape[0]} does not match block_table batch {B}")
    if not (isinstance(win, int) and -1 <= win < 2**31 - 4096) or (win_left is not None and win_left < 0):
        raise ValueError(f"win_left must be None or a key count, got {win_left}")
    if not 0 < scale <= 1e30:
        raise ValueError(f"sm_scale must be positive, got {sm_scale}")

    def lens(name, x):
        if x is None:
            return None
        t = torch.as_tensor(x)
        if not _lib.is_integer(t) or t.numel() != B:
            raise ValueError(f"{name} must hold B={B} integers, got {tuple(t.shape)} {t.dtype}")
        return _lib.saturated_int32(t).reshape(-1)

    ql = lens("actual_seq_lengths_query", actual_seq_lengths_query)
    kl = lens("actual_seq_lengths_kv", actual_seq_lengths_kv)
    if packed and ql.device.type == "cpu" and bool((ql[1:] < ql[:-1]).any()):
        raise ValueError("actual_seq_lengths_query must be non-decreasing prefix sums")
    dev = _lib.require_device(q, k_cache, v_cache, block_table, sinks)
    if sinks is not None and (sinks.dtype != torch.float32 or tuple(sinks.shape) != (H,)):
        raise ValueError(f"sinks must be [{H}] float32, got {tuple(sinks.shape)} {sinks.dtype}")
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
        _lib.require_contiguous(name, t)
    for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
        if t.data_ptr() % 16 != 0:
            raise ValueError(f"{name} must start on 16 bytes")

    with torch.cuda.device(dev):
        ql, kl = (None if x is None else x.to(dev).contiguous() for x in (ql, kl))
        bt = _lib.saturated_int32(block_table).contiguous()
        sk = None if sinks is None else sinks.contiguous()
        T = q.shape[0] if packed else B * q.shape[1]
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev)
        lib = _lib.load_library()
        ws_bytes = lib.dsa_paged_gqa_workspace_size(T, B, H, G, D, bt.shape[1] * block_size)
        ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev) if ws_bytes else None
        rc = lib.dsa_paged_gqa_fwd(_KINDS[q.dtype], _lib.ptr(q), _lib.ptr(k_cache), _lib.ptr(v_cache), _lib.ptr(bt),
                                   _lib.ptr(ql) if packed else None, None if packed else _lib.ptr(ql), _lib.ptr(kl),
                                   T, B, 0 if packed else q.shape[1], H, G, D, num_blocks, block_size, bt.shape[1],
                                   1 if is_causal else 0, win, _lib.ptr(sk), float(scale), _lib.ptr(out),
                                   _lib.ptr(lse), _lib.ptr(ws), ws_bytes, _lib.stream_handle(dev))
        _lib.check(rc, "dsa_paged_gqa_fwd")
    return out, lse
