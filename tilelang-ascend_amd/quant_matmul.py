"""8-bit matrix product with a scale for each token and each output channel, gfx950.

``quant_matmul(x, weight, x_scale, weight_scale)`` multiplies rows as
``act_quant(..., dtype=torch.int8)`` writes them -- activations with a scale per
token, weights [N, K] with a scale per output channel -- in int32 (exact) and
returns ``x weight^T * x_scale * weight_scale^T + bias`` rounded once to
``dtype``: the projections of an 8-bit layer between the quantiser and the
attention kernels.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_OUT = {torch.bfloat16: _lib.KIND_BF16, torch.float16: _lib.KIND_FP16, torch.float32: _lib.KIND_FP32}
MAX_K = 131071  # int32 sums of products of at most 2^14


def quant_matmul(x: torch.Tensor, weight: torch.Tensor, x_scale: torch.Tensor, weight_scale: torch.Tensor,
                 bias: Optional[torch.Tensor] = None, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[..., N] in ``dtype`` (bfloat16, float16 or float32) from x [..., K] int8 (x_scale: one fp32 per row, as
    ``act_quant`` returns it), weight [N, K] int8 (weight_scale: one fp32 per row) and bias [N] or None."""
    res = _lib.host_path().quant_matmul(x, weight, x_scale, weight_scale, bias, _OUT.get(dtype))
    if res is not None:
        return _lib.returned(res, "dsa_quant_matmul")
    if dtype not in _OUT:
        raise ValueError(f"dtype must be torch.bfloat16, torch.float16 or torch.float32, got {dtype}")
    for name, t in (("x", x), ("weight", weight)):
        if t.dtype != torch.int8:
            raise ValueError(f"{name} must be int8, got {t.dtype}")
    for name, t in (("x_scale", x_scale), ("weight_scale", weight_scale)):
        if t.dtype != torch.float32:
            raise ValueError(f"{name} must be float32, got {t.dtype}")
    if x.dim() < 2 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if not 1 <= K <= MAX_K:
        raise ValueError(f"K must be in [1, {MAX_K}], got {K}")
    M = x.numel() // K
    if x_scale.numel() != M:
        raise ValueError(f"x_scale must have one entry per row ({M}), got {x_scale.numel()}")
    if weight_scale.numel() != N:
        raise ValueError(f"weight_scale must have one entry per output channel ({N}), got {weight_scale.numel()}")
    if bias is not None and (tuple(bias.shape) != (N,) or not bias.dtype.is_floating_point):
        raise ValueError(f"bias must be [{N}] in a floating-point type, got {tuple(bias.shape)} {bias.dtype}")
    dev = _lib.require_device(x, weight, x_scale, weight_scale, bias)
    for name, t in (("x", x), ("weight", weight), ("x_scale", x_scale), ("weight_scale", weight_scale)):
        _lib.require_contiguous(name, t)
    with torch.cuda.device(dev):
        bias = None if bias is None else bias.to(torch.float32).contiguous()
        out = torch.empty(x.shape[:-1] + (N,), dtype=dtype, device=dev)
        if M and N:
            lib = _lib.load_library()
            aligned = (x.data_ptr() | weight.data_ptr()) % 16 == 0
            ws_bytes = lib.dsa_quant_matmul_workspace_size(M, N, K, 1 if aligned else 0)
            ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev) if ws_bytes else None
            rc = lib.dsa_quant_matmul(_OUT[dtype], _lib.ptr(x), _lib.ptr(weight), _lib.ptr(x_scale),
                                      _lib.ptr(weight_scale), _lib.ptr(bias), M, N, K, _lib.ptr(out), _lib.ptr(ws),
                                      ws_bytes, _lib.stream_handle(dev))
            _lib.check(rc, "dsa_quant_matmul")
    return out
