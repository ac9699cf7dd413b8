"""Paged KV-cache layout read by the forest cascade kernels.

One cache tensor per layer, shape ``[2, num_blocks, num_kv_heads, block_size * head_dim]``
(plane 0 = K, plane 1 = V), block_size fixed at 16 tokens.  Inside one (block, kv head)
tile the element order is the MFMA operand order of gfx950, so a wavefront can load its
operands with one contiguous 16-byte read per lane and no shuffle:

* K tile: ``[head_dim / x, 16 tokens, x]`` with ``x = 16 bytes / element size`` (8 for bf16,
  16 for fp8).  For one 16-byte slice of the head dimension the 16 tokens are adjacent.
* V tile: ``[head_dim, 16 tokens]``.  For one channel the 16 tokens are adjacent, which is
  the contraction order of the ``P @ V`` product.

This is the split layout the vLLM ROCm paged-attention path uses for its cache, so a
stock ROCm backend can serve the prefill side of the same cache.

A float8_e4m3fn cache comes in two forms: with one scale per KV head, given by the caller, or
block-scaled: a fp32 table ``[num_blocks, num_kv_heads, 2]`` beside the cache holds one scale per
block, KV head and plane (K's, V's), which the cache writer takes from the data.

The attention-backend hook ``get_kv_cache_shape`` of the engine that the platform starts
(``arctic_platform/common/ray_server.py:395-404``) is where this shape is announced.
"""

from __future__ import annotations

import torch

BLOCK_SIZE = 16


def x_width(dtype: torch.dtype) -> int:
    """Elements per 16-byte slice of the head dimension in a K tile."""
    return 16 // torch.empty((), dtype=dtype).element_size()


def kv_cache_shape(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int):
    if block_size != BLOCK_SIZE:
        raise ValueError(f"forest cascade attention supports block_size={BLOCK_SIZE} only, got {block_size}")
    return (2, num_blocks, num_kv_heads, block_size * head_dim)


def block_scales_shape(num_blocks: int, num_kv_heads: int):
    """Shape of the fp32 scale table of a block-scaled cache.  The table needs no initial values (a
    block's scales are written with its first token); zeros are a good choice."""
    return (num_blocks, num_kv_heads, 2)


def pack_blocks(k: torch.Tensor, v: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Token-major blocks ``[num_blocks, 16, num_kv_heads, head_dim]`` -> cache tensor."""
    if k.shape != v.shape or k.dim() != 4 or k.shape[1] != BLOCK_SIZE:
        raise ValueError("k and v must both be [num_blocks, 16, num_kv_heads, head_dim]")
    dtype = dtype or k.dtype
    nb, bs, hkv, d = k.shape
    x = x_width(dtype)
    if d % x:
        raise ValueError(f"head_dim {d} is not a multiple of {x}")
    cache = torch.empty(kv_cache_shape(nb, bs, hkv, d), dtype=dtype, device=k.device)
    # K: [nb, tok, h, d/x, x] -> [nb, h, d/x, tok, x]
    cache[0].view(nb, hkv, d // x, bs, x).copy_(k.view(nb, bs, hkv, d // x, x).permute(0, 2, 3, 1, 4))
    # V: [nb, tok, h, d] -> [nb, h, d, tok]
    cache[1].view(nb, hkv, d, bs).copy_(v.permute(0, 2, 3, 1))
    return cache


def unpack_blocks(cache: torch.Tensor, head_dim: int):
    """Cache tensor -> token-major ``(k, v)`` blocks ``[num_blocks, 16, num_kv_heads, head_dim]``."""
    two, nb, hkv, tile = cache.shape
    if two != 2 or tile != BLOCK_SIZE * head_dim:
        raise ValueError("not a forest-cascade KV cache tensor")
    x = x_width(cache.dtype)
    k = cache[0].view(nb, hkv, head_dim // x, BLOCK_SIZE, x).permute(0, 3, 1, 2, 4).reshape(nb, BLOCK_SIZE, hkv, head_dim)
    v = cache[1].view(nb, hkv, head_dim, BLOCK_SIZE).permute(0, 3, 1, 2)
    return k, v


def convert_cache(cache: torch.Tensor, head_dim: int, dtype: torch.dtype) -> torch.Tensor:
    """Re-pack a cache for another element type (the slice width ``x`` depends on it)."""
    k, v = unpack_blocks(cache, head_dim)
    return pack_blocks(k.to(dtype), v.to(dtype), dtype)


E4M3_MAX = 448.0
SCALE_EXP_MIN, SCALE_EXP_MAX = -100, 120


def block_scale_for(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two s with ``amax <= 448 s``, kept within [2**-100, 2**120] (fp32)."""
    m, e = torch.frexp(amax.float())  # amax = m * 2**e with m in [0.5, 1); 448 = 0.875 * 2**9
    e = torch.where(m > 0.875, e + 1, e) - 9
    e = torch.where(amax > 0, e, torch.full_like(e, SCALE_EXP_MIN)).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def quantize_blocks(k: torch.Tensor, v: torch.Tensor):
    """Token-major blocks ``[num_blocks, 16, num_kv_heads, head_dim]`` -> ``(cache, block_scales)`` as
    ``append_kv(..., block_scales=)`` leaves them when whole blocks are written."""
    codes, scales = [], []
    for x in (k.float(), v.float()):
        finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
        s = block_scale_for(finite.amax(dim=(1, 3)))
        codes.append((x / s[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn))
        scales.append(s)
    return pack_blocks(*codes), torch.stack(scales, dim=-1).contiguous()


def dequantize_blocks(cache: torch.Tensor, block_scales: torch.Tensor, head_dim: int):
    """The way back: fp32 token-major ``(k, v)`` blocks of a block-scaled cache."""
    k, v = unpack_blocks(cache, head_dim)
    return k.float() * block_scales[:, None, :, 0:1], v.float() * block_scales[:, None, :, 1:2]
