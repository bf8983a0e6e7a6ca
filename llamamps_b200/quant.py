"""Q4 weight format (utils/pack_weights.py) -- packing on the host or device.

Format (utils/pack_weights.py:18-46): the tensor is flattened row-major,
zero-padded to a multiple of 32, and split into groups of 32; scale =
max|w|/7 in fp32 (0 -> 1.0); code = round-half-even(w/scale) clamped to
[-8, 7]; nibble = code + 8; byte b = nib[2b] | nib[2b+1] << 4; scales are
stored fp16.  ``pack_q4`` runs the CUDA packer for device tensors and a torch
implementation for host tensors (the offline converter path; decode never
packs).
"""
from __future__ import annotations

import torch

GROUP = 32


def pack_q4_host(w: torch.Tensor):
    """Host packer (offline conversion): returns (uint8[n_pad/2], float16[n_pad/32])."""
    flat = w.detach().to(torch.float32).reshape(-1).cpu()
    pad = (GROUP - flat.numel() % GROUP) % GROUP
    if pad:
        flat = torch.cat([flat, torch.zeros(pad, dtype=torch.float32)])
    blocks = flat.view(-1, GROUP)
    scales = blocks.abs().amax(dim=1) / 7.0
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    codes = torch.round(blocks / scales[:, None]).clamp_(-8, 7).to(torch.int16) + 8
    u = codes.to(torch.uint8).reshape(-1)
    packed = u[0::2] | (u[1::2] << 4)
    return packed.contiguous(), scales.to(torch.float16)


def pack_q4(w: torch.Tensor):
    """Pack ``w`` into the Q4 format on the tensor's own device."""
    if w.is_cuda:
        from .kernels import q4_pack_device
        return q4_pack_device(w.detach().to(torch.float32).contiguous())
    return pack_q4_host(w)


def unpack_q4(packed: torch.Tensor, scales: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """The fp16 [rows, k] values of a Q4 matrix (code * scale, rounded once)."""
    p = packed.reshape(-1, GROUP // 2)
    c = torch.stack([p & 15, p >> 4], dim=-1).flatten(-2).to(torch.float32) - 8.0
    return (c * scales.reshape(-1, 1).to(torch.float32)).to(torch.float16).reshape(rows, k)


# -- rows of the 4-bit KV cache (include/llamamps_b200.h, "4-bit KV cache") ----
KV_ROW_BYTES = 72     # 64 code bytes and 4 fp16 scales for 128 elements


def quantise_kv_rows(x: torch.Tensor):
    """fp16 rows [..., 128] as the cache holds them: (uint8 codes [..., 64],
    fp16 scales [..., 4]).  The scale of a group of 32 is the smallest number
    with 8 significant bits (and multiple of 2^-24, at most 9344) that is >=
    max|x| / 7, or 1 for a zero group, so code * scale is exact in fp16; a row
    that is not finite gets NaN scales."""
    g = x.to(torch.float64).unflatten(-1, (-1, GROUP))
    finite = torch.isfinite(g).all(dim=-1).all(dim=-1)[..., None]
    g = torch.where(finite[..., None], g, torch.zeros_like(g))
    top = g.abs().amax(dim=-1)
    m, e = torch.frexp(top / 7.0)
    scale = torch.ldexp(torch.ceil(m * 256.0), e - 8)
    scale = torch.where(scale < 2.0 ** -16, torch.ceil(scale * 2.0 ** 24) * 2.0 ** -24, scale).clamp(max=9344.0)
    scale = torch.where(top == 0, torch.ones_like(scale), scale)
    n = (torch.round(g / scale[..., None]).clamp(-7, 7).flatten(-2) + 8).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), torch.where(finite, scale, torch.nan).to(torch.float16)


def dequantise_kv_rows(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp16 values of cached rows: (codes [..., 64], scales [..., 4]) -> [..., 128] (exact)."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(torch.float32) - 8.0
    return (c.unflatten(-1, (-1, GROUP)) * scales.to(torch.float32)[..., None]).flatten(-2).to(torch.float16)
