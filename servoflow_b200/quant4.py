"""4-bit formats of libsfb200: packed codes, the K/V cache held in 4 bits
(KV4Cache, read by B200Backend.kv4_attention) and weights with group scales
(pack_w4, read by B200Backend.w4a16_linear).

Codes are integers c in [-8, 7]. Eight consecutive values of the contiguous
dimension make one little-endian 32-bit word: value 2i of the eight sits in
bits [4i, 4i+4), value 2i+1 in bits [16+4i, 16+4i+4); the nibble is c + 8.

pack_codes, unpack_codes, pack_w4 and KV4Cache.dequantize are setup-time and
test helpers in plain torch, on any device; the serving operators are kernels.
"""
from __future__ import annotations

import torch

from . import _capi

GROUP = 32                  # channels per scale of the K/V cache


def pack_codes(codes: torch.Tensor) -> torch.Tensor:
    """Integer codes in [-8, 7], [..., n] with n % 8 == 0 -> uint8 [..., n / 2]."""
    if codes.shape[-1] % 8:
        raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "the packed dimension must be a multiple of 8")
    n = (codes + 8).to(torch.uint8).unflatten(-1, (-1, 8))
    # byte j of a word holds nibbles 2j, 2j+1: values (0,2) (4,6) (1,3) (5,7)
    lo, hi = n[..., [0, 4, 1, 5]], n[..., [2, 6, 3, 7]]
    return (lo | (hi << 4)).flatten(-2)


def unpack_codes(packed: torch.Tensor) -> torch.Tensor:
    """uint8 [..., n / 2] -> int8 codes [..., n]."""
    b = packed.unflatten(-1, (-1, 4))
    out = torch.empty(*b.shape[:-1], 8, dtype=torch.int8, device=packed.device)
    out[..., [0, 4, 1, 5]] = (b & 15).to(torch.int8) - 8
    out[..., [2, 6, 3, 7]] = (b >> 4).to(torch.int8) - 8
    return out.flatten(-2)


def pack_w4(w: torch.Tensor, group: int = 128, scale_dtype: torch.dtype = torch.float16):
    """Quantises a float weight [N, K] to 4 bits per group of `group` inputs:
    s = max|w| / 7 rounded to scale_dtype, c = clamp(round(w / s), -7, 7), 0
    where s is 0. Returns (codes uint8 [N, K / 2], scales [N, K / group])."""
    if w.dim() != 2 or group not in (32, 64, 128) or w.shape[1] % group:
        raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "w must be [N, K] with K a multiple of group (32, 64 or 128)")
    if scale_dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise _capi.SfbError(_capi.SFB_ERR_DTYPE, f"scale dtype {scale_dtype}")
    g = w.float().unflatten(1, (-1, group))
    s = (g.abs().amax(-1) / 7.0).to(scale_dtype)
    f = s.float().unsqueeze(-1)
    c = torch.where(f > 0, torch.round(g / f).clamp(-7, 7), torch.zeros_like(g))
    return pack_codes(c.flatten(1).to(torch.int32)), s


class KV4Cache:
    """K and V of `batch` sessions in 4 bits: codes uint8 [batch, heads_kv,
    capacity, head_dim / 2] and scales fp16 [batch, heads_kv, capacity,
    head_dim / 32], the last two dimensions contiguous, K and V with the same
    strides. Owns nothing but the four tensors; `allocate` makes them."""

    __slots__ = ("k_codes", "v_codes", "k_scale", "v_scale")

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor):
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale

    @classmethod
    def allocate(cls, batch: int, heads_kv: int, capacity: int, head_dim: int, device="cuda") -> "KV4Cache":
        """A zeroed cache (every value 0); capacity is rounded up to a multiple of 32 slots."""
        if head_dim not in (64, 128) or batch < 0 or heads_kv < 1 or capacity < 0:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "head_dim must be 64 or 128")
        cap = (capacity + 31) // 32 * 32
        code = lambda: torch.full((batch, heads_kv, cap, head_dim // 2), 0x88, dtype=torch.uint8, device=device)
        scale = lambda: torch.zeros(batch, heads_kv, cap, head_dim // GROUP, dtype=torch.float16, device=device)
        return cls(code(), code(), scale(), scale())

    @property
    def shape(self):
        """(batch, heads_kv, capacity, head_dim)."""
        b, h, c, d2 = self.k_codes.shape
        return b, h, c, 2 * d2

    def dequantize(self):
        """(K, V) as fp32 [batch, heads_kv, capacity, head_dim], in plain torch."""
        out = []
        for c, s in ((self.k_codes, self.k_scale), (self.v_codes, self.v_scale)):
            out.append((unpack_codes(c).float().unflatten(-1, (-1, GROUP)) * s.float().unsqueeze(-1)).flatten(-2))
        return tuple(out)

    def pack(self):
        """(sfb_kv4_cache as bytes, batch, heads_kv, capacity, head_dim, device
        index); raises where the tensors do not fit it."""
        kc, vc, ks, vs = self.k_codes, self.v_codes, self.k_scale, self.v_scale
        shape, sshape, st, ss = kc.shape, ks.shape, kc.stride(), ks.stride()
        if len(shape) != 4 or len(sshape) != 4 or vc.shape != shape or vs.shape != sshape \
                or sshape[:3] != shape[:3] or sshape[3] * 16 != shape[3]:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "inconsistent cache shapes")
        if kc.dtype is not torch.uint8 or vc.dtype is not torch.uint8 or ks.dtype is not torch.float16 \
                or vs.dtype is not torch.float16:
            raise _capi.SfbError(_capi.SFB_ERR_DTYPE, "cache codes are uint8, scales fp16")
        if vc.stride() != st or vs.stride() != ss:
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "K and V of a cache share their strides")
        B, H, C, D2 = shape
        if st[3] != 1 or ss[3] != 1 or (C > 1 and (st[2] != D2 or ss[2] != sshape[3])):
            raise _capi.SfbError(_capi.SFB_ERR_SHAPE, "the last two dimensions of a cache are contiguous")
        dev = kc.get_device()
        if dev < 0 or vc.get_device() != dev or ks.get_device() != dev or vs.get_device() != dev:
            raise ValueError("the cache's tensors must be on one CUDA device")
        return (_capi.KV4_CACHE.pack(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), st[0], st[1],
                                     ss[0], ss[1], B, H, C, 2 * D2), B, H, C, 2 * D2, dev)
