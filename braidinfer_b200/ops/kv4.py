"""The 4-bit paged KV cache: its format, its PyTorch restatement and read-back.

A layer is a :class:`KV4Layer` of two tensors,

* ``codes``  uint8 ``[P, 2, Hkv, page, D/2]``: rows of ``D`` 4-bit codes, K in
  slab 0 and V in slab 1 (the slabs of the bf16 pool, ``ops/attention.py``);
* ``scales`` bf16 ``[P, 2, Hkv, page, D/64, 2]``: a pair (step ``s``, offset
  ``z``) for each group of 64 elements.

An element stands for ``s * c + z``.  A group with least element ``a`` and
largest ``b`` has ``s = bf16((b - a) * r)`` with ``r`` the fp32 number next to
1/15 and the product rounded to fp32 first, ``z = bf16(a)`` and
``c = round((x - z) / s)`` clamped to 0..15 (0 where ``s`` is 0), so a value is
off by at most half a step plus what rounding ``s`` and ``z`` to bf16 shifts the
ends of the range: ``|x' - x| <= s / 2 + 2**-8 * (|a| + |b|)``.  A group that
holds a NaN or an infinity reads as NaN throughout.  Steps are per token, KV
head and 64 elements: an outlier coarsens its own group alone.  A row of 128
elements takes 72 bytes instead of 256.

A row of codes is ``D / 8`` little-endian 32-bit words; word ``2 i + h`` holds
elements ``8 i + h D / 2`` and the seven after it, element ``j`` in bits
``4 j .. 4 j + 3`` (the order in which the attention kernels read them).

Attention over the cache on CUDA takes rotated query elements up to 2**100 in
magnitude, steps of V from 2**-60 on (0 included) and, where a group of V is
constant, values up to 2**50; beyond that its sums may overflow or lose bits.
"""
from __future__ import annotations

from typing import NamedTuple, Tuple

import torch

from ._ext import ext

KV4_GROUP = 64


class KV4Layer(NamedTuple):
    """One layer of a 4-bit paged KV cache (see the module's text)."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def page_size(self) -> int:
        return self.codes.shape[3]

    @property
    def head_dim(self) -> int:
        return self.codes.shape[4] * 2


class KV4Cache:
    """All layers' 4-bit cache; ``cache[i]`` is layer ``i`` as a :class:`KV4Layer`."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int,
                 device=None):
        if head_dim not in (64, 128):
            raise ValueError(f"4-bit KV cache: head_dim must be 64 or 128, got {head_dim}")
        shape = (num_layers, num_pages, 2, num_kv_heads, page_size)
        self.codes = torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device)
        self.scales = torch.zeros(*shape, head_dim // KV4_GROUP, 2, dtype=torch.bfloat16, device=device)

    def __getitem__(self, i: int) -> KV4Layer:
        return KV4Layer(self.codes[i], self.scales[i])

    def __len__(self) -> int:
        return self.codes.shape[0]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @staticmethod
    def row_bytes(head_dim: int) -> int:
        """Bytes of one (token, KV head) of K or of V."""
        return head_dim // 2 + head_dim // KV4_GROUP * 4


def kv4_pack_ref(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes ``[..., D/2]`` and scales ``[..., D/64, 2]`` of ``x [..., D]`` (fp32 arithmetic)."""
    d = x.shape[-1]
    g = x.float().unflatten(-1, (d // KV4_GROUP, KV4_GROUP))
    a, b = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    fine = g.isfinite().all(-1, keepdim=True) & (b - a).isfinite()
    nan = torch.full_like(a, float("nan"))
    fifteenth = torch.tensor(1 / 15, dtype=torch.float32, device=a.device)  # a product, as on CUDA: not a division
    s, z = torch.where(fine, (b - a) * fifteenth, nan).bfloat16(), torch.where(fine, a, nan).bfloat16()
    step = s.float()
    c = torch.where(fine & (step > 0), (g - z.float()) / torch.where(step > 0, step, torch.ones_like(step)),
                    torch.zeros_like(g))
    c = c.round().clamp(0, 15).to(torch.uint8).reshape(*x.shape[:-1], 2, d // 16, 8)
    c = c.transpose(-3, -2).reshape(*x.shape[:-1], d // 2, 2)
    return c[..., 0] | (c[..., 1] << 4), torch.cat([s, z], -1)


def kv4_unpack_ref(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values (fp32 ``[..., D]``) that codes and scales stand for."""
    d = codes.shape[-1] * 2
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], d // 16, 2, 8)
    c = c.transpose(-3, -2).reshape(*codes.shape[:-1], d // KV4_GROUP, KV4_GROUP).float()
    s = scales.float()
    return (s[..., :1] * c + s[..., 1:]).reshape(*codes.shape[:-1], d)


def kv4_read(kv_layer: KV4Layer, slots: torch.Tensor) -> torch.Tensor:
    """The K and V that the cache holds at ``slots [T]`` (int32 flat slots,
    ``page * page_size + offset``) as ``[T, 2, Hkv, D]`` bf16, rounded once;
    zeros for a slot outside the cache."""
    codes, scales = kv_layer
    if slots.dim() != 1:
        raise ValueError("kv4_read: slots must be one-dimensional")
    if codes.is_cuda:
        return ext().kv4_read(codes, scales, slots)
    P, ps, s = codes.shape[0], codes.shape[3], slots.long()
    ok = (s >= 0) & (s < P * ps)
    s = torch.where(ok, s, torch.zeros_like(s))
    v = kv4_unpack_ref(codes[s // ps, :, :, s % ps], scales[s // ps, :, :, s % ps])
    return torch.where(ok[:, None, None, None], v, torch.zeros_like(v)).bfloat16()
