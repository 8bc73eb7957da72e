"""The 4-bit key / value cache's tensors and format (csrc/cache4.hip has its kernels, ``reference`` its oracles)."""
from __future__ import annotations

from typing import NamedTuple

import torch

SCALE_BYTES = 4  # of a key's row of scales, D / 32 of them used
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class Cache4(NamedTuple):
    """Keys and values in 4 bits: codes uint8 [..., slots, Hkv, max_seq, D / 2] (element 2 j of a row in the low half of byte j;
    a code is a sign and one of ``MAGNITUDES``), scales uint8 [..., slots, Hkv, max_seq, 4], one for 32 elements along the head:
    2^(byte - 127), 255 for a block that holds an inf or a NaN (elements from 1.75 2^127 on read as inf). A leading dimension is the layer (``layer`` takes one)."""
    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    def layer(self, i: int) -> "Cache4":
        return Cache4(self.k[i], self.k_scale[i], self.v[i], self.v_scale[i])


def new_cache4(slots: int, Hkv: int, max_seq: int, D: int, device, layers: int | None = None) -> Cache4:
    if D not in (64, 96, 128):
        raise ValueError(f"head dim {D}: a 4-bit cache holds 64, 96 or 128")
    lead = (slots, Hkv, max_seq) if layers is None else (layers, slots, Hkv, max_seq)
    zeros = lambda n: torch.zeros((*lead, n), dtype=torch.uint8, device=device)  # noqa: E731
    return Cache4(zeros(D // 2), zeros(SCALE_BYTES), zeros(D // 2), zeros(SCALE_BYTES))


def cache4_bytes(slots: int, Hkv: int, max_seq: int, D: int, layers: int = 1) -> int:
    return layers * slots * Hkv * max_seq * 2 * (D // 2 + SCALE_BYTES)
