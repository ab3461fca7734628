"""The 8-bit KV cache: one byte per element and one fp32 scale per (token, kv head), K and V apart.

``QuantKV`` is a pair of tensors that the runner and the models hand around where an fp16 cache is one tensor: ``data`` uint8
``[..., blocks, 2 (K, V), kv heads, block size, head dim]`` and ``scale`` fp32 ``[..., blocks, 2, kv heads, block size]``.  An
element stands for ``(data - 128) * scale``; ``data`` is 1 .. 255 where something was written, and a row of zeros has scale 0.
Bytes with an offset instead of signed ones: the attention kernel makes fp16 numbers of them with one byte permutation.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

KV_DTYPES = ("float16", "int8")
HEAD_DIMS = (64, 96, 128, 256)          # what the kernels are built for


class QuantKV:
    """The whole cache (a leading ``layers`` dimension) or one layer of it; ``kv[i]`` is layer i."""

    __slots__ = ("data", "scale")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor):
        if data.dtype is not torch.uint8 or scale.dtype is not torch.float32:
            raise TypeError(f"an 8-bit cache is uint8 data and float32 scales, not {data.dtype} and {scale.dtype}")
        shape = data.shape
        if len(shape) < 5 or shape[:-1] != scale.shape or shape[-4] != 2:
            raise ValueError(f"data [.., blocks, 2, kv heads, block size, head dim] and scales of its leading dimensions are "
                             f"needed, not {tuple(shape)} and {tuple(scale.shape)}")
        if data.get_device() != scale.get_device():
            raise ValueError(f"data on {data.device}, scales on {scale.device}")
        self.data, self.scale = data, scale

    @classmethod
    def zeros(cls, shape: Tuple[int, ...], device=None) -> "QuantKV":
        return cls(torch.zeros(shape, dtype=torch.uint8, device=device),
                   torch.zeros(shape[:-1], dtype=torch.float32, device=device))

    def __getitem__(self, layer: int) -> "QuantKV":
        return QuantKV(self.data[layer], self.scale[layer])

    @property
    def shape(self) -> torch.Size:
        return self.data.shape

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def num_blocks(self) -> int:
        return self.data.shape[-5]

    @property
    def kv_heads(self) -> int:
        return self.data.shape[-3]

    @property
    def block_size(self) -> int:
        return self.data.shape[-2]

    @property
    def head_dim(self) -> int:
        return self.data.shape[-1]

    def copy_block(self, src: int, dst: int) -> None:
        """Copies a block of every layer."""
        self.data[:, dst].copy_(self.data[:, src])
        self.scale[:, dst].copy_(self.scale[:, src])


def refuses(config) -> Optional[str]:
    """Why a model cannot keep its cache in 8 bits, or None where it can."""
    if config.is_gemma or config.is_latent or config.is_hybrid:
        return f"'{config.arch}' keeps its cache at 16 bits or more"
    if config.head_dim not in HEAD_DIMS:
        return f"head dimension {config.head_dim} (8-bit caches: {', '.join(map(str, HEAD_DIMS))})"
    if config.num_heads // config.num_kv_heads > 16:
        return f"{config.num_heads // config.num_kv_heads} query heads per kv head (8-bit caches: up to 16)"
    rot = config.head_dim if not config.partial_rotary_factor else 2 * int(config.partial_rotary_factor * config.head_dim // 2)
    if rot % 16:
        return f"{rot} rotated dimensions of a head (8-bit caches: a multiple of 16)"
    return None
