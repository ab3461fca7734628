"""Rows and weights in 8-bit floating point (e4m3) with fp32 scales, as ``ops.backend``'s ``*_fp8`` operators take them.

``Fp8Rows``: activations.  ``data`` e4m3 ``[rows, columns]`` and ``scale`` ``[blocks of 128 columns, rows]``: an element stands for
``data * scale``, and what the operators write has the scale max|x| / 448 of its block (0 where that is not above 1e-30; a block that
holds an infinity or a NaN reads back as NaN).

``Fp8Weight``: a linear layer.  ``data`` e4m3 ``[N, K]`` and ``scale`` ``[blocks of 128 rows, blocks of 128 columns]``, the layout that
checkpoints of such weights have.  With ``glu`` it is a gate and an up weight of N / 2 rows each, one after the other, and the up
weight begins blocks of its own.

The operators write memory of its own: data and scales (and ``add_rmsnorm_fp8``'s residual and ``normed``) that share bytes with anything
else of the call are refused on the GPU.  Columns of the same buffer side by side are fine, and so is ``normed`` in the place of ``add``.
"""
from __future__ import annotations

from typing import Optional

import torch

BLOCK, TOP, LEAST = 128, 448.0, 1e-30
F8, F32 = torch.float8_e4m3fn, torch.float32
BIAS_TYPES = frozenset((torch.float16, torch.bfloat16, F32))


def blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


class Fp8Rows:
    __slots__ = ("data", "scale")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor):
        shape = data.shape
        if data.dtype is not F8 or scale.dtype is not F32:
            raise TypeError(f"rows in 8 bits are float8_e4m3fn data and float32 scales, not {data.dtype} and {scale.dtype}")
        if len(shape) != 2 or scale.shape != ((shape[1] + 127) // 128, shape[0]):
            raise ValueError(f"data [rows, columns] and scales [blocks of {BLOCK} columns, rows] are needed, not {tuple(shape)} and "
                             f"{tuple(scale.shape)}")
        if data.get_device() != scale.get_device():
            raise ValueError(f"data on {data.device}, scales on {scale.device}")
        self.data, self.scale = data, scale

    @classmethod
    def empty(cls, rows: int, columns: int, device=None) -> "Fp8Rows":
        return cls(torch.empty(rows, columns, dtype=F8, device=device), torch.empty(blocks(columns), rows, dtype=F32, device=device))

    @property
    def shape(self) -> torch.Size:
        return self.data.shape

    def __getitem__(self, rows: slice) -> "Fp8Rows":
        return Fp8Rows(self.data[rows], self.scale[:, rows])

    def dequant(self) -> torch.Tensor:
        """The rows as fp32."""
        return self.data.float() * self.scale.t().repeat_interleave(BLOCK, 1)[:, : self.data.shape[1]]


class Fp8Weight:
    __slots__ = ("data", "scale", "bias", "glu")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, bias: Optional[torch.Tensor] = None, glu: bool = False):
        shape = data.shape
        if data.dtype is not F8 or scale.dtype is not F32:
            raise TypeError(f"a weight in 8 bits is float8_e4m3fn data and float32 scales, not {data.dtype} and {scale.dtype}")
        if len(shape) != 2 or (glu and shape[0] % 2) or scale.shape != (
                2 * ((shape[0] // 2 + 127) // 128) if glu else (shape[0] + 127) // 128, (shape[1] + 127) // 128):
            raise ValueError(f"data [N, K] and scales of blocks of {BLOCK} x {BLOCK}{' of each half' if glu else ''} are needed, not "
                             f"{tuple(shape)} and {tuple(scale.shape)}")
        device = data.get_device()
        if not scale.is_contiguous() or device != scale.get_device():
            raise ValueError("the scales have to be contiguous, and on the device of the data")
        if bias is not None and (glu or bias.dtype not in BIAS_TYPES or bias.shape != shape[:1]
                                 or (bias.stride() != (1,) and shape[0] != 1) or bias.get_device() != device):
            raise ValueError(f"a bias of {shape[0]} numbers in fp16, bfloat16 or fp32 is expected beside the data, none for a gate and up weight")
        self.data, self.scale, self.bias, self.glu = data, scale, bias, glu

    @classmethod
    def from_dense(cls, w: torch.Tensor, bias: Optional[torch.Tensor] = None, glu: bool = False) -> "Fp8Weight":
        """Quantises ``w`` [N, K], once: a block's largest becomes 448."""
        if w.dim() != 2 or (glu and w.shape[0] % 2):
            raise ValueError(f"a weight [N, K] is expected, of two halves for a gate and up weight, not {tuple(w.shape)}")
        data, scales = [], []
        for part in w.chunk(2) if glu else [w]:
            n, k = part.shape
            x = torch.zeros(blocks(n) * BLOCK, blocks(k) * BLOCK, device=w.device)
            x[:n, :k] = part
            x = x.view(blocks(n), BLOCK, blocks(k), BLOCK)
            top = x.abs().amax((1, 3))
            steps = torch.where(top <= LEAST, torch.zeros_like(top), TOP / top)
            data.append((x * steps[:, None, :, None]).view(blocks(n) * BLOCK, -1)[:n, :k].to(F8))
            scales.append(torch.where(top <= LEAST, torch.zeros_like(top), top / TOP))
        return cls(torch.cat(data).contiguous(), torch.cat(scales), bias, glu)

    @property
    def N(self) -> int:
        return self.data.shape[0]

    @property
    def K(self) -> int:
        return self.data.shape[1]

    def dequant(self) -> torch.Tensor:
        """The weight as fp32."""
        rows = self.N // 2 if self.glu else self.N
        s = self.scale.repeat_interleave(BLOCK, 1)[:, : self.K].view(-1, blocks(rows), 1, self.K)
        return self.data.float() * s.expand(-1, -1, BLOCK, -1).reshape(s.shape[0], -1, self.K)[:, :rows].reshape(-1, self.K)
