"""A weight in microscaled 4-bit floating point (MXFP4) on the device.

The 4-bit base of a Linear whose product runs on the scaled matrix instruction of gfx950 (ops.linear_mxfp4, its input
quantised to the same format), next to the NF4 base of vpt.sdxl (which has to be dequantised first). A frozen LoRA base
too: vpt.sdxl.LoRALinearNF4 takes an MXFP4Weight in its "dequant" and "resident" modes.
"""

from __future__ import annotations

import torch

from . import ops

BF16 = torch.bfloat16


class MXFP4Weight:
    """A [N, K] tensor as `codes` u8 [N, 64 c] and `scales` u8 [N, 4 c], c = ceil(K / 128): rows padded with zeros to a
    multiple of 128 values, blocks of 32 (ops.mxfp4_quantize). Where K is a multiple of 128 these are the plain [N, K / 2]
    and [N, K / 32] of the format."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        self.shape = tuple(int(s) for s in shape)
        if len(self.shape) != 2 or self.shape[0] < 1 or self.shape[1] < 1:
            raise ValueError(f"MXFP4Weight: shape [N, K] expected, got {self.shape}")
        ops._mx_parts(codes, scales, *self.shape, "MXFP4Weight")
        self.codes, self.scales = codes, scales
        self.numel = self.shape[0] * self.shape[1]
        self.resident = None  # bf16 copies of the "resident" LoRA base mode, as NF4Weight's
        self.resident_qkv = None

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "MXFP4Weight":
        """From a [N, K] tensor (bf16, f16 or f32) on the device."""
        codes, scales = ops.mxfp4_quantize(w)
        return cls(codes, scales, w.shape)

    @classmethod
    def from_parts(cls, codes: torch.Tensor, scales: torch.Tensor, shape) -> "MXFP4Weight":
        """From unpadded parts ([N, ceil(K / 2)] codes, [N, ceil(K / 32)] scales, e.g. of a checkpoint): padded where K is
        not a multiple of 128, otherwise as they are. What lies behind K in the last block of a row is cleared."""
        N, K = (int(s) for s in shape)
        cs, ss = ops.mxfp4_shapes(N, K)
        for t, want, name in ((codes, (N, (K + 1) // 2), "codes"), (scales, (N, (K + 31) // 32), "scales")):
            if t.dtype != torch.uint8 or tuple(t.shape) != want:
                raise ValueError(f"MXFP4Weight.from_parts: {name} u8 {want} expected, got {t.dtype} {tuple(t.shape)}")
        if K % 128:
            c, s = codes.new_zeros(cs), scales.new_zeros(ss)
            c[:, :codes.shape[1]] = codes
            s[:, :scales.shape[1]] = scales
            if K % 2:
                c[:, K // 2] &= 15
            codes, scales = c, s
        return cls(codes.contiguous(), scales.contiguous(), (N, K))

    def dequantize(self, out: torch.Tensor | None = None) -> torch.Tensor:
        return ops.mxfp4_dequantize(self.codes, self.scales, self.shape[1],
                                    None if out is None else out.view(self.shape), BF16)

    def to(self, device) -> "MXFP4Weight":
        """On `device`: itself where it is there already."""
        codes, scales = self.codes.to(device), self.scales.to(device)
        return self if codes is self.codes and scales is self.scales else MXFP4Weight(codes, scales, self.shape)
