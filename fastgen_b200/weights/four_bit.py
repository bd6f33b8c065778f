"""Matrices of 4-bit weights with a scale for each group of columns of a row.

``W[n, k] = (code[n, k] - 8) * scale[n, k // group]``: codes 0..15, groups of 32, 64 or 128 columns, scales in
bfloat16.  :meth:`Weight4.quantize` makes one from a matrix, as a model's projections become 4-bit weights when they are
bound; codes and scales that a program has already go through the constructor.  :meth:`fastgen_b200.csrc.ops.Ops.linear` multiplies by it as by an ordinary matrix.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

GROUPS = (32, 64, 128)


class Weight4:
    """``codes`` [N, K / 2] uint8, two columns a byte, the even column in the low half; ``scales`` [N, K / group] bfloat16."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor) -> None:
        if codes.dtype != torch.uint8 or codes.dim() != 2 or codes.shape[0] == 0:
            raise ValueError(f"4-bit codes are uint8 [rows, columns / 2], got {codes.dtype} {tuple(codes.shape)}")
        n, k = codes.shape[0], 2 * codes.shape[1]
        if scales.dtype != torch.bfloat16 or scales.dim() != 2 or scales.shape[0] != n or scales.device != codes.device:
            raise ValueError(f"scales of 4-bit weights are bfloat16 [{n}, columns / group], got {scales.dtype} {tuple(scales.shape)}")
        groups = scales.shape[1]
        if groups == 0 or k % groups or k // groups not in GROUPS:
            raise ValueError(f"{k} columns in {groups} groups: groups of 4-bit weights have one of {GROUPS} columns")
        self._set(self._packed(codes), scales.contiguous(), k // groups)

    def _set(self, packed: torch.Tensor, scales: torch.Tensor, group: int) -> None:
        #: int32 [N, K / 8]: a word's nibbles are the columns 0, 2, 4, 6, 1, 3, 5, 7 of its eight, lowest first
        self.packed = packed
        self.scales = scales
        self.group = group
        self.rows, self.columns = packed.shape[0], 8 * packed.shape[1]

    @staticmethod
    def _packed(codes: torch.Tensor) -> torch.Tensor:
        n, half = codes.shape
        four = codes.reshape(n, half // 4, 4)  # bytes of eight columns: even columns low, odd ones high
        even, odd = four & 15, four >> 4
        pairs = torch.stack([even, odd], dim=2)  # [n, words, 2, 4]: the low half's nibbles, then the high half's
        out = pairs[..., 0::2] | (pairs[..., 1::2] << 4)  # [n, words, 2, 2]
        return out.reshape(n, half).contiguous().view(torch.int32)

    @property
    def shape(self) -> Tuple[int, int]:
        return self.rows, self.columns

    @property
    def device(self) -> torch.device:
        return self.packed.device

    def numel(self) -> int:
        n, k = self.shape
        return n * k

    def nbytes(self) -> int:
        return 4 * self.packed.numel() + 2 * self.scales.numel()

    def __getitem__(self, rows: slice) -> "Weight4":
        """Some neighbouring rows, without a copy."""
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("4-bit weights are cut into neighbouring rows only")
        out = object.__new__(Weight4)
        out._set(self.packed[rows], self.scales[rows], self.group)
        return out

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The matrix that the codes and scales stand for."""
        n, k = self.shape
        b = self.packed.view(torch.uint8).view(n, k // 8, 2, 2)
        nibbles = torch.stack([b & 15, b >> 4], dim=4).view(n, k // 8, 2, 4)
        codes = nibbles.transpose(2, 3).reshape(n, k)
        w = (codes.to(torch.float32) - 8.0).view(n, -1, self.group) * self.scales.float().unsqueeze(2)
        return w.view(n, k).to(dtype)

    @staticmethod
    def why_not(k: int, group: int = 128) -> Optional[str]:
        """``None``, or why a matrix of ``k`` columns cannot be held in groups of ``group``."""
        if group not in GROUPS:
            return f"groups of {group} columns: 4-bit weights take one of {GROUPS}"
        if k <= 0 or k % group:
            return f"{k} columns are no multiple of the group of {group}"
        return None

    @staticmethod
    def quantize(w: torch.Tensor, group: int = 128) -> "Weight4":
        """The nearest codes of ``w`` [N, K] (finite numbers) under a scale of a seventh of a group's largest magnitude,
        rounded to bfloat16; a group of zeros has scale zero."""
        if w.dim() != 2 or not w.is_floating_point():
            raise ValueError(f"quantize takes a matrix of floating numbers, got {w.dtype} {tuple(w.shape)}")
        n, k = w.shape
        why = Weight4.why_not(k, group)
        if why is not None:
            raise ValueError(why)
        packed, scales = [], []
        rows = max(1, (1 << 26) // k)
        for r in range(0, n, rows):
            part = w[r : r + rows].float().reshape(-1, k // group, group)
            s = (part.abs().amax(2) / 7.0).to(torch.bfloat16)
            # (a scale below bfloat16's range is zero, as if the group were)
            c = torch.round(torch.where(s.float().unsqueeze(2) > 0, part / s.float().unsqueeze(2), torch.zeros_like(part)))
            c = (c.clamp(-8, 7) + 8).to(torch.uint8).view(-1, k)
            packed.append(Weight4._packed(c[:, 0::2] | (c[:, 1::2] << 4)))
            scales.append(s)
        out = object.__new__(Weight4)
        out._set(torch.cat(packed), torch.cat(scales), group)
        return out
